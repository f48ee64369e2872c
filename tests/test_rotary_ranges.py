"""Rotary positions: factors at and beyond what 32 bits hold."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_amd import apply_rotary, rotary_frequencies
from test_rotary import base_args


@pytest.mark.parametrize("factor", [float("inf"), float("-inf"), float("nan"), 1e39])
def test_factors_that_are_no_finite_float_are_refused(fta_lib, factor):
    assert fta_lib.fta_rotary(C.byref(base_args(attention_factor=factor)), None) == -9


@pytest.mark.gpu
def test_the_wrapper_refuses_them_too():
    q, at, inv_freq = torch.ones(1, 1, 1, 32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), rotary_frequencies(32, device="cuda")[0]
    for _ in range(2):
        for factor in (1e39, -1e39, float("inf")):
            with pytest.raises(ValueError):
                apply_rotary(q, None, at, inv_freq, attention_factor=factor)
        assert torch.equal(apply_rotary(q, None, at, inv_freq, attention_factor=3e38)[0], q * 3e38)
