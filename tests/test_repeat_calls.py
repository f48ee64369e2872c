"""Repeat calls (`_binding.recall`, csrc/binding.cpp): what has a signature and what does not (CPU), and calls of the
operators from remembered signatures (GPU)."""
import pytest
import torch
from torch.autograd import forward_ad

from flash_tree_attn_amd import _lib, apply_rotary, rotary_frequencies, shaped_tree_attention, token_logprobs
from flash_tree_attn_amd.flash_decoding import _refuse_derivatives

DEV = "cuda"


def test_tensors_with_tangents_have_no_signature():
    t = torch.ones(2, 3)
    plain = _lib.binding().recall({}, "name", t)
    assert isinstance(plain, bytes)
    _refuse_derivatives("f", t, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, torch.ones_like(t))
        assert _lib.binding().recall({}, "name", dual) is None
        assert _lib.binding().recall({}, "name", t) == plain
        _refuse_derivatives("f", t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            _refuse_derivatives("f", None, dual)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            _refuse_derivatives("f", dual)
    with pytest.raises(RuntimeError, match="no_grad"):
        _refuse_derivatives("f", t.clone().requires_grad_())


@pytest.mark.gpu
def test_tangents_are_refused():
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)
    q, k, cache, lens, mask = r(1, 2, 3, 64), r(1, 2, 3, 64), r(1, 2, 70, 64), torch.tensor([70], device=DEV), torch.zeros(3, 3, device=DEV)
    inv_freq, _ = rotary_frequencies(64, device=DEV)
    at = torch.arange(3, device=DEV)
    calls = (lambda x: apply_rotary(x, k, at, inv_freq), lambda x: token_logprobs(x, top_k=2),
             lambda x: shaped_tree_attention(x, cache, cache, k, k, mask, lens, softcap=3.0))
    for call in calls:
        for _ in range(2):      # the second time it is remembered
            call(q)
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(q, torch.ones_like(q))
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call(dual)
            call(q)
