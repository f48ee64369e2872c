"""Repeat calls (`_binding.recall`, csrc/binding.cpp): what has a signature and what does not (CPU), and calls of the
operators from remembered signatures (GPU)."""
import pytest
import torch
from torch.autograd import forward_ad

from flash_tree_attn_amd import _lib, apply_rotary, rotary_frequencies, shaped_tree_attention, token_logprobs
from flash_tree_attn_amd.flash_decoding import _refuse_derivatives

DEV = "cuda"
pytestmark = pytest.mark.filterwarnings("ignore::DeprecationWarning")      # torch's own, at the first tangent


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


def remember(cache, signature):
    _lib.binding().remember(cache, signature, 0, bytes(64), (), (), 0, 0, 0)      # never launched


def test_signatures_are_kept_up_to_a_bound():
    cache = {}
    for n in range(1, 300):
        signature = _lib.binding().recall(cache, "name", n, torch.empty(n, 2))
        assert isinstance(signature, bytes) and signature not in cache
        remember(cache, signature)
        assert len(cache) == (n if n <= 256 else n - 256)


def test_what_tells_signatures_apart():
    base = torch.zeros(64)
    calls = [(base[:16],), (base[1:17],), (base[4:20].view(4, 4),), (base[:32:2],), (base[:16].double(),), (base[:16].int(),), (base[:16], None), (base[:16], 0),
             (base[:16], 0.0), (base[:16], False), (base[:16], 1), (base[:16], "0"), (base[:16], torch.int32), (base[:16].clone().requires_grad_(),)]
    signatures = [_lib.binding().recall({}, "name", *c) for c in calls]
    assert len(set(signatures)) == len(calls)
    assert _lib.binding().recall({}, "name", base[4:20]) == signatures[0]      # elsewhere, alike
    with torch.no_grad():
        assert _lib.binding().recall({}, "name", calls[-1][0]) == signatures[0]
    for odd in (1 << 70, [], torch.zeros(2, 2).to_sparse()):
        assert _lib.binding().recall({}, "name", base, odd) is None


@pytest.mark.gpu
def test_known_shapes_at_other_alignments_and_strides():
    g = torch.Generator().manual_seed(2)
    store = torch.randn(4096, generator=g).to(DEV)
    inv_freq, at = rotary_frequencies(64, device=DEV)[0], torch.arange(3, device=DEV)
    for _ in range(2):
        for offset in (0, 4, 1, 8, 3):      # elements: 16-byte aligned or not
            q = store[offset:offset + 384].view(1, 2, 3, 64)
            assert torch.equal(apply_rotary(q, None, at, inv_freq)[0], apply_rotary(q.clone(), None, at, inv_freq)[0])
            x = store[offset:offset + 1500].view(2, 750)
            for a, b in zip(token_logprobs(x, top_k=3)[1:], token_logprobs(x.clone(), top_k=3)[1:]):
                torch.testing.assert_close(a, b, atol=2e-5, rtol=1e-6)
        wide = store[:768].view(1, 2, 3, 128)[..., :64]      # the same sizes, other strides
        assert torch.equal(apply_rotary(wide, None, at, inv_freq)[0], apply_rotary(wide.contiguous(), None, at, inv_freq)[0])


@pytest.mark.gpu
def test_more_signatures_than_are_kept():
    """A loop whose sizes grow with every step, twice: every call gives what a fresh tensor's gives."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(400, generator=g).to(DEV)
    for _ in range(2):
        for n in range(20, 320):
            got = token_logprobs(x[:n], top_k=1)
            assert int(got.top_ids) == int(x[:n].argmax())
