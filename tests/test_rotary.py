"""Rotary positions (`fta_rotary`, `apply_rotary`): frequencies, refusals and the kernel's source on host threads (CPU),
parity with the 64-bit definition on the GPU."""
import ctypes as C
import math

import pytest
import torch

from flash_tree_attn_amd import _lib, apply_rotary, rotary_frequencies, tree_depths
from oracle.step_oracle import rotary_oracle
from step_host import host_step_lib  # noqa: F401  (fixture)

DEV = "cuda"
DTYPES = {torch.float32: _lib.FTA_F32, torch.float16: _lib.FTA_F16, torch.bfloat16: _lib.FTA_BF16}


def check(got, x, ref, factor=1.0):
    """Half a step of the output type, plus the 32-bit arithmetic: cos and sin are off by at most 2 steps and the rounding
    of the reduced angle (pi 2^-25), 4e-7 in all, the two products and their sum by 3 half steps, 2e-7: 6e-7 (|a| + |b|),
    and |a| + |b| <= 2 max |x| of the row. fp16 results below 2^-14 have half steps of 2^-25."""
    bound = torch.finfo(got.dtype).eps / 2 * ref.abs() + 6e-7 * factor * 2 * x.double().abs().amax(-1, keepdim=True) + 2.0 ** -25
    bad = (got.double() - ref).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float(((got.double() - ref).abs() / bound).max()):.2f} bounds"


# ---------------------------------------------------------------- CPU
def test_frequencies():
    inv, factor = rotary_frequencies(64)
    assert inv.dtype == torch.float64 and factor == 1.0
    assert inv.tolist() == pytest.approx([10000.0 ** (-2 * t / 64) for t in range(32)], rel=1e-15)
    lin, _ = rotary_frequencies(64, scaling="linear", factor=4.0)
    assert torch.equal(lin, inv / 4)
    base, _ = rotary_frequencies(64, scaling="base", factor=4.0)
    assert base[0] == 1.0 and float(base[-1] * 4) == pytest.approx(float(inv[-1]), rel=1e-12)
    parts, factor = rotary_frequencies(64, scaling="by_parts", factor=4.0, original_len=4096)
    assert factor == pytest.approx(1 + 0.1 * math.log(4.0))
    turns = 4096 * inv / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], inv[turns >= 32]) and torch.equal(parts[turns <= 1], (inv / 4)[turns <= 1])
    assert bool(((parts <= inv) & (parts >= inv / 4)).all())
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(rotary_dim=8, base=0.0), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="by_parts"), dict(rotary_dim=8, factor=-1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_tree_depths():
    assert tree_depths([-1, 0, 0, 1, 3, -1, 5]).tolist() == [0, 1, 1, 2, 3, 0, 1]
    with pytest.raises(ValueError):
        tree_depths([-1, 2, 0])


def base_args(**kw):
    a = _lib.FtaRotaryArgs()
    for f in ("q", "k", "out_q", "out_k", "positions", "inv_freq"):
        setattr(a, f, 0x1000)
    cfg = dict(bsz=2, num_q_heads=4, num_kv_heads=2, q_len=3, head_dim=64, rotary_dim=64, dtype=_lib.FTA_BF16, attention_factor=1.0)
    cfg.update(kw)
    for k, v in cfg.items():
        setattr(a, k, v)
    for s in ("q_stride", "k_stride", "out_q_stride", "out_k_stride"):
        getattr(a, s)[:] = [4 * 3 * 64, 3 * 64, 64]
    a.pos_stride[:] = [0, 1]
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(head_dim=96), -2), (dict(dtype=5), -6), (dict(pos_dtype=2), -6), (dict(len_dtype=9), -6), (dict(bsz=0), -7), (dict(q_len=0), -7),
    (dict(rotary_dim=0), -7), (dict(rotary_dim=7), -7), (dict(rotary_dim=66), -7), (dict(num_kv_heads=0), -7), (dict(q=None), -1),
    (dict(out_k=None), -1), (dict(positions=None), -1), (dict(inv_freq=None), -1), (dict(k=None, out_k=None), -7), (dict(q=0x1004), -8),
    (dict(inv_freq=0x1004, freq_is_f64=1), -8),
])
def test_argument_errors_without_touching_the_gpu(fta_lib, kw, status):
    assert fta_lib.fta_rotary(C.byref(base_args(**kw)), None) == status


def test_stride_errors_and_missing_device(fta_lib):
    assert fta_lib.fta_rotary(None, None) == -1
    a = base_args()
    a.q_stride[2] = 68
    assert fta_lib.fta_rotary(C.byref(a), None) == -8
    a = base_args()
    a.pos_stride[1] = -1
    assert fta_lib.fta_rotary(C.byref(a), None) == -8
    if not torch.cuda.is_available():
        assert fta_lib.fta_rotary(C.byref(base_args()), None) == -11
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        apply_rotary(torch.zeros(1, 1, 1, 32), None, torch.zeros(1, dtype=torch.int32), torch.ones(16))


SHAPES = [
    # bsz hq hk L  D   rd   interleaved inverse dtype  factor
    (1, 3, 1, 1, 32, 32, False, False, torch.float32, 1.0),
    (2, 4, 2, 5, 64, 64, True, False, torch.bfloat16, 1.0),
    (3, 2, 1, 7, 128, 64, False, True, torch.float16, 1.25),
    (1, 5, 5, 3, 64, 22, False, False, torch.bfloat16, 1.0),      # halves of 11: one pair per thread
    (2, 2, 1, 4, 128, 2, True, True, torch.float32, 0.5),         # one pair
    (1, 8, 2, 9, 256, 254, True, False, torch.float16, 1.0),
    (2, 3, 3, 2, 256, 128, False, False, torch.float32, 1.0),
    (1, 2, 1, 3, 32, 8, False, False, torch.float32, 2.0),        # one turning unit, three that copy
    (2, 2, 1, 3, 128, 112, False, False, torch.bfloat16, 1.0),
    (1, 2, 2, 5, 64, 8, True, False, torch.float16, 3.0),
]


def make(shape, seed=0, device="cpu"):
    bsz, hq, hk, L, D, rd, interleaved, inverse, dtype, factor = shape
    g = torch.Generator().manual_seed(seed)
    x = dict(q=torch.randn(bsz, hq, L, D, generator=g).to(dtype), k=torch.randn(bsz, hk, L, D, generator=g).to(dtype),
             positions=torch.randint(0, 9, (bsz, L), generator=g, dtype=torch.int32),
             kv_seq_len=torch.randint(0, 1 << 20, (bsz,), generator=g), inv_freq=rotary_frequencies(rd)[0])
    return {n: t.to(device) for n, t in x.items()}, dict(interleaved=interleaved, inverse=inverse, attention_factor=factor)


@pytest.mark.parametrize("shape", SHAPES)
def test_kernel_source_on_host_threads(host_step_lib, shape):
    x, opt = make(shape)
    a = _lib.FtaRotaryArgs()
    oq, ok = torch.full_like(x["q"], float("nan")), torch.full_like(x["k"], float("nan"))
    a.q, a.k, a.out_q, a.out_k = x["q"].data_ptr(), x["k"].data_ptr(), oq.data_ptr(), ok.data_ptr()
    a.positions, a.kv_seq_len, a.inv_freq = x["positions"].data_ptr(), x["kv_seq_len"].data_ptr(), x["inv_freq"].data_ptr()
    a.bsz, a.num_q_heads, a.q_len, a.head_dim = x["q"].shape
    a.num_kv_heads, a.rotary_dim, a.dtype = x["k"].size(1), 2 * x["inv_freq"].numel(), DTYPES[x["q"].dtype]
    a.pos_dtype, a.len_dtype, a.freq_is_f64 = _lib.FTA_I32, _lib.FTA_I64, 1
    a.interleaved, a.inverse, a.attention_factor = opt["interleaved"], opt["inverse"], opt["attention_factor"]
    a.q_stride[:], a.out_q_stride[:] = x["q"].stride()[:3], oq.stride()[:3]
    a.k_stride[:], a.out_k_stride[:] = x["k"].stride()[:3], ok.stride()[:3]
    a.pos_stride[:] = x["positions"].stride()
    assert host_step_lib.fta_rotary(C.byref(a), None) == 0
    for got, name in ((oq, "q"), (ok, "k")):
        check(got, x[name], rotary_oracle(x[name], x["positions"], x["inv_freq"], x["kv_seq_len"], **opt), opt["attention_factor"])


# ---------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES + [(2, 32, 8, 300, 128, 128, False, False, torch.bfloat16, 1.0),
                                            (64, 40, 8, 130, 128, 96, True, False, torch.float16, 1.0),
                                            (64, 16, 4, 130, 128, 64, False, False, torch.float16, 1.0)])
def test_matches_the_definition(shape):
    x, opt = make(shape, 1, DEV)
    for seed in (1, 2):     # the second call runs from the remembered signature
        x, opt = make(shape, seed, DEV)
        q, k = apply_rotary(x["q"], x["k"], x["positions"], x["inv_freq"], kv_seq_len=x["kv_seq_len"], **opt)
        for got, name in ((q, "q"), (k, "k")):
            check(got, x[name], rotary_oracle(x[name], x["positions"], x["inv_freq"], x["kv_seq_len"], **opt), opt["attention_factor"])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [False, True])
def test_values_behind_rotary_dim_are_copied_as_they_are(interleaved):
    q = torch.randn(2, 3, 5, 64, device=DEV).half()
    q[..., 32:] = torch.tensor([float("nan"), float("inf"), -float("inf"), -0.0], device=DEV).half().repeat(8)
    out, _ = apply_rotary(q, None, torch.arange(5, device=DEV), rotary_frequencies(32, device=DEV)[0], interleaved=interleaved, attention_factor=0.5)
    assert torch.equal(out[..., 32:].view(torch.int16), q[..., 32:].view(torch.int16)) and out[..., :32].isfinite().all()


@pytest.mark.gpu
def test_strided_rows_in_place_and_back():
    """q and k as slices of one projection [bsz, L, heads, D], turned in place (other heads untouched), then turned back."""
    g = torch.Generator().manual_seed(5)
    fused = torch.randn(3, 6, 8 + 2 + 2, 64, generator=g).to(DEV)
    before = fused.clone()
    q, k = fused[:, :, :8].transpose(1, 2), fused[:, :, 8:10].transpose(1, 2)
    q0, k0 = q.clone(), k.clone()
    pos, inv = torch.arange(6, device=DEV), rotary_frequencies(48, device=DEV)[0].float()
    oq, ok = apply_rotary(q, k, pos, inv, out_q=q, out_k=k)
    assert oq is q and ok is k and torch.equal(fused[:, :, 10:], before[:, :, 10:])
    check(q, q0, rotary_oracle(q0, pos, inv))
    check(k, k0, rotary_oracle(k0, pos, inv))
    apply_rotary(q, k, pos, inv, inverse=True, out_q=q, out_k=k)
    assert (fused - before).abs().max() < 2e-6
    only, none = apply_rotary(q0, None, pos, inv)
    assert none is None
    check(only, q0, rotary_oracle(q0, pos, inv))
    odd = torch.randn(2, 3, 4, 65, device=DEV)[..., 1:]     # rows at odd offsets are copied
    got, _ = apply_rotary(odd, None, pos[:4], inv)
    check(got, odd, rotary_oracle(odd, pos[:4], inv))


@pytest.mark.gpu
def test_refusals():
    q, pos, inv = torch.zeros(2, 4, 3, 64, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV), torch.ones(32, device=DEV)
    ok = lambda **kw: apply_rotary(kw.get("q", q), kw.get("k"), kw.get("pos", pos), kw.get("inv", inv), **{n: v for n, v in kw.items() if n not in ("q", "k", "pos", "inv")})
    ok()
    for kw in (dict(q=q[0]), dict(q=q.double()), dict(k=q[:1]), dict(k=q.half()), dict(pos=pos.float()), dict(pos=pos[:2]), dict(pos=pos.cpu()),
               dict(inv=inv.half()), dict(inv=torch.ones(33, device=DEV)), dict(inv=inv[:0]), dict(kv_seq_len=pos), dict(attention_factor=float("nan")),
               dict(out_q=q.half()), dict(out_q=q[:1].expand(2, 4, 3, 64)), dict(out_k=q), dict(q=torch.zeros(1, 1, 3, 48, device=DEV))):
        with pytest.raises(ValueError):
            ok(**kw)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
        ok(q=q.clone().requires_grad_())
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
        ok(inv=inv.clone().requires_grad_())
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):   # the same signature, remembered by now
        ok(q=q.clone().requires_grad_())
