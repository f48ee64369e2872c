"""`apply_rotary`: rotary positions for the rows that enter a tree-attention call, and `rotary_frequencies`, the
inverse frequencies it takes (plain, or scaled for contexts longer than the model was trained on).

A tree node stands at (keys in the cache) + (its depth in the tree): pass `kv_seq_len` and the depths
(`tree_mask.tree_depths`), and no position tensor has to be formed. Runs a gfx950 kernel through the C ABI
(`fta_rotary`, include/fta.h); GPU tensors only, no fallback, no autograd.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib
from .flash_decoding import _DTYPES, _as_rows, _calls, _check, _current_stream, _refuse_derivatives, _remember_call, _rows_ok

_INT_DTYPES = {torch.int32: _lib.FTA_I32, torch.int64: _lib.FTA_I64}


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       original_len: Optional[int] = None, low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> Tuple[torch.Tensor, float]:
    """(inv_freq float64 [rotary_dim / 2] in radians per position, attention_factor) for `apply_rotary`.

    scaling  None        base ** (-2 t / rotary_dim)
             "linear"    the same divided by `factor` (positions interpolated)
             "base"      base raised to base * factor ** (rotary_dim / (rotary_dim - 2)): the fastest pair keeps its
                         frequency, the slowest is divided by `factor`
             "by_parts"  pairs that turn at least `high_turns` times over `original_len` positions keep their
                         frequency, pairs below `low_turns` are divided by `factor`, those between are blended;
                         attention_factor = 1 + 0.1 ln(factor)
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even and at least 2, got {rotary_dim}")
    if not (base > 0 and factor > 0):
        raise ValueError("base and factor must be positive")
    if scaling not in (None, "linear", "base", "by_parts"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'base' or 'by_parts'")
    if scaling == "base":
        base = base * factor ** (rotary_dim / max(rotary_dim - 2, 1))
    inv = torch.tensor(float(base), dtype=torch.float64) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    attention_factor = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "by_parts":
        if original_len is None or original_len <= 0 or not high_turns > low_turns:
            raise ValueError("scaling by parts needs original_len > 0 and high_turns > low_turns")
        keep = ((original_len * inv / (2 * math.pi) - low_turns) / (high_turns - low_turns)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1 - keep)
        attention_factor = 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    return (inv.to(device) if device is not None else inv), attention_factor


def _out_rows(name: str, out: Optional[torch.Tensor], like: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(like.shape, dtype=like.dtype, device=like.device)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must have its input's shape, dtype and device")
    if not _rows_ok(out) or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{name} needs unit inner stride, 16-byte aligned rows and a place of its own for every value")
    return out


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, *,
                 kv_seq_len: Optional[torch.Tensor] = None, interleaved: bool = False, attention_factor: float = 1.0,
                 inverse: bool = False, out_q: Optional[torch.Tensor] = None,
                 out_k: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Turns the first 2 * len(inv_freq) values of every row by its position; the others are copied.

      q          [bsz, num_heads, q_len, head_dim], head_dim 32, 64, 128 or 256, fp32, fp16 or bf16
      k          [bsz, num_kv_heads, q_len, head_dim] of q's dtype, or None
      positions  int32 / int64 [q_len] or [bsz, q_len]; with `kv_seq_len` (int32 / int64 [bsz]) row i of sequence b
                 stands at kv_seq_len[b] + positions[b, i]
      inv_freq   float64 or float32 [rotary_dim / 2] on q's device, radians per position (`rotary_frequencies`)
      interleaved       pairs (2t, 2t + 1) instead of (t, t + rotary_dim / 2)
      attention_factor  multiplies the turned values
      inverse           turns back (angles negated; the factor still multiplies)
    Angles are formed in 64 bits. Returns (q, k) turned, in `out_q` / `out_k` where given; these may be q and k
    themselves, and must not overlap the inputs otherwise.
    """
    lib = _lib.load()
    hit = _lib.binding().recall(_calls(), "rotary", q, k, positions, inv_freq, kv_seq_len, interleaved, attention_factor, inverse, out_q, out_k)
    if hit.__class__ is tuple:
        if hit[0]:
            _check(hit[0])
        return hit[1], hit[2] if k is not None else None

    if q.dim() != 4:
        raise ValueError(f"q must be [bsz, num_heads, q_len, head_dim], got {tuple(q.shape)}")
    dev = q.device
    if dev.type != "cuda":
        raise RuntimeError("apply_rotary runs on the GPU only; there is no CPU fallback")
    _refuse_derivatives("apply_rotary", q, k, inv_freq)
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    bsz, hq, L, D = q.shape
    if k is not None and (k.dim() != 4 or (k.size(0), k.size(2), k.size(3)) != (bsz, L, D) or k.dtype != q.dtype or k.device != dev):
        raise ValueError("k must be [bsz, num_kv_heads, q_len, head_dim] with q's dtype and device")
    if k is None and out_k is not None:
        raise ValueError("out_k without k")
    if positions.dtype not in _INT_DTYPES or positions.device != dev or tuple(positions.shape) not in ((L,), (bsz, L), (1, L)):
        raise ValueError("positions must be an int32 / int64 tensor [q_len] or [bsz, q_len] on q's device")
    if inv_freq.dim() != 1 or inv_freq.dtype not in (torch.float64, torch.float32) or inv_freq.device != dev:
        raise ValueError("inv_freq must be a float64 / float32 tensor [rotary_dim / 2] on q's device")
    if not 2 <= 2 * inv_freq.numel() <= D:
        raise ValueError(f"rotary_dim 2 * {inv_freq.numel()} must be between 2 and head_dim {D}")
    if kv_seq_len is not None and (kv_seq_len.dtype not in _INT_DTYPES or kv_seq_len.device != dev or kv_seq_len.numel() != bsz):
        raise ValueError("kv_seq_len must be an int32 / int64 tensor of bsz elements on q's device")
    if not math.isfinite(attention_factor):
        raise ValueError("attention_factor must be finite")
    given = (q, k, positions, inv_freq, kv_seq_len)
    oq = _out_rows("out_q", out_q, q)
    ok = None if k is None else _out_rows("out_k", out_k, k)
    q = _as_rows(q)
    k = None if k is None else _as_rows(k)
    inv_freq = inv_freq.contiguous()
    kv_seq_len = None if kv_seq_len is None else kv_seq_len.contiguous()

    a = _lib.FtaRotaryArgs()
    a.q, a.out_q, a.positions, a.inv_freq = q.data_ptr(), oq.data_ptr(), positions.data_ptr(), inv_freq.data_ptr()
    a.bsz, a.num_q_heads, a.q_len, a.head_dim, a.rotary_dim = bsz, hq, L, D, 2 * inv_freq.numel()
    a.q_stride[:], a.out_q_stride[:] = q.stride()[:3], oq.stride()[:3]
    if k is not None:
        a.k, a.out_k, a.num_kv_heads = k.data_ptr(), ok.data_ptr(), k.size(1)
        a.k_stride[:], a.out_k_stride[:] = k.stride()[:3], ok.stride()[:3]
    if kv_seq_len is not None:
        a.kv_seq_len, a.len_dtype = kv_seq_len.data_ptr(), _INT_DTYPES[kv_seq_len.dtype]
    a.dtype, a.pos_dtype, a.freq_is_f64 = _DTYPES[q.dtype], _INT_DTYPES[positions.dtype], inv_freq.dtype == torch.float64
    a.interleaved, a.inverse, a.attention_factor = bool(interleaved), bool(inverse), float(attention_factor)
    per_sequence = positions.dim() == 2 and positions.size(0) > 1
    a.pos_stride[:] = (positions.stride(0) if per_sequence else 0, positions.stride(-1))
    with torch.cuda.device(dev):
        _check(lib.fta_rotary(C.byref(a), _current_stream(dev.index)))
    outputs = (("out_q", -1 if out_q is None else 9, oq),) + (() if k is None else (("out_k", -1 if out_k is None else 10, ok),))
    read = (q, k, positions, inv_freq, kv_seq_len)
    _remember_call(hit, lib.fta_rotary, a, dev, tuple(zip(("q", "k", "positions", "inv_freq", "kv_seq_len"), range(1, 6), given, read)), outputs)
    return oq, ok
