"""`shaped_tree_attention`: tree attention whose scores are shaped before the softmax, for models that cap them with a
tanh, let them fall with distance, look back through a sliding window, or pack several documents into a cache row.

Same tensors as `flash_decoding_attention`; runs gfx950 kernels of its own through the C ABI (`fta_shaped_decode`,
include/fta.h). GPU tensors only, no fallback, no autograd.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from .flash_decoding import (_DTYPES, FtaAssertionError, _as_rows, _calls, _check, _current_stream, _num_cus, _prepare_mask,
                             _refuse_derivatives, _remember_call, _rows_ok)


def shaped_tree_attention(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, current_k: torch.Tensor, current_v: torch.Tensor,
    mask: torch.Tensor, kv_seq_len: torch.Tensor, *,
    softcap: float = 0.0, slopes: Optional[torch.Tensor] = None, window: int = 0, first_key: Optional[torch.Tensor] = None,
    depths: Optional[torch.Tensor] = None, max_seq_len_in_batch: Optional[int] = None, output: Optional[torch.Tensor] = None,
    sm_scale: Optional[float] = None, kv_group_num: int = 1, block_tables: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """softmax over the cached keys and the tree's of
        y - slopes[head] * (p_i - p_j) (+ mask[i, j] for a tree key),   y = softcap * tanh(x / softcap), x = sm_scale q_i . k_j
    times V. A cached key j stands at position j, tree node i at kv_seq_len[b] + depths[i].

      q [bsz, num_heads, q_len, head_dim]; k_cache / v_cache [bsz, num_kv_heads, ctx, head_dim], or page pools with
      `block_tables`; current_k / current_v [bsz, num_kv_heads (or num_heads), q_len, head_dim]; mask and kv_seq_len: as
      `flash_decoding_attention` takes them. fp32, fp16 or bf16; head_dim 32, 64, 128 or 256.
      softcap    0 (none) or the cap of the scores
      slopes     float32 [num_heads]: how much a score falls per position of distance, or None
      window     0 (none), or: keys at a distance of `window` or more are left out (1: a node sees itself only)
      first_key  int32 [bsz]: cached keys in front of it belong to another document and are left out, or None
      depths     int32 [q_len] or [bsz, q_len]: depth of every node (`tree_mask.tree_depths`); None = 0, 1, 2, ... (a
                 chain). Only distances depend on it: needed with slopes or a window
    A row that sees nothing yields zeros. Returns [bsz, num_heads, q_len, head_dim] in q's dtype (in `output` if given).
    """
    lib = _lib.load()
    hit = _lib.binding().recall(_calls(), "shaped", q, k_cache, v_cache, current_k, current_v, mask, kv_seq_len, slopes, first_key, depths, block_tables,
                                output, softcap, window, max_seq_len_in_batch, sm_scale, kv_group_num)
    if hit.__class__ is tuple:
        if hit[0]:
            _check(hit[0])
        return hit[1]

    if q.dim() != 4:
        raise ValueError(f"q must be [bsz, num_heads, q_len, head_dim], got {tuple(q.shape)}")
    bsz, hq, L, D = q.shape
    dev = q.device
    if dev.type != "cuda":
        raise RuntimeError("shaped_tree_attention runs on the GPU only; there is no CPU fallback")
    _refuse_derivatives("shaped_tree_attention", q, k_cache, v_cache, current_k, current_v, mask, slopes)
    if q.dtype not in _DTYPES:
        raise ValueError(f"unsupported dtype {q.dtype}")
    paged = block_tables is not None
    for name, t in (("k_cache", k_cache), ("v_cache", v_cache), ("current_k", current_k), ("current_v", current_v)):
        if t.dim() != 4:
            raise ValueError(f"{name} must be 4-dimensional, got {tuple(t.shape)}")
        if t.dtype != q.dtype or t.device != dev:
            raise ValueError(f"{name} must have q's dtype and device")
        pool = paged and name.endswith("cache")
        if (t.size(0) != bsz and not pool) or t.size(3) != D:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, incompatible with q {tuple(q.shape)}")
    if k_cache.shape != v_cache.shape:
        raise FtaAssertionError("k_cache and v_cache must have the same shape")
    hkv = k_cache.size(1)
    if hkv * int(kv_group_num) != hq:
        raise ValueError(f"num_heads {hq} != num_kv_heads {hkv} * kv_group_num {kv_group_num}")
    if current_k.shape != current_v.shape or current_k.size(2) != L or current_k.size(1) not in (hkv, hq):
        raise ValueError("current_k/current_v must be [bsz, num_kv_heads (or num_heads), q_len, head_dim]")
    if kv_seq_len.device != dev or kv_seq_len.dtype not in (torch.int32, torch.int64) or kv_seq_len.numel() != bsz:
        raise ValueError("kv_seq_len must be an int32/int64 tensor of bsz elements on q's device")
    if paged and (block_tables.dim() != 2 or block_tables.size(0) != bsz or block_tables.dtype != torch.int32 or block_tables.device != dev):
        raise ValueError("block_tables must be an int32 tensor [bsz, pages per sequence] on q's device")
    if not (softcap >= 0 and math.isfinite(softcap)):
        raise ValueError("softcap must be 0 (none) or positive and finite")
    if not 0 <= int(window) < 1 << 31:
        raise ValueError("window must be 0 (none) or positive")
    if slopes is not None and (slopes.dtype != torch.float32 or slopes.device != dev or tuple(slopes.shape) != (hq,)):
        raise ValueError("slopes must be a float32 tensor [num_heads] on q's device")
    if first_key is not None and (first_key.dtype != torch.int32 or first_key.device != dev or first_key.numel() != bsz):
        raise ValueError("first_key must be an int32 tensor of bsz elements on q's device")
    if depths is not None and (depths.dtype != torch.int32 or depths.device != dev or tuple(depths.shape) not in ((L,), (1, L), (bsz, L))):
        raise ValueError("depths must be an int32 tensor [q_len] or [bsz, q_len] on q's device")
    scale = 1.0 / (D ** 0.5) if sm_scale is None else float(sm_scale)
    if not math.isfinite(scale):
        raise ValueError("sm_scale must be finite")
    if output is None:
        out = torch.empty((bsz, hq, L, D), dtype=q.dtype, device=dev)
    else:
        out = output
        if out.shape != (bsz, hq, L, D) or out.dtype != q.dtype or out.device != dev:
            raise FtaAssertionError("output must be [bsz, num_heads, q_len, head_dim] with q's dtype and device")
        if not _rows_ok(out) or any(s == 0 and n > 1 for s, n in zip(out.stride(), out.shape)):
            raise ValueError("output needs unit inner stride, 16-byte aligned rows and a place of its own for every value")

    given = (q, k_cache, v_cache, current_k, current_v, mask, kv_seq_len, slopes, first_key, depths, block_tables)
    q, k_cache, v_cache, current_k, current_v = (_as_rows(t) for t in (q, k_cache, v_cache, current_k, current_v))
    mask = _prepare_mask(mask, bsz, hq, L, dev)
    kv_seq_len = kv_seq_len.contiguous().view(-1)
    slopes = None if slopes is None else slopes.contiguous()
    first_key = None if first_key is None else first_key.contiguous().view(-1)
    if depths is not None and depths.stride(-1) != 1 and L > 1:
        depths = depths.contiguous()
    if paged and block_tables.stride(1) != 1 and block_tables.size(1) > 1:
        block_tables = block_tables.contiguous()

    a = _lib.FtaShapedArgs()
    a.q, a.k_cache, a.v_cache = q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    a.cur_k, a.cur_v, a.mask, a.kv_seq_len, a.out = current_k.data_ptr(), current_v.data_ptr(), mask.data_ptr(), kv_seq_len.data_ptr(), out.data_ptr()
    a.bsz, a.num_q_heads, a.num_kv_heads, a.cur_heads, a.q_len, a.head_dim = bsz, hq, hkv, current_k.size(1), L, D
    if paged:
        a.page_size, a.cache_len = k_cache.size(2), block_tables.size(1) * k_cache.size(2)
        a.block_table, a.block_table_stride = block_tables.data_ptr(), block_tables.stride(0)
    else:
        a.cache_len = k_cache.size(2)
    if slopes is not None:
        a.slopes = slopes.data_ptr()
    if first_key is not None:
        a.first_key = first_key.data_ptr()
    if depths is not None:
        a.depths, a.depth_stride = depths.data_ptr(), depths.stride(0) if depths.dim() == 2 and depths.size(0) > 1 else 0
    a.max_seq_len_hint = 0 if max_seq_len_in_batch is None else min(max(int(max_seq_len_in_batch), 1), 0x7fffffff)
    a.dtype, a.len_dtype = _DTYPES[q.dtype], _lib.FTA_I64 if kv_seq_len.dtype == torch.int64 else _lib.FTA_I32
    a.mask_kind = _lib.MASK_PACKED_U64 if mask.dtype == torch.int64 else _lib.MASK_ADDITIVE_F32
    a.window, a.softcap, a.sm_scale = int(window), float(softcap), scale
    for name, t in (("q_stride", q), ("k_stride", k_cache), ("v_stride", v_cache), ("ck_stride", current_k), ("cv_stride", current_v),
                    ("mask_stride", mask), ("out_stride", out)):
        getattr(a, name)[:] = t.stride()[:3]
    need = C.c_int64()
    _check(lib.fta_shaped_workspace(C.byref(a), _num_cus(dev), C.byref(need)))
    a.workspace_bytes = need.value
    if need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=dev)
        a.workspace = workspace.data_ptr()
    with torch.cuda.device(dev):
        _check(lib.fta_shaped_decode(C.byref(a), _current_stream(dev.index)))
    read = (q, k_cache, v_cache, current_k, current_v, mask, kv_seq_len, slopes, first_key, depths, block_tables)
    fields = ("q", "k_cache", "v_cache", "cur_k", "cur_v", "mask", "kv_seq_len", "slopes", "first_key", "depths", "block_table")
    _remember_call(hit, lib.fta_shaped_decode, a, dev, tuple(zip(fields, range(1, 12), given, read)), (("out", -1 if output is None else 12, out),))
    return out
