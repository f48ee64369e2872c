"""What follows the model's logits in a speculative-decoding step: `token_logprobs` (log probabilities of given tokens,
entropy, top alternatives) and `accept_tree_path` (the accepted path of the draft tree, in the form that
`append_accepted_kv` takes). Both run gfx950 kernels through the C ABI (`fta_logprobs`, `fta_accept_path`,
include/fta.h); GPU tensors only, no fallback, no autograd.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from .flash_decoding import _DTYPES, _calls, _check, _current_stream, _refuse_derivatives, _remember_call

_INT_DTYPES = {torch.int32: _lib.FTA_I32, torch.int64: _lib.FTA_I64}
MAX_TOP_K = 128


class TokenLogprobs(NamedTuple):
    logprobs: Optional[torch.Tensor]   # float32 [..., num_ids], None without token_ids
    entropy: torch.Tensor              # float32 [...]
    lse: torch.Tensor                  # float32 [...]: log-sum-exp of the scaled logits
    top_logprobs: torch.Tensor         # float32 [..., top_k], descending
    top_ids: torch.Tensor              # int64 [..., top_k]


def _logprob_outputs(lead, num_ids, top_k, dev):
    new = lambda shape, dtype=torch.float32: torch.empty(shape, dtype=dtype, device=dev)
    return (None if num_ids is None else new(lead + (num_ids,)), new(lead), new(lead), new(lead + (top_k,)), new(lead + (top_k,), torch.int64))


def _fill_outputs(a, out):
    a.logprobs = out[0].data_ptr() if out[0] is not None else None
    a.entropy, a.lse, a.top_logprobs, a.top_ids = out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), out[4].data_ptr()


def token_logprobs(logits: torch.Tensor, token_ids: Optional[torch.Tensor] = None, *, top_k: int = 0,
                   temperature: float = 1.0) -> TokenLogprobs:
    """Log probabilities under softmax(logits / temperature), in one read of the logits.

      logits     [..., vocab], fp32, fp16 or bf16, inner stride 1 (rows of any stride and alignment)
      token_ids  int32 / int64 [..., num_ids]: the tokens to score, or None. An id outside [0, vocab) scores -inf
      top_k      0 .. 128: the largest logits per row, descending, equal logits by ascending id
    Sums are held in 32 bits. A logit of -inf adds nothing; a row of nothing but -inf has lse -inf, entropy 0 and log
    probabilities of -inf; a NaN or +inf makes its row's lse, entropy and log probabilities NaN.
    """
    lib = _lib.load()
    hit = _lib.binding().recall(_calls(), "logprobs", logits, token_ids, top_k, temperature)
    if hit.__class__ is tuple:
        if hit[0]:
            _check(hit[0])
        return TokenLogprobs(*hit[1:]) if token_ids is not None else TokenLogprobs(None, *hit[1:])

    dev = logits.device
    if dev.type != "cuda":
        raise RuntimeError("token_logprobs runs on the GPU only; there is no CPU fallback")
    _refuse_derivatives("token_logprobs", logits)
    if logits.dim() < 1 or logits.dtype not in _DTYPES or logits.numel() == 0:
        raise ValueError("logits must be a non-empty fp32, fp16 or bf16 tensor [..., vocab]")
    vocab = logits.size(-1)
    if vocab > 1 << 30:
        raise ValueError("a row may hold up to 2^30 logits")
    top_k = int(top_k)
    if not 0 <= top_k <= min(vocab, MAX_TOP_K):
        raise ValueError(f"top_k {top_k} is not between 0 and min(vocab, {MAX_TOP_K})")
    if not (temperature > 0 and math.isfinite(temperature) and math.isfinite(1.0 / temperature)):
        raise ValueError("temperature must be positive and finite")
    if token_ids is not None:
        if token_ids.dtype not in _INT_DTYPES or token_ids.device != dev or token_ids.shape[:-1] != logits.shape[:-1] or token_ids.dim() != logits.dim():
            raise ValueError("token_ids must be an int32 / int64 tensor [..., num_ids] with the logits' leading sizes and device")
    lead = logits.shape[:-1]
    rows = logits.reshape(-1, vocab)                       # a view where the leading dimensions fold into one stride
    if rows.stride(1) != 1 and vocab > 1:
        rows = rows.contiguous()
    ids = None if token_ids is None else token_ids.reshape(rows.size(0), -1) if token_ids.numel() else token_ids.new_empty(rows.size(0), 0)

    a = _lib.FtaLogprobArgs()
    a.logits, a.rows, a.vocab, a.logits_stride = rows.data_ptr(), rows.size(0), vocab, rows.stride(0)
    a.dtype, a.top_k, a.inv_temperature = _DTYPES[logits.dtype], top_k, 1.0 / temperature
    if ids is not None:
        a.token_ids, a.num_ids, a.id_dtype = ids.data_ptr(), ids.size(1), _INT_DTYPES[ids.dtype]
        a.id_stride[:] = ids.stride()
    need = C.c_int64()
    _check(lib.fta_logprobs_workspace(C.byref(a), C.byref(need)))
    out = _logprob_outputs(lead, None if token_ids is None else token_ids.size(-1), top_k, dev)
    _fill_outputs(a, out)
    a.workspace_bytes = need.value
    if need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=dev)
        a.workspace = workspace.data_ptr()
    with torch.cuda.device(dev):
        _check(lib.fta_logprobs(C.byref(a), _current_stream(dev.index)))
    fields = ("logprobs", "entropy", "lse", "top_logprobs", "top_ids")
    _remember_call(hit, lib.fta_logprobs, a, dev, (("logits", 1, logits, rows), ("token_ids", 2, token_ids, ids)),
                   tuple((f, -1, t) for f, t in zip(fields, out) if t is not None))
    return TokenLogprobs(*out)


def accept_tree_path(tree_tokens: torch.Tensor, parents: torch.Tensor, target_tokens: torch.Tensor, *,
                     max_accept: Optional[int] = None, len_dtype: torch.dtype = torch.int64) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Walks every draft tree from its root along the nodes whose token is what the model picked.

      tree_tokens    int32 / int64 [bsz, q_len]: the token of every node; node 0 is the root, the last certain token
      parents        int32 / int64 [q_len] or [bsz, q_len]: parent of every node, parents before children, root -1.
                     A node > 0 whose parent is not in [0, its own index) hangs nowhere (padding) and is not accepted
      target_tokens  int32 / int64 [bsz, q_len]: the token the model picks after each node (the largest logit's,
                     `token_logprobs(...).top_ids[..., 0]`, or a sample of its distribution)
      max_accept     nodes to accept at most, the root included (default q_len)
    The root is always accepted; from an accepted node the path goes on to its first child, in index order, that
    holds the node's target token. Returns
      accept_idx   int32 [bsz, max_accept]: the path's nodes, 0 behind them     } what `append_accepted_kv` takes
      accept_len   [bsz] in `len_dtype` (int32 or int64, as the cache lengths)  }
      next_token   [bsz] in target_tokens' dtype: the target at the path's last node
    """
    lib = _lib.load()
    hit = _lib.binding().recall(_calls(), "accept", tree_tokens, parents, target_tokens, max_accept, len_dtype)
    if hit.__class__ is tuple:
        if hit[0]:
            _check(hit[0])
        return hit[1:]
    dev = tree_tokens.device
    if dev.type != "cuda":
        raise RuntimeError("accept_tree_path runs on the GPU only; there is no CPU fallback")
    if tree_tokens.dim() != 2 or tree_tokens.numel() == 0 or target_tokens.shape != tree_tokens.shape:
        raise ValueError("tree_tokens and target_tokens must be [bsz, q_len]")
    bsz, L = tree_tokens.shape
    if tuple(parents.shape) not in ((L,), (1, L), (bsz, L)):
        raise ValueError("parents must be [q_len] or [bsz, q_len]")
    for name, t in (("tree_tokens", tree_tokens), ("parents", parents), ("target_tokens", target_tokens)):
        if t.dtype not in _INT_DTYPES or t.device != dev:
            raise ValueError(f"{name} must be an int32 / int64 tensor on tree_tokens' device")
    if max_accept is not None and not 1 <= int(max_accept) <= 1 << 30:
        raise ValueError("max_accept must be between 1 (the root) and 2^30")
    if len_dtype not in _INT_DTYPES:
        raise ValueError("len_dtype must be torch.int32 or torch.int64")
    a = _lib.FtaAcceptArgs()
    a.bsz, a.q_len, a.max_accept = bsz, L, L if max_accept is None else int(max_accept)
    a.token_dtype, a.target_dtype = _INT_DTYPES[tree_tokens.dtype], _INT_DTYPES[target_tokens.dtype]
    a.parent_dtype, a.len_dtype = _INT_DTYPES[parents.dtype], _INT_DTYPES[len_dtype]
    a.token_stride[:], a.target_stride[:] = tree_tokens.stride(), target_tokens.stride()
    per_sequence = parents.dim() == 2 and parents.size(0) > 1
    a.parent_stride[:] = (parents.stride(0) if per_sequence else 0, parents.stride(-1))
    idx = torch.empty((a.bsz, a.max_accept), dtype=torch.int32, device=dev)
    count = torch.empty(a.bsz, dtype=len_dtype, device=dev)
    token = torch.empty(a.bsz, dtype=target_tokens.dtype, device=dev)
    a.tree_tokens, a.parents, a.target_tokens = tree_tokens.data_ptr(), parents.data_ptr(), target_tokens.data_ptr()
    a.accept_idx, a.accept_len, a.next_token = idx.data_ptr(), count.data_ptr(), token.data_ptr()
    with torch.cuda.device(dev):
        _check(lib.fta_accept_path(C.byref(a), _current_stream(dev.index)))
    _remember_call(hit, lib.fta_accept_path, a, dev, (("tree_tokens", 1, tree_tokens, tree_tokens), ("parents", 2, parents, parents),
                                                      ("target_tokens", 3, target_tokens, target_tokens)),
                   (("accept_idx", -1, idx), ("accept_len", -1, count), ("next_token", -1, token)))
    return idx, count, token
