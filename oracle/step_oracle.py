"""Oracles of the operators around one tree-attention call: rotary positions, token log probabilities, the accepted path
and attention with shaped scores.

TEST INFRASTRUCTURE ONLY: the shipped package never imports this module. Plain torch in 64 bits (or Python loops), from
the formulas in include/fta.h, on whatever device the inputs live on. The reference has none of these operators: parity
is unpinned, the definitions are this library's own.
"""
from __future__ import annotations

from typing import Optional

import torch


def rotary_oracle(x, positions, inv_freq, kv_seq_len=None, interleaved=False, attention_factor=1.0, inverse=False):
    """x [bsz, heads, L, D] -> float64 of the same shape."""
    bsz, _, L, _ = x.shape
    pos = positions.reshape(-1, L).expand(bsz, L).double()
    if kv_seq_len is not None:
        pos = pos + kv_seq_len.reshape(bsz, 1).double()
    angle = pos[:, None, :, None] * inv_freq.double() * (-1.0 if inverse else 1.0)
    half = inv_freq.numel()
    y = x.double().clone()
    t = torch.arange(half, device=x.device)
    first, second = (2 * t, 2 * t + 1) if interleaved else (t, t + half)
    a, b = y[..., first], y[..., second]
    y[..., first] = attention_factor * (a * angle.cos() - b * angle.sin())
    y[..., second] = attention_factor * (b * angle.cos() + a * angle.sin())
    return y


def logprobs_oracle(logits, token_ids=None, top_k=0, temperature=1.0):
    """(logprobs, entropy, lse, top_logprobs, top_ids) in float64 / int64, rows of [..., vocab]."""
    y = logits.double() / temperature
    vocab = y.size(-1)
    empty = (y == float("-inf")).all(-1)
    lse = torch.logsumexp(y, -1)
    logp = torch.where(empty[..., None], float("-inf"), y - lse[..., None])
    p = logp.exp()
    entropy = -torch.where(p == 0, 0.0, p * logp).sum(-1)
    ids = None
    if token_ids is not None:
        inside = (token_ids >= 0) & (token_ids < vocab)
        ids = torch.where(inside, torch.gather(logp, -1, token_ids.long().clamp(0, vocab - 1)), float("-inf"))
    rank = logits.double()
    rank = torch.where(rank.isnan(), float("-inf"), rank)     # (tests keep NaN rows' top_k within their numbers)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :top_k]
    return ids, entropy, lse, torch.gather(logp, -1, order), order


def accept_path_oracle(tree_tokens, parents, target_tokens, max_accept=None):
    """Python loops: (accept_idx int32, accept_len int64, next_token)."""
    bsz, L = tree_tokens.shape
    width = L if max_accept is None else max_accept
    parents = parents.reshape(-1, L).expand(bsz, L).tolist()
    tokens, targets = tree_tokens.tolist(), target_tokens.tolist()
    idx = torch.zeros(bsz, width, dtype=torch.int32)
    count, following = [], []
    for b in range(bsz):
        node, path = 0, [0]
        while len(path) < width:
            child = next((i for i in range(node + 1, L) if parents[b][i] == node and tokens[b][i] == targets[b][node]), None)
            if child is None:
                break
            node = child
            path.append(node)
        idx[b, : len(path)] = torch.tensor(path, dtype=torch.int32)
        count.append(len(path))
        following.append(targets[b][node])
    return idx, torch.tensor(count), torch.tensor(following, dtype=target_tokens.dtype)


def shaped_attention_oracle(q, k_cache, v_cache, current_k, current_v, mask, kv_seq_len, *, softcap=0.0, slopes=None, window=0,
                            first_key=None, depths=None, sm_scale=None, block_tables=None):
    """Float64 [bsz, Hq, L, D]. `mask` additive or bool, broadcastable to [bsz, Hq, L, L]. Rows that see nothing are zero."""
    bsz, hq, L, D = q.shape
    hkv = k_cache.size(1)
    scale = D ** -0.5 if sm_scale is None else sm_scale
    if mask.dtype == torch.bool:
        mask = torch.zeros(mask.shape, dtype=torch.float64, device=q.device).masked_fill(~mask, float("-inf"))
    mask = mask.double().expand(bsz, hq, L, L)
    depth = torch.arange(L, device=q.device) if depths is None else depths
    depth = depth.reshape(-1, L).expand(bsz, L).double()
    out = torch.zeros(bsz, hq, L, D, dtype=torch.float64, device=q.device)
    for b in range(bsz):
        if block_tables is not None:
            k, v = (c[block_tables[b].long()].transpose(0, 1).reshape(hkv, -1, D) for c in (k_cache, v_cache))
        else:
            k, v = k_cache[b], v_cache[b]
        T = min(max(int(kv_seq_len[b]), 0), k.size(1))
        first = min(max(int(first_key[b]), 0), T) if first_key is not None else 0
        q_pos = T + depth[b]
        k_pos = torch.cat([torch.arange(first, T, device=q.device).double(), q_pos])
        away = q_pos[:, None] - k_pos[None, :]
        for h in range(hq):
            c = h // (hq // hkv)
            ch = h // (hq // current_k.size(1))
            keys = torch.cat([k[c, first:T], current_k[b, ch]]).double()
            values = torch.cat([v[c, first:T], current_v[b, ch]]).double()
            z = torch.matmul(q[b, h].double(), keys.t().contiguous()) * scale
            if softcap:
                z = softcap * torch.tanh(z / softcap)
            if slopes is not None:
                z = z - float(slopes[h]) * away
            z[:, T - first:] = torch.where(mask[b, h] == float("-inf"), float("-inf"), z[:, T - first:] + mask[b, h])
            if window:
                z = z.masked_fill(away >= window, float("-inf"))
            top = z.amax(-1, keepdim=True)
            p = torch.where(top == float("-inf"), 0.0, torch.exp(z - torch.where(top == float("-inf"), 0.0, top)))
            values = torch.where((p > 0).any(0)[:, None], values, 0.0)     # what no row sees adds nothing, whatever it holds
            out[b, h] = torch.matmul(p, values) / p.sum(-1, keepdim=True).clamp_min(1e-300)
    return out
