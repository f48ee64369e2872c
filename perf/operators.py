"""Cases for measuring the operators around one tree-attention call of speculative decoding: rotary positions of the
tree's queries and keys, tree attention with shaped scores (cap, distance bias, window, document start), log
probabilities with entropy and top alternatives, and the accepted path.

With `own` false, `run` computes an operator in elementary torch operations in 32 bits (rotary angles in 64); with
`own` true it makes the calls a user makes of this package. `exact` is the definition in 64 bits."""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------------------------- cases
def _attention(name, **kw):
    case = dict(op="attention", bsz=1, heads=8, kv_heads=8, q_len=4, head_dim=64, cache=256, shortest=256, dtype="bf16",
                softcap=0.0, slopes=False, window=0, first_key=False, page=0, packed=False)
    case.update(kw)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the smallest verification call: one short sequence in fp32, a chain of four tokens, a capped score
        _attention("attn_short_fp32", dtype="f32", softcap=30.0, window=128),
        # plain decode of one token on a grouped-query model with capped scores, eight sequences
        _attention("attn_one_token_bf16", bsz=8, heads=32, kv_heads=8, q_len=1, head_dim=128, cache=4096, shortest=1024, softcap=50.0),
        # a draft tree of 26 nodes on a multi-head model with distance biases, paged cache, ragged lengths
        _attention("attn_tree26_paged_f16", bsz=4, heads=32, kv_heads=32, q_len=26, head_dim=128, cache=4096, shortest=1024, dtype="f16",
                   slopes=True, page=64, packed=True),
        # a tree of 64 nodes on a grouped-query model, 8192 cached keys, capped scores: the compute-heavy middle
        _attention("attn_tree64_8k_bf16", bsz=8, heads=32, kv_heads=8, q_len=64, head_dim=128, cache=8192, shortest=8192, softcap=50.0),
        # a large ragged batch with documents that start inside the cache rows: the largest call
        _attention("attn_ragged_32k_bf16", bsz=64, heads=64, kv_heads=8, q_len=16, head_dim=128, cache=32768, shortest=512, softcap=30.0,
                   slopes=True, first_key=True),
        # one token far into a long cache, on the interleaved layout (latency)
        dict(op="rotary", name="rotary_one_token_bf16", bsz=1, heads=32, kv_heads=8, q_len=1, head_dim=128, rotary_dim=128, dtype="bf16",
             interleaved=True, scaling="none", cache=131072, inverse=False),
        # a prompt chunk: half layout, part of the head, positions scaled by parts for a long context
        dict(op="rotary", name="rotary_chunk_f16", bsz=8, heads=32, kv_heads=8, q_len=2048, head_dim=128, rotary_dim=64, dtype="f16",
             interleaved=False, scaling="by_parts", cache=32768, inverse=False),
        # one step of one sequence: a single row of logits, the token's log probability and five alternatives
        dict(op="logprobs", name="logprobs_one_row_f32", rows=1, q_len=1, vocab=32000, ids=1, top_k=5, temperature=1.0, dtype="f32", banned=False),
        # a batch of small trees, a vocabulary that is no multiple of anything, some tokens banned, a temperature
        dict(op="logprobs", name="logprobs_tree26_f16", rows=4, q_len=26, vocab=50001, ids=4, top_k=10, temperature=0.7, dtype="f16", banned=True),
        # a batch of trees of 64 over a large vocabulary
        dict(op="logprobs", name="logprobs_tree64_bf16", rows=8, q_len=64, vocab=131072, ids=1, top_k=20, temperature=1.0, dtype="bf16", banned=False),
        # one tree of 26 nodes (latency)
        dict(op="accept", name="accept_tree26", bsz=1, q_len=26, max_accept=26, wide=False),
        # a large batch of trees, each with a shape of its own
        dict(op="accept", name="accept_batch256", bsz=256, q_len=256, max_accept=64, wide=True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "logprobs", "accept"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([32, 64, 128, 256])
        q_len = _log_int(rng, 1, 160)
        cache = _log_int(rng, 64, 32768)
        most = 64 * 64 * 16 * 32768 * 128 // (16 if dtype == "f32" else 1)   # fp32 products run at a sixteenth of the rate
        room = max(1, most // (heads * q_len * head_dim * cache))
        room = min(room, max(1, 64 * 8 * 32768 * 128 // (kv_heads * cache * head_dim)))
        bsz = _log_int(rng, 1, min(64, room))
        page = rng.choice([0, 0, 16, 32, 64, 128])
        return _attention(None, bsz=bsz, heads=heads, kv_heads=kv_heads, q_len=q_len, head_dim=head_dim, cache=cache,
                          shortest=rng.randint(0, cache), dtype=dtype, softcap=rng.choice([0.0, 20.0, 50.0]), slopes=rng.random() < 0.5,
                          window=rng.choice([0, 0, rng.randint(1, cache)]), first_key=rng.random() < 0.3, page=page, packed=rng.random() < 0.4)
    if op == "rotary":
        kv_heads = rng.choice([1, 2, 4, 8, 16])
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([32, 64, 128, 256])
        q_len = _log_int(rng, 1, 2048)
        room = max(1, 8 * 40 * 2048 * 128 // ((heads + kv_heads) * q_len * head_dim) // (2 if dtype == "f32" else 1))
        return dict(op="rotary", bsz=_log_int(rng, 1, min(64, room)), heads=heads, kv_heads=kv_heads, q_len=q_len, head_dim=head_dim,
                    rotary_dim=rng.choice([head_dim, head_dim // 2, 2 * rng.randint(1, head_dim // 2)]), dtype=dtype,
                    interleaved=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "base", "by_parts"]),
                    cache=_log_int(rng, 1, 1048576), inverse=rng.random() < 0.2)
    if op == "logprobs":
        vocab = _log_int(rng, 100, 200000)
        q_len = _log_int(rng, 1, 64)
        room = max(1, 8 * 64 * 131072 // (vocab * q_len) // (2 if dtype == "f32" else 1))
        return dict(op="logprobs", rows=_log_int(rng, 1, min(64, room)), q_len=q_len, vocab=vocab, ids=rng.randint(1, 6),
                    top_k=rng.randint(1, 32), temperature=rng.choice([1.0, 0.6, 1.7]), dtype=dtype, banned=rng.random() < 0.5)
    q_len = _log_int(rng, 1, 512)
    return dict(op="accept", bsz=_log_int(rng, 1, 256 * 256 // max(q_len, 256)), q_len=q_len, max_accept=rng.randint(1, q_len), wide=rng.random() < 0.5)


def _visible_keys(case):
    """Expected visible cache keys over the batch, per row (lengths are uniform between `shortest` and `cache`)."""
    keys = case["bsz"] * (case["shortest"] + case["cache"]) / 2
    if case["first_key"]:
        keys *= 0.875      # documents start in the first quarter of their row
    if case["window"]:
        keys = min(keys, case["bsz"] * case["window"])
    return keys


def work(case):
    if case["op"] == "attention":
        es, d = _BYTES[case["dtype"]], case["head_dim"]
        keys = _visible_keys(case)
        rows = case["bsz"] * case["q_len"]
        moved = 2 * case["kv_heads"] * (keys + rows) * d * es + 2 * case["heads"] * rows * d * es
        moved += case["q_len"] * (8 * ((case["q_len"] + 63) // 64) if case["packed"] else 4 * case["q_len"])
        return {"bytes": moved, "flops": 4 * case["heads"] * case["q_len"] * d * (keys + rows)}
    if case["op"] == "rotary":
        n = case["bsz"] * (case["heads"] + case["kv_heads"]) * case["q_len"]
        return {"bytes": 2 * n * case["head_dim"] * _BYTES[case["dtype"]], "flops": 3 * n * case["rotary_dim"]}
    if case["op"] == "logprobs":
        n = case["rows"] * case["q_len"]
        return {"bytes": n * (case["vocab"] * _BYTES[case["dtype"]] + case["ids"] * 12 + case["top_k"] * 12 + 8), "flops": 6 * n * case["vocab"]}
    n = case["bsz"] * case["q_len"]
    return {"bytes": 20 * n + 4 * case["bsz"] * case["max_accept"] + 16 * case["bsz"], "flops": n}


# --------------------------------------------------------------------------------------------- inputs
def _tree(bsz, q_len, gen, dev, reach):
    """Parents of random trees: node i hangs below one of the `reach` nodes in front of it. [bsz, q_len], root -1."""
    i = torch.arange(q_len, device=dev)
    back = torch.randint(1, reach + 1, (bsz, q_len), generator=gen, device=dev)
    return torch.where(i > 0, (i - back).clamp_min(0), -1)


def _ancestors(parents):
    """Boolean [.., L, L]: j is i or an ancestor of i. Paths double with every squaring."""
    q_len = parents.size(-1)
    a = torch.eye(q_len, device=parents.device) + torch.nn.functional.one_hot(parents.clamp_min(0), q_len).float() * (parents >= 0).unsqueeze(-1)
    for _ in range(max(1, (q_len - 1).bit_length())):
        a = (torch.matmul(a, a.contiguous()) > 0).float()
    return a > 0


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    state = dict(case=case)
    if case["op"] == "attention":
        dt, b, h, hk, n, d, t = _DTYPES[case["dtype"]], case["bsz"], case["heads"], case["kv_heads"], case["q_len"], case["head_dim"], case["cache"]
        normal = lambda *shape: torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dt)
        state.update(q=normal(b, h, n, d), current_k=normal(b, hk, n, d), current_v=normal(b, hk, n, d))
        if case["page"]:
            per = -(-t // case["page"])
            state["tables"] = torch.randperm(b * per, generator=gen, device=dev).to(torch.int32).view(b, per)
            state.update(k=normal(b * per, hk, case["page"], d), v=normal(b * per, hk, case["page"], d))
        else:
            state.update(k=normal(b, hk, t, d), v=normal(b, hk, t, d), tables=None)
        # lengths spread evenly over the range, in an order of their own
        spread = torch.linspace(case["shortest"], t, b, device=dev, dtype=torch.float64) if b > 1 else torch.tensor([float(t)], device=dev)
        state["lens"] = spread.round().long()[torch.randperm(b, generator=gen, device=dev)]
        parents = _tree(1, n, gen, dev, 4)[0]
        seen = _ancestors(parents)
        state["depths"] = (seen.sum(-1) - 1).to(torch.int32)
        state["seen"] = seen
        state["mask"] = torch.zeros(n, n, device=dev).masked_fill_(~seen, float("-inf"))
        if case["packed"]:
            bits = torch.nn.functional.pad(seen, (0, -n % 64)).view(n, -1, 64).long()
            state["mask"] = (bits << torch.arange(64, device=dev)).sum(-1)
        state["slopes"] = 2.0 ** (-8.0 * torch.arange(1, h + 1, device=dev, dtype=torch.float32) / h) if case["slopes"] else None
        state["first"] = (state["lens"].double() * torch.rand(b, generator=gen, device=dev, dtype=torch.float64) / 4).int() if case["first_key"] else None
        state["scale"] = d ** -0.5
    elif case["op"] == "rotary":
        dt, b, n, d = _DTYPES[case["dtype"]], case["bsz"], case["q_len"], case["head_dim"]
        state["q"] = torch.randn(b, case["heads"], n, d, generator=gen, device=dev).to(dt)
        state["k"] = torch.randn(b, case["kv_heads"], n, d, generator=gen, device=dev).to(dt)
        state["depths"] = torch.arange(n, device=dev, dtype=torch.int32)
        state["lens"] = torch.randint(case["cache"] // 2, case["cache"], (b,), generator=gen, device=dev)
        state["inv_freq"], state["factor"] = _frequencies(case)
        state["inv_freq"] = state["inv_freq"].to(dev)
    elif case["op"] == "logprobs":
        dt, n, vocab = _DTYPES[case["dtype"]], case["rows"], case["vocab"]
        x = torch.randn(n, case["q_len"], vocab, generator=gen, device=dev)
        # sharper in some rows than in others, as next-token logits are
        x = x * (1.0 + 3.0 * torch.rand(n, case["q_len"], 1, generator=gen, device=dev))
        if case["banned"]:
            x.masked_fill_(torch.rand(vocab, generator=gen, device=dev) < 0.3, float("-inf"))
            x[..., vocab // 2] = 0.5
        state["logits"] = x.to(dt)
        state["ids"] = torch.randint(0, vocab, (n, case["q_len"], case["ids"]), generator=gen, device=dev)
    else:
        b, n = case["bsz"], case["q_len"]
        state["parents"] = _tree(b if case["wide"] else 1, n, gen, dev, 3).to(torch.int32)
        state["ancestors"] = _ancestors(state["parents"].long())
        # few distinct tokens, so that siblings repeat; most nodes' targets are a child's token, so that paths get long
        state["tokens"] = torch.randint(0, 50, (b, n), generator=gen, device=dev)
        target = torch.randint(0, 50, (b, n), generator=gen, device=dev)
        parents = state["parents"].long().expand(b, n)
        row = torch.arange(b, device=dev).unsqueeze(1).expand(b, n)
        keep = (torch.rand(b, n, generator=gen, device=dev) < 0.95) & (parents >= 0)
        # the last child in index order that is kept sets the target (one writer each: deterministic)
        order = torch.arange(n, device=dev).expand(b, n)
        last = torch.full((b, n), -1, device=dev).scatter_reduce_(1, parents.clamp_min(0), torch.where(keep, order, -1), "amax")
        state["target"] = torch.where(last >= 0, state["tokens"][row, last.clamp_min(0)], target)
    return state


def _frequencies(case):
    """What a model's configuration gives: inverse frequencies of the pairs and the factor on the rotated values."""
    rd, base, scaling, factor = case["rotary_dim"], 10000.0, case["scaling"], 8.0
    if scaling == "base":
        base *= factor ** (rd / max(rd - 2, 1))
    inv = base ** (-torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    if scaling == "linear":
        return inv / factor, 1.0
    if scaling == "by_parts":
        turns = 4096 * inv / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        return inv * keep + inv / factor * (1 - keep), 0.1 * math.log(factor) + 1.0
    return inv, 1.0


# ------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "rotary": _plain_rotary, "logprobs": _plain_logprobs, "accept": _plain_accept}[state["case"]["op"]](state)


def _own(s):
    import flash_tree_attn_amd as fta
    c = s["case"]
    if c["op"] == "attention":
        return fta.shaped_tree_attention(s["q"], s["k"], s["v"], s["current_k"], s["current_v"], s["mask"], s["lens"], softcap=c["softcap"],
                                         slopes=s["slopes"], window=c["window"], first_key=s["first"], depths=s["depths"],
                                         sm_scale=s["scale"], kv_group_num=c["heads"] // c["kv_heads"], block_tables=s["tables"])
    if c["op"] == "rotary":
        return fta.apply_rotary(s["q"], s["k"], s["depths"], s["inv_freq"], kv_seq_len=s["lens"], interleaved=c["interleaved"],
                                attention_factor=s["factor"], inverse=c["inverse"])
    if c["op"] == "logprobs":
        r = fta.token_logprobs(s["logits"], s["ids"], top_k=c["top_k"], temperature=c["temperature"])
        return [r.logprobs, r.entropy, r.top_logprobs, r.top_ids]
    return list(fta.accept_tree_path(s["tokens"], s["parents"], s["target"], max_accept=c["max_accept"]))


def _plain_attention(s):
    c = s["case"]
    b, h, n, d = s["q"].shape
    hk, g = c["kv_heads"], c["heads"] // c["kv_heads"]
    k, v = s["k"], s["v"]
    if s["tables"] is not None:      # [pages, heads, page, d] -> [b, heads, t, d]
        k = k[s["tables"].long()].permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
        v = v[s["tables"].long()].permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)
    t = k.size(2)
    keys = torch.cat([k, s["current_k"]], 2).float().transpose(2, 3).contiguous()
    values = torch.cat([v, s["current_v"]], 2).float()
    z = torch.matmul(s["q"].float().view(b, hk, g * n, d), keys).view(b, h, n, t + n) * s["scale"]
    del keys
    if c["softcap"]:
        z = torch.tanh(z / c["softcap"]) * c["softcap"]
    rows = s["lens"].view(b, 1) + s["depths"]                                              # positions of the queries [b, n]
    cols = torch.cat([torch.arange(t, device=z.device).expand(b, t), rows], 1)             # and of the keys [b, t + n]
    dist = rows.unsqueeze(2) - cols.unsqueeze(1)                                           # [b, n, t + n]
    if s["slopes"] is not None:
        z -= s["slopes"].view(1, h, 1, 1) * dist.float().unsqueeze(1)
    j = torch.arange(t, device=z.device)
    cached = j < s["lens"].view(b, 1)
    if s["first"] is not None:
        cached = cached & (j >= s["first"].view(b, 1))
    seen = torch.cat([cached.unsqueeze(1).expand(b, n, t), s["seen"].expand(b, n, n)], 2)
    if c["window"]:
        seen = seen & (dist < c["window"])
    z.masked_fill_(~seen.unsqueeze(1), float("-inf"))
    z -= z.amax(-1, keepdim=True)
    z.exp_()
    total = z.sum(-1, keepdim=True)
    out = torch.matmul(z.view(b, hk, g * n, t + n), values.contiguous()).view(b, h, n, d) / total
    return out.to(s["q"].dtype)


def _plain_rotary(s):
    c = s["case"]
    rd = c["rotary_dim"]
    pos = (s["lens"].view(-1, 1) + s["depths"]).double()
    angle = pos.unsqueeze(-1) * s["inv_freq"]
    sin = torch.sin(angle) * (-1.0 if c["inverse"] else 1.0)
    cos, sin = (torch.cos(angle) * s["factor"]).float().unsqueeze(1), (sin * s["factor"]).float().unsqueeze(1)      # [b, 1, n, rd / 2]

    def turn(x):
        y = x[..., :rd].float()
        if c["interleaved"]:
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        else:
            a, b = y[..., : rd // 2], y[..., rd // 2:]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        return torch.cat([y.to(x.dtype), x[..., rd:]], -1)

    return turn(s["q"]), turn(s["k"])


def _plain_logprobs(s):
    c = s["case"]
    raw = s["logits"].float()
    x = raw / c["temperature"]
    x = x - x.amax(-1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(-1, keepdim=True)
    logp = x - torch.log(total)
    entropy = torch.log(total).squeeze(-1) - torch.where(e > 0, e * x, 0.0).sum(-1) / total.squeeze(-1)
    top = torch.sort(raw, dim=-1, descending=True, stable=True).indices[..., : c["top_k"]]
    return [torch.gather(logp, -1, s["ids"]), entropy, torch.gather(logp, -1, top), top]


def _plain_accept(s):
    c = s["case"]
    b, n = s["tokens"].shape
    parents = s["parents"].long().expand(b, n)
    i = torch.arange(n, device=parents.device)
    match = (torch.gather(s["target"], 1, parents.clamp_min(0)) == s["tokens"]) & (parents >= 0)
    # of several matching children of one parent the first in index order counts
    first = torch.full((b, n), n, device=parents.device).scatter_reduce_(1, parents.clamp_min(0), torch.where(match, i, n), "amin")
    match = match & (torch.gather(first, 1, parents.clamp_min(0)) == i)
    match[:, 0] = True
    depth = s["ancestors"].sum(-1) - 1
    on_path = ((s["ancestors"] & ~match.unsqueeze(1)).sum(-1) == 0) & (depth < c["max_accept"])
    order = torch.where(on_path, i, n).sort(1).values[:, : c["max_accept"]]
    accept_len = on_path.sum(1)
    last = torch.where(on_path, i, 0).amax(1, keepdim=True)
    return [torch.where(order < n, order, 0).to(torch.int32), accept_len, torch.gather(s["target"], 1, last).squeeze(1)]


# ------------------------------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    if case["op"] == "logprobs":
        x = s["logits"].double() / case["temperature"]
        lse = torch.logsumexp(x, -1, keepdim=True)
        p = torch.exp(x - lse)
        entropy = torch.special.entr(p).sum(-1)
        best = torch.sort(s["logits"].double(), dim=-1, descending=True, stable=True).values[..., : case["top_k"]] / case["temperature"]
        return [torch.gather(x, -1, s["ids"]) - lse, entropy, best - lse, None]
    return None


def _exact_attention(case, s):
    b, h, n, d = s["q"].shape
    hk, g = case["kv_heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(b, h, n, d, dtype=torch.float64, device=s["q"].device)
    for i in range(b):
        length = int(s["lens"][i])
        first = int(s["first"][i]) if s["first"] is not None else 0
        if s["tables"] is not None:
            rows = [x[s["tables"][i].long()].transpose(0, 1).reshape(hk, -1, d) for x in (s["k"], s["v"])]
        else:
            rows = [s["k"][i], s["v"][i]]
        k, v = (torch.cat([x[:, first:length], y[i]], 1).double() for x, y in zip(rows, (s["current_k"], s["current_v"])))
        q_pos = length + s["depths"].double()
        k_pos = torch.cat([torch.arange(first, length, device=k.device, dtype=torch.float64), q_pos])
        allowed = torch.cat([torch.ones(n, length - first, dtype=torch.bool, device=k.device), s["seen"]], 1)
        away = q_pos[:, None] - k_pos[None, :]
        if case["window"]:
            allowed &= away < case["window"]
        for head in range(hk):       # one group of query heads at a time
            q = s["q"][i, head * g:(head + 1) * g].double()
            z = torch.matmul(q.reshape(g * n, d), k[head].t().contiguous()).view(g, n, -1) * s["scale"]
            if case["softcap"]:
                z = case["softcap"] * torch.tanh(z / case["softcap"])
            if s["slopes"] is not None:
                z = z - s["slopes"][head * g:(head + 1) * g].double().view(g, 1, 1) * away
            p = torch.softmax(z.masked_fill(~allowed, float("-inf")), -1)
            out[i, head * g:(head + 1) * g] = torch.matmul(p.view(g * n, -1), v[head].contiguous()).view(g, n, d)
    return out


def _exact_rotary(case, s):
    rd = case["rotary_dim"]
    pos = s["lens"].view(-1, 1, 1, 1).double() + s["depths"].view(1, 1, -1, 1).double()
    angle = pos * s["inv_freq"] * (-1 if case["inverse"] else 1)
    turn = torch.polar(torch.full_like(angle, s["factor"]), angle)
    got = []
    for x in (s["q"].double(), s["k"].double()):
        half = x[..., :rd].unflatten(-1, (-1, 2)) if case["interleaved"] else x[..., :rd].unflatten(-1, (2, -1)).transpose(-1, -2)
        pair = torch.view_as_real(torch.view_as_complex(half.contiguous()) * turn)
        pair = pair if case["interleaved"] else pair.transpose(-1, -2)
        got.append(torch.cat([pair.flatten(-2), x[..., rd:]], -1))
    return tuple(got)
