"""Token log probabilities (`fta_logprobs`, `token_logprobs`) and the accepted path (`fta_accept_path`,
`accept_tree_path`): refusals and the kernels' source on host threads (CPU), parity with the 64-bit definitions on the
GPU."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_amd import TokenLogprobs, _lib, accept_tree_path, random_tree_parents, token_logprobs
from oracle.step_oracle import accept_path_oracle, logprobs_oracle
from step_host import host_step_lib  # noqa: F401  (fixture)

DEV = "cuda"
DTYPES = {torch.float32: _lib.FTA_F32, torch.float16: _lib.FTA_F16, torch.bfloat16: _lib.FTA_BF16}


def check(got, logits, ids, top_k, temperature=1.0):
    """Bound of the 32-bit arithmetic. An exponent d = (x - m) / T log2 e carries 2 half steps: under the softmax the mean
    of |d| is at most log2 e (ln vocab + 1), so a sum of weights is off by 2^-23 (ln vocab + 1) relative, 2^-23 more for
    exp2 and, per thread, at most 129 additions in turn, 129 half steps; then some 20 more in the reductions: 150 half
    steps + 2^-23 (ln vocab + 2) < 1.2e-5 up to 2^20 tokens. ln and the entropy's quotient carry that error once each (the
    entropy's relative to its size); a log probability adds 3 half steps of (x - m) / T and of itself."""
    ref_ids, ref_entropy, ref_lse, ref_top, ref_top_ids = logprobs_oracle(logits, ids, top_k, temperature)
    near = lambda a, b, size: bool(((a.double() - b).abs() <= 1.2e-5 + 2.0 ** -22 * size + 1.2e-5 * size.clamp_max(20)).all())

    def same(a, b, size):
        a, finite = a.double(), b.isfinite()
        assert torch.equal(a[~finite].nan_to_num(1e300), b[~finite].nan_to_num(1e300))
        assert near(a[finite], b[finite], size[finite]), float((a[finite] - b[finite]).abs().max())

    same(got.entropy, ref_entropy, ref_entropy.abs())
    same(got.lse, ref_lse, ref_lse.abs())
    assert torch.equal(got.top_ids, ref_top_ids)
    same(got.top_logprobs, ref_top, ref_top.abs())
    if ids is not None:
        same(got.logprobs, ref_ids, ref_ids.abs())


# ---------------------------------------------------------------- CPU: refusals
def logprob_args(**kw):
    a = _lib.FtaLogprobArgs()
    for f in ("logits", "token_ids", "logprobs", "entropy", "lse", "top_logprobs", "top_ids"):
        setattr(a, f, 0x1000)
    cfg = dict(rows=2, vocab=100, num_ids=1, top_k=3, dtype=_lib.FTA_BF16, id_dtype=_lib.FTA_I64, inv_temperature=1.0, logits_stride=100)
    cfg.update(kw)
    for k, v in cfg.items():
        setattr(a, k, v)
    a.id_stride[:] = [1, 1]
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(logits=None), -1), (dict(entropy=None), -1), (dict(lse=None), -1), (dict(token_ids=None), -1), (dict(logprobs=None), -1), (dict(top_ids=None), -1),
    (dict(dtype=3), -6), (dict(id_dtype=4), -6), (dict(rows=0), -7), (dict(vocab=0), -7), (dict(num_ids=-1), -7), (dict(top_k=101), -7),
    (dict(top_k=129, vocab=1000), -9), (dict(inv_temperature=0.0), -9), (dict(inv_temperature=float("inf")), -9), (dict(inv_temperature=float("nan")), -9),
    (dict(vocab=(1 << 30) + 1), -9), (dict(logits_stride=-1), -8), (dict(logits=0x1001), -8), (dict(rows=1000, vocab=100000, logits_stride=100000), -1),
])
def test_logprob_argument_errors(fta_lib, kw, status):
    assert fta_lib.fta_logprobs(C.byref(logprob_args(**kw)), None) == status


def test_logprob_workspace(fta_lib):
    need = C.c_int64(-5)
    a = logprob_args(rows=1000, vocab=100000, logits_stride=100000)
    assert fta_lib.fta_logprobs_workspace(C.byref(a), C.byref(need)) == 0 and need.value > 0
    a.workspace, a.workspace_bytes = 0x1000, need.value - 1
    assert fta_lib.fta_logprobs(C.byref(a), None) == -5
    a.workspace, a.workspace_bytes = 0x1008, need.value
    assert fta_lib.fta_logprobs(C.byref(a), None) == -8
    assert fta_lib.fta_logprobs_workspace(C.byref(logprob_args()), C.byref(need)) == 0 and need.value == 0
    assert fta_lib.fta_logprobs_workspace(C.byref(logprob_args(rows=-1)), C.byref(need)) == -7
    if not torch.cuda.is_available():
        assert fta_lib.fta_logprobs(C.byref(logprob_args()), None) == -11


def accept_args(**kw):
    a = _lib.FtaAcceptArgs()
    for f in ("tree_tokens", "target_tokens", "parents", "accept_idx", "accept_len", "next_token"):
        setattr(a, f, 0x1000)
    cfg = dict(bsz=2, q_len=5, max_accept=5)
    cfg.update(kw)
    for k, v in cfg.items():
        setattr(a, k, v)
    for s in ("token_stride", "target_stride", "parent_stride"):
        getattr(a, s)[:] = [5, 1]
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(tree_tokens=None), -1), (dict(next_token=None), -1), (dict(token_dtype=2), -6), (dict(len_dtype=-1), -6), (dict(bsz=0), -7), (dict(q_len=0), -7),
    (dict(max_accept=0), -7), (dict(q_len=16385), -9), (dict(max_accept=(1 << 30) + 1), -9),
])
def test_accept_argument_errors(fta_lib, kw, status):
    assert fta_lib.fta_accept_path(C.byref(accept_args(**kw)), None) == status
    assert fta_lib.fta_accept_path(None, None) == -1


def test_python_wrappers_reject_cpu_tensors():
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_logprobs(torch.zeros(2, 10))
    z = torch.zeros(1, 3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        accept_tree_path(z, z[0], z)


# ---------------------------------------------------------------- inputs
LOGIT_CASES = [
    # rows vocab dtype ids top_k temperature kind
    (1, 1, torch.float32, 1, 1, 1.0, "plain"),
    (2, 7, torch.bfloat16, 2, 7, 0.7, "plain"),               # fewer logits than one granule
    (3, 1001, torch.float16, 3, 40, 1.0, "plain"),            # odd rows: every alignment of the first logit
    (5, 333, torch.float32, 1, 5, 2.0, "banned"),             # two thirds -inf
    (2, 4100, torch.bfloat16, 1, 128, 1.0, "equal"),          # every logit the same: more candidates than slots
    (2, 1500, torch.float16, 2, 33, 1.0, "empty row"),
    (2, 900, torch.float32, 1, 4, 1.0, "peaked"),
    (3, 600, torch.bfloat16, 1, 6, 1.0, "nan"),
    (2, 777, torch.float32, 0, 0, 1.0, "plain"),
    (3, 153, torch.bfloat16, 1, 22, 1.0, "banned"),           # fewer groups of threads with logits than alternatives
    (2, 400, torch.float16, 1, 60, 1.0, "plain"),
    (2, 2000, torch.float32, 1, 30, 1.0, "nearly empty"),     # fewer finite logits than alternatives
    (2, 5000, torch.bfloat16, 1, 12, 1.0, "one corner"),      # finite logits in few threads
]


def make_logits(case, seed, device="cpu"):
    rows, vocab, dtype, num_ids, _, _, kind = case
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * 3
    if kind == "banned":
        x[torch.rand(rows, vocab, generator=g) < 0.67] = float("-inf")
        x[:, vocab - 1] = 1.0
    elif kind == "equal":
        x[:] = -0.25
    elif kind == "empty row":
        x[rows - 1] = float("-inf")
    elif kind == "peaked":
        x[:, vocab // 3] = 90.0
    elif kind == "nearly empty":
        x[:, 7:] = float("-inf")
    elif kind == "one corner":
        x[:, 40:] = float("-inf")
    elif kind == "nan":
        x[0, 17] = float("nan")
    x = x.to(dtype)
    if kind == "plain" and vocab > 4:
        x[..., 1], x[..., 3] = 0.0, -0.0          # equal values: ascending ids
    ids = torch.randint(0, vocab, (rows, num_ids), generator=g)
    if num_ids > 1:
        ids[0, 0], ids[0, 1] = -1, vocab         # outside: -inf
    return x.to(device), ids.to(device)


# ---------------------------------------------------------------- CPU: host threads
@pytest.mark.parametrize("case", LOGIT_CASES + [
    (1, 170001, torch.float32, 2, 100, 1.0, "plain"),      # 11 chunks, joined in two rounds of keys
    (1, 140000, torch.bfloat16, 1, 20, 1.0, "equal"),
])
def test_logprob_kernel_source_on_host_threads(host_step_lib, case):
    rows, vocab, dtype, num_ids, top_k, temperature, _ = case
    x, ids = make_logits(case, 3)
    run_host(host_step_lib, x, ids, top_k, temperature)


def run_host(lib, x, ids, top_k, temperature):
    rows = x.size(0)
    a = _lib.FtaLogprobArgs()
    out = dict(logprobs=torch.full((rows, ids.size(1)), 7.0), entropy=torch.full((rows,), 7.0), lse=torch.full((rows,), 7.0),
               top_logprobs=torch.full((rows, top_k), 7.0), top_ids=torch.full((rows, top_k), -7))
    a.logits, a.rows, a.vocab, a.logits_stride = x.data_ptr(), rows, x.size(1), x.stride(0)
    a.token_ids, a.num_ids, a.id_dtype = ids.data_ptr(), ids.size(1), _lib.FTA_I64
    a.id_stride[:] = ids.stride()
    for n, t in out.items():
        setattr(a, n, t.data_ptr())
    a.dtype, a.top_k, a.inv_temperature = DTYPES[x.dtype], top_k, 1.0 / temperature
    need = C.c_int64()
    assert lib.fta_logprobs_workspace(C.byref(a), C.byref(need)) == 0
    ws = torch.full((need.value // 8 + 2,), -1, dtype=torch.int64)
    a.workspace, a.workspace_bytes = (ws.data_ptr() + 15) // 16 * 16, need.value
    assert lib.fta_logprobs(C.byref(a), None) == 0
    got = TokenLogprobs(**out)
    nan = x.isnan().any(-1)
    if nan.any():
        assert bool(got.entropy[nan].isnan().all() and got.lse[nan].isnan().all() and got.top_logprobs[nan].isnan().all())
        assert torch.equal(got.top_ids[nan], logprobs_oracle(x, None, top_k)[4][nan])
    keep = ~nan
    check(TokenLogprobs(*(t[keep] for t in got)), x[keep], ids[keep], top_k, temperature)


def tree_case(seed, bsz, L, one_tree=False, padded=False, distinct=4, int32=False):
    g = torch.Generator().manual_seed(seed)
    parents = torch.stack([random_tree_parents(L, g) for _ in range(1 if one_tree else bsz)])
    if padded:
        parents[:, L - L // 3:] = -1
        if L > 6:
            parents[0, 4], parents[0, 5] = 4, L + 3      # a node below itself, a parent out of range: hang nowhere
    tokens, targets = torch.randint(0, distinct, (bsz, L), generator=g), torch.randint(0, distinct, (bsz, L), generator=g)
    if int32:
        parents, tokens, targets = parents.int(), tokens.int(), targets.int()
    return tokens, parents[0] if one_tree else parents, targets


TREE_CASES = [(1, 1, 1, True, False, 1), (2, 3, 26, True, False, 2), (3, 5, 70, False, True, 1), (4, 2, 300, False, False, 1), (5, 4, 64, False, True, 3)]


@pytest.mark.parametrize("seed, bsz, L, one_tree, padded, distinct", TREE_CASES)
def test_accept_kernel_source_on_host_threads(host_step_lib, seed, bsz, L, one_tree, padded, distinct):
    tokens, parents, targets = tree_case(seed, bsz, L, one_tree, padded, distinct, int32=seed % 2 == 1)
    for width in sorted({L, 1, max(1, L // 2), L + 5}):
        a = _lib.FtaAcceptArgs()
        i64 = tokens.dtype == torch.int64
        idx, count, token = torch.full((bsz, width), -9, dtype=torch.int32), torch.full((bsz,), -9), torch.full((bsz,), -9, dtype=targets.dtype)
        a.tree_tokens, a.parents, a.target_tokens = tokens.data_ptr(), parents.data_ptr(), targets.data_ptr()
        a.accept_idx, a.accept_len, a.next_token = idx.data_ptr(), count.data_ptr(), token.data_ptr()
        a.bsz, a.q_len, a.max_accept = bsz, L, width
        a.token_dtype = a.target_dtype = a.parent_dtype = _lib.FTA_I64 if i64 else _lib.FTA_I32
        a.len_dtype = _lib.FTA_I64
        a.token_stride[:], a.target_stride[:] = tokens.stride(), targets.stride()
        a.parent_stride[:] = (0 if one_tree else L, 1)
        assert host_step_lib.fta_accept_path(C.byref(a), None) == 0
        for got, ref in zip((idx, count, token), accept_path_oracle(tokens, parents, targets, width)):
            assert torch.equal(got, ref)


# ---------------------------------------------------------------- GPU
@pytest.mark.gpu
@pytest.mark.parametrize("case", LOGIT_CASES + [
    (3, 50001, torch.float16, 4, 10, 0.7, "banned"), (200, 50001, torch.float32, 2, 20, 1.0, "plain"), (130, 131072, torch.bfloat16, 1, 32, 1.0, "plain"),
    (1, 131072, torch.bfloat16, 1, 5, 1.0, "peaked"), (1, 150000, torch.float16, 1, 128, 1.3, "plain"), (150, 40000, torch.bfloat16, 1, 64, 1.0, "equal"),
    (140, 70000, torch.float32, 2, 3, 1.0, "empty row"), (2, 600000, torch.float32, 1, 100, 1.0, "plain"),
])
def test_logprobs_match_the_definition(case):
    rows, vocab, dtype, num_ids, top_k, temperature, kind = case
    for seed in (1, 2):      # the second call runs from the remembered signature
        x, ids = make_logits(case, seed, DEV)
        got = token_logprobs(x, ids, top_k=top_k, temperature=temperature)
        again = token_logprobs(x, ids, top_k=top_k, temperature=temperature)
        for a, b in zip(got, again):
            assert torch.equal(a.nan_to_num(1e30), b.nan_to_num(1e30))      # the same bits every time
        nan = x.isnan().any(-1)
        if nan.any():
            assert bool(got.entropy[nan].isnan().all() and got.lse[nan].isnan().all() and got.logprobs[nan].isnan().all())
            assert torch.equal(got.top_ids[nan], logprobs_oracle(x, None, top_k)[4][nan])
        keep = ~nan
        check(type(got)(*(t[keep] for t in got)), x[keep], ids[keep], top_k, temperature)


@pytest.mark.gpu
def test_logprobs_of_strided_and_leading_dimensions():
    g = torch.Generator().manual_seed(9)
    big = torch.randn(3, 4, 1010, generator=g).to(torch.bfloat16).to(DEV)
    for x in (big[:, -1:, 3:1000], big[:, :, :999], big[0, 1], big.transpose(0, 1)):
        ids = torch.randint(0, x.size(-1), (*x.shape[:-1], 2), generator=g, dtype=torch.int32).to(DEV)
        got = token_logprobs(x, ids, top_k=3)
        assert got.logprobs.shape == ids.shape and got.entropy.shape == x.shape[:-1] and got.top_ids.shape == (*x.shape[:-1], 3)
        check(got, x, ids, 3)
    got = token_logprobs(big)
    assert got.logprobs is None and got.top_ids.shape == (3, 4, 0)
    check(got, big, None, 0)


@pytest.mark.gpu
def test_accept_matches_the_walk():
    for seed, bsz, L, one_tree, padded, distinct in TREE_CASES + [(6, 300, 64, False, True, 2), (7, 2, 5000, True, False, 1)]:
        for int32 in (False, True):
            tokens, parents, targets = tree_case(seed, bsz, L, one_tree, padded, distinct, int32)
            for width in (None, 3):
                for _ in range(2):
                    got = accept_tree_path(tokens.to(DEV), parents.to(DEV), targets.to(DEV), max_accept=width, len_dtype=torch.int32)
                ref = accept_path_oracle(tokens, parents, targets, width)
                assert got[0].dtype == torch.int32 and got[1].dtype == torch.int32 and got[2].dtype == targets.dtype
                assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu().long(), ref[1]) and torch.equal(got[2].cpu(), ref[2])


@pytest.mark.gpu
def test_refusals():
    x, ids = torch.zeros(2, 50, device=DEV), torch.zeros(2, 1, dtype=torch.int64, device=DEV)
    for args, kw in (((x.double(),), {}), ((x[:0],), {}), ((x, ids.float()), {}), ((x, ids[:1]), {}), ((x, ids.cpu()), {}), ((x, ids[0]), {}),
                     ((x,), dict(top_k=51)), ((x,), dict(top_k=-1)), ((torch.zeros(1, 500, device=DEV),), dict(top_k=129)),
                     ((x,), dict(temperature=0.0)), ((x,), dict(temperature=float("nan"))), ((x,), dict(temperature=-1.0))):
        with pytest.raises(ValueError):
            token_logprobs(*args, **kw)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
        token_logprobs(x.clone().requires_grad_())
    t = torch.zeros(2, 5, dtype=torch.int64, device=DEV)
    for args, kw in (((t[0], t, t), {}), ((t, t[:, :4], t), {}), ((t, t, t[:, :4]), {}), ((t.float(), t, t), {}), ((t, t.cpu(), t), {}), ((t, t, t), dict(max_accept=0)), ((t, t, t), dict(max_accept=1 << 32)), ((t, t, t), dict(max_accept=(1 << 30) + 1)),
                     ((t, t, t), dict(len_dtype=torch.int16)), ((t[:, :0], t[:, :0], t[:, :0]), {})):
        with pytest.raises(ValueError):
            accept_tree_path(*args, **kw)
