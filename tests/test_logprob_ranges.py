"""Token log probabilities at the ends of what logits and temperatures may be (the kernel's source on host threads, and on
the GPU): tokens banned with the type's lowest value, temperatures near 0."""
import ctypes as C

import pytest
import torch

from flash_tree_attn_amd import TokenLogprobs, _lib, token_logprobs
from step_host import host_step_lib  # noqa: F401  (fixture)

DEV = "cuda"
DTYPES = {torch.float32: _lib.FTA_F32, torch.float16: _lib.FTA_F16, torch.bfloat16: _lib.FTA_BF16}


def definition(x, ids, top_k, temperature):
    """In 64 bits, relative to the rows' maxima: next to 3e38 even 64 bits would lose a sum's logarithm."""
    y = x.double()
    top = y.amax(-1, keepdim=True)
    d = (y - top) / temperature
    log_sum = torch.logsumexp(d, -1, keepdim=True)
    logp = d - log_sum
    order = torch.sort(y, dim=-1, descending=True, stable=True).indices[..., :top_k]
    entropy = torch.special.entr(logp.exp()).sum(-1)
    return torch.gather(logp, -1, ids), entropy, (top / temperature + log_sum).squeeze(-1), torch.gather(logp, -1, order), order


def check(got, x, ids, top_k, temperature):
    """Against the definition in 64 bits, rounded to the outputs' 32 (what they cannot hold is an infinity there). Sums of up
    to 2^20 weights are off by 1.2e-5 relative, and the entropy and the logarithm by as much once each; a log probability
    adds the half steps of 1 / T (2^-24), of the difference to the maximum, of their product and of itself: 2^-22 of its
    size. Infinities and NaN have to be where the definition has them."""
    ref_logp, ref_entropy, ref_lse, ref_top, ref_ids = definition(x, ids, top_k, temperature)
    assert torch.equal(got.top_ids, ref_ids)
    for name, a, b in (("logprobs", got.logprobs, ref_logp), ("entropy", got.entropy, ref_entropy), ("lse", got.lse, ref_lse), ("top", got.top_logprobs, ref_top)):
        a, b = a.double(), b.float().double()
        finite = b.isfinite()
        assert torch.equal(a[~finite], b[~finite]), name
        far = (a[finite] - b[finite]).abs() - (1.2e-5 + 2.0 ** -22 * b[finite].abs() + 1.2e-5 * b[finite].abs().clamp_max(20))
        assert bool((far <= 0).all()), (name, a, b)


def host_call(lib, x, ids, top_k, temperature):
    rows = x.size(0)
    out = TokenLogprobs(torch.full((rows, ids.size(1)), 7.0), torch.full((rows,), 7.0), torch.full((rows,), 7.0), torch.full((rows, top_k), 7.0),
                        torch.full((rows, top_k), -7))
    a = _lib.FtaLogprobArgs()
    a.logits, a.rows, a.vocab, a.logits_stride = x.data_ptr(), rows, x.size(1), x.stride(0)
    a.token_ids, a.num_ids, a.id_dtype = ids.data_ptr(), ids.size(1), _lib.FTA_I64
    a.id_stride[:] = ids.stride()
    a.logprobs, a.entropy, a.lse, a.top_logprobs, a.top_ids = (t.data_ptr() for t in out)
    a.dtype, a.top_k, a.inv_temperature = DTYPES[x.dtype], top_k, 1.0 / temperature
    need = C.c_int64()
    assert lib.fta_logprobs_workspace(C.byref(a), C.byref(need)) == 0
    ws = torch.full((need.value // 8 + 2,), -1, dtype=torch.int64)
    a.workspace, a.workspace_bytes = (ws.data_ptr() + 15) // 16 * 16, need.value
    assert lib.fta_logprobs(C.byref(a), None) == 0
    return out


def banned(vocab, dtype, seed=0, device="cpu"):
    """Three rows: all but 35 tokens banned with the type's lowest value (in a row of several pieces, whole pieces of them),
    every token banned so, and a third of them."""
    g = torch.Generator().manual_seed(seed)
    x = (2 * torch.randn(3, vocab, generator=g)).to(dtype)
    low = torch.finfo(dtype).min
    allowed = torch.randperm(min(vocab, 3000), generator=g)[:35]
    x[0] = torch.full((vocab,), low, dtype=dtype).index_copy(0, allowed, x[0, allowed])
    x[1] = low
    x[2, torch.rand(vocab, generator=g) < 0.3] = low
    ids = torch.stack([torch.stack([allowed[3], torch.tensor(vocab - 1)])] * 3)
    return x.to(device), ids.to(device)


BANNED = [(700, torch.float32), (700, torch.bfloat16), (701, torch.float16), (40000, torch.float32), (70001, torch.bfloat16), (70000, torch.float16)]


@pytest.mark.parametrize("temperature", [1.0, 0.7, 2.0])
@pytest.mark.parametrize("vocab, dtype", BANNED)
def test_banned_with_the_lowest_value_on_host_threads(host_step_lib, vocab, dtype, temperature):  # noqa: F811
    x, ids = banned(vocab, dtype)
    check(host_call(host_step_lib, x, ids, 9, temperature), x, ids, 9, temperature)


def logits(rows, vocab, dtype, seed=0, device="cpu"):
    """Maxima between 21 and 33, the largest logit twice in the last row."""
    g = torch.Generator().manual_seed(seed)
    x = (5 * torch.randn(rows, vocab, generator=g)).to(dtype)
    x[torch.arange(rows), torch.randint(0, vocab, (rows,), generator=g)] = torch.linspace(21, 33, rows).to(dtype)
    x[-1, vocab // 2] = x[-1].max()
    ids = torch.stack([x.float().argmax(-1), torch.randint(0, vocab, (rows,), generator=g)], -1)
    return x.to(device), ids.to(device)


COLD = [(6, 900, torch.float32), (4, 1201, torch.bfloat16), (2, 30000, torch.float32), (2, 40001, torch.float16)]
TEMPERATURES = (1e-3, 1e-6, 1e-8, 1e-10, 1e-30)


@pytest.mark.parametrize("temperature", TEMPERATURES)
@pytest.mark.parametrize("rows, vocab, dtype", COLD)
def test_temperatures_near_zero_on_host_threads(host_step_lib, rows, vocab, dtype, temperature):  # noqa: F811
    x, ids = logits(rows, vocab, dtype)
    check(host_call(host_step_lib, x, ids, 3, temperature), x, ids, 3, temperature)


@pytest.mark.parametrize("inv_temperature, status", [(1.0, 0), (2.3e38, 0), (2.4e38, -9), (3.4e38, -9), (1e-44, 0)])
def test_a_temperature_whose_inverse_in_units_of_log2_e_does_not_fit_is_refused(fta_lib, inv_temperature, status):
    a = _lib.FtaLogprobArgs()
    a.rows, a.vocab, a.logits_stride, a.dtype, a.id_dtype, a.inv_temperature = 1, 10, 10, _lib.FTA_F32, _lib.FTA_I64, inv_temperature
    assert fta_lib.fta_logprobs_workspace(C.byref(a), C.byref(C.c_int64())) == status


@pytest.mark.parametrize("temperature", [4.4e-39, 1e38])
def test_the_least_and_largest_temperatures_on_host_threads(host_step_lib, temperature):  # noqa: F811
    x, ids = logits(3, 500, torch.float32, 2)
    check(host_call(host_step_lib, x, ids, 3, temperature), x, ids, 3, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("rows, vocab, dtype", COLD + [(300, 50001, torch.bfloat16), (70, 131072, torch.float32)])
def test_temperatures_near_zero(rows, vocab, dtype):
    for temperature in TEMPERATURES:
        x, ids = logits(rows, vocab, dtype, 1, DEV)
        check(token_logprobs(x, ids, top_k=3, temperature=temperature), x, ids, 3, temperature)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab, dtype", BANNED + [(131072, torch.float32), (131072, torch.bfloat16)])
def test_banned_with_the_lowest_value(vocab, dtype):
    for temperature in (1.0, 0.7, 2.0):
        for rows in (1, 100):      # few rows are cut into smaller pieces than many
            x, ids = banned(vocab, dtype, 1, DEV)
            x, ids = x.repeat(rows, 1), ids.repeat(rows, 1)
            check(token_logprobs(x, ids, top_k=9, temperature=temperature), x, ids, 9, temperature)


@pytest.mark.gpu
def test_rows_of_more_logits_than_an_int_counts_are_refused():
    for vocab in ((1 << 30) + 1, (1 << 32) + 5):
        with pytest.raises(ValueError, match="2\\^30"):
            token_logprobs(torch.zeros(1, 1, device=DEV, dtype=torch.bfloat16).expand(1, vocab))
