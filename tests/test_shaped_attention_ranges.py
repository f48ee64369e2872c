"""Shaped tree attention at the ends of what its arguments may be (the kernel's source on host threads, and on the GPU):
finite masks, from soft ones to the type's lowest value, in front of keys that count; caps that bind hardly or not at all;
many keys far below the one that leads."""
import pytest
import torch

from test_shaped_attention import case_inputs, check, gpu_call, host_call, host_lib, make, options, oracle  # noqa: F401  (host_lib: fixture)

DEV = "cuda"

# (bsz hq hkv L D cache dtype lens), options(): every way in which a wave may meet masked keys before those that count
MASKED = {
    "two waves a row, 48 nodes f32": ((1, 1, 1, 48, 64, 150, torch.float32, [150]), {}),
    "two waves a row, 48 nodes bf16": ((1, 1, 1, 48, 64, 150, torch.bfloat16, [150]), {}),
    "four waves a row": ((1, 1, 1, 30, 64, 200, torch.float32, [190]), dict(softcap=20.0)),
    "one wave a row, two tree tiles": ((1, 2, 1, 100, 64, 130, torch.bfloat16, [130]), dict(slopes=True)),
    "one wave a row, f32": ((1, 2, 1, 70, 128, 70, torch.float32, [70]), dict(softcap=30.0, slopes=True)),
    "cut, fp16": ((2, 2, 1, 6, 32, 600, torch.float16, [600, 70]), dict(softcap=30.0)),
    "cut, f32": ((1, 1, 1, 9, 32, 1030, torch.float32, [1030]), dict(slopes=True)),
}
VALUES = (torch.finfo(torch.float32).min, -1e9, -1e6, -1e4, -200.0)


def masked(name, value, seed=5, device="cpu"):
    """The tree's mask with `value` for -inf; the last node is padding: it sees no tree key, not even itself."""
    shape, opt = MASKED[name]
    x = make(seed, *shape, device=device)
    x["mask"][:, :, -1] = float("-inf")
    x["mask"] = x["mask"].masked_fill(x["mask"] == float("-inf"), value)
    return x, options(shape[1], shape[0], device=device, **opt)


@pytest.mark.parametrize("name, value", [(n, v) for n in MASKED for v in (VALUES[0], -1e9, -1e4) if v == -1e9 or not n.startswith("cut")])
def test_keys_behind_finite_masks_on_host_threads(host_lib, name, value):  # noqa: F811
    x, opt = masked(name, value)
    check(host_call(host_lib, x, opt), oracle(x, opt), x, opt)


@pytest.mark.gpu
@pytest.mark.parametrize("name", MASKED)
def test_keys_behind_finite_masks(name):
    for value in VALUES:
        x, opt = masked(name, value, device=DEV)
        got = gpu_call(x, opt)
        check(got, oracle(x, opt), x, opt)
        x["mask"] = x["mask"].masked_fill(x["mask"] == value, float("-inf"))
        if value < -1e5:      # such a key weighs nothing next to any other
            check(got, oracle(x, opt), x, opt)


# softcap, (bsz hq hkv L D cache dtype lens), options()
CAPPED = [(cap, shape, opt) for cap in (200.0, 300.0, 1e3, 1e5, 1e8, 2e38) for shape, opt in (
    ((1, 2, 1, 5, 64, 130, torch.float16, [130]), {}),
    ((1, 2, 1, 40, 64, 100, torch.bfloat16, [100]), dict(slopes=True)),
    ((1, 2, 1, 3, 32, 100, torch.float32, [97]), {}),
)]


def check_capped(got, x, opt):
    """`check`, with a cap that large counted as the scores are: |cap tanh(x / cap)| <= |x|, and no step of the arithmetic may
    be larger than what it gives. The scores are up to 20: 16-bit calls may put 2^-21 of a cap up to 256 into an exponent
    (under 2^-13, a quarter of fp16's half step of the weights, which `check` counts twice over)."""
    check(got, oracle(x, opt), x, dict(opt, softcap=min(opt["softcap"], 20.0)))


@pytest.mark.parametrize("cap, shape, opt", CAPPED)
def test_large_caps_on_host_threads(host_lib, cap, shape, opt):  # noqa: F811
    x = make(7, *shape)
    x["q"] = x["q"] * 3
    opt = options(shape[1], shape[0], softcap=cap, **opt)
    check_capped(host_call(host_lib, x, opt), x, opt)


@pytest.mark.gpu
@pytest.mark.parametrize("cap, shape, opt", CAPPED + [(c, (2, 8, 2, 64, 128, 2000, t, [2000, 1500]), {}) for c in (255.0, 257.0, 1e6) for t in (torch.float16, torch.bfloat16)])
def test_large_caps(cap, shape, opt):
    x = make(7, *shape, device=DEV)
    opt = options(shape[1], shape[0], softcap=cap, device=DEV, **opt)
    check_capped(gpu_call(x, opt), x, opt)


def far_below(keys, dtype, below, device="cpu"):
    """One token whose own key leads and `keys` cached ones whose scores are `below` lower; their values differ from its."""
    D = 64
    x = make(9, 1, 1, 1, 1, D, keys, dtype, [keys], device=device)
    x["q"].zero_()[..., 0] = 8.0      # times the scale of 1 / 8: the scores are the keys' first values
    x["k_cache"][..., 0], x["current_k"][..., 0] = -below, 0.0
    x["v_cache"].fill_(1.0)
    x["current_v"].fill_(-1.0)
    return x, {}


# In units of log2 e the scores are 14.4, 25.07 and 27.4 lower: of fp16's weights the last two are below its least number, 2^-24,
# next to a leading weight of 1. All of them together move the result by up to 2 keys e^-below.
FAR = [(torch.float16, 10.0), (torch.float16, 17.375), (torch.float16, 19.0), (torch.bfloat16, 17.375), (torch.float32, 17.375)]


class OneStretch:
    """The library with a bound of the lengths that does not hold: one workgroup walks over all of a sequence's keys, as in a
    batch that gives every one its own."""

    def __init__(self, lib):
        self.lib = lib

    def fta_shaped_workspace(self, a, cus, need):
        a._obj.max_seq_len_hint = 1
        return self.lib.fta_shaped_workspace(a, cus, need)

    def fta_shaped_decode(self, a, stream):
        return self.lib.fta_shaped_decode(a, stream)


@pytest.mark.parametrize("dtype, below", FAR[1:2])
def test_many_keys_far_below_on_host_threads(host_lib, dtype, below):  # noqa: F811
    x, opt = far_below(60000, dtype, below)
    check(host_call(OneStretch(host_lib), x, opt), oracle(x, opt), x, opt)


def check_far(got, x, keys):
    """`check` in 16 bits. In 32, what bounds such a row are the sums: each addition to O or l rounds by up to 2^-24 of what is
    there, at most l max |v| and l with max |v| = 1, a product adds two keys at a time and a wave at most every key: keys / 2
    additions in a row for either, keys * 2^-24 of the result, and next to it the exponents' 2^-23 (score + bound of the
    score's own sum) < 2^-23 * 200 (scores below 20 from products of up to 8 * 20) on values that differ by 2."""
    if got.dtype != torch.float32:
        check(got, oracle(x, {}), x, {})
    else:
        assert float((got.double() - oracle(x, {})).abs().max()) <= keys * 2.0 ** -24 + 2 * 200 * 2.0 ** -23


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, below", FAR)
def test_many_keys_far_below(dtype, below):
    for keys in (30000, 131072, 1000000):
        x, opt = far_below(keys, dtype, below, DEV)
        check_far(gpu_call(x, opt), x, keys)
        if keys < 1000000:
            check_far(gpu_call(x, opt, max_seq_len_in_batch=1), x, keys)
