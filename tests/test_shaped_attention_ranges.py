"""Shaped tree attention at the ends of what its arguments may be (the kernel's source on host threads, and on the GPU):
finite masks, from soft ones to the type's lowest value, in front of keys that count."""
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
