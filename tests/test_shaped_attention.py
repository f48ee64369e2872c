"""Tree attention with shaped scores (`fta_shaped_decode`, `shaped_tree_attention`): refusals and the kernel's source on
host threads (CPU), parity with the 64-bit definition on the GPU."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from flash_tree_attn_amd import (_lib, additive_mask_from_parents, pack_mask, random_tree_parents, shaped_tree_attention, tree_depths)
from flash_tree_attn_amd import build as fta_build
from oracle.step_oracle import shaped_attention_oracle
from step_host import CLANG, HERE

DEV = "cuda"
DTYPES = {torch.float32: _lib.FTA_F32, torch.float16: _lib.FTA_F16, torch.bfloat16: _lib.FTA_BF16}


def check(got, ref, x, opt):
    """|out - ref| elementwise against three terms. (1) Half a step of the output type. (2) Weights: rounded to the type
    for the second product and summed as rounded, so every one is off by half a step relative to the others, which moves
    the mean of V by at most eps / 2 times the weights' mean deviation of V, <= 2 max |v|. (3) The exponents, 32-bit: a score
    is off by about 2^-23 (|x| sqrt(D) + cap), and the bias, whose magnitude is at most slope * reach, by 2^-23 of that
    for keys whose weight counts (a weight e^-d only counts d e^-d < 1 of its bias' error); all by 2 max |v| again."""
    eps = torch.finfo(got.dtype).eps
    vmax = max(float(x["v_cache"].float().nan_to_num(0, 0, 0).abs().max()) if x["v_cache"].numel() else 0.0, float(x["current_v"].float().nan_to_num(0, 0, 0).abs().max()))
    size = float(x["q"].float().norm(dim=-1).max()) * max(float(x["k_cache"].float().nan_to_num(0, 0, 0).norm(dim=-1).max()) if x["k_cache"].numel() else 0.0,
                                                        float(x["current_k"].float().nan_to_num(0, 0, 0).norm(dim=-1).max())) * abs(opt.get("sm_scale") or got.size(-1) ** -0.5)
    exponent = 2.0 ** -23 * (4 * size + 4 * opt.get("softcap", 0.0) + 64)
    weight = 0.0 if got.dtype == torch.float32 else eps / 2
    bound = eps / 2 * ref.abs() + 2 * vmax * (weight + exponent) + 2.0 ** -24
    far = ((got.double() - ref).abs() / bound).nan_to_num(1e9)
    assert got.isfinite().all() and float(far.max()) <= 1.0, f"worst {float(far.max()):.2f} bounds"
    return float(far.max())


# ---------------------------------------------------------------- inputs
def make(seed, bsz, hq, hkv, L, D, cache, dtype, lens, page=0, cur_heads=None, depths="tree", device="cpu", mask="tree"):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    ch = hkv if cur_heads is None else cur_heads
    x = dict(q=r(bsz, hq, L, D), current_k=r(bsz, ch, L, D), current_v=r(bsz, ch, L, D))
    parents = [random_tree_parents(L, g) for _ in range(bsz)]
    if page:
        per = -(-cache // page)
        x["k_cache"], x["v_cache"] = r(bsz * per, hkv, page, D), r(bsz * per, hkv, page, D)
        x["block_tables"] = torch.randperm(bsz * per, generator=g).to(torch.int32).view(bsz, per)
    else:
        x["k_cache"], x["v_cache"] = r(bsz, hkv, cache, D), r(bsz, hkv, cache, D)
    x["mask"] = torch.stack([additive_mask_from_parents(p) for p in parents])[:, None]
    if mask == "shared":
        x["mask"] = x["mask"][0, 0]
    x["kv_seq_len"] = torch.tensor(lens, dtype=torch.int64)
    if depths == "tree":
        x["depths"] = torch.stack([tree_depths(p) for p in parents])
    elif depths == "shared":
        x["depths"] = tree_depths(parents[0])
    return {n: t.to(device) for n, t in x.items()}


def options(hq, bsz, softcap=0.0, slopes=False, window=0, first=None, device="cpu", falling=True, **kw):
    opt = dict(softcap=softcap, window=window, **kw)
    if slopes:
        opt["slopes"] = (2.0 ** (-8.0 * torch.arange(1, hq + 1) / hq)).to(device) * (1.0 if falling else -1.0)
    if first is not None:
        opt["first_key"] = torch.tensor(first, dtype=torch.int32, device=device)
    return opt


CASES = {
    # name: (bsz hq hkv L D cache dtype lens, make(), options())
    "one token, grouped heads": ((2, 4, 1, 1, 64, 200, torch.bfloat16, [200, 65]), {}, dict(softcap=20.0)),
    "tree, slopes, two tiles of rows": ((1, 4, 2, 40, 128, 150, torch.float16, [150]), {}, dict(slopes=True)),
    "window across tiles, odd": ((2, 2, 2, 7, 128, 300, torch.bfloat16, [299, 130]), {}, dict(window=77, slopes=True)),
    "window of one, empty cache": ((3, 2, 1, 5, 64, 128, torch.float16, [0, 128, 1]), {}, dict(window=1)),
    "documents": ((3, 4, 2, 9, 32, 260, torch.bfloat16, [260, 100, 70]), {}, dict(first=[130, 100, -3], softcap=30.0)),
    "everything, paged 16": ((2, 4, 2, 13, 64, 256, torch.float16, [250, 33]), dict(page=16), dict(softcap=15.0, slopes=True, window=100, first=[180, 0])),
    "paged 128, two tree tiles": ((1, 2, 1, 70, 64, 384, torch.bfloat16, [300]), dict(page=128), dict(softcap=50.0)),
    "f32": ((2, 4, 2, 6, 64, 120, torch.float32, [120, 31]), {}, dict(softcap=10.0, slopes=True)),
    "f32 paged, window, D 128": ((1, 2, 1, 35, 128, 96, torch.float32, [90]), dict(page=32), dict(window=40)),
    "f32, 64 keys a tile": ((1, 2, 1, 25, 128, 150, torch.float32, [150]), {}, dict(softcap=30.0, slopes=True, window=101)),
    "f32, 128 keys a tile, paged": ((2, 2, 2, 9, 32, 304, torch.float32, [300, 129]), dict(page=16), dict(softcap=4.0, first=[140, 3])),
    "f32, 130 rows": ((1, 2, 1, 65, 32, 70, torch.float32, [70]), {}, dict(slopes=True)),
    "rising bias, capped": ((1, 2, 1, 3, 64, 900, torch.bfloat16, [900]), {}, dict(softcap=2.0, slopes=True, falling=False)),
    "head_dim 256": ((1, 2, 1, 3, 256, 140, torch.bfloat16, [129]), {}, dict(softcap=25.0, slopes=True)),
    "f32 head_dim 256": ((1, 1, 1, 2, 256, 64, torch.float32, [50]), {}, dict(slopes=True)),
    "head_dim 32, 130 rows": ((1, 2, 1, 65, 32, 128, torch.float16, [128]), {}, dict(window=90)),
    "negative scale": ((1, 2, 1, 4, 64, 100, torch.float16, [100]), {}, dict(softcap=5.0, sm_scale=-0.2)),
    "tree K/V per query head": ((1, 4, 2, 6, 64, 70, torch.bfloat16, [70]), dict(cur_heads=4), dict(softcap=9.0)),
    "lengths beyond the cache": ((3, 2, 1, 4, 64, 100, torch.float16, [1000, -4, 64]), {}, dict(slopes=True)),
    "chain depths, shared mask": ((2, 2, 1, 10, 64, 90, torch.bfloat16, [90, 64]), dict(depths=None, mask="shared"), dict(window=33)),
    "long, cut in stretches": ((2, 2, 1, 3, 64, 1500, torch.bfloat16, [1500, 700]), {}, dict(softcap=30.0)),
    "long, f32, ragged": ((3, 1, 1, 2, 32, 1100, torch.float32, [1100, 5, 900]), {}, dict(slopes=True, first=[200, 0, 899])),
}
POSITIONAL = ("q", "k_cache", "v_cache", "current_k", "current_v", "mask", "kv_seq_len")


def case_inputs(name, device="cpu", seed=0):
    shape, how, opt = CASES[name]
    x = make(seed, *shape, device=device, **how)
    o = options(shape[1], shape[0], device=device, **opt)
    if how.get("depths", "tree") is None:
        chain = torch.arange(shape[3])
        x["mask"] = torch.zeros(shape[3], shape[3]).masked_fill(chain[:, None] < chain, float("-inf")).to(device)
    return x, o


def oracle(x, opt):
    return shaped_attention_oracle(*(x[n] for n in POSITIONAL), depths=x.get("depths"), block_tables=x.get("block_tables"), **opt)


# ---------------------------------------------------------------- CPU: host threads
@pytest.fixture(scope="module")
def host_lib(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no host clang++")
    out = tmp_path_factory.mktemp("host_shaped")
    src = out / "shaped_host.cpp"
    src.write_text('#include "fta_device.h"\n#include "shaped_attn_ops_host.h"\n#include "shaped_attn.hip"\n'
                   'extern "C" void host_block_loads_land_late(int late) { host_block::loads_land_late() = late != 0; }\n')
    flags = ["-x", "c++", "-std=c++20", "-O1", "-fPIC", "-pthread", "-I", os.path.join(HERE, "host_block"), "-I", fta_build.INCLUDE, "-I", fta_build.CSRC]
    path = str(out / "libfta_host_shaped.so")
    run = subprocess.run([CLANG, *flags, "-shared", str(src), "-o", path], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-3000:]
    lib = C.CDLL(path)
    lib.fta_shaped_decode.argtypes = [C.POINTER(_lib.FtaShapedArgs), C.c_void_p]
    lib.fta_shaped_workspace.argtypes = [C.POINTER(_lib.FtaShapedArgs), C.c_int, C.POINTER(C.c_int64)]
    return lib


def host_call(lib, x, opt):
    a = _lib.FtaShapedArgs()
    q = x["q"]
    out = torch.full_like(q, float("nan"))
    bsz, hq, L, D = q.shape
    mask = x["mask"].expand(bsz, hq, L, x["mask"].size(-1))
    a.q, a.k_cache, a.v_cache, a.cur_k, a.cur_v = (x[n].data_ptr() for n in POSITIONAL[:5])
    a.mask, a.kv_seq_len, a.out = mask.data_ptr(), x["kv_seq_len"].data_ptr(), out.data_ptr()
    a.bsz, a.num_q_heads, a.q_len, a.head_dim = q.shape
    a.num_kv_heads, a.cur_heads = x["k_cache"].size(1), x["current_k"].size(1)
    a.cache_len = x["k_cache"].size(2)
    if "block_tables" in x:
        a.page_size, a.cache_len = x["k_cache"].size(2), x["block_tables"].size(1) * x["k_cache"].size(2)
        a.block_table, a.block_table_stride = x["block_tables"].data_ptr(), x["block_tables"].stride(0)
    if "slopes" in opt:
        a.slopes = opt["slopes"].data_ptr()
    if "first_key" in opt:
        a.first_key = opt["first_key"].data_ptr()
    if "depths" in x:
        a.depths, a.depth_stride = x["depths"].data_ptr(), x["depths"].stride(0) if x["depths"].dim() == 2 else 0
    a.dtype, a.len_dtype, a.mask_kind = DTYPES[q.dtype], _lib.FTA_I64, _lib.MASK_PACKED_U64 if mask.dtype == torch.int64 else _lib.MASK_ADDITIVE_F32
    a.window, a.softcap, a.sm_scale = opt.get("window", 0), opt.get("softcap", 0.0), opt.get("sm_scale", D ** -0.5)
    for n, t in (("q_stride", q), ("k_stride", x["k_cache"]), ("v_stride", x["v_cache"]), ("ck_stride", x["current_k"]), ("cv_stride", x["current_v"]),
                 ("mask_stride", mask), ("out_stride", out)):
        getattr(a, n)[:] = t.stride()[:3]
    need = C.c_int64()
    assert lib.fta_shaped_workspace(C.byref(a), 256, C.byref(need)) == 0
    ws = torch.full((need.value // 4 + 8,), float("nan"))
    a.workspace, a.workspace_bytes = (ws.data_ptr() + 15) // 16 * 16, need.value
    assert lib.fta_shaped_decode(C.byref(a), None) == 0
    return out


@pytest.mark.parametrize("name", CASES)
def test_kernel_source_on_host_threads(host_lib, name):
    x, opt = case_inputs(name)
    host_lib.host_block_loads_land_late(len(name) % 2)      # half of the cases with loads that land as late as the waits allow
    check(host_call(host_lib, x, opt), oracle(x, opt), x, opt)
    host_lib.host_block_loads_land_late(0)


@pytest.mark.parametrize("name", ["f32", "f32, 64 keys a tile", "f32, 130 rows", "paged 128, two tree tiles", "tree, slopes, two tiles of rows"])
def test_packed_masks_on_host_threads(host_lib, name):
    x, opt = case_inputs(name)
    check(host_call(host_lib, {**x, "mask": pack_mask(x["mask"])}, opt), oracle(x, opt), x, opt)


def test_rows_that_see_nothing_and_what_nobody_sees(host_lib):
    x, opt = blind_case()
    got = host_call(host_lib, x, opt)
    assert bool((got[0, :, 2] == 0).all() and (got[1, :, 3] == 0).all())
    check(got, oracle(x, opt), x, opt)


def blind_case(device="cpu"):
    """Row 2 of sequence 0 sees nothing (its cache part begins behind the last key); tree nodes 5 and 6 hold NaN and infinity
    and are seen by nobody, nor are the cache rows behind a length or in front of a document, which hold NaN."""
    x = make(3, 2, 4, 2, 7, 64, 140, torch.bfloat16, [130, 64])
    nan, inf = float("nan"), float("inf")
    x["mask"][:, :, 5:] = -inf
    x["mask"][:, :, :, 5:] = -inf
    x["mask"][0, :, 2] = -inf
    x["mask"][1, :, 3] = -inf
    for n in ("current_k", "current_v"):
        x[n][:, :, 5], x[n][:, :, 6] = nan, inf
    for n in ("k_cache", "v_cache"):
        x[n][0, :, 130:], x[n][1, :, 64:], x[n][0, :, :130], x[n][1, :, :40] = nan, inf, nan, nan
    opt = options(4, 2, softcap=20.0, slopes=True, first=[130, 40])     # sequence 0: nothing of the cache is left
    opt["first_key"][1] = 64                                             # nor of sequence 1's
    x["k_cache"][1, :, :64], x["v_cache"][1, :, :64] = nan, nan
    return {n: t.to(device) for n, t in x.items()}, {n: t.to(device) if torch.is_tensor(t) else t for n, t in opt.items()}


def lowest_value_case(device="cpu"):
    """An empty cache and rows whose mask holds nothing but the type's lowest value: all of their keys count alike."""
    x = make(4, 1, 2, 1, 6, 64, 64, torch.float16, [0])
    x["mask"] = torch.full((6, 6), torch.finfo(torch.float32).min)
    x["mask"][0, 1:] = float("-inf")
    return {n: t.to(device) for n, t in x.items()}, {}


def test_masks_of_the_lowest_value(host_lib):
    x, opt = lowest_value_case()
    got = host_call(host_lib, x, opt)
    check(got, oracle(x, opt), x, opt)
    torch.testing.assert_close(got[0, :, 3].float(), x["current_v"][0].float().mean(1).expand(2, -1), atol=2e-3, rtol=2e-3)


def shaped_args(**kw):
    a = _lib.FtaShapedArgs()
    for f in ("q", "k_cache", "v_cache", "cur_k", "cur_v", "mask", "kv_seq_len", "out"):
        setattr(a, f, 0x1000)
    cfg = dict(bsz=2, num_q_heads=8, num_kv_heads=2, cur_heads=2, q_len=4, head_dim=128, cache_len=256, dtype=_lib.FTA_BF16, len_dtype=_lib.FTA_I64, sm_scale=0.1)
    cfg.update(kw)
    for n, v in cfg.items():
        setattr(a, n, v)
    for n in ("q_stride", "k_stride", "v_stride", "ck_stride", "cv_stride", "out_stride"):
        getattr(a, n)[:] = [1 << 16, 1 << 12, 128]
    return a


@pytest.mark.parametrize("kw, status", [
    (dict(q=None), -1), (dict(mask=None), -1), (dict(out=None), -1), (dict(head_dim=96), -2), (dict(dtype=7), -6), (dict(len_dtype=2), -6), (dict(mask_kind=2), -6),
    (dict(bsz=0), -7), (dict(q_len=0), -7), (dict(window=-1), -7), (dict(num_q_heads=9), -7), (dict(cur_heads=4), -7), (dict(cache_len=-1), -7),
    (dict(softcap=-1.0), -9), (dict(softcap=float("nan")), -9), (dict(softcap=float("inf")), -9), (dict(softcap=3e38), -9), (dict(softcap=1e-40), -9), (dict(sm_scale=float("nan")), -9),
    (dict(block_table=0x1000, page_size=48, block_table_stride=100), -3), (dict(block_table=0x1000, page_size=64, block_table_stride=1), -7),
    (dict(block_table=0x1000, page_size=64, block_table_stride=9, cache_len=0), -7), (dict(k_cache=0x1008), -8), (dict(mask=0x1002), -8), (dict(depth_stride=-1), -8),
])
def test_argument_errors_without_touching_the_gpu(fta_lib, kw, status):
    assert fta_lib.fta_shaped_decode(C.byref(shaped_args(**kw)), None) == status
    assert fta_lib.fta_shaped_decode(None, None) == -1


def test_workspace_and_stride_errors(fta_lib):
    need = C.c_int64(-1)
    assert fta_lib.fta_shaped_workspace(C.byref(shaped_args()), 256, C.byref(need)) == 0 and need.value == 0      # short: one launch, nothing cut
    a = shaped_args(cache_len=8192)
    assert fta_lib.fta_shaped_workspace(C.byref(a), 256, C.byref(need)) == 0 and need.value > 0
    assert fta_lib.fta_shaped_workspace(C.byref(shaped_args(cache_len=8192, window=64)), 256, C.byref(need)) == 0 and need.value == 0
    assert fta_lib.fta_shaped_workspace(C.byref(shaped_args(cache_len=8192, max_seq_len_hint=300)), 256, C.byref(need)) == 0 and need.value == 0
    assert fta_lib.fta_shaped_workspace(C.byref(shaped_args(head_dim=5)), 256, C.byref(need)) == -2
    assert fta_lib.fta_shaped_workspace(None, 256, C.byref(need)) == -1
    a = shaped_args()
    a.v_stride[2] = 132
    assert fta_lib.fta_shaped_decode(C.byref(a), None) == -8
    a = shaped_args()
    a.k_stride[2] = 1 << 27
    assert fta_lib.fta_shaped_decode(C.byref(a), None) == -9
    if not torch.cuda.is_available():
        assert fta_lib.fta_shaped_decode(C.byref(shaped_args()), None) == -11


def test_python_wrapper_rejects_cpu_tensors():
    x, opt = case_inputs("f32")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        shaped_tree_attention(*(x[n] for n in POSITIONAL), kv_group_num=2, **opt)


# ---------------------------------------------------------------- GPU
def gpu_call(x, opt, **kw):
    extra = {n: x[n] for n in ("depths", "block_tables") if n in x}
    return shaped_tree_attention(*(x[n] for n in POSITIONAL), kv_group_num=x["q"].size(1) // x["k_cache"].size(1), **extra, **opt, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("name", CASES)
def test_matches_the_definition(name):
    for seed in (1, 2):      # the second call runs from the remembered signature
        x, opt = case_inputs(name, DEV, seed)
        got = gpu_call(x, opt)
        check(got, oracle(x, opt), x, opt)
        for _ in range(3):
            assert torch.equal(gpu_call(x, opt), got)      # the same bits every time


@pytest.mark.gpu
def test_blind_rows_and_lowest_masks():
    x, opt = blind_case(DEV)
    got = gpu_call(x, opt)
    assert bool((got[0, :, 2] == 0).all() and (got[1, :, 3] == 0).all())
    check(got, oracle(x, opt), x, opt)
    x, opt = lowest_value_case(DEV)
    check(gpu_call(x, opt), oracle(x, opt), x, opt)


LARGE = {
    # bsz hq hkv L D cache dtype lens, make, options
    "grouped, 64 nodes": ((2, 8, 2, 64, 128, 4096, torch.bfloat16, [4096, 3000]), {}, dict(softcap=50.0)),
    "ragged batch of 70": ((70, 4, 1, 5, 64, 2000, torch.float16, [(i * 397) % 2001 for i in range(70)]), {}, dict(slopes=True, softcap=30.0)),
    "one long sequence, paged, window": ((1, 8, 2, 16, 128, 40000, torch.bfloat16, [39999]), dict(page=64), dict(window=5000, slopes=True)),
    "three blocks of rows": ((1, 8, 1, 50, 128, 3000, torch.float16, [2999]), {}, dict(softcap=20.0)),
    "f32 long": ((2, 8, 2, 20, 128, 3000, torch.float32, [3000, 1234]), dict(page=16), dict(softcap=30.0, slopes=True)),
    "head_dim 256, 64 nodes": ((2, 4, 2, 64, 256, 2000, torch.bfloat16, [2000, 77]), {}, dict(softcap=30.0)),
    "uneven stretches": ((3, 16, 4, 20, 64, 40000, torch.bfloat16, [40000, 7, 33333]), {}, dict(softcap=30.0, slopes=True)),
    "even stretches": ((4, 16, 4, 20, 64, 20000, torch.float16, [20000] * 4), dict(page=128), dict(slopes=True)),
    "head_dim 32": ((3, 16, 4, 33, 32, 5000, torch.float16, [5000, 1, 2500]), {}, dict(slopes=True)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", LARGE)
def test_larger_calls_match_the_definition(name):
    shape, how, opt = LARGE[name]
    x = make(5, *shape, device=DEV, **how)
    opt = options(shape[1], shape[0], device=DEV, **opt)
    got = gpu_call(x, opt)
    check(got, oracle(x, opt), x, opt)
    assert torch.equal(gpu_call(x, opt), got)


@pytest.mark.gpu
def test_mask_forms_strides_output_and_hint():
    x, opt = case_inputs("everything, paged 16", DEV, 7)
    want = gpu_call(x, opt)
    packed = dict(x, mask=pack_mask(x["mask"].cpu()).to(DEV))
    boolean = dict(x, mask=x["mask"] == 0)
    assert torch.equal(gpu_call(packed, opt), want) and torch.equal(gpu_call(boolean, opt), want)
    assert torch.equal(gpu_call(dict(x, kv_seq_len=x["kv_seq_len"].int()), opt), want)
    out = torch.empty(2, 13, 4, 64, dtype=torch.float16, device=DEV).transpose(1, 2)       # [bsz, L, heads, D] as a caller's layer holds it
    assert gpu_call(x, opt, output=out) is out and torch.equal(out, want)
    strided = dict(x, q=x["q"].transpose(1, 2).contiguous().transpose(1, 2), current_k=torch.cat([x["current_k"]] * 2, -1)[..., :64])
    assert torch.equal(gpu_call(strided, opt), want)
    odd = dict(x, q=torch.cat([x["q"][..., :1], x["q"]], -1)[..., 1:])                     # unaligned rows are copied
    assert torch.equal(gpu_call(odd, opt), want)
    y, o = case_inputs("long, cut in stretches", DEV, 8)
    check(gpu_call(y, o, max_seq_len_in_batch=1500), oracle(y, o), y, o)
    check(gpu_call(y, o, max_seq_len_in_batch=100), oracle(y, o), y, o)                    # a bound that does not hold only costs speed


@pytest.mark.gpu
def test_plain_scores_agree_with_flash_decoding_attention():
    from flash_tree_attn_amd import flash_decoding_attention
    for shape in ((2, 8, 2, 16, 128, 1000, torch.bfloat16, [1000, 640]), (2, 4, 4, 9, 64, 300, torch.float16, [300, 0])):
        x = make(11, *shape, device=DEV)
        a = gpu_call(x, {})
        b = flash_decoding_attention(*(x[n] for n in POSITIONAL), 64, kv_group_num=shape[1] // shape[2])
        torch.testing.assert_close(a, b, atol=2 * 2e-3, rtol=2e-2)      # each is within 2e-3 / 1e-2 of the exact result


@pytest.mark.gpu
def test_other_stream_and_graph_replays():
    x, opt = case_inputs("long, cut in stretches", DEV, 9)
    want = gpu_call(x, opt)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = gpu_call(x, opt)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs, each with workspace of its own from its pool; replays between eager calls
    outs, graphs = [], []
    for _ in range(2):
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            gpu_call(x, opt, output=out)
        outs.append(out)
        graphs.append(graph)
    for k in range(4):
        x["q"].copy_(torch.randn_like(x["q"].float()).to(x["q"].dtype))
        x["kv_seq_len"].copy_(torch.tensor([1500 - 100 * k, 300 * k]))
        eager = gpu_call(x, opt)
        for out, graph in zip(outs, graphs):
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for out in outs:
            assert torch.equal(out, eager)


@pytest.mark.gpu
def test_refusals():
    x, opt = case_inputs("f32", DEV)
    call = lambda x=x, **kw: gpu_call(x, dict(opt, **kw))
    call()
    t = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=DEV)
    for kw in (dict(softcap=-1.0), dict(softcap=float("nan")), dict(window=-1), dict(window=1 << 31), dict(slopes=t(3)), dict(slopes=t(4).half()), dict(first_key=t(2)),
               dict(first_key=t(3, dtype=torch.int32)), dict(sm_scale=float("inf"))):
        with pytest.raises(ValueError):
            call(**kw)
    for change in (dict(depths=t(6, dtype=torch.int64)), dict(depths=t(3, 6, dtype=torch.int32)), dict(q=x["q"].double()), dict(q=x["q"][0]), dict(k_cache=x["k_cache"].half()),
                   dict(v_cache=x["v_cache"][:, :, :100]), dict(current_k=x["current_k"][:, :1]), dict(kv_seq_len=x["kv_seq_len"][:1]), dict(mask=t(5, 5)),
                   dict(kv_seq_len=x["kv_seq_len"].cpu()), dict(block_tables=t(2, 3)), dict(current_v=x["current_v"][:, :, :5])):
        with pytest.raises(ValueError):
            call(dict(x, **change))
    with pytest.raises(ValueError):
        call(dict(x, q=torch.zeros(2, 4, 6, 48, device=DEV)))
    for out in (t(2, 4, 6, 32), t(1, 4, 6, 64).expand(2, 4, 6, 64), t(2, 4, 6, 128)[..., ::2]):
        with pytest.raises(ValueError):
            gpu_call(x, opt, output=out)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
        call(dict(x, q=x["q"].clone().requires_grad_()))
    for again in range(2):      # also where the same call without a gradient is remembered
        with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
            call(slopes=opt["slopes"].clone().requires_grad_())
        with torch.enable_grad(), pytest.raises(RuntimeError, match="no_grad"):
            call(dict(x, mask=x["mask"].clone().requires_grad_()))
        call(slopes=opt["slopes"].clone())
