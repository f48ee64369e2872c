"""The kernels of csrc/shaped_attn.hip for large caps in 16-bit types, through the same walk over the compiler's output as
the others (test_shaped_attn_asm.py): no register is touched while its LDS read is in flight, nothing is spilled."""
import os
import re
import subprocess

import pytest

from flash_tree_attn_amd import build as fta_build
from test_shaped_attn_asm import HOST, touched_in_flight

KERNELS = {"__bf16": [(64, 2, 1), (128, 1, 0), (128, 2, 0), (256, 1, 1)], "_Float16": [(32, 1, 0), (128, 1, 1), (256, 2, 0)]}   # head_dim, waves per 32 rows, paged


@pytest.mark.parametrize("dtype", KERNELS)
def test_no_register_is_touched_while_its_read_is_in_flight(dtype, tmp_path):
    source = open(os.path.join(fta_build.CSRC, "shaped_attn.hip")).read()
    wanted = [f"template __global__ void shaped_kernel<{dtype}, {d}, {waves}, {'true' if paged else 'false'}, true>(const ShapedParams);"
              for d, waves, paged in KERNELS[dtype]]
    src, out = tmp_path / "shaped.hip", tmp_path / "shaped.s"
    src.write_text(source[:source.index(HOST)] + "\n".join(wanted) + "\n}  // namespace\n}  // namespace fta\n")
    subprocess.run([fta_build.HIPCC, *fta_build.FLAGS, "--cuda-device-only", "-S", "-x", "hip", str(src), "-o", str(out)], check=True, capture_output=True)
    text = out.read_text()
    kernels = re.findall(r"^(_ZN3fta\S*shaped_kernel[^:\s]*):[^\n]*\n(.*?)^\.Lfunc_end", text, flags=re.S | re.M)
    assert len(kernels) == len(wanted)
    for name, body in kernels:
        reads, bad = touched_in_flight(body)
        assert reads >= 8 and not bad, (name, sorted(bad)[:3])
    assert re.findall(r"\.vgpr_spill_count:\s+(\d+)", text) == ["0"] * len(wanted)
