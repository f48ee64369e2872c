"""Where csrc/shaped_attn.hip cuts its line of tiles. The kernel and the join compute the bounds for themselves, each in a
compilation of its own: they have to agree whether or not a compiler fuses a product with the sum behind it."""
import os
import subprocess

import pytest

from flash_tree_attn_amd import build as fta_build
from step_host import CLANG

PROGRAM = r"""
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
using std::max; using std::min;
#define __device__
#define __forceinline__ inline __attribute__((always_inline))
constexpr int kMinStretch = 4;
struct ShapedParams { int groups, lead_groups, lead_share; };
inline float fast_rcp(float x) { return 1.f / x; }
%s
int main() {
  std::srand(1);
  for (int k = 0; k < 4000; ++k) {
    ShapedParams p{};
    p.groups = 1 + std::rand() %% 512;
    p.lead_groups = k %% 2 && p.groups > 1 ? p.groups / 2 : 0;
    p.lead_share = p.lead_groups ? 584 : 0;
    const int bits = 3 + k %% 28, total = (1 << bits) + (std::rand() & ((1 << bits) - 1));
    if (total >= 1 << 30) continue;
    const Stretches s = cut_line(p, total);
    unsigned long long sum = 0;
    for (int g = 0; g <= s.groups; ++g) {
      sum = sum * 1000003 + static_cast<unsigned>(s.start(g));
      if (s.start(g) < 0 || s.start(g) > total || (g && s.start(g) <= s.start(g - 1))) { std::printf("not ascending\n"); return 1; }
    }
    if (s.start(0) != 0 || s.start(s.groups) != total) { std::printf("not the whole line\n"); return 1; }
    for (int i = 0; i < 8; ++i) {
      const int x = i < 2 ? (i ? total - 1 : 0) : std::rand() %% total, g = s.holder(x);
      if (s.start(g) > x || s.start(g + 1) <= x) { std::printf("holder\n"); return 1; }
    }
    std::printf("%%d %%d %%llu\n", p.groups, total, sum);
  }
}
"""


def test_bounds_do_not_depend_on_what_the_compiler_fuses(tmp_path):
    if not os.path.exists(CLANG):
        pytest.skip("no host clang++")
    if "fma" not in open("/proc/cpuinfo").read():
        pytest.skip("no fused multiply-add on this machine")
    text = open(os.path.join(fta_build.CSRC, "shaped_attn.hip")).read()
    start = text.index("struct Stretches {")
    end = text.index("\n}\n", text.index(" cut_line(", start)) + 3
    src = tmp_path / "cut.cpp"
    src.write_text(PROGRAM % text[start:end])
    results = []
    for contract in ("off", "fast"):
        exe = str(tmp_path / contract)
        subprocess.run([CLANG, "-std=c++17", "-O2", "-mfma", f"-ffp-contract={contract}", str(src), "-o", exe], check=True, capture_output=True)
        run = subprocess.run([exe], capture_output=True, text=True)
        assert run.returncode == 0, run.stdout[-200:]
        results.append(run.stdout)
    assert results[0] == results[1]
