"""The operand reads of csrc/shaped_attn.hip are LDS reads in inline assembly whose waits the source places itself: the
compiler takes a read's registers as written at once. This walks the compiler's output along every branch and checks
that no instruction touches a register while its read is in flight, and that nothing is spilled (a spill is such an
instruction). Cross-compiles for gfx950, no GPU."""
import os
import re
import subprocess

import pytest

from flash_tree_attn_amd import build as fta_build

HOST = "// ---------------------------------------------------------------------------------------------- host"
KERNELS = {   # type: head_dim, waves per 32 rows, paged
    "__bf16": [(32, 1, 0), (64, 2, 1), (128, 1, 0), (128, 1, 1), (128, 2, 0), (256, 1, 1), (256, 2, 0)],
    "float": [(32, 4, 0), (64, 4, 1), (64, 2, 0), (128, 2, 0), (128, 1, 1), (256, 1, 0)],
}


def registers(text):
    out = set()
    for m in re.finditer(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        if m.group(1):
            out |= {(m.group(1), i) for i in range(int(m.group(2)), int(m.group(3)) + 1)}
        else:
            out.add((m.group(4), int(m.group(5))))
    return frozenset(out)


def blocks_of(text):
    """{label: [(instruction, written as assembly)]}, in order."""
    blocks, current, ours = {"": []}, "", False
    for line in text.split("\n"):
        if ";;#ASMSTART" in line or ";;#ASMEND" in line:
            ours = ";;#ASMSTART" in line
            continue
        line = line.split(";")[0].strip()
        if line.endswith(":"):
            current = line[:-1]
            blocks[current] = []
        elif line and not line.startswith("."):
            blocks[current].append((line, ours))
    return blocks


def touched_in_flight(text):
    """(reads walked over, instructions that touch a register in flight). LDS reads land in order: a wait for n of them
    leaves the last n in flight (every LDS access of the compiler's own is waited for in the same way, so counting only
    ours is on the safe side)."""
    blocks = blocks_of(text)
    order = list(blocks)
    after = dict(zip(order, order[1:] + [None]))
    seen, bad, reads, work = set(), set(), 0, [("", ())]
    while work:
        label, flight = work.pop()
        if (label, flight) in seen:
            continue
        seen.add((label, flight))
        flight, ended = list(flight), False
        for line, ours in blocks[label]:
            op, rest = (line.split(None, 1) + [""])[:2]
            if op == "s_waitcnt":
                m = re.search(r"lgkmcnt\((\d+)\)", line)
                if m:
                    flight = flight[max(len(flight) - int(m.group(1)), 0):]
                continue
            if op.startswith("s_cbranch") or op == "s_branch":
                work.append((rest.strip(), tuple(flight)))
                if op == "s_branch":
                    ended = True
                    break
                continue
            if op == "s_endpgm":
                ended = True
                if flight:
                    bad.add((label, line))
                break
            used = registers(rest)
            if any(used & destination for destination in flight):
                bad.add((label, line))
            if ours and op.startswith("ds_read"):
                flight.append(registers(rest.split(",")[0]))
                reads += 1
        if not ended and after[label] is not None:
            work.append((after[label], tuple(flight)))
    return reads, bad


def test_the_walk_finds_a_read_that_is_not_waited_for():
    body = ";;#ASMSTART\nds_read_b128 v[0:3], v9\n;;#ASMEND\n%s\nv_add_f32 v5, v3, v4\ns_endpgm\n"
    assert touched_in_flight(body % ";;#ASMSTART\ns_waitcnt lgkmcnt(0)\n;;#ASMEND") == (1, set())
    assert touched_in_flight(body % "s_nop 0")[1]
    assert touched_in_flight(body % "s_cbranch_scc1 there\ns_waitcnt lgkmcnt(0)\nthere:")[1]


@pytest.mark.parametrize("dtype", KERNELS)
def test_no_register_is_touched_while_its_read_is_in_flight(dtype, tmp_path):
    source = open(os.path.join(fta_build.CSRC, "shaped_attn.hip")).read()
    assert source.count(HOST) == 1
    wanted = [f"template __global__ void shaped_kernel<{dtype}, {d}, {waves}, {'true' if paged else 'false'}>(const ShapedParams);"
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
