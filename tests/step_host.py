"""The kernels around a tree-attention call (rotary positions, token log probabilities, accepted path), compiled for the
host from the product sources and run on host threads (tests/host_block). A module-scoped fixture; the build lives in a
temporary directory and nothing under flash_tree_attn_amd/ knows of it."""
import ctypes as C
import os
import subprocess

import pytest

from flash_tree_attn_amd import _lib
from flash_tree_attn_amd import build as fta_build

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = os.path.join(os.path.dirname(fta_build.HIPCC), "..", "llvm", "bin", "clang++")


@pytest.fixture(scope="module")
def host_step_lib(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no host clang++")
    out = tmp_path_factory.mktemp("host_step")
    flags = ["-x", "c++", "-std=c++20", "-O1", "-fPIC", "-pthread", "-I", os.path.join(HERE, "host_block"), "-I", fta_build.INCLUDE, "-I", fta_build.CSRC,
             "-include", os.path.join(HERE, "host_block", "step_ops_host.h")]
    procs, objs = [], []
    for src in ("rotary.hip", "token_logprobs.hip", "accept_path.hip"):
        objs.append(str(out / (src + ".o")))
        procs.append(subprocess.Popen([CLANG, *flags, "-c", os.path.join(fta_build.CSRC, src), "-o", objs[-1]], stdout=subprocess.PIPE, stderr=subprocess.STDOUT))
    for proc in procs:
        log = proc.communicate()[0]
        assert proc.returncode == 0, log.decode()[-3000:]
    path = str(out / "libfta_host_step.so")
    subprocess.run([CLANG, "-shared", "-pthread", *objs, "-o", path], check=True, capture_output=True)
    lib = C.CDLL(path)
    for name, args in (("fta_rotary", _lib.FtaRotaryArgs), ("fta_logprobs", _lib.FtaLogprobArgs), ("fta_accept_path", _lib.FtaAcceptArgs)):
        getattr(lib, name).argtypes = [C.POINTER(args), C.c_void_p]
    lib.fta_logprobs_workspace.argtypes = [C.POINTER(_lib.FtaLogprobArgs), C.POINTER(C.c_int64)]
    return lib
