"""CPU tests: which kernel the MXFP4 products of the GPU tests take, so that a changed rule that leaves a kernel or a part of
one untested fails here.  The library's two launchers are replaced by ones that note which was called; nothing is launched."""
import json
import os
import shutil
import subprocess
import sys

import pytest

from test_gpu_mx_paths import CASES, IDS, PREFIXES, edges

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "hip-kernels_amd", "csrc")
STUB = """
#include "mx_kernels.h"
extern "C" {
const char* way = "";
}
namespace gxmoe {
hipError_t launch_mx_tile(const MxProductArgs&, MxTile kind, hipStream_t) {
  way = kind == MxTile::large ? "large" : kind == MxTile::middle ? "middle" : "low";
  return hipSuccess;
}
hipError_t launch_mx_stream(const MxProductArgs&, bool wide, bool split, hipStream_t) {
  way = wide ? (split ? "wide split stream" : "wide stream") : split ? "split stream" : "stream";
  return hipSuccess;
}
}
"""
CHILD = """
import ctypes, json, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # before the library: its calls go there
sys.path.insert(0, sys.argv[2])
import gptoss_moe as g
way = ctypes.c_char_p.in_dll(stub, "way")
at = lambda i: (i + 1) << 42  # addresses that nothing reads
out = []
for experts, rows, N, K, quantize in json.load(sys.stdin):
    r = g.Mxfp4Result(0, 1.0, 7.0, 0, None if quantize else at(9), N, at(9) if quantize else None, at(10) if quantize else None)
    if experts:
        g.check(g.lib.gptoss_moe_grouped_mxfp4_matmul(at(0), at(1), rows, None, at(3), experts, rows, at(4), at(5), at(6), N, K,
                                                      ctypes.byref(r), None))
    else:
        g.check(g.lib.gptoss_mxfp4_matmul(at(0), at(1), rows, at(4), at(5), at(6), N, K, ctypes.byref(r), None))
    out.append(way.value.decode())
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def ways(tmp_path_factory):
    """[(experts or 0, rows, N, K, quantize)] to the kernels' names."""
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    where = tmp_path_factory.mktemp("mx")
    (where / "stub.cpp").write_text(STUB)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-D__HIP_PLATFORM_AMD__", "-I" + os.path.join(rocm, "include"), "-I" + CSRC, "-shared",
                    "-fPIC", str(where / "stub.cpp"), "-o", str(where / "stub.so")], check=True)

    def ask(calls):
        r = subprocess.run([sys.executable, "-c", CHILD, str(where / "stub.so"), os.path.join(ROOT, "hip-kernels_amd")],
                           input=json.dumps(calls), capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        return json.loads(r.stdout.splitlines()[-1])

    return ask


def test_the_kernels_of_the_cases(ways):
    calls = [(name, way, (len(counts) if len(counts) > 1 else 0, sum(edges(counts)) + sum(counts), N, K, quantize))
             for name, (way, counts, N, K) in zip(IDS, CASES) for quantize in ((False, True) if N % 32 == 0 else (False,))]
    got = ways([call for _, _, call in calls])
    for (name, way, call), have in zip(calls, got):
        if call[-1] and "stream" in way and "wide" not in way:  # the stream makes MXFP4 of 32 columns a wave
            way = "wide " + way
        assert have == way, (name, call)
    assert set(got) == {"large", "middle", "low", "stream", "wide stream", "split stream", "wide split stream"}


def test_the_kernels_of_the_prefixes(ways):
    calls = [(way, (0, n, N, K, False)) for way, N, K, rows in PREFIXES for n in rows]
    assert ways([call for _, call in calls]) == [way for way, _ in calls]
