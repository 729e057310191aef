"""Which kernel a call of heatvit_amd.lm.gemm_f8 takes, from the rule of
heatvit_amd/csrc/hv_lm_plan.h, built for the host."""

import ctypes as C
import functools
import subprocess
import tempfile
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
NAMES = ("rows16", "rows16x2", "rows32", "rows64", "tile64", "tile128deep", "tile128", "tile256")
# those that a float32 output and a 16-bit one can take
F32 = ("rows16", "rows16x2", "rows32", "rows64", "tile64", "tile128")
F16 = ("rows16", "rows16x2", "rows32", "tile64", "tile128deep", "tile128", "tile256")


@functools.lru_cache(None)
def _library():
    with tempfile.TemporaryDirectory() as d:
        so = Path(d) / "f8_kernel.so"
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", str(so),
                        "-I", str(ROOT / "heatvit_amd" / "csrc"),
                        str(ROOT / "tests" / "device_math" / "f8_kernel.cpp")], check=True)
        L = C.CDLL(str(so))
    L.f8_kernel.argtypes = [C.c_int, C.c_int, C.c_int, C.c_longlong]
    return L


def kernel_of(f32, m, n, lda):
    return NAMES[_library().f8_kernel(int(f32), m, n, lda)]
