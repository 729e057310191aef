"""Where rows and keys lie and which kernel a call of the attention takes, from
heatvit_amd/csrc/hv_lm_paged.h and hv_lm_attn_plan.h, built for the host."""

import ctypes as C
import functools
import subprocess
import tempfile
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
NAMES = ("few", "few in shares", "tiles", "tiles in shares")


@functools.lru_cache(None)
def library():
    with tempfile.TemporaryDirectory() as d:
        so = Path(d) / "paged.so"
        subprocess.run(["g++", "-O1", "-fwrapv", "-std=c++17", "-shared", "-fPIC", "-o", str(so),
                        "-I", str(ROOT / "heatvit_amd" / "csrc"),
                        str(ROOT / "tests" / "device_math" / "paged.cpp")], check=True)
        L = C.CDLL(str(so))
    i, p, n = C.c_int, C.c_void_p, C.c_longlong
    L.seq_rows_of.argtypes = [p, i, i, p]
    L.keys_of.argtypes = [i] * 4
    L.page_at.argtypes = [i, i, i, p, n]
    L.row_at.argtypes = [i] * 5 + [n]
    L.row_at.restype = n
    L.seen_at.argtypes = [i] * 5 + [p]
    L.attention_shape.argtypes = [i] * 5 + [n]
    L.attention_workspace.argtypes = [i] * 5
    L.attention_workspace.restype = n
    L.tile_of_cost.argtypes = L.cost_before.argtypes = [i] * 4
    L.part_of_tiles.argtypes = [i] * 3
    L.attention_run.argtypes = [i] * 6
    L.place_in_runs.argtypes = [i] * 2
    L.share_numbers.argtypes = [i] * 5 + [p]
    L.table_keys.argtypes, L.table_keys.restype = [i, n], n
    L.packed_keys.argtypes, L.packed_keys.restype = [i, n, i], n
    return L


def kernel_of(rows, batch, heads, kv_heads, width, most_keys):
    return NAMES[library().attention_shape(rows, batch, heads, kv_heads, width, most_keys)]
