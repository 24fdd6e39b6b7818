"""The rule that takes a work-group's shape for an int8 product (csrc/w8a8_shapes.h), compiled for the host."""
import ctypes
import functools
import pathlib
import shutil
import subprocess
import tempfile

CSRC = pathlib.Path(__file__).resolve().parents[1] / "xestrata-win_amd" / "csrc"
NAMES = ["16x16 ring", "32x32 ring", "64x32 ring", "64x64 ring", "64x64", "64x128", "128x128", "128x256", "256x256"]


@functools.lru_cache(None)
def _rule():
    with tempfile.TemporaryDirectory() as d:
        src, so = pathlib.Path(d) / "rule.cpp", pathlib.Path(d) / "rule.so"
        src.write_text('#include "w8a8_shapes.h"\nextern "C" int pick(int t, int k, int n, int g) { return xs::pick_shape(t, k, n, g != 0); }\n'
                       'extern "C" int count() { return xs::kShapeCount; }\n')
        subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(CSRC), "-o", str(so), str(src)],
                       check=True, capture_output=True)
        lib = ctypes.CDLL(str(so))
    assert lib.count() == len(NAMES)
    return lib.pick


def shape(n_tok, n_in, n_out, gated=False):
    """The name of the shape that a call takes: tokens x weight rows (gated: half as many outputs)."""
    return NAMES[_rule()(n_tok, n_in, n_out, int(gated))]


# a call on each shape, its last tiles and its last step cut: (shape, tokens, n_in, outputs, gated); for the smallest one of up to 16
# tokens and one of more
CALLS = [("16x16 ring", 9, 272, 75, False), ("16x16 ring", 17, 272, 40, False), ("32x32 ring", 261, 272, 284, False),
         ("64x32 ring", 505, 1040, 528, False), ("64x64 ring", 749, 2064, 711, False), ("64x64", 505, 272, 529, False),
         ("64x128", 1054, 272, 1017, False), ("128x128", 1420, 400, 1443, False), ("128x256", 2040, 3500, 4090, False),
         ("256x256", 3500, 272, 3517, False),
         ("16x16 ring", 9, 272, 75, True), ("16x16 ring", 20, 200, 301, True), ("32x32 ring", 17, 272, 40, True),
         ("64x32 ring", 383, 1040, 345, True), ("64x64 ring", 505, 2064, 529, True), ("64x64", 383, 272, 345, True),
         ("64x128", 749, 272, 711, True), ("128x128", 1054, 400, 1017, True), ("128x256", 2040, 3500, 2041, True),
         ("256x256", 2457, 272, 2481, True)]
IDS = [f"{'gated ' if c[4] else ''}{c[0]} {c[1]}" for c in CALLS]
