"""By which entry of its table a run of keys in pages is found (csrc/pages.h), without a GPU: the key's own, and none past the last
key's, whatever tile is asked for."""
import ctypes as C
import os
import subprocess

import pytest

import perseus_amd as pa

CSRC = os.path.join(os.path.dirname(pa.__file__), "csrc")
SOURCE = """
#include "pages.h"
extern "C" uint32_t entry32(int t, int run, int log, int len) { return pch::clear::entry_of<32>(t, run, log, len); }
extern "C" uint32_t entry64(int t, int run, int log, int len) { return pch::clear::entry_of<64>(t, run, log, len); }
"""


@pytest.fixture(scope="module")
def entry(tmp_path_factory):
    at = tmp_path_factory.mktemp("pages")
    (at / "pages.cpp").write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", CSRC, str(at / "pages.cpp"), "-o", str(at / "pages.so")], check=True)
    lib = C.CDLL(str(at / "pages.so"))
    for f in (lib.entry32, lib.entry64):
        f.restype = C.c_uint32
    return {32: lib.entry32, 64: lib.entry64}


@pytest.mark.parametrize("keys", [32, 64])
@pytest.mark.parametrize("log", [4, 5, 6, 7, 12, 30])
def test_no_entry_past_the_last_key_s(entry, keys, log):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 100, 127, 128, 129, 1000, 4096, 2 ** 31 - 64, 2 ** 31 - 1]
    for n in lens:
        tiles = -(-n // keys)
        for t in sorted({x for x in (0, 1, 2, tiles // 2, tiles - 2, tiles - 1, tiles, tiles + 1) if 0 <= x <= tiles + 1}):
            for run in range(0, keys, 16):
                j, got = t * keys + run, entry[keys](t, run, log, n)
                assert got == min(j, n - 1) >> log, f"tile {t} run {run} of {n} keys"
