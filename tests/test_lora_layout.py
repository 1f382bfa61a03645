"""Every index of the adapter kernels' workspace, followed on the host from the
functions that the kernels themselves use: z as it is written and as expand
reads it lies within grimoire_lora_workspace_bytes for every max_rank, rank,
split and number of rows."""
import ctypes as C
import os
import subprocess

import pytest

from grimoire_amd import _abi, build

PROGRAM = r"""
#include "lora_layout.hpp"
#include <algorithm>
using namespace grim;

// end of the last byte of z that shrink writes (at[0]) and expand reads
// (at[1]) for `rows` rows; 1 if a rank's code is too short
extern "C" int z_ends(int K, int R, int rows, int64_t* at) {
    const int splits = lora_splits(K, rows), mc = lora_max_chunks(R);
    const int64_t tiles = (int64_t(rows) + kLoraRows - 1) / kLoraRows;
    at[0] = at[1] = 0;
    for (int rank = 1; rank <= R; ++rank) {
        for (int f = 0; f < (rank + 15) / 16; ++f)
            at[0] = std::max(at[0], (lora_z_run(R, rows, splits - 1, tiles - 1, f >> 1, 1) + 1) * kLoraRunBytes);
        int code = 1;
        while (!lora_code_is(code, mc, rank)) code *= 2;
        if (code * 32 < rank) return 1;
        for (int c = 0; c < code; ++c)
            at[1] = std::max(at[1], (lora_z_run(R, rows, splits - 1, tiles - 1, c, 1) + 1) * kLoraRunBytes);
    }
    return 0;
}
"""


@pytest.fixture(scope="module")
def z_ends(tmp_path_factory):
    d = tmp_path_factory.mktemp("lora_layout")
    (d / "p.cc").write_text(PROGRAM)
    subprocess.run([build.CXX, "-std=c++17", "-O1", "-shared", "-fPIC", "-I", str(build.CSRC), "-o", str(d / "p.so"),
                    str(d / "p.cc")], check=True)
    fn = C.CDLL(os.fspath(d / "p.so")).z_ends
    fn.argtypes = [C.c_int, C.c_int, C.c_int, C.POINTER(C.c_int64)]

    def ends(K, R, rows):
        at = (C.c_int64 * 2)()
        assert fn(K, R, rows, at) == 0, (K, R, rows)
        return at[0], at[1]
    return ends


@pytest.mark.parametrize("R", range(16, 257, 16))
def test_z_lies_in_the_workspace(z_ends, R):
    for K in (8, 64, 512, 520, 1032, 2048, 2880, 7168):
        L = _abi.Lora(K=K, N=32, slots=1, max_rank=R)
        for rows in (1, 15, 16, 17, 20, 33, 96, 511, 512, 513, 700, 1031, 4096, 5000, 9000, 100001):
            need = int(_abi.lib().grimoire_lora_workspace_bytes(C.byref(L), rows))
            written, read = z_ends(K, R, rows)
            assert written <= need and read <= need, (K, rows, written, read, need)
