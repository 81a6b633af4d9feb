"""How rows of scores and 8-bit scores are shared out (vq_amd/csrc/score_rules.hpp), compiled by g++ and asked without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

from scores_sizes import SIZES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN = """
#include "score_rules.hpp"
typedef long long i64;
extern "C" {
int plan(i64 n, int k, int top, int bytes, i64 *out) {
    const vq::RowPlan p = vq::plan_rows(n, k, top, bytes); out[0] = p.lanes, out[1] = p.per_lane, out[2] = p.parts, out[3] = p.codes; return 0; }
i64 parts_taken(i64 n, int k, int top) {
    const vq::RowPlan p = vq::plan_rows(n, k, top, 2);
    return p.parts == 1 ? 0 : std::min<int64_t>(n, vq::logprob_rows_of_a_launch(p, top)) * p.parts * vq::part_bytes(top); }
i64 parts_provided(i64 n, int k, int top) { return vq::part_workspace(n, k, top); }
int way(i64 n, int k, int dim) { return vq::score_way(n, k, dim); }
}
"""
LENGTHS = [1, 2, 3, 4, 7, 8, 9, 15, 16, 17, 63, 64, 65, 128, 129, 160, 168, 200, 255, 256, 257, 512, 513, 1023, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384,
           16385, 50021, 65536, 262144, 524288, 524289, 1000003, 1 << 20]
ROWS = [1, 2, 3, 15, 16, 17, 64, 255, 1023, 1024, 2047, 2048, 4095, 4096, 16384, 16385, 100_000, 1 << 30]
TOPS = [0, 1, 2, 7, 8, 15, 16, 20, 31, 32]


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("plans") / "plans.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-static-libubsan", "-x", "c++", "-", "-I", os.path.join(ROOT, "vq_amd", "csrc"), "-o", so], input=MAIN, text=True, check=True)
    lib = C.CDLL(so)
    lib.plan.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_int, C.c_void_p]
    for f in (lib.parts_taken, lib.parts_provided):
        f.argtypes, f.restype = [C.c_longlong, C.c_int, C.c_int], C.c_longlong
    lib.way.argtypes = [C.c_longlong, C.c_int, C.c_int]
    return lib


@pytest.mark.parametrize("bytes_", [2, 4])
def test_every_code_of_a_row_has_a_lane(lib, bytes_):
    """By the size of an element: every code has a register, and where lanes read whole vectors a row has one."""
    out = (C.c_longlong * 4)()
    for k in LENGTHS:
        for n in ROWS:
            for top in TOPS:
                lib.plan(n, k, top, bytes_, out)
                lanes, per_lane, parts, codes = out
                assert parts * codes >= k and (parts - 1) * codes < k and codes <= lanes * per_lane
                assert parts <= 64 and (parts == 1 or (lanes == 256 and codes == lanes * per_lane))
                assert per_lane in {1: (16,), 4: (16,), 8: (32,), 64: (8, 16, 32, 64), 256: (32, 64)}[lanes]
                assert k >= 16 // bytes_ or lanes == 1


def test_sizes_of_the_tests_reach_every_way(lib):
    assert set(SIZES) == set(range(7))
    for way, sizes in SIZES.items():
        for n, dim, k in sizes:
            assert lib.way(n, k, dim) == way, (n, dim, k)


def test_a_smaller_call_needs_no_more(lib):
    """The workspace of a call holds what its plan takes, and what any call takes that is larger in none of rows, codes and
    alternatives."""
    grid = {(n, k, top): lib.parts_provided(n, k, top) for n in ROWS for k in LENGTHS for top in TOPS}
    for (n, k, top), held in grid.items():
        assert lib.parts_taken(n, k, top) <= held <= 64 << 20
        i, j, t = ROWS.index(n), LENGTHS.index(k), TOPS.index(top)
        for less in ((ROWS[i - 1] if i else n, k, top), (n, LENGTHS[j - 1] if j else k, top), (n, k, TOPS[t - 1] if t else top)):
            assert grid[less] <= held
    assert any(lib.parts_taken(n - 1, k, 2) > lib.parts_taken(n, k, 2) for n, k in ((1024, 65536), (2048, 16385)))
