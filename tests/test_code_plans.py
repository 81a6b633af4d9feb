"""How the work of the calls of models over codes is shared out (vq_amd/csrc/code_rules.hpp), compiled by g++ and asked without a GPU: what the kernels
count on beside what test_code_rules.py asks."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MAIN = """
#include "code_rules.hpp"
typedef long long i64;
extern "C" {
int plan(i64 n, int k, int grad, i64 *out) { const vq::DistillPlan p = vq::plan_distill(n, k, grad); out[0] = p.waves, out[1] = p.parts;
    out[2] = vq::distill_rows_of_a_launch(p); return 0; }
int lists(i64 n, int k, int m, i64 *out) { const vq::ListPlan p = vq::plan_lists(n, k, m); out[0] = p.buckets, out[1] = p.shares,
    out[2] = vq::list_lds(p.width, true), out[3] = vq::list_lds(p.width, false), out[4] = vq::kListBeside; return 0; }
i64 distill_bytes(i64 n, int k) { return vq::distill_work(n, k); }
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rules") / "plans.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-static-libubsan", "-x", "c++", "-", "-I", os.path.join(ROOT, "vq_amd", "csrc"), "-o", so], input=MAIN, text=True, check=True)
    lib = C.CDLL(so)
    lib.plan.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_void_p]
    lib.distill_bytes.argtypes, lib.distill_bytes.restype = [C.c_longlong, C.c_int], C.c_longlong
    return lib


def test_rows_in_parts_have_their_sums_and_five_numbers(lib):
    """m, L, log R, and the rest's largest score and sum, for the gradient behind the parts' results; at most 2^22 rows, so that the gradient of a
    launch's rows is a launch, too."""
    out = (C.c_longlong * 3)()
    for k in (16385, 20000, 32768, 32769, 50021, 65536, 65537, 100_003, 524_288, 524_289, 1 << 20):
        for n in (1, 63, 64, 1000, 5000, 1 << 20, 1 << 22, 1 << 23, 1 << 24, 1 << 30):
            for grad in (0, 1):
                lib.plan(n, k, grad, out)
                waves, parts, rows = out
                if waves == 0:
                    assert parts >= 2 and rows <= 1 << 22
                    assert lib.distill_bytes(n, k) >= min(n, rows) * (parts * 8 + 20)


def test_two_workgroups_that_list_positions_fit_a_compute_unit(lib):
    """By all of their LDS, the 160 KB of a compute unit: what a launch asks for and what the kernel has beside.  Shares are cut where that makes at
    most 1024 workgroups."""
    lib.lists.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_void_p]
    out = (C.c_longlong * 5)()
    for n in (0, 1, 1024, 32768, 32769, 100_000, 1_000_000, 1 << 24):
        for k in (1, 2, 255, 256, 257, 480, 481, 8379, 65536, 262_144, 1 << 20):
            for m in (1, 4, 8, 64):
                lib.lists(n, k, m, out)
                buckets, shares, lds, count_lds, beside = out
                assert lds + beside <= 80 * 1024 and count_lds + beside <= 80 * 1024
                assert shares == 1 or buckets * m * shares <= 1024
