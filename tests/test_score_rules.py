"""What the calls on 8-bit scores and log probabilities of codes refuse (vq_amd/csrc/score_rules.hpp), compiled by g++ and
asked without a GPU: the entry points return these before they touch the device."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -4
MAIN = """
#include "score_rules.hpp"
#define P(v) ((const void *)(v))
typedef long long i64;
extern "C" {
int rows(int type, i64 x, i64 n, i64 ld, int dim, i64 q, i64 ldq, i64 s) {
    return vq::check_rows_i8(type, P(x), n, ld, dim, P(q), ldq, P(s)).status; }
int scores(i64 x, i64 xs, i64 n, i64 ldx, i64 w, i64 ws, int k, i64 ldw, int dim, i64 b, int type, i64 out, i64 ldo) {
    return vq::check_scores_i8(P(x), P(xs), n, ldx, P(w), P(ws), k, ldw, dim, P(b), type, P(out), ldo).status; }
int logprobs(int type, i64 s, i64 n, i64 ld, int k, float beta, int cb, i64 c, i64 cs, int top, i64 lp, i64 m, i64 l, i64 h, i64 tl, i64 tc) {
    return vq::check_code_logprobs(type, P(s), n, ld, k, beta, cb, P(c), cs, top, P(lp), P(m), P(l), P(h), P(tl), P(tc)).status; }
int plan(i64 n, int k, int top, i64 *out) { const vq::RowPlan p = vq::plan_rows(n, k, top); out[0] = p.lanes, out[1] = p.per_lane, out[2] = p.parts, out[3] = p.codes; return 0; }
int way(i64 n, int k, int dim) { return vq::score_way(n, k, dim); }
i64 launch_rows(int k) { return vq::score_rows_of_a_launch(k); }
int pack(i64 n, int k, int dim) { return vq::score_pack(n, k, dim); }
int lanes(int length, int bytes) { const vq::LanePlan p = vq::plan_lanes(length, bytes); return p.lanes * p.vectors * 16 / bytes; }
int grad(int type, i64 s, i64 n, i64 ld, int k, float beta, int cb, i64 c, i64 cs, i64 m, i64 l, i64 h, i64 gl, i64 gh, i64 g, i64 ldg) {
    return vq::check_code_logprobs_grad(type, P(s), n, ld, k, beta, cb, P(c), cs, P(m), P(l), P(h), P(gl), P(gh), P(g), ldg).status; }
}
"""
A = 1 << 20  # the arrays' addresses are far apart


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rules") / "rules.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-static-libubsan", "-x", "c++", "-", "-I", os.path.join(ROOT, "vq_amd", "csrc"), "-o", so], input=MAIN, text=True, check=True)
    lib = C.CDLL(so)
    i, q, f = C.c_int, C.c_longlong, C.c_float
    lib.rows.argtypes = [i, q, q, q, i, q, q, q]
    lib.scores.argtypes = [q, q, q, q, q, q, i, q, i, q, i, q, q]
    lib.logprobs.argtypes = [i, q, q, q, i, f, i, q, q, i, q, q, q, q, q, q]
    lib.grad.argtypes = [i, q, q, q, i, f, i, q, q, q, q, q, q, q, q, q]
    return lib


ROWS = dict(type=0, x=A, n=4, ld=100, dim=100, q=2 * A, ldq=112, s=3 * A)
SCORES = dict(x=A, xs=2 * A, n=4, ldx=112, w=3 * A, ws=4 * A, k=10, ldw=112, dim=100, b=5 * A, type=0, out=6 * A, ldo=10)
LOGPROBS = dict(type=0, s=A, n=4, ld=100, k=100, beta=1.0, cb=4, c=2 * A, cs=1, top=3, lp=3 * A, m=4 * A, l=5 * A, h=6 * A, tl=7 * A, tc=8 * A)
GRAD = dict(type=0, s=A, n=4, ld=100, k=100, beta=1.0, cb=4, c=2 * A, cs=1, m=3 * A, l=4 * A, h=5 * A, gl=6 * A, gh=7 * A, g=8 * A, ldg=100)
CALLS = dict(rows=ROWS, scores=SCORES, logprobs=LOGPROBS, grad=GRAD)

REFUSED = [
    ("rows", dict(type=3), INVALID), ("rows", dict(type=-1), INVALID), ("rows", dict(n=-1), INVALID), ("rows", dict(dim=0), INVALID),
    ("rows", dict(dim=131072, ld=131072, ldq=131072), UNSUPPORTED), ("rows", dict(ld=99), INVALID), ("rows", dict(ldq=99), INVALID),
    ("rows", dict(x=0), INVALID), ("rows", dict(q=0), INVALID), ("rows", dict(s=0), INVALID), ("rows", dict(x=A + 2), INVALID),
    ("rows", dict(s=3 * A + 1), INVALID), ("rows", dict(q=A + 4 * 399), INVALID), ("rows", dict(s=A), INVALID), ("rows", dict(s=2 * A + 96), INVALID),
    ("rows", dict(n=1 << 56, ld=1 << 10), INVALID), ("rows", dict(n=2, ldq=1 << 62), INVALID),
    ("scores", dict(k=0), INVALID), ("scores", dict(dim=-1), INVALID), ("scores", dict(type=7), INVALID), ("scores", dict(k=(1 << 24) + 1, ldo=1 << 25), UNSUPPORTED),
    ("scores", dict(dim=131072, ldx=131072, ldw=131072), UNSUPPORTED), ("scores", dict(ldx=99), INVALID), ("scores", dict(ldw=99), INVALID),
    ("scores", dict(ldo=9), INVALID), ("scores", dict(xs=0), INVALID), ("scores", dict(ws=0), INVALID), ("scores", dict(out=0), INVALID),
    ("scores", dict(b=5 * A + 2), INVALID), ("scores", dict(out=6 * A + 2), INVALID), ("scores", dict(out=A), INVALID),
    ("scores", dict(out=3 * A + 1000), INVALID), ("scores", dict(out=5 * A), INVALID), ("scores", dict(n=1 << 61), INVALID),
    ("logprobs", dict(k=0), INVALID), ("logprobs", dict(ld=99), INVALID), ("logprobs", dict(beta=0.0), INVALID), ("logprobs", dict(beta=-1.0), INVALID),
    ("logprobs", dict(beta=float("nan")), INVALID), ("logprobs", dict(beta=float("inf")), INVALID), ("logprobs", dict(beta=1e31), INVALID), ("logprobs", dict(beta=1e-31), INVALID), ("logprobs", dict(cb=3), INVALID),
    ("logprobs", dict(cb=8), INVALID), ("logprobs", dict(cs=0), INVALID), ("logprobs", dict(c=2 * A + 2), INVALID), ("logprobs", dict(c=0), INVALID),
    ("logprobs", dict(lp=0), INVALID), ("logprobs", dict(top=-1), INVALID), ("logprobs", dict(top=33), UNSUPPORTED), ("logprobs", dict(tl=0), INVALID),
    ("logprobs", dict(tc=0), INVALID), ("logprobs", dict(s=0), INVALID), ("logprobs", dict(s=A + 1), INVALID), ("logprobs", dict(m=4 * A + 2), INVALID),
    ("logprobs", dict(k=(1 << 20) + 1, ld=1 << 25), UNSUPPORTED), ("logprobs", dict(h=A + 8), INVALID), ("logprobs", dict(tl=8 * A), INVALID),
    ("logprobs", dict(lp=4 * A + 12), INVALID), ("logprobs", dict(tc=2 * A), INVALID),
    ("grad", dict(ldg=99), INVALID), ("grad", dict(m=0), INVALID), ("grad", dict(l=0), INVALID), ("grad", dict(h=0), INVALID), ("grad", dict(g=0), INVALID),
    ("grad", dict(gl=0, gh=0), INVALID), ("grad", dict(c=0), INVALID), ("grad", dict(g=A + 400), INVALID), ("grad", dict(g=A, ldg=101), INVALID),
    ("grad", dict(g=3 * A), INVALID), ("grad", dict(g=2 * A), INVALID), ("grad", dict(beta=0.0), INVALID), ("grad", dict(gl=6 * A + 1), INVALID),
    ("grad", dict(g=8 * A + 2), INVALID), ("grad", dict(type=2, s=A + 1), INVALID),
]
TAKEN = [
    ("rows", {}), ("rows", dict(n=0, x=0, q=0, s=0)), ("rows", dict(type=2, x=A + 2)), ("rows", dict(q=2 * A + 1, ldq=101)), ("rows", dict(dim=1, ld=1, ldq=1)),
    ("rows", dict(dim=131071, ld=131071, ldq=131071, q=8 * A, s=16 * A)),
    ("scores", {}), ("scores", dict(n=0, x=0, xs=0, w=0, ws=0, out=0)), ("scores", dict(b=0)), ("scores", dict(x=A + 3, ldx=101)), ("scores", dict(type=1, out=6 * A + 2)),
    ("scores", dict(xs=4 * A)),  # inputs may share memory
    ("logprobs", {}), ("logprobs", dict(n=0, s=0, c=0, lp=0, m=0, l=0, h=0, tl=0, tc=0)), ("logprobs", dict(top=0, tl=0, tc=0)), ("logprobs", dict(c=0, lp=0)),
    ("logprobs", dict(m=0, l=0, h=0)), ("logprobs", dict(cb=1, c=2 * A + 1, cs=16)), ("logprobs", dict(top=32, k=2, ld=2)), ("logprobs", dict(beta=1.1e-30)),
    ("grad", {}), ("grad", dict(g=A)), ("grad", dict(gl=0, c=0)), ("grad", dict(gh=0, h=0)), ("grad", dict(n=0, s=0, g=0, m=0)),
]


@pytest.mark.parametrize("call,change,status", REFUSED)
def test_refused(lib, call, change, status):
    assert getattr(lib, call)(*{**CALLS[call], **change}.values()) == status


@pytest.mark.parametrize("call,change", TAKEN)
def test_taken(lib, call, change):
    assert getattr(lib, call)(*{**CALLS[call], **change}.values()) == 0


def test_every_code_of_a_row_has_a_lane(lib):
    lib.plan.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_void_p]
    out = (C.c_longlong * 4)()
    for k in [1, 2, 3, 7, 8, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1023, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 50021, 65536, 262144, 1000003, 1 << 20]:
        for n in (1, 2, 3, 15, 16, 17, 64, 255, 1024, 100_000, 1 << 30):
            for top in (0, 2, 8, 32):
                lib.plan(n, k, top, out)
                lanes, per_lane, parts, codes = out
                assert codes <= lanes * per_lane and parts * codes >= k and (parts - 1) * codes < k and (parts == 1 or (lanes == 256 and codes % 64 == 0))
                assert parts <= 64 and (parts == 1 or codes == lanes * per_lane)
                assert per_lane in {1: (16,), 4: (16,), 8: (32,), 64: (8, 16, 32, 64), 256: (32, 64)}[lanes]
                assert lanes < 64 or k >= 8  # a vector of 16 bytes at least


def test_tiles_fit_their_launches(lib):
    """Rows and codes of a workgroup, and its lanes, by way: a grid has fewer than 2^32 lanes and at most 65,535 workgroups in its
    second dimension, which k_scores_any and FEW use for the rows."""
    lib.way.argtypes, lib.launch_rows.argtypes, lib.launch_rows.restype = [C.c_longlong, C.c_int, C.c_int], [C.c_int], C.c_longlong
    lib.pack.argtypes = [C.c_longlong, C.c_int, C.c_int]
    size = [(16, 16, 256), (64, 64, 256), (64, 64, 256), (64, 128, 512), (128, 128, 512), (256, 256, 512), (128, 128, 512)]
    seen = set()
    for k in [1, 2, 16, 24, 64, 65, 127, 128, 129, 256, 777, 1024, 4096, 65536, 262144, 1 << 24]:
        most = lib.launch_rows(k)
        assert most >= 64 and most % 64 == 0 and most // 64 <= 65535 and most // 64 * -(-k // 64) * 256 < 1 << 32
        for n in [1, 2, 16, 17, 64, 65, 128, 129, 300, 1000, 4099, 16384, 100_000, most - 1, most]:
            for dim in (1, 128, 8192, 131071):
                if n <= most:
                    w = lib.way(n, k, dim)
                    rows, codes, wg = size[w]
                    tiles = -(-n // rows) * -(-k // codes)
                    assert tiles * wg < 1 << 32 and (w or -(-n // 16) <= 65535)
                    seen.add(w)
                if lib.pack(n, k, dim):
                    assert k * (dim + 15) <= (1 << 30) + 15 * k and n * k * dim >= 1 << 28
    assert seen == set(range(7))


def test_rows_in_registers(lib):
    for size in (2, 4):
        for length in [1, 3, 4, 7, 8, 64, 65, 128, 129, 512, 513, 1024, 1025, 2048, 2049, 8192, 8193, 16384, 16385, 131071]:
            held = lib.lanes(length, size)
            assert held >= length if 16 // size <= length <= 2048 * 16 // size else held == 0


def test_a_missing_context_is_an_error():
    from vq_amd import _ffi
    lib = _ffi.lib()
    assert lib.vq_rows_i8(None, 0, None, 0, 1, 1, None, 1, None) == INVALID
    assert lib.vq_scores_i8(None, None, None, 0, 1, None, None, 1, 1, 1, None, 0, None, 1) == INVALID
    assert lib.vq_code_logprobs(None, 0, None, 0, 1, 1, 1.0, 4, None, 1, 0, None, None, None, None, None, None) == INVALID
    assert lib.vq_code_logprobs_grad(None, 0, None, 0, 1, 1, 1.0, 4, None, 1, None, None, None, None, None, None, 1) == INVALID
