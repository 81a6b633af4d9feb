"""What the calls of models over codes refuse and how their work is shared out (vq_amd/csrc/code_rules.hpp), compiled by g++ and
asked without a GPU: the entry points return these before they touch the device."""
import ctypes as C
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INVALID, UNSUPPORTED = -1, -4
MAIN = """
#include "code_rules.hpp"
#define P(v) ((const void *)(v))
typedef long long i64;
extern "C" {
int embed(int type, i64 t, int k, i64 ldt, int dim, int m, int cb, i64 c, i64 n, i64 cs, float scale, int out_type, i64 o, i64 ldo) {
    return vq::check_code_embed(type, P(t), k, ldt, dim, m, cb, P(c), n, cs, scale, out_type, P(o), ldo).status; }
int embed_grad(int type, i64 g, i64 n, i64 ldg, int dim, int m, int cb, i64 c, i64 cs, float scale, int k, int acc, int out_type, i64 o, i64 ldo) {
    return vq::check_code_embed_grad(type, P(g), n, ldg, dim, m, cb, P(c), cs, scale, k, acc, out_type, P(o), ldo).status; }
int distill(int type, i64 s, i64 n, i64 ld, int k, float beta, int top, i64 lp, i64 c, i64 ldt, int rest, i64 loss, i64 m, i64 l, i64 r, i64 gl, i64 g, i64 ldg) {
    return vq::check_code_distill(type, P(s), n, ld, k, beta, top, P(lp), P(c), ldt, rest, P(loss), P(m), P(l), P(r), P(gl), P(g), ldg).status; }
int back(int type, i64 s, i64 n, i64 ld, int k, float beta, int top, i64 lp, i64 c, i64 ldt, int rest, i64 m, i64 l, i64 r, i64 gl, i64 g, i64 ldg) {
    return vq::check_code_distill_grad(type, P(s), n, ld, k, beta, top, P(lp), P(c), ldt, rest, P(m), P(l), P(r), P(gl), P(g), ldg).status; }
int verify(int type, i64 t, i64 ldt, float beta, i64 q, i64 ldq, float bq, i64 n, int d, int k, int cb, i64 c, i64 cs, i64 u, i64 ldu, i64 a, i64 o, i64 ldo) {
    return vq::check_code_verify(type, P(t), ldt, beta, P(q), ldq, bq, n, d, k, cb, P(c), cs, P(u), ldu, P(a), P(o), ldo).status; }
i64 embed_bytes(i64 n, int k, int dim, int m) { return vq::embed_work(n, k, dim, m).bytes; }
int few(i64 n, int k, int m, i64 across) { return vq::embed_few(n, k, m, across); }
int lists(i64 n, int k, int m, i64 *out) { const vq::ListPlan p = vq::plan_lists(n, k, m); out[0] = p.width, out[1] = p.buckets, out[2] = p.share, out[3] = p.shares;
    const vq::EmbedWork w = vq::embed_work(n, k, 100, m); out[4] = w.below - w.counts, out[5] = w.partial - w.below, out[6] = w.counts - w.edges;
    out[7] = vq::list_lds(p.width, true); return 0; }
int plan(i64 n, int k, int grad, i64 *out) { const vq::DistillPlan p = vq::plan_distill(n, k, grad); out[0] = p.waves, out[1] = p.per_lane, out[2] = p.parts;
    out[3] = vq::distill_rows_of_a_launch(p); return 0; }
i64 distill_bytes(i64 n, int k) { return vq::distill_work(n, k); }
i64 verify_rows(int d, int k) { return vq::verify_sequences_of_a_launch(d, k); }
i64 verify_bytes(i64 n, int d, int k) { return vq::verify_work(n, d, k); }
int verify_parts(int k) { return vq::verify_parts(k); }
}
"""
A = 1 << 22  # the arrays' addresses are far apart


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("rules") / "codes.so")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover=all",
                    "-static-libubsan", "-x", "c++", "-", "-I", os.path.join(ROOT, "vq_amd", "csrc"), "-o", so], input=MAIN, text=True, check=True)
    lib = C.CDLL(so)
    i, q, f = C.c_int, C.c_longlong, C.c_float
    lib.embed.argtypes = [i, q, i, q, i, i, i, q, q, q, f, i, q, q]
    lib.embed_grad.argtypes = [i, q, q, q, i, i, i, q, q, f, i, i, i, q, q]
    lib.distill.argtypes = [i, q, q, q, i, f, i, q, q, q, i, q, q, q, q, q, q, q]
    lib.back.argtypes = [i, q, q, q, i, f, i, q, q, q, i, q, q, q, q, q, q]
    lib.verify.argtypes = [i, q, q, f, q, q, f, q, i, i, i, q, q, q, q, q, q, q]
    lib.embed_bytes.argtypes, lib.embed_bytes.restype = [q, i, i, i], q
    lib.plan.argtypes = [q, i, i, C.c_void_p]
    lib.distill_bytes.argtypes, lib.distill_bytes.restype = [q, i], q
    lib.verify_rows.argtypes, lib.verify_rows.restype = [i, i], q
    lib.verify_bytes.argtypes, lib.verify_bytes.restype = [q, i, i], q
    return lib


EMBED = dict(type=0, t=A, k=10, ldt=100, dim=100, m=2, cb=4, c=2 * A, n=4, cs=2, scale=1.0, out_type=0, o=3 * A, ldo=100)
EMBED_GRAD = dict(type=0, g=A, n=4, ldg=100, dim=100, m=2, cb=4, c=2 * A, cs=2, scale=1.0, k=10, acc=0, out_type=0, o=3 * A, ldo=100)
DISTILL = dict(type=0, s=A, n=4, ld=100, k=100, beta=1.0, top=3, lp=2 * A, c=3 * A, ldt=3, rest=1, loss=4 * A, m=5 * A, l=6 * A, r=7 * A, gl=8 * A, g=9 * A, ldg=100)
BACK = {k: v for k, v in DISTILL.items() if k != "loss"}
VERIFY = dict(type=0, t=A, ldt=100, beta=1.0, q=2 * A, ldq=100, bq=1.0, n=4, d=3, k=100, cb=4, c=3 * A, cs=3, u=4 * A, ldu=4, a=5 * A, o=6 * A, ldo=4)
CALLS = dict(embed=EMBED, embed_grad=EMBED_GRAD, distill=DISTILL, back=BACK, verify=VERIFY)
NAN, INF = float("nan"), float("inf")

REFUSED = [
    ("embed", dict(type=3), INVALID), ("embed", dict(out_type=-1), INVALID), ("embed", dict(n=-1), INVALID), ("embed", dict(k=0), INVALID), ("embed", dict(dim=0), INVALID),
    ("embed", dict(m=0), INVALID), ("embed", dict(m=65, cs=65), UNSUPPORTED), ("embed", dict(k=(1 << 20) + 1), UNSUPPORTED),
    ("embed", dict(dim=(1 << 20) + 1, ldt=1 << 21, ldo=1 << 21), UNSUPPORTED), ("embed", dict(ldt=99), INVALID), ("embed", dict(ldo=99), INVALID),
    ("embed", dict(cb=3), INVALID), ("embed", dict(cs=1), INVALID), ("embed", dict(c=2 * A + 2), INVALID), ("embed", dict(scale=NAN), INVALID), ("embed", dict(scale=INF), INVALID),
    ("embed", dict(scale=-INF), INVALID), ("embed", dict(t=0), INVALID), ("embed", dict(c=0), INVALID), ("embed", dict(o=0), INVALID), ("embed", dict(t=A + 2), INVALID),
    ("embed", dict(o=3 * A + 1), INVALID), ("embed", dict(o=A + 7996), INVALID), ("embed", dict(o=2 * A), INVALID), ("embed", dict(n=1 << 50), INVALID),
    ("embed", dict(ldt=1 << 60), INVALID), ("embed", dict(cs=1 << 60), INVALID),
    ("embed_grad", dict(type=7), INVALID), ("embed_grad", dict(n=-1), INVALID), ("embed_grad", dict(acc=2), INVALID), ("embed_grad", dict(n=(1 << 29) + 1), UNSUPPORTED),
    ("embed_grad", dict(g=0), INVALID), ("embed_grad", dict(c=0), INVALID), ("embed_grad", dict(o=0), INVALID), ("embed_grad", dict(n=0, o=0), INVALID),
    ("embed_grad", dict(o=A), INVALID), ("embed_grad", dict(o=2 * A), INVALID), ("embed_grad", dict(ldo=99), INVALID), ("embed_grad", dict(ldg=99), INVALID),
    ("embed_grad", dict(scale=NAN), INVALID), ("embed_grad", dict(g=A + 1), INVALID), ("embed_grad", dict(o=3 * A + 2), INVALID), ("embed_grad", dict(k=0), INVALID),
    ("distill", dict(type=5), INVALID), ("distill", dict(k=0), INVALID), ("distill", dict(k=(1 << 20) + 1, ld=1 << 21, ldg=1 << 21), UNSUPPORTED), ("distill", dict(ld=99), INVALID),
    ("distill", dict(beta=0.0), INVALID), ("distill", dict(beta=NAN), INVALID), ("distill", dict(beta=1e31), INVALID), ("distill", dict(top=0), INVALID),
    ("distill", dict(top=65, ldt=65), UNSUPPORTED), ("distill", dict(ldt=2), INVALID), ("distill", dict(rest=2), INVALID), ("distill", dict(rest=-1), INVALID),
    ("distill", dict(s=0), INVALID), ("distill", dict(lp=0), INVALID), ("distill", dict(c=0), INVALID), ("distill", dict(gl=0), INVALID), ("distill", dict(g=0), INVALID),
    ("distill", dict(lp=2 * A + 2), INVALID), ("distill", dict(loss=4 * A + 1), INVALID), ("distill", dict(loss=A), INVALID), ("distill", dict(m=4 * A + 8), INVALID),
    ("distill", dict(r=9 * A), INVALID), ("distill", dict(l=2 * A), INVALID), ("distill", dict(g=A + 400), INVALID), ("distill", dict(g=A, ldg=101), INVALID),
    ("distill", dict(g=3 * A), INVALID), ("distill", dict(ldg=99), INVALID), ("distill", dict(g=9 * A + 2), INVALID), ("distill", dict(n=1 << 50), INVALID),
    ("back", dict(m=0), INVALID), ("back", dict(l=0), INVALID), ("back", dict(r=0), INVALID), ("back", dict(gl=0), INVALID), ("back", dict(g=0), INVALID),
    ("back", dict(g=5 * A), INVALID), ("back", dict(g=7 * A), INVALID), ("back", dict(r=7 * A + 2), INVALID), ("back", dict(top=0), INVALID), ("back", dict(ldg=1), INVALID),
    ("verify", dict(type=3), INVALID), ("verify", dict(n=-1), INVALID), ("verify", dict(d=-1), INVALID), ("verify", dict(d=64, cs=64, ldu=65, ldo=65), UNSUPPORTED),
    ("verify", dict(k=0), INVALID), ("verify", dict(k=(1 << 20) + 1, ldt=1 << 21, ldq=1 << 21), UNSUPPORTED), ("verify", dict(n=(1 << 30) + 1), UNSUPPORTED),
    ("verify", dict(ldt=99), INVALID), ("verify", dict(ldq=99), INVALID), ("verify", dict(beta=0.0), INVALID), ("verify", dict(bq=-1.0), INVALID), ("verify", dict(bq=NAN), INVALID),
    ("verify", dict(cb=8), INVALID), ("verify", dict(cs=2), INVALID), ("verify", dict(c=3 * A + 2), INVALID), ("verify", dict(ldu=3), INVALID), ("verify", dict(ldo=3), INVALID),
    ("verify", dict(t=0), INVALID), ("verify", dict(c=0), INVALID), ("verify", dict(u=0), INVALID), ("verify", dict(a=0), INVALID), ("verify", dict(o=0), INVALID),
    ("verify", dict(t=A + 2), INVALID), ("verify", dict(q=2 * A + 1), INVALID), ("verify", dict(a=6 * A + 4), INVALID), ("verify", dict(o=A + 4), INVALID),
    ("verify", dict(a=4 * A), INVALID), ("verify", dict(o=3 * A), INVALID), ("verify", dict(ldt=1 << 60), INVALID),
]
TAKEN = [
    ("embed", {}), ("embed", dict(n=0, t=0, c=0, o=0)), ("embed", dict(type=1, t=A + 2)), ("embed", dict(cb=1, c=2 * A + 1)), ("embed", dict(scale=0.0)), ("embed", dict(scale=-3e38)),
    ("embed", dict(m=64, cs=64)),
    ("embed_grad", {}), ("embed_grad", dict(acc=1)), ("embed_grad", dict(n=0, g=0, c=0)), ("embed_grad", dict(n=0, g=0, c=0, o=0, acc=1)), ("embed_grad", dict(out_type=2, o=3 * A + 2)),
    ("distill", {}), ("distill", dict(gl=0, g=0, ldg=0)), ("distill", dict(g=A)), ("distill", dict(loss=0, m=0, l=0, r=0)), ("distill", dict(n=0, s=0, lp=0, c=0)),
    ("distill", dict(ldt=64, top=64)), ("distill", dict(type=2, s=A + 2, g=9 * A + 2)), ("distill", dict(lp=3 * A)),  # inputs may share memory
    ("back", {}), ("back", dict(g=A)), ("back", dict(rest=0, r=0)), ("back", dict(n=0, s=0, lp=0, c=0, m=0, gl=0)),
    ("verify", {}), ("verify", dict(q=0, ldq=0, bq=0.0)), ("verify", dict(d=0, c=0, cb=0, cs=0)), ("verify", dict(n=0, t=0, q=0, c=0, u=0, a=0, o=0)),
    ("verify", dict(d=63, cs=63, ldu=64, ldo=64)), ("verify", dict(q=A)),
]


@pytest.mark.parametrize("call,change,status", REFUSED)
def test_refused(lib, call, change, status):
    assert getattr(lib, call)(*{**CALLS[call], **change}.values()) == status


@pytest.mark.parametrize("call,change", TAKEN)
def test_taken(lib, call, change):
    assert getattr(lib, call)(*{**CALLS[call], **change}.values()) == 0


SIZES = [1, 2, 3, 15, 16, 17, 255, 256, 257, 511, 512, 513, 1024, 1025, 2048, 2049, 4096, 4097, 8192, 8193, 16384, 16385, 32768, 32769, 50021, 65536, 65537, 262144, 524289, 1 << 20]


def test_buckets_and_shares_hold_every_code_and_position(lib):
    lib.lists.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_void_p]
    out = (C.c_longlong * 8)()
    for k in SIZES:
        for n in (0, 1, 63, 1024, 1025, 4096, 32768, 32769, 50000, 100_000, 1_000_000, 16_777_216, 1 << 30):
            for m in (1, 4, 64):
                if n * m > 1 << 30:
                    continue
                lib.lists(n, k, m, out)
                width, buckets, share, shares, counts, below, edges, lds = out
                assert 1 <= width <= 512 and (buckets - 1) * width < k <= buckets * width and buckets * 1024 < 1 << 32 and lds <= 65536
                assert share * shares >= n and (shares == 1 or (shares - 1) * share < n) and shares <= 256 and share < 1 << 31
                if shares > 1:
                    assert counts >= 4 * m * shares * k and below >= 4 * m * shares * buckets
                assert edges >= 4 * m * -(-n // 1024)


def test_every_code_of_a_row_has_a_lane(lib):
    out = (C.c_longlong * 4)()
    for k in SIZES:
        for n in (1, 2, 63, 64, 100, 1023, 1024, 4096, 1 << 30):
            for grad in (0, 1):
                lib.plan(n, k, grad, out)
                waves, per_lane, parts, rows = out
                assert per_lane in {0: (32, 64), 1: (8, 16, 32, 64), 4: (32, 64), 16: (32, 64)}[waves]
                held = (64 * waves if waves else 256) * per_lane
                assert parts * held >= k and (parts - 1) * held < k and parts <= 64 and (waves == 0 or parts == 1)
                assert rows >= 1
                lanes = 64 * waves if waves > 1 else 64 if waves else 256
                assert rows * parts * lanes < 1 << 32
                if waves == 0:  # the parts' sums, and three numbers per row for the gradient
                    assert lib.distill_bytes(n, k) >= min(n, rows) * (parts * 8 + 12)


def test_drafts_fit_their_launches(lib):
    for k in SIZES:
        assert (lib.verify_parts(k) - 1) * 4096 < k <= lib.verify_parts(k) * 4096 and lib.verify_parts(k) <= 256
        for d in (0, 1, 5, 63):
            most = lib.verify_rows(d, k)
            assert most >= 1 and most * (2 * d + 1) * lib.verify_parts(k) * 256 < 1 << 32
            for n in (1, 5, 1000, 1 << 30):
                assert lib.verify_bytes(n, d, k) >= min(n, most) * (lib.verify_parts(k) * ((2 * d + 1) * 16 + 8) + 64)


def test_workspaces_grow_with_every_size(lib):
    """A call that is smaller in no size finds no larger workspace than the one before left."""
    for k in SIZES:
        for n in (1, 63, 64, 1000, 1024, 1025, 5000, 100_000):
            for up in (n, n + 1, 2 * n):
                for more in (k, min(k + 1, 1 << 20), min(2 * k, 1 << 20)):
                    assert lib.distill_bytes(up, more) >= lib.distill_bytes(n, k)
                    for d in (0, 3, 63):
                        assert lib.verify_bytes(up, d, more) >= lib.verify_bytes(n, d, k) and lib.verify_bytes(up, min(d + 1, 63), more) >= lib.verify_bytes(n, d, k)
                    assert lib.embed_bytes(up, more, 100, 2) >= lib.embed_bytes(n, k, 100, 2) and lib.embed_bytes(up, more, 101, 3) >= lib.embed_bytes(n, k, 100, 2)


def test_a_missing_context_is_an_error():
    from vq_amd import _ffi
    lib = _ffi.lib()
    assert lib.vq_code_embed(None, 0, None, 1, 1, 1, 1, 4, None, 0, 1, 1.0, 0, None, 1) == INVALID
    assert lib.vq_code_embed_grad(None, 0, None, 0, 1, 1, 1, 4, None, 1, 1.0, 1, 0, 0, None, 1) == INVALID
    assert lib.vq_code_distill(None, 0, None, 0, 1, 1, 1.0, 1, None, None, 1, 0, None, None, None, None, None, None, 1) == INVALID
    assert lib.vq_code_distill_grad(None, 0, None, 0, 1, 1, 1.0, 1, None, None, 1, 0, None, None, None, None, None, 1) == INVALID
    assert lib.vq_code_verify(None, 0, None, 1, 1.0, None, 1, 1.0, 0, 0, 1, 4, None, 1, None, 1, None, None, 1) == INVALID


def test_lists_of_their_own_stay_so_for_smaller_calls(lib):
    """A call without a buffer is followed by none, smaller in every size, that needs one."""
    lib.few.argtypes = [C.c_longlong, C.c_int, C.c_int, C.c_longlong]
    for k in SIZES:
        for m in (1, 2, 8, 64):
            for across in (1, 2, 5, 40):
                for n in (0, 1, 1000, 1024):
                    codes = lib.few(n, k, m, across)
                    assert codes in (0, 4, 16, 64)
                    if codes:
                        assert -(-k // codes) * m * across <= 1024
                        assert all(lib.few(a, b, c, d) for a, b, c, d in ((n // 2, k, m, across), (n, max(1, k - 1), m, across), (n, k // 2 + 1, m, across), (n, k, max(1, m - 1), across),
                                                                          (n, k, m, max(1, across - 1))))
                assert not lib.few(1025, k, m, across)
