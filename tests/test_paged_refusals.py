"""What ghip_rope, ghip_kv_append and ghip_flash_attn_paged refuse, and that what
they accept stores inside its buffers, on a context without a device; and the
index arithmetic of the paged kernels in a host build."""
import ctypes as C
import os
import random
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = [i << 40 for i in range(1, 10)]  # addresses: compared, never read


@pytest.fixture()
def ctx():
    import ghip
    L = ghip.lib()
    L.ghip_init_dry_run.restype = C.c_int
    L.ghip_init_dry_run.argtypes = [C.POINTER(C.c_void_p)]
    c = C.c_void_p()
    assert L.ghip_init_dry_run(C.byref(c)) == 0
    yield c
    L.ghip_free(c)


def T(ty, ne, data, e=None, nb=None):
    import ghip
    t = ghip.Tensor()
    t.type = ty
    e = e or ghip.BLOCK[ty][1]
    ne = list(ne) + [1] * (4 - len(ne))
    t.ne[:] = ne
    t.nb[:] = nb or [e, e * ne[0], e * ne[0] * ne[1], e * ne[0] * ne[1] * ne[2]]
    t.data = data
    return t


def ref(t):
    return C.byref(t) if t is not None else None


def rope_params(n_dims=64, mode=2, sections=(0, 0, 0, 0), **kw):
    import ghip
    return ghip.Rope(n_dims, mode, sections=sections, **kw).params


def run_rope(ctx, D=64, H=4, N=9, n_dims=64, mode=2, sections=(0, 0, 0, 0), xty=0, dty=None, pos=None, factors=None, dst=None, x=None, **kw):
    import ghip
    x = T(xty, [D, H, N], A[0]) if x is None else x
    d = T(xty if dty is None else dty, [D, H, N], A[1]) if dst is None else dst
    pos = T(ghip.I32, [N, 4 if sum(sections) else 1], A[2]) if pos is None else pos
    r = rope_params(n_dims, mode, sections, **kw)
    st = ghip.lib().ghip_rope(ctx, ref(x), ref(pos), ref(factors), C.byref(r), ref(d), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


def test_rope_accepts(ctx):
    import ghip
    for N in (0, 1, 9, 5000):
        for ty in (ghip.F32, ghip.F16, ghip.BF16):
            for D, n, mode, s in ((64, 64, 2, (0,) * 4), (80, 20, 0, (0,) * 4), (128, 128, 8, (16, 24, 24, 0)),
                                  (128, 128, 40, (24, 20, 20, 0)), (80, 40, 24, (20, 20, 0, 0)), (33, 12, 2, (0,) * 4)):
                st, msg = run_rope(ctx, D=D, n_dims=n, mode=mode, sections=s, N=N, xty=ty)
                assert st == 0, msg


def test_rope_refuses(ctx):
    import ghip
    for want, kw in [
            ("mode", dict(mode=1)), ("n_dims", dict(n_dims=63)), ("n_dims", dict(n_dims=0)), ("n_dims", dict(n_dims=66)),
            ("n_dims", dict(mode=24, sections=(9, 9, 0, 0))), ("freq_base", dict(freq_base=0.0)),
            ("freq_base", dict(freq_base=float("inf"))), ("freq_scale", dict(freq_scale=-1.0)),
            ("sections", dict(mode=8)), ("sections", dict(mode=40, sections=(4, -1, 4, 0))),
            ("ext_factor", dict(ext_factor=1.0)), ("ext_factor", dict(ext_factor=float("nan"))),
            ("F32, F16 or BF16", dict(xty=ghip.I32)), ("of its type", dict(dty=ghip.F16)),
            ("shape", dict(dst=T(ghip.F32, [64, 4, 8], A[1]))), ("null data", dict(dst=T(ghip.F32, [64, 4, 9], None))),
            ("fewer positions", dict(pos=T(ghip.I32, [8], A[2]))), ("I32", dict(pos=T(ghip.F32, [9], A[2]))),
            ("each axis", dict(mode=8, sections=(8, 8, 16, 0), pos=T(ghip.I32, [9, 2], A[2]))),
            ("factors", dict(factors=T(ghip.F32, [31], A[3]))), ("factors", dict(factors=T(ghip.F16, [32], A[3]))),
            ("apart", dict(dst=T(ghip.F32, [64, 4, 9], A[0] + 256))),
            ("strides", dict(dst=T(ghip.F32, [64, 4, 9], A[0], nb=[4, 512, 2048, 20480]))),
            ("rows of elements", dict(x=T(ghip.F32, [64, 4, 9], A[0], nb=[8, 512, 2048, 20480]))),
            ("[D, H, T]", dict(x=T(ghip.F32, [64, 4, 9, 2], A[0]), dst=T(ghip.F32, [64, 4, 9, 2], A[1])))]:
        st, msg = run_rope(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)
    L = ghip.lib()
    x, pos, r = T(0, [64, 4, 9], A[0]), T(ghip.I32, [9], A[2]), rope_params()
    for args in ((None, ref(pos), None, C.byref(r), ref(x)), (ref(x), None, None, C.byref(r), ref(x)), (ref(x), ref(pos), None, None, ref(x)),
                 (ref(x), ref(pos), None, C.byref(r), None)):
        assert L.ghip_rope(ctx, *args, None) != 0
    assert L.ghip_rope(None, ref(x), ref(pos), None, C.byref(r), ref(x), None) != 0


def run_append(ctx, D=64, Hkv=2, N=9, kty=0, vty=None, cty=1, page=16, pages=5, slots=None, kv=None, v=None, k=None, rope=True, pos=True, factors=None, **kw):
    import ghip
    k = T(kty, [D, Hkv, N], A[0]) if k is None else k
    v = T(kty if vty is None else vty, [D, Hkv, N], A[1]) if v is None else v
    slots = T(ghip.I64, [N], A[2]) if slots is None else slots
    kv = T(cty, [2 * D, Hkv, page, pages], A[3]) if kv is None else kv
    p = T(ghip.I32, [N], A[4]) if pos is True else pos
    r = rope_params(**kw) if rope else None
    st = ghip.lib().ghip_kv_append(ctx, ref(k), ref(v), ref(slots), ref(p), ref(factors), ref(r), ref(kv), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


def test_append(ctx):
    import ghip
    for N in (0, 1, 9, 8192):
        for kty, cty in ((0, 1), (0, 30), (1, 1), (30, 30)):
            for page, pages in ((1, 4), (24, 600), (16, 0)):
                st, msg = run_append(ctx, N=N, kty=kty, cty=cty, page=page, pages=pages)
                assert st == 0, msg
    st, msg = run_append(ctx, rope=False, pos=None)
    assert st == 0, msg
    st, msg = run_append(ctx, kv=T(1, [128, 2, 16, 5], A[3], nb=[2, 300, 600, 20000]))
    assert st == 0, msg
    for want, kw in [
            ("kv must be F16", dict(cty=0)), ("kv's type", dict(kty=1, cty=30)), ("kv's type", dict(vty=1)),
            ("same shape", dict(v=T(0, [64, 2, 8], A[1]))), ("head size", dict(D=264)),
            ("2 D", dict(kv=T(1, [64, 2, 16, 5], A[3]))), ("2 D", dict(kv=T(1, [128, 3, 16, 5], A[3]))),
            ("I64", dict(slots=T(ghip.I32, [9], A[2]))), ("I64", dict(slots=T(ghip.I64, [8], A[2]))),
            ("need a rotation", dict(rope=False)), ("n_dims", dict(n_dims=128)), ("pos", dict(pos=None)),
            ("null data", dict(slots=T(ghip.I64, [9], None))), ("apart", dict(kv=T(1, [128, 2, 16, 5], A[0] + 64))),
            ("factors", dict(factors=T(ghip.F32, [9], A[5])))]:
        st, msg = run_append(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)


def run_paged(ctx, D=64, H=8, Hkv=2, N=9, B=3, per=7, cty=1, page=16, pages=50, q=None, kv=None, seqs=None, sinks=None, dst=None, scale=0.1, window=0,
              n_first=0, n_shared=0, max_q=3):
    import ghip
    q = T(0, [D, H, N], A[0]) if q is None else q
    kv = T(cty, [2 * D, Hkv, page, pages], A[1]) if kv is None else kv
    seqs = T(ghip.I32, [3 + per, B], A[2]) if seqs is None else seqs
    dst = T(0, [D, H, N], A[3]) if dst is None else dst
    pp = ghip.PagedParams(scale, window, n_first, n_shared, max_q)
    st = ghip.lib().ghip_flash_attn_paged(ctx, ref(q), ref(kv), ref(seqs), ref(sinks), C.byref(pp), ref(dst), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


def test_paged_stores_inside_its_buffers(ctx):
    rng = random.Random(5)
    for _ in range(300):
        Hkv = rng.choice([1, 2, 4, 8])
        N = rng.choice([1, 3, 40, 700, 5000])
        st, msg = run_paged(ctx, D=rng.choice([8, 64, 80, 96, 120, 128, 256]), Hkv=Hkv, H=Hkv * rng.choice([1, 3, 4, 8, 16, 40]), N=N, B=rng.choice([1, 2, 64, 300]),
                            per=rng.choice([1, 9, 1000]), cty=rng.choice([1, 30]), page=rng.choice([1, 24, 64, 256]), pages=rng.choice([0, 1, 9000]),
                            window=rng.choice([0, 1, 4096]), n_first=rng.choice([0, 4]), n_shared=rng.choice([0, 1]), max_q=rng.choice([0, 1, 5, 60, 5000]))
        assert st == 0, msg


def test_paged_refuses(ctx):
    import ghip
    for want, kw in [
            ("F32 rows", dict(q=T(1, [64, 8, 9], A[0]))), ("shape", dict(dst=T(0, [64, 8, 8], A[3]))), ("head size", dict(D=60)), ("head size", dict(D=264)),
            ("kv must be F16", dict(cty=0)), ("2 D", dict(kv=T(1, [64, 2, 16, 50], A[1]))), ("16 bytes", dict(kv=T(1, [128, 2, 16, 50], A[1] + 8))),
            ("16 bytes", dict(kv=T(1, [128, 2, 16, 50], A[1], nb=[2, 264, 528, 8448]))), ("H_kv", dict(H=9)), ("seqs", dict(seqs=T(ghip.I64, [10, 3], A[2]))),
            ("seqs", dict(seqs=T(ghip.I32, [2, 3], A[2]))), ("sinks", dict(sinks=T(0, [7], A[4]))), ("sinks", dict(sinks=T(1, [8], A[4]))),
            ("scale", dict(scale=float("nan"))), ("scale", dict(scale=float("inf"))), ("window", dict(window=-1)), ("n_first", dict(n_first=-1)), ("n_shared", dict(n_shared=-1)),
            ("n_shared", dict(n_shared=113)), ("max_q", dict(max_q=-1)), ("apart", dict(dst=T(0, [64, 8, 9], A[0] + 4096))),
            ("null data", dict(seqs=T(ghip.I32, [10, 3], None))), ("[D, H, T]", dict(q=T(0, [64, 8, 9, 2], A[0]), dst=T(0, [64, 8, 9, 2], A[3])))]:
        st, msg = run_paged(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)
    q, kv, s, pp = T(0, [64, 8, 9], A[0]), T(1, [128, 2, 16, 50], A[1]), T(ghip.I32, [10, 3], A[2]), ghip.PagedParams(1.0, 0, 0, 0, 3)
    L = ghip.lib()
    for args in ((None, ref(kv), ref(s), None, C.byref(pp), ref(q)), (ref(q), None, ref(s), None, C.byref(pp), ref(q)),
                 (ref(q), ref(kv), None, None, C.byref(pp), ref(q)), (ref(q), ref(kv), ref(s), None, None, ref(q)), (ref(q), ref(kv), ref(s), None, C.byref(pp), None)):
        assert L.ghip_flash_attn_paged(ctx, *args, None) != 0


def test_binding_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    import ghip
    for t in (torch.zeros(3), torch.zeros(3, dtype=torch.float64)):
        with pytest.raises(ghip.GhipError):
            ghip._view(t)


HOST = r"""
#include "ghip_paged.h"
extern "C" void seq(int q0, int nq, int nkv, int T, int max_q, long long *o) {
    PagedSeq s = paged_seq(q0, nq, nkv, T, max_q); o[0] = s.q0; o[1] = s.nq; o[2] = s.pos0; }
extern "C" void keys(long long p0, long long p1, int w, int f, long long *o) {
    PagedKeys k = paged_keys(p0, p1, w, f); o[0] = k.first; o[1] = k.lo; o[2] = k.hi; }
extern "C" unsigned divide(unsigned n, unsigned d) { return paged_div(n, paged_divisor(d)); }
extern "C" void tiles(long long p0, long long p1, int w, int f, int from, int to, int kt, int nz, int *o) {
    PagedTiles t = paged_tiles(p0, p1, w, f, from, to, kt);
    o[0] = t.a0; o[1] = t.a1; o[2] = t.b0; o[3] = t.b1; o[4] = t.na; o[5] = t.n; o[6] = paged_share(t.n, nz); }
extern "C" int seen(long long p, long long j, int w, int f) { return paged_seen(p, j, w, f); }
"""


def test_index_arithmetic(tmp_path):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("no C++ compiler")
    src, so = tmp_path / "idx.cpp", str(tmp_path / "idx.so")
    src.write_text(HOST)
    subprocess.run([cc, "-shared", "-fPIC", "-Wno-unused-function", "-I", os.path.join(ROOT, "llama.rust_amd", "csrc"), "-o", so, str(src)], check=True)
    L = C.CDLL(so)
    o = (C.c_longlong * 3)()
    ll = C.c_longlong
    rng = random.Random(1)
    big = [0, 1, -1, 5, 2 ** 31 - 1, -2 ** 31]
    for _ in range(3000):
        q0, nq, nkv = (rng.choice(big) if rng.random() < 0.3 else rng.randint(-5, 60) for _ in range(3))
        n, mq = rng.randint(0, 50), rng.randint(0, 50)
        L.seq(q0, nq, nkv, n, min(mq, n), o)
        assert o[2] == nkv - nq and 0 <= o[1] <= min(mq, n)
        if o[1]:
            assert o[0] == q0 >= 0 and q0 + o[1] <= n
        assert o[1] == len([i for i in range(max(0, min(nq, min(mq, n)))) if 0 <= q0 < n and q0 + i < n])
    for _ in range(3000):
        p0 = rng.randint(-20, 60)
        p1 = p0 + rng.randint(0, 30)
        w, f = rng.choice([0, 1, 7, 64, 2 ** 31 - 1]), rng.choice([0, 1, 9, 200, 2 ** 31 - 1])
        L.keys(ll(p0), ll(p1), w, f, o)
        first, lo, hi = o[0], o[1], o[2]
        for j in range(100):
            some = any(j <= p and (not w or j > p - w or j < f) for p in range(p0, p1 + 1))
            assert some == any(L.seen(ll(p), ll(j), w, f) for p in range(p0, p1 + 1))
            assert some == (j < first or lo <= j < hi), (p0, p1, w, f, j)
        assert 0 <= first <= lo <= hi or hi == 0
    L.divide.restype = C.c_uint
    for d in [1, 2, 3, 7, 16, 24, 64, 100, 255, 256, 257, 641, 2 ** 16 + 1, 2 ** 30, 2 ** 31 - 1]:
        for n in [0, 1, d - 1, d, d + 1, 3 * d - 1, 2 ** 31 - 1, 2 ** 32 - 1] + [rng.randrange(2 ** 32) for _ in range(200)]:
            n %= 2 ** 32
            assert L.divide(C.c_uint(n), C.c_uint(d)) == n // d, (n, d)
    o7 = (C.c_int * 7)()
    for _ in range(3000):
        p0 = rng.randint(-20, 60)
        p1 = p0 + rng.randint(0, 30)
        w, f = rng.choice([0, 1, 7, 64]), rng.choice([0, 1, 9, 200])
        fr = rng.choice([0, 0, 5, 40])
        to, kt, nz = fr + rng.randint(0, 90), rng.choice([4, 8, 32]), rng.randint(1, 9)
        L.tiles(ll(p0), ll(p1), w, f, fr, to, kt, nz, o7)
        a0, a1, b0, b1, na, n, share = o7
        keys = []  # as the kernels walk them: tile t, then its keys below the range's end
        for t in range(n):
            k0, ke = (a0 + t * kt, a1) if t < na else (b0 + (t - na) * kt, b1)
            assert k0 < ke
            keys += range(k0, min(k0 + kt, ke))
        want = [j for j in range(fr, to) if any(L.seen(ll(p), ll(j), w, f) for p in range(p0, p1 + 1))]
        assert keys == want, (p0, p1, w, f, fr, to, kt)
        assert share * nz >= n


def test_null_data_is_refused(ctx):
    """A tensor that is given has data: without it factors and sinks would be left out
    (and the rotation's table read as another one)."""
    import ghip
    for st, msg in (run_rope(ctx, factors=T(ghip.F32, [32], None)), run_append(ctx, factors=T(ghip.F32, [32], None)),
                    run_paged(ctx, sinks=T(ghip.F32, [8], None))):
        assert st != 0 and "null data" in msg, msg


def test_outputs_lie_apart_from_what_is_read(ctx):
    import ghip
    for want, (st, msg) in [
            ("kv", run_paged(ctx, dst=T(ghip.F32, [64, 8, 9], A[1] + 64))), ("seqs", run_paged(ctx, dst=T(ghip.F32, [64, 8, 9], A[2] - 64))),
            ("sinks", run_paged(ctx, sinks=T(ghip.F32, [8], A[3] + 4096))), ("pos", run_rope(ctx, pos=T(ghip.I32, [9], A[1] + 8))),
            ("factors", run_rope(ctx, factors=T(ghip.F32, [32], A[1] + 8))), ("slots", run_append(ctx, slots=T(ghip.I64, [9], A[3] + 8))),
            ("pos", run_append(ctx, pos=T(ghip.I32, [9], A[3] + 8))), ("factors", run_append(ctx, factors=T(ghip.F32, [32], A[3] + 8)))]:
        assert st != 0 and "apart" in msg and want in msg, (want, msg)
    # an empty cache lies nowhere
    st, msg = run_paged(ctx, pages=0, dst=T(ghip.F32, [64, 8, 9], A[1]))
    assert st == 0, msg


def test_strides_of_axes_of_one_element_do_not_count(ctx):
    """What is never stepped over may have any stride: one token of a batch's slots, one
    head of several, one page, positions of one token by axis."""
    import ghip
    odd = 4 * 7 + 1
    one = lambda ty, ne, e, data: T(ty, ne, data, nb=[e if n > 1 else odd for n in (list(ne) + [1] * 4)[:4]])
    for st, msg in (
            run_rope(ctx, N=1, H=1, x=T(0, [64, 1, 1], A[0], nb=[4, odd, odd, odd]), dst=T(0, [64, 1, 1], A[0], nb=[4, 256, 256, 256])),
            run_rope(ctx, N=1, pos=T(ghip.I32, [1], A[2], nb=[32, odd, odd, odd])),
            run_rope(ctx, N=1, mode=8, sections=(8, 8, 8, 8), pos=T(ghip.I32, [1, 4], A[2], nb=[16, 4, 16, 16])),
            run_rope(ctx, D=2, n_dims=2, factors=one(ghip.F32, [1], 4, A[3])),
            run_append(ctx, N=1, slots=one(ghip.I64, [1], 8, A[2]), kv=T(1, [128, 2, 16, 1], A[3], nb=[2, 256, 512, odd])),
            run_append(ctx, D=1, rope=False, pos=None, k=T(0, [1, 2, 9], A[0], nb=[odd, 4, 8, 72]), v=T(0, [1, 2, 9], A[1], nb=[odd, 4, 8, 72])),
            run_paged(ctx, H=1, Hkv=1, sinks=one(ghip.F32, [1], 4, A[4]), kv=T(1, [128, 1, 16, 50], A[1], nb=[2, odd, 256, 4096])),
            run_paged(ctx, page=1, pages=1, kv=T(1, [128, 2, 1, 1], A[1], nb=[2, 256, odd, odd])),
            run_paged(ctx, B=1, N=1, H=2, q=T(0, [64, 2, 1], A[0], nb=[4, 256, odd, odd]), dst=T(0, [64, 2, 1], A[3], nb=[4, 256, odd, odd]),
                      seqs=T(ghip.I32, [10, 1], A[2], nb=[4, odd, odd, odd]))):
        assert st == 0, msg
    # where they are stepped over they do
    for want, (st, msg) in (("I32", run_rope(ctx, N=2, pos=T(ghip.I32, [2], A[2], nb=[32, 64, 64, 64]))),
                            ("I64", run_append(ctx, N=2, slots=T(ghip.I64, [2], A[2], nb=[32, 64, 64, 64]))),
                            ("16 bytes", run_paged(ctx, kv=T(1, [128, 2, 16, 50], A[1], nb=[2, 256, 512, 8196])))):
        assert st != 0 and want in msg, msg


def test_binding_refuses_numbers_that_do_not_fit():
    """A window or a size past 32 bits would be taken for its low bits."""
    pytest.importorskip("torch")
    import ghip
    for kw in (dict(scale=1e39), dict(window=2 ** 32 + 5), dict(n_first=2 ** 31), dict(n_shared=-2 ** 31 - 1), dict(max_q=2 ** 40), dict(window=1.5)):
        with pytest.raises(ghip.GhipError, match="32 bits"):
            ghip.paged_params(**{**dict(scale=1.0, window=0, n_first=0, n_shared=0, max_q=1), **kw})
    for kw in (dict(n_dims=2 ** 32 + 64), dict(n_dims=64, mode=2 ** 32), dict(n_dims=64, sections=(2 ** 33, 0, 0, 0)), dict(n_dims=64, n_ctx_orig=2 ** 31)):
        with pytest.raises(ghip.GhipError, match="32 bits"):
            ghip.Rope(**kw)
    assert bytes(ghip.PagedParams(0.5, 7, 4, 3, 2)) == ghip.paged_params(0.5, 7, 4, 3, 2)


def test_more_workgroups_than_a_launch_takes_are_refused(ctx, monkeypatch):
    """A launch has fewer than 2^32 threads: refused before anything runs, not by the join."""
    monkeypatch.setenv("GHIP_FAP_SHARED", "1")
    for N, ok in ((1 << 19, True), (1 << 20, False), (1 << 22, False)):
        st, msg = run_paged(ctx, D=8, H=32, Hkv=8, N=N, B=2, n_shared=16, max_q=N)
        assert (st == 0) == ok and (ok or "too many rows" in msg), msg
