"""What the calls on a quantized KV cache refuse, and that what they accept stores
inside its buffers, on a context without a device."""
import ctypes as C

import pytest

from test_paged_refusals import A, T, ctx, ref, rope_params  # noqa: F401


def codes(ty, ne, data, nb=None):
    """a tensor of codes: strides in bytes"""
    import ghip
    row = ne[0] * (1 if ty == ghip.E4M3 else 0.5)
    return T(ty, ne, data, 1, nb or [1, int(row), int(row * ne[1]), int(row * ne[1] * ne[2])])


def scales_of(D, Hkv, page, pages, data, nb=None):
    import ghip
    S = 1 if D <= 32 else 2 if D <= 64 else 4 if D <= 128 else 8
    return T(ghip.E8M0, [2 * S, Hkv, page, pages], data, 1, nb)


def run_append(ctx, D=64, Hkv=2, N=9, kty=0, vty=None, cty=256, page=16, pages=5, slots=None, kv=None, sc=None, v=None, k=None, rope=True,
               pos=True, factors=None, **kw):
    import ghip
    k = T(kty, [D, Hkv, N], A[0]) if k is None else k
    v = T(kty if vty is None else vty, [D, Hkv, N], A[1]) if v is None else v
    slots = T(ghip.I64, [N], A[2]) if slots is None else slots
    kv = codes(cty, [2 * D, Hkv, page, pages], A[3]) if kv is None else kv
    sc = scales_of(D, Hkv, page, pages, A[5]) if sc is None else sc
    p = T(ghip.I32, [N], A[4]) if pos is True else pos
    kw.setdefault("n_dims", min(64, D))
    r = rope_params(**kw) if rope else None
    st = ghip.lib().ghip_kv_append_mx(ctx, ref(k), ref(v), ref(slots), ref(p), ref(factors), ref(r), ref(kv), ref(sc), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


def run_read(ctx, D=64, Hkv=2, N=9, oty=0, cty=256, page=16, pages=5, slots=None, kv=None, sc=None, dst=None):
    import ghip
    slots = T(ghip.I64, [N], A[2]) if slots is None else slots
    kv = codes(cty, [2 * D, Hkv, page, pages], A[3]) if kv is None else kv
    sc = scales_of(D, Hkv, page, pages, A[5]) if sc is None else sc
    dst = T(oty, [2 * D, Hkv, N], A[0]) if dst is None else dst
    st = ghip.lib().ghip_kv_read_mx(ctx, ref(kv), ref(sc), ref(slots), ref(dst), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


# what is wrong with a cache, whatever the call
def wrong_caches():
    import ghip
    e4, e2 = ghip.E4M3, ghip.E2M1
    return [
        ("E4M3 or E2M1", dict(cty=ghip.F16)), ("multiple of 16", dict(D=24)), ("multiple of 16", dict(D=272)), ("multiple of 16", dict(D=8)),
        ("2 D", dict(kv=codes(e4, [64, 2, 16, 5], A[3]))), ("2 D", dict(kv=codes(e4, [128, 3, 16, 5], A[3]), sc=scales_of(64, 3, 16, 5, A[5]))),
        ("2 D", dict(kv=codes(e4, [128, 2, 16, 5], A[3], [2, 256, 512, 8192]))),
        ("16 bytes", dict(kv=codes(e4, [128, 2, 16, 5], A[3] + 8))), ("16 bytes", dict(kv=codes(e4, [128, 2, 16, 5], A[3], [1, 136, 272, 4352]))),
        ("16 bytes", dict(kv=codes(e2, [128, 2, 16, 5], A[3], [1, 72, 144, 2304]))),
        ("scales must be E8M0", dict(sc=T(ghip.F32, [4, 2, 16, 5], A[5]))),
        ("S = 1, 2, 4 or 8", dict(sc=scales_of(128, 2, 16, 5, A[5]))), ("S = 1, 2, 4 or 8", dict(sc=scales_of(64, 2, 16, 4, A[5]))),
        ("S = 1, 2, 4 or 8", dict(sc=scales_of(64, 2, 8, 5, A[5]))), ("S = 1, 2, 4 or 8", dict(sc=scales_of(64, 1, 16, 5, A[5]))),
        ("S = 1, 2, 4 or 8", dict(sc=scales_of(64, 2, 16, 5, A[5], [2, 8, 16, 256]))),
        ("2 S bytes", dict(sc=scales_of(64, 2, 16, 5, A[5] + 2))), ("2 S bytes", dict(sc=scales_of(64, 2, 16, 5, A[5], [1, 6, 12, 192]))),
        ("null data", dict(kv=codes(e4, [128, 2, 16, 5], None))), ("null data", dict(sc=scales_of(64, 2, 16, 5, None)))]


def test_append(ctx):
    import ghip
    for N in (0, 1, 9, 8192):
        for kty in (0, 1, 30):
            for cty in (ghip.E4M3, ghip.E2M1):
                for D, page, pages in ((64, 1, 4), (128, 24, 600), (80, 16, 0), (16, 16, 3), (256, 64, 3)):
                    st, msg = run_append(ctx, N=N, kty=kty, cty=cty, D=D, page=page, pages=pages)
                    assert st == 0, msg
    st, msg = run_append(ctx, rope=False, pos=None)
    assert st == 0, msg
    st, msg = run_append(ctx, kv=codes(256, [128, 2, 16, 5], A[3], nb=[1, 160, 640, 16384]), sc=scales_of(64, 2, 16, 5, A[5], [1, 4, 12, 256]))
    assert st == 0, msg
    for want, kw in wrong_caches() + [
            ("of one type", dict(kty=ghip.I32)), ("of one type", dict(vty=1)), ("same shape", dict(v=T(0, [64, 2, 8], A[1]))),
            ("[D, H_kv, T]", dict(k=T(0, [64, 2, 9, 2], A[0]), v=T(0, [64, 2, 9, 2], A[1]))),
            ("rows of elements", dict(k=T(0, [64, 2, 9], A[0], nb=[8, 512, 1024, 9216]))),
            ("I64", dict(slots=T(ghip.I32, [9], A[2]))), ("I64", dict(slots=T(ghip.I64, [8], A[2]))),
            ("need a rotation", dict(rope=False)), ("n_dims", dict(n_dims=128)), ("pos", dict(pos=None)),
            ("null data", dict(slots=T(ghip.I64, [9], None))), ("null data", dict(pos=T(ghip.I32, [9], None))),
            ("lie apart", dict(kv=codes(256, [128, 2, 16, 5], A[0] + 64))), ("lie apart", dict(sc=scales_of(64, 2, 16, 5, A[2] + 64))),
            ("lie apart", dict(sc=scales_of(64, 2, 16, 5, A[3] + 4096))), ("lie apart", dict(kv=codes(256, [128, 2, 16, 5], A[4]))),
            ("factors", dict(factors=T(ghip.F32, [9], A[6]))), ("null data", dict(factors=T(ghip.F32, [32], None)))]:
        st, msg = run_append(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)
    L, none = ghip.lib(), None
    for i in range(9):
        args = [ref(T(0, [64, 2, 9], A[0])), ref(T(0, [64, 2, 9], A[1])), ref(T(ghip.I64, [9], A[2])), none, none, none,
                ref(codes(256, [128, 2, 16, 5], A[3])), ref(scales_of(64, 2, 16, 5, A[5]))]
        if i < 8 and args[i] is not None:
            args[i] = None
            assert L.ghip_kv_append_mx(ctx, *args, None) != 0
    assert L.ghip_kv_append_mx(None, *args, None) != 0


def test_read(ctx):
    import ghip
    for N in (0, 1, 9, 20000):
        for oty in (0, 1, 30):
            for cty in (ghip.E4M3, ghip.E2M1):
                for D, page, pages in ((64, 1, 4), (128, 24, 600), (80, 16, 0), (16, 16, 3), (256, 64, 3)):
                    st, msg = run_read(ctx, N=N, oty=oty, cty=cty, D=D, page=page, pages=pages)
                    assert st == 0, msg
    st, msg = run_read(ctx, dst=T(0, [128, 2, 9], A[0], nb=[4, 540, 2000, 18000]))
    assert st == 0, msg
    for want, kw in wrong_caches() + [
            ("dst must be F32", dict(oty=ghip.I32)), ("rows of elements", dict(dst=T(0, [128, 2, 9], A[0], nb=[8, 1024, 2048, 20480]))),
            ("[2 D, H_kv, T]", dict(dst=T(0, [128, 2, 9, 2], A[0]))), ("[2 D, H_kv", dict(dst=T(0, [128, 3, 9], A[0]))),
            ("I64", dict(slots=T(ghip.I32, [9], A[2]))), ("I64", dict(slots=T(ghip.I64, [8], A[2]))),
            ("null data", dict(dst=T(0, [128, 2, 9], None))), ("null data", dict(slots=T(ghip.I64, [9], None))),
            ("lie apart", dict(dst=T(0, [128, 2, 9], A[3] + 256))), ("lie apart", dict(dst=T(0, [128, 2, 9], A[5]))),
            ("lie apart", dict(dst=T(0, [128, 2, 9], A[2])))]:
        st, msg = run_read(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)
    L = ghip.lib()
    args = [ref(codes(256, [128, 2, 16, 5], A[3])), ref(scales_of(64, 2, 16, 5, A[5])), ref(T(ghip.I64, [9], A[2])), ref(T(0, [128, 2, 9], A[0]))]
    for i in range(4):
        assert L.ghip_kv_read_mx(ctx, *[None if j == i else a for j, a in enumerate(args)], None) != 0
    assert L.ghip_kv_read_mx(None, *args, None) != 0


def test_binding_refuses():
    """Codes and scales of other dtypes or shapes, before any call."""
    import ghip
    torch = pytest.importorskip("torch")
    kv, sc = ghip.mx_cache(3, 16, 2, 64, 8, device="cpu")
    assert kv.shape == (3, 16, 2, 128) and kv.dtype == torch.float8_e4m3fn and sc.shape == (3, 16, 2, 4) and (sc == 27).all()
    kv4, sc4 = ghip.mx_cache(3, 16, 2, 80, 4, device="cpu")
    assert kv4.shape == (3, 16, 2, 80) and kv4.dtype == torch.uint8 and sc4.shape == (3, 16, 2, 8)
    for a, b, why in ((kv.float(), sc, "not supported"), (kv, sc.float(), "scales"), (kv, sc, "GPU")):
        with pytest.raises(ghip.GhipError, match=why):
            ghip._view_mx(a, b)
    with pytest.raises(ghip.GhipError, match="4 or 8"):
        ghip.mx_cache(3, 16, 2, 64, 6, device="cpu")


def run_paged(ctx, D=64, H=8, Hkv=2, N=9, B=3, per=7, cty=256, page=16, pages=5, q=None, kv=None, sc=None, seqs=None, sinks=None, dst=None, scale=0.1,
              window=0, n_first=0, n_shared=0, max_q=3, workspace=False):
    import ghip
    q = T(0, [D, H, N], A[0]) if q is None else q
    kv = codes(cty, [2 * D, Hkv, page, pages], A[3]) if kv is None else kv
    sc = scales_of(D, Hkv, page, pages, A[5]) if sc is None else sc
    seqs = T(ghip.I32, [3 + per, B], A[2]) if seqs is None else seqs
    dst = T(0, [D, H, N], A[6]) if dst is None else dst
    pp = ghip.PagedParams(scale, window, n_first, n_shared, max_q)
    if workspace:
        n = C.c_size_t()
        return ghip.lib().ghip_flash_attn_paged_mx_workspace(ref(q), ref(kv), ref(sc), ref(seqs), C.byref(pp), ref(dst), C.byref(n)), n.value
    st = ghip.lib().ghip_flash_attn_paged_mx(ctx, ref(q), ref(kv), ref(sc), ref(seqs), ref(sinks), C.byref(pp), ref(dst), None)
    return st, ghip.lib().ghip_last_error(ctx).decode()


def test_paged_stores_inside_its_buffers(ctx):
    import random
    import ghip
    rng = random.Random(5)
    for _ in range(300):
        Hkv = rng.choice([1, 2, 4, 8])
        N = rng.choice([1, 3, 40, 700, 5000])
        kw = dict(D=rng.choice([16, 64, 80, 96, 112, 128, 256]), Hkv=Hkv, H=Hkv * rng.choice([1, 3, 4, 8, 16, 40]), N=N, B=rng.choice([1, 2, 64, 300]),
                  per=rng.choice([1, 9, 1000]), cty=rng.choice([ghip.E4M3, ghip.E2M1]), page=rng.choice([1, 24, 64, 256]), pages=rng.choice([0, 1, 9000]),
                  window=rng.choice([0, 1, 4096]), n_first=rng.choice([0, 4]), n_shared=rng.choice([0, 1]), max_q=rng.choice([0, 1, 5, 60, 5000]))
        st, msg = run_paged(ctx, **kw)
        assert st == 0, msg
        assert run_paged(ctx, workspace=True, **kw)[0] == 0


def test_paged_refuses(ctx):
    import ghip
    wrong = [(want, kw) for want, kw in wrong_caches() if not ("sc" in kw and "kv" in kw)]
    for want, kw in wrong + [
            ("H_kv", dict(H=9)), ("F32 rows", dict(q=T(1, [64, 8, 9], A[0]))), ("shape", dict(dst=T(0, [64, 8, 8], A[6]))),
            ("seqs", dict(seqs=T(ghip.I64, [10, 3], A[2]))), ("seqs", dict(seqs=T(ghip.I32, [2, 3], A[2]))), ("sinks", dict(sinks=T(0, [7], A[4]))),
            ("scale", dict(scale=float("nan"))), ("window", dict(window=-1)), ("n_first", dict(n_first=-1)), ("n_shared", dict(n_shared=-1)),
            ("n_shared", dict(n_shared=113)), ("max_q", dict(max_q=-1)), ("apart", dict(dst=T(0, [64, 8, 9], A[0] + 4096))),
            ("apart from kv", dict(dst=T(0, [64, 8, 9], A[3] + 4096))), ("apart from scales", dict(dst=T(0, [64, 8, 9], A[5] + 256))),
            ("null data", dict(seqs=T(ghip.I32, [10, 3], None))), ("null data", dict(sinks=T(0, [8], None)))]:
        st, msg = run_paged(ctx, **kw)
        assert st != 0 and want in msg, (want, kw, msg)
        if "sinks" not in kw:
            assert run_paged(ctx, workspace=True, **kw)[0] != 0
    L = ghip.lib()
    pp = ghip.PagedParams(1.0, 0, 0, 0, 3)
    args = [ref(T(0, [64, 8, 9], A[0])), ref(codes(256, [128, 2, 16, 5], A[3])), ref(scales_of(64, 2, 16, 5, A[5])), ref(T(ghip.I32, [10, 3], A[2])), None,
            C.byref(pp), ref(T(0, [64, 8, 9], A[6]))]
    for i in range(7):
        if args[i] is not None:
            assert L.ghip_flash_attn_paged_mx(ctx, *[None if j == i else a for j, a in enumerate(args)], None) != 0
    assert L.ghip_flash_attn_paged_mx(None, *args, None) != 0
    # the cache of the other call
    st = L.ghip_flash_attn_paged(ctx, args[0], args[1], args[3], None, args[5], args[6], None)
    assert st != 0 and "F16 or BF16" in L.ghip_last_error(ctx).decode()


def test_append_of_more_than_can_be_counted(ctx):
    """Tokens times heads past what 64 bits of threads hold (strides of 0)."""
    import ghip
    n = 2 ** 31 - 1
    k, v = (T(0, [256, n, n], a, 4, [4, 0, 0, 0]) for a in (A[0], A[1]))
    kv, sc = codes(ghip.E4M3, [512, n, 1, 1], A[3], [1, 0, 0, 0]), scales_of(256, n, 1, 1, A[5], [1, 0, 0, 0])
    st, msg = run_append(ctx, D=256, Hkv=n, N=n, k=k, v=v, kv=kv, sc=sc, slots=T(ghip.I64, [n], A[2]), rope=False, pos=None)
    assert st != 0 and "k too large" in msg, msg
