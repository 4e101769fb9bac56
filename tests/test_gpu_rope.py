"""ghip_rope and ghip_kv_append against the rotation's formula in 64 bits.

The angle's reduction is exact up to one rounding of the last eighth turn
(2^-24 radians); sin, cos and the products add three roundings of 2^-24 each, so
an element is within 2^-21 of |x0| + |x1|, plus half a step of its own type."""
import itertools

import pytest

import paged_oracle as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def _mode(mode):
    import ghip
    return {"norm": ghip.ROPE_NORM, "neox": ghip.ROPE_NEOX, "mrope": ghip.ROPE_MROPE, "imrope": ghip.ROPE_IMROPE,
            "vision": ghip.ROPE_VISION}[mode]


def _tol(y, mag, dtype):
    half = torch.finfo(dtype).eps / 2
    return mag * 2.0 ** -21 + y.abs() * half * 1.01 + torch.finfo(dtype).smallest_normal * half


def _sections(mode, n):
    p = n if mode == "vision" else n // 2
    return {"mrope": (p // 4, p - p // 4 - p // 3, p // 3, 0), "imrope": (p - 2 * (p // 3), p // 3, p // 3, 0),
            "vision": (p // 2, p - p // 2, 0, 0)}.get(mode, (0, 0, 0, 0))


def _positions(T, axes, start, g):
    return (start + torch.randint(0, 5000, (axes, T), generator=g)).to(torch.int32)


def check(be, T, H, D, n, mode, dtype, sections=None, base=10000.0, start=0, factors=False, seed=0, **yarn):
    import ghip
    g = torch.Generator().manual_seed(seed)
    sections = _sections(mode, n) if sections is None else sections
    axes = 1 if mode in ("norm", "neox") else 4
    x = torch.randn((T, H, D), generator=g).to(TYPES[dtype])
    pos = _positions(T, axes, start, g)
    pairs = n if mode == "vision" else n // 2
    f = (1 + torch.rand(pairs, generator=g) * 7) if factors else None
    kw = dict(scale=yarn.get("freq_scale", 1.0), ext=yarn.get("ext_factor", 0.0), attn=yarn.get("attn_factor", 1.0),
              n_ctx=yarn.get("n_ctx_orig", 0))
    want, mag = P.rope(x, pos, mode, n, base, sections, f, **kw)
    r = ghip.Rope(n, _mode(mode), freq_base=base, sections=sections, **yarn)
    print(f"rope T={T} H={H} D={D} n={n} {mode} {dtype} start={start} {yarn}", flush=True)
    got = be.rope(x.cuda(), pos.cuda() if axes > 1 else pos[0].cuda(), r, factors=f.cuda() if factors else None)
    err = (got.cpu().double() - want).abs()
    tol = _tol(want, mag, TYPES[dtype])
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("mode", ["norm", "neox", "mrope", "imrope", "vision"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("T,H,D,n", [(1, 1, 2, 2), (1, 32, 128, 128), (7, 3, 80, 40), (5, 5, 96, 24), (3, 2, 33, 12),
                                     (65, 7, 256, 256), (2, 1, 10, 4)])
def test_modes(be, T, H, D, n, mode, dtype):
    if mode == "vision":
        n = max(2, min(n, D // 2) // 2 * 2)
        if 2 * n > D:
            pytest.skip("no vision pairs in this head size")
    s = _sections(mode, n)
    if mode == "vision" and D == 2:
        pytest.skip("no vision pairs in this head size")
    check(be, T, H, D, n, mode, dtype, sections=s if sum(s) or mode in ("norm", "neox") else (1, 0, 0, 0))


def test_many_heads_share_angles(be):
    """Sizes where a thread takes four heads, the last group of them short."""
    check(be, 700, 31, 128, 128, "imrope", "f32", base=5e6)
    check(be, 1100, 30, 96, 36, "norm", "f16")
    check(be, 1100, 14, 80, 40, "vision", "bf16")


@pytest.mark.parametrize("start", [100000, 2000000, 2 ** 31 - 6000])
def test_far_positions(be, start):
    check(be, 9, 2, 128, 128, "neox", "f32", start=start, base=1e6)


def test_negative_positions_turn_back(be):
    check(be, 9, 2, 64, 64, "neox", "f32", start=-4000)


def test_factors_and_context_extension(be):
    check(be, 33, 4, 128, 128, "neox", "f32", factors=True, start=9000, base=5e5)
    check(be, 33, 4, 128, 128, "norm", "f32", start=30000, freq_scale=0.25)
    check(be, 33, 4, 128, 96, "neox", "f32", start=30000, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=8192, attn_factor=0.9)
    check(be, 33, 4, 128, 128, "mrope", "f32", start=3000, freq_scale=0.5, ext_factor=0.7, n_ctx_orig=4096)


def test_sections_repeat(be):
    check(be, 6, 2, 128, 128, "mrope", "f32", sections=(3, 0, 5, 2))
    check(be, 6, 2, 128, 128, "imrope", "f32", sections=(5, 1, 3, 4))
    check(be, 6, 2, 128, 64, "vision", "f32", sections=(7, 9, 2, 1))


def test_strides_and_in_place(be):
    """A view of a wider projection, every other head, rotated where it lies."""
    import ghip
    g = torch.Generator().manual_seed(3)
    w = torch.randn((11, 2, 6, 72), generator=g)
    pos = _positions(11, 1, 70, g)
    want, mag = P.rope(w[:, 1, ::2, 3:67], pos, "neox", 64, 10000.0)
    wd = w.cuda()
    x = wd[:, 1, ::2, 3:67]
    be.rope(x, pos[0].cuda(), ghip.Rope(64), out=x)
    got = wd.cpu()
    assert ((got[:, 1, ::2, 3:67].double() - want).abs() <= _tol(want, mag, torch.float32)).all()
    rest = torch.ones_like(w, dtype=torch.bool)
    rest[:, 1, ::2, 3:67] = False
    assert torch.equal(got[rest], w[rest])


def test_nothing_to_rotate(be):
    import ghip
    x = torch.empty((0, 4, 64), device="cuda")
    assert be.rope(x, torch.empty(0, dtype=torch.int32, device="cuda"), ghip.Rope(64)).shape == (0, 4, 64)


# ---------------------------------------------------------------- KV append

def append(be, T, Hkv, D, n, mode, dtype, ctype, page, pages, factors=False, rope=True, seed=0, pad=0, strided=False):
    import ghip
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn((T, Hkv, D), generator=g).to(TYPES[dtype]) for _ in range(2))
    axes = 1 if mode in ("norm", "neox") else 4
    pos = _positions(T, axes, 100, g)
    slots = torch.randperm(page * pages, generator=g)[:T].clone()
    if pad:
        slots[::pad] = torch.tensor([-1, page * pages, 2 ** 40, -2 ** 63])[torch.arange(len(slots[::pad])) % 4]
    sec = _sections(mode, n)
    pairs = n if mode == "vision" else n // 2
    f = (1 + torch.rand(pairs, generator=g) * 7) if factors else None
    big = torch.randn((pages, page + (2 if strided else 0), Hkv, 2 * D), generator=g).to(TYPES[ctype])
    kv = big[:, :page]
    want, mag = kv.double().clone(), torch.zeros(kv.shape, dtype=torch.float64)
    y, m = P.rope(k, pos, mode, n, 10000.0, sec, f) if rope else (k.double(), torch.zeros(k.shape, dtype=torch.float64))
    written = torch.zeros(kv.shape[:2], dtype=torch.bool)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < page * pages:
            written[s // page, s % page] = True
            want[s // page, s % page, :, :D], mag[s // page, s % page, :, :D] = y[t], m[t]
            want[s // page, s % page, :, D:] = v[t].double()
    bd = big.cuda()
    print(f"append T={T} Hkv={Hkv} D={D} n={n} {mode} {dtype}->{ctype} page={page} strided={strided}", flush=True)
    be.kv_append(k.cuda(), v.cuda(), slots.cuda(), bd[:, :page], pos=pos.cuda() if rope else None,
                 rope=ghip.Rope(n, _mode(mode), sections=sec) if rope else None, factors=f.cuda() if factors else None)
    out = bd.cpu()
    got = out[:, :page]
    err, tol = (got.double() - want).abs(), _tol(want, mag, TYPES[ctype])
    assert (err <= tol).all(), float((err / tol).max())
    assert torch.equal(got[~written], kv[~written])
    assert torch.equal(out[:, page:], big[:, page:])


@pytest.mark.parametrize("mode", ["norm", "neox", "mrope", "imrope"])
@pytest.mark.parametrize("dtype,ctype", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,Hkv,D,n,page", [(1, 1, 64, 64, 1), (7, 8, 128, 128, 16), (33, 3, 80, 20, 24), (5, 2, 15, 6, 3)])
def test_append(be, T, Hkv, D, n, page, mode, dtype, ctype):
    append(be, T, Hkv, D, n, mode, dtype, ctype, page, T // page + 3)


def test_append_large_padded_strided(be):
    append(be, 1500, 8, 128, 128, "neox", "f32", "f16", 64, 40, factors=True, pad=7)
    append(be, 1500, 7, 96, 96, "mrope", "f32", "bf16", 16, 128, pad=5, strided=True)


def test_append_without_rotation(be):
    append(be, 9, 2, 64, 64, "neox", "f32", "f16", 8, 4, rope=False)
    append(be, 9, 2, 21, 6, "neox", "bf16", "bf16", 8, 4, rope=False)


def test_append_nothing(be):
    kv = torch.ones((2, 4, 1, 128), dtype=torch.float16, device="cuda")
    e = torch.empty((0, 1, 64), device="cuda")
    be.kv_append(e, e, torch.empty(0, dtype=torch.int64, device="cuda"), kv)
    assert (kv == 1).all()


def test_far_slots(be):
    """A cache past 2^32 bytes: the last slots' offsets need 64 bits."""
    import ghip
    D, Hkv, page, pages = 128, 8, 64, 18000  # 4.7 GB
    kv = torch.zeros((pages, page, Hkv, 2 * D), dtype=torch.float16, device="cuda")
    k = torch.randn((3, Hkv, D), device="cuda")
    slots = torch.tensor([page * pages - 1, page * (pages - 5) + 3, 7], device="cuda")
    be.kv_append(k, -k, slots, kv)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(kv[s // page, s % page], torch.cat([k[t], -k[t]], -1).half())
    assert int((kv != 0).any(-1).sum()) == 3 * Hkv


def test_streams_and_graph(be):
    """Calls on another stream than the inputs' own, captured: replays follow what
    positions and slots hold by then."""
    import ghip
    r = ghip.Rope(64, ghip.ROPE_NEOX)
    x = torch.randn((5, 4, 64), device="cuda")
    kv = torch.zeros((4, 8, 4, 128), dtype=torch.bfloat16, device="cuda")
    pos = torch.arange(5, dtype=torch.int32, device="cuda")
    slots = torch.arange(5, device="cuda")
    out = torch.empty_like(x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        be.rope(x, pos, r, out=out)
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            be.rope(x, pos, r, out=out)
            be.kv_append(x, x, slots, kv, pos=pos, rope=r)
    for i, (p0, s0) in enumerate(itertools.product((0, 1000), (0, 9, 27))):
        pos.copy_(torch.arange(5, device="cuda") + p0)
        slots.copy_(torch.arange(5, device="cuda") + s0)
        x.copy_(torch.randn((5, 4, 64), device="cuda"))
        kv.zero_()
        g.replay()
        torch.cuda.synchronize()
        eager, kv2 = be.rope(x, pos, r), torch.zeros_like(kv)
        be.kv_append(x, x, slots, kv2, pos=pos, rope=r)
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and torch.equal(kv, kv2), i


def test_one_token_of_strided_tables(be):
    """Positions by axis as a column, a slot out of a longer table: the strides of axes
    of one element do not count."""
    import ghip
    r = ghip.Rope(64, ghip.ROPE_MROPE, sections=(8, 8, 16, 0))
    x = torch.randn((1, 4, 64), device="cuda")
    pos = torch.tensor([[7, 3, 900, 1]], dtype=torch.int32, device="cuda").t()
    slots = torch.arange(8, device="cuda")[3:4]
    wide = torch.arange(64, device="cuda").view(8, 8)[3:4, ::4][:, :1].t()[0]
    kv, kv2 = (torch.zeros((2, 8, 4, 128), dtype=torch.float16, device="cuda") for _ in range(2))
    assert torch.equal(be.rope(x, pos, r), be.rope(x, pos.contiguous(), r))
    be.kv_append(x, x, wide, kv, pos=pos, rope=r)
    be.kv_append(x, x, torch.full_like(slots, 24) % 16, kv2, pos=pos.contiguous(), rope=r)
    torch.cuda.synchronize()
    assert not kv.any() and int(wide[0]) == 24  # (past the 16 slots of this cache)
    be.kv_append(x, x, torch.arange(32, device="cuda")[8:16:8], kv, pos=pos, rope=r)
    assert torch.equal(kv, kv2) and kv2.any()


@pytest.mark.parametrize("dtype,ctype", [("f32", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("T,Hkv,D,page", [(9, 2, 80, 16), (600, 4, 128, 24), (5, 3, 36, 1)])
def test_append_of_patches(be, T, Hkv, D, page, dtype, ctype):
    append(be, T, Hkv, D, D // 2, "vision", dtype, ctype, page, T // page + 3)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("D", [64, 80, 36])
def test_rows_at_odd_elements(be, D, dtype):
    """16-bit rows whose addresses are no multiples of 4 bytes, read and written by vectors."""
    import ghip
    g = torch.Generator().manual_seed(7)
    w = torch.randn((300, 6, D + 3), generator=g).to(TYPES[dtype])
    pos = _positions(300, 1, 70, g)
    r = ghip.Rope(D, ghip.ROPE_NEOX)
    for T, at in ((3, 1), (300, 3)):
        x = w[:T, :, at:at + D]
        want, mag = P.rope(x, pos[:, :T], "neox", D, 10000.0)
        out = torch.full((T, 6, D + 5), 7.0, dtype=TYPES[dtype], device="cuda")
        be.rope(w.cuda()[:T, :, at:at + D], pos[0, :T].cuda(), r, out=out[:, :, 3:3 + D])
        got = out.cpu()
        assert ((got[:, :, 3:3 + D].double() - want).abs() <= _tol(want, mag, TYPES[dtype])).all()
        got[:, :, 3:3 + D] = 7.0
        assert (got == 7.0).all()


@pytest.mark.parametrize("fast,slow", [(8.0, 0.25), (64.0, 4.0), (1.0, 1.0)])
def test_context_extension_between_other_wavelengths(be, fast, slow):
    import ghip
    g = torch.Generator().manual_seed(5)
    x, pos = torch.randn((20, 3, 128), generator=g), _positions(20, 1, 30000, g)
    want, mag = P.rope(x, pos, "neox", 128, 1e4, scale=0.25, ext=1.0, n_ctx=8192, fast=fast, slow=slow)
    r = ghip.Rope(128, ghip.ROPE_NEOX, freq_scale=0.25, ext_factor=1.0, n_ctx_orig=8192, beta_fast=fast, beta_slow=slow)
    got = be.rope(x.cuda(), pos[0].cuda(), r).cpu()
    assert ((got.double() - want).abs() <= _tol(want, mag, torch.float32)).all()
