"""A quantized KV cache: what ghip_kv_append_mx writes and ghip_kv_read_mx reads,
against the definition in 64 bits (mx_oracle, paged_oracle).

The kernels round a rotation formed in 64 bits, so their bytes are the
definition's; an element may only differ where its value is so near to a border that
the angle decides: an angle of position p is off by p 2^-53 (the oracle's product)
and p 2^-64 turns (the kernel's fraction of a turn), sin, cos and the products by
2^-44 together, relative to the pair, which may be as large as the block's largest
times sqrt(2)."""
import pytest

import mx_oracle as M
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


def rope_of(mode, n, base, sections):
    import ghip
    m = {"norm": ghip.ROPE_NORM, "neox": ghip.ROPE_NEOX, "mrope": ghip.ROPE_MROPE, "imrope": ghip.ROPE_IMROPE, "vision": ghip.ROPE_VISION}
    return ghip.Rope(n, m[mode], freq_base=base, sections=sections)


def tokens(T, H, D, ty, g, strided=False):
    """projections with a few strong channels; strided: as slices of wider rows"""
    w = D + 5 if strided else D
    x = torch.randn((T, H + strided, w), generator=g) * torch.exp(torch.randn((1, 1, w), generator=g))
    return x.to(TYPES[ty]).cuda()[:, strided:, w - D:]


def check_append(be, bits, ty, T, H, D, page, mode=None, n=None, sections=(0, 0, 0, 0), base=10000.0, start=0, factors=False,
                 strided=False, seed=0, layers=1):
    g = torch.Generator().manual_seed(seed)
    k, v = tokens(T, H, D, ty, g, strided), tokens(T, H, D, ty, g, strided)
    pages = max(1, (T + page - 1) // page) + 2
    whole = [M.cache(pages, page, H * layers, D, bits, g)[i].cuda() for i in (0, 1)]
    kv, sc = (t[:, :, H * (layers - 1):] for t in whole)  # the last layer's heads of a cache of all layers
    before = [t.cpu().clone() for t in whole]
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[T // 3::7] = -1 - slots[T // 3::7]  # padding
    if T > 4:
        slots[2] = pages * page  # outside the cache
    kw, mag = {}, torch.zeros((), dtype=torch.float64)
    want_k = k.cpu().double()
    tol = torch.zeros((T, 1, 1), dtype=torch.float64)
    if mode:
        axes = 4 if sum(sections) else 1
        pos = (start + torch.arange(T) * 3 + 50 * torch.arange(axes).view(-1, 1)).to(torch.int32)
        f = torch.linspace(1.0, 5.0, n if mode == "vision" else n // 2) if factors else None
        kw = dict(pos=pos.cuda() if axes > 1 else pos[0].cuda(), rope=rope_of(mode, n, base, sections), factors=f.cuda() if factors else None)
        want_k, mag = P.rope(k.cpu(), pos, mode, n, base, sections, f)
        # (a factor's quotient: 2^-53 more of the angle)
        far = pos.double().abs().amax(0)
        tol = (far * 3 * 2.0 ** -53 * 6.3 + 2.0 ** -43 * (far > 0)).view(T, 1, 1)  # (position 0: exact)
    print(f"append {bits} {ty} T={T} H={H} D={D} page={page} {mode} n={n} start={start} strided={strided}", flush=True)
    be.kv_append(k, v, slots.cuda(), kv, scales=sc, **kw)
    got, gsc = M.unpack(whole[0].cpu(), bits), whole[1].cpu().long()
    wc, wsc = M.unpack(before[0], bits), before[1].long()
    S = M.scale_bytes(D)
    h0 = H * (layers - 1)
    off = torch.zeros_like(wc, dtype=torch.bool)
    for part, x, t in ((0, want_k, tol), (1, v.cpu().double(), torch.zeros_like(tol))):
        c, sb, room = M.encode(x, bits)
        # (twice: of both a pair and a block's largest; what is not rotated is exact)
        near = (room < t * 2) & (mag > 0) if part == 0 else torch.zeros_like(room, dtype=torch.bool)
        # few: but a 16-bit element that is not rotated and the largest of its block lies on a border
        # of the scale once in 128, and then all 32 are near one
        assert near.double().mean() < 2.0 ** -7
        for i in range(T):
            s = int(slots[i])
            if not 0 <= s < pages * page:
                continue
            at = (s // page, s % page, slice(h0, h0 + H))
            wc[at + (slice(part * D, part * D + D),)] = c[i]
            off[at + (slice(part * D, part * D + D),)] = near[i]
            wsc[at + (slice(part * S, part * S + S),)] = sb[i]
    same = (got == wc) | off
    assert same.all(), [(tuple(int(v) for v in i), int(got[tuple(i)]), int(wc[tuple(i)])) for i in (~same).nonzero()[:5]]
    assert ((gsc == wsc) | off.any()).all()
    # (next to a border: one code apart at most)
    assert (got == wc)[~off].all()


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 128, 240, 256])
def test_append_as_it_is(be, bits, ty, D):
    check_append(be, bits, ty, 37, 3, D, 16)


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("mode,D,n,sections", [
    ("neox", 128, 128, (0, 0, 0, 0)), ("norm", 128, 128, (0, 0, 0, 0)), ("neox", 64, 16, (0, 0, 0, 0)), ("neox", 80, 20, (0, 0, 0, 0)),
    ("norm", 80, 20, (0, 0, 0, 0)), ("norm", 96, 22, (0, 0, 0, 0)), ("neox", 96, 2, (0, 0, 0, 0)), ("neox", 256, 250, (0, 0, 0, 0)),
    ("mrope", 128, 128, (16, 24, 24, 0)), ("imrope", 128, 128, (24, 20, 20, 0)), ("vision", 80, 40, (20, 20, 0, 0)),
    ("vision", 256, 128, (64, 64, 0, 0)), ("mrope", 64, 32, (1, 2, 3, 10)), ("neox", 16, 16, (0, 0, 0, 0)), ("norm", 256, 256, (0, 0, 0, 0))])
def test_append_rotated(be, bits, mode, D, n, sections):
    for ty, T, H, page in (("f32", 33, 2, 24), ("bf16", 5, 5, 1), ("f16", 1, 1, 64)):
        check_append(be, bits, ty, T, H, D, page, mode, n, sections, 500000.0, start=9000, factors=T == 33)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_many_heads_share_angles(be, bits):
    """Enough tokens for four heads a thread, with heads left over."""
    for H in (4, 5, 7):
        check_append(be, bits, "f32", 2600, H, 64, 16, "neox", 64, start=100)
        check_append(be, bits, "bf16", 2600, H, 64, 16, "norm", 60, start=100)
    check_append(be, bits, "f32", 2600, 5, 80, 16, "neox", 20, start=100)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_far_and_negative_positions(be, bits):
    check_append(be, bits, "f32", 20, 2, 128, 16, "neox", 128, base=1e6, start=2 ** 24)
    check_append(be, bits, "f32", 20, 2, 128, 16, "norm", 128, start=-500)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_strided(be, bits):
    check_append(be, bits, "f32", 21, 2, 64, 16, "neox", 64, strided=True, layers=3)
    check_append(be, bits, "bf16", 21, 2, 128, 24, "norm", 128, strided=True, layers=2)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_borders(be, bits):
    """Every border between two codes, the values next to it, both signs; blocks at the borders of
    their scales; the smallest and largest blocks; infinities and NaN."""
    g = M.grid(bits)
    mid = ((g[1:] + g[:-1]) / 2).float()
    xs = [torch.cat([mid, torch.nextafter(mid, torch.tensor(0.0)), torch.nextafter(mid, torch.tensor(1e9)), g.float()])]
    rows = []
    for e in (-90, -20, 0, 3, 100):
        v = torch.cat([xs[0], -xs[0]])
        for i in range(0, len(v), 31):
            b = torch.zeros(32)
            b[0] = M.TOP[bits]
            b[1:1 + len(v[i:i + 31])] = v[i:i + 31]
            rows.append(b * 2.0 ** e)
    top = torch.tensor(M.TOP[bits])
    for e in (-109, -100, -50, 0, 100):
        for x in (top, torch.nextafter(top, torch.tensor(0.0)), torch.nextafter(top, torch.tensor(1e9)), top / 2, top * 0.75):
            rows.append((torch.linspace(-1, 1, 32) * x.float()) * 2.0 ** e)
    rows += [torch.zeros(32), -torch.zeros(32), torch.full((32,), 1e-45), torch.full((32,), 3.4028234e38), torch.full((32,), -1e-38)]
    for bad in (float("inf"), -float("inf"), float("nan")):
        r = torch.randn(32)
        r[17] = bad
        rows.append(r)
    while len(rows) % 4:
        rows.append(torch.randn(32))
    x = torch.stack(rows).view(-1, 1, 128)
    T = x.shape[0]
    import ghip
    kv, sc = ghip.mx_cache(T, 1, 1, 128, bits)
    be.kv_append(x.cuda(), x.flip(0).cuda(), torch.arange(T).cuda(), kv, scales=sc)
    for part, y in ((0, x), (1, x.flip(0))):
        c, sb, _ = M.encode(y.double(), bits)
        assert torch.equal(sc.cpu().long().view(T, 1, 8)[..., 4 * part:4 * part + 4], sb)
        got = M.unpack(kv.cpu(), bits).view(T, 1, 256)[..., 128 * part:128 * part + 128]
        assert torch.equal(got, c), (got != c).nonzero()[:5]
    back = be.kv_read(kv, torch.arange(T).cuda(), sc).cpu()
    bad = ~torch.isfinite(x.view(-1, 32)).all(1)
    assert torch.equal(torch.isnan(back[:, 0, :128].reshape(-1, 32)), bad.view(-1, 1).expand(-1, 32))


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("ty", ["f32", "f16", "bf16"])
def test_read_every_code(be, bits, ty):
    """Every code under scales of every size: the value in 64 bits, rounded once to the output's type."""
    D, codes = 256, 256 if bits == 8 else 16
    sb = torch.tensor([20, 64, 100, 111, 112, 118, 126, 127, 128, 134, 135, 142, 143, 200, 246, 255])
    kv = (torch.arange(16 * 2 * D).view(16, 1, 1, 2 * D) % codes)
    sc = sb.view(16, 1, 1, 1).expand(16, 1, 1, 16).clone()
    sc[..., 1::2] = sb.flip(0).view(16, 1, 1, 1)
    p = M.pack(kv, bits).cuda()
    got = be.kv_read(p.view(torch.float8_e4m3fn) if bits == 8 else p, torch.arange(16).cuda(), sc.to(torch.uint8).cuda(), dtype=TYPES[ty])
    want = M.decode(kv, sc, D, bits).view(16, 1, 2 * D)
    w = want.to(TYPES[ty])
    if ty == "bf16" and bits == 8:
        w = want.float().to(TYPES[ty])  # (4 significant bits: exact either way)
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(w))
    fine = ~torch.isnan(w)
    assert torch.equal(got.cpu()[fine], w[fine])
    e8m0 = sc.to(torch.uint8).view(torch.float8_e8m0fnu).cuda()
    again = be.kv_read(p.view(torch.float8_e4m3fn) if bits == 8 else p, torch.arange(16).cuda(), e8m0, dtype=TYPES[ty])
    assert torch.equal(again.cpu()[fine], w[fine])


@pytest.mark.parametrize("bits", [8, 4])
@pytest.mark.parametrize("D", [16, 48, 64, 80, 128, 256])
def test_read(be, bits, D):
    """Slots in any order, twice, padding and outside the cache; pages of any size; views; many rows."""
    g = torch.Generator().manual_seed(D)
    for T, H, page, ty in ((1, 1, 1, "f32"), (50, 3, 24, "bf16"), (333, 2, 16, "f16"), (9000, 4, 64, "f32"), (9001, 4, 64, "bf16")):
        pages = min(40, T) + 2
        kv, sc = M.cache(pages, page, H, D, bits, g)
        slots = torch.randint(-3, pages * page + 3, (T,), generator=g)
        out = torch.full((T, H, 2 * D + 4), 7.0, dtype=TYPES[ty], device="cuda")[:, :, 2:-2]
        be.kv_read(kv.cuda(), slots.cuda(), sc.cuda(), out=out)
        rows = M.values(kv, sc, bits).view(-1, H, 2 * D)
        there = (slots >= 0) & (slots < pages * page)
        want = torch.where(there.view(T, 1, 1), rows[slots.clamp(0, pages * page - 1)], torch.full((), 7.0, dtype=torch.float64)).to(TYPES[ty])
        assert torch.equal(out.cpu(), want)
        base = out._base if out._base is not None else out
        assert (base[..., :2] == 7).all() and (base[..., -2:] == 7).all()


def test_nothing_to_do(be):
    import ghip
    kv, sc = ghip.mx_cache(3, 16, 2, 64, 8)
    none = torch.zeros((0, 2, 64), device="cuda")
    be.kv_append(none, none, torch.zeros(0, dtype=torch.int64, device="cuda"), kv, scales=sc)
    assert be.kv_read(kv, torch.zeros(0, dtype=torch.int64, device="cuda"), sc).shape == (0, 2, 128)
    assert (sc == 27).all() and (kv.view(torch.uint8) == 0).all()
    no, ns = ghip.mx_cache(0, 16, 2, 64, 4)
    out = be.kv_read(no, torch.arange(3).cuda(), ns)
    assert (out == 0).all()


@pytest.mark.parametrize("bits", [8, 4])
def test_shift_of_a_context(be, bits):
    """Rows read back, rotated by the distance they move and written to other slots, in a captured
    graph that is replayed over a cache whose contents and slots have changed."""
    import ghip
    g = torch.Generator().manual_seed(5)
    T, H, D = 40, 2, 64
    kv, sc = (t.cuda() for t in M.cache(8, 16, H, D, bits, g))
    rope = rope_of("neox", 64, 10000.0, (0, 0, 0, 0))
    src, dst = torch.arange(20, 60).cuda(), torch.arange(64, 104).cuda()
    pos = torch.full((T,), -20, dtype=torch.int32).cuda()
    rows = torch.zeros((T, H, 2 * D), device="cuda")

    def shift():
        be.kv_read(kv, src, sc, out=rows)
        be.kv_append(rows[..., :D], rows[..., D:], dst, kv, pos=pos, rope=rope, scales=sc)

    def want():
        old = M.values(kv, sc, bits).view(-1, H, 2 * D)[src.cpu()]
        k, _ = P.rope(old[..., :D].float(), pos.cpu().view(1, -1), "neox", 64, 10000.0)
        return [M.encode(y, bits) for y in (k, old[..., D:])]

    def same(w):
        for part, (c, sb, room) in enumerate(w):
            got = M.unpack(kv.cpu(), bits).view(-1, H, 2 * D)[dst.cpu()][..., part * D:part * D + D]
            assert ((got == c) | (room < 2.0 ** -40)).all()
            assert torch.equal(sc.cpu().long().view(-1, H, 4)[dst.cpu()][..., 2 * part:2 * part + 2], sb)

    w = want()
    shift()
    same(w)
    graph, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=s):
        shift()
    for i in range(4):
        fresh = M.cache(8, 16, H, D, bits, g)
        kv.copy_(fresh[0].cuda()) if bits == 4 else kv.view(torch.uint8).copy_(fresh[0].view(torch.uint8).cuda())
        sc.copy_(fresh[1].cuda())
        src.copy_(torch.randperm(60, generator=g)[:T])
        pos.fill_(-7 - i)
        torch.cuda.synchronize()
        w = want()
        graph.replay()
        torch.cuda.synchronize()
        same(w)
        shift()
        torch.cuda.synchronize()
        same(w)
