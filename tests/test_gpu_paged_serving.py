"""The serving example end to end, step by step against 64 bits: prompts, shared
pages and generated tokens on one cache; and the workspace that attention takes."""
import os
import sys

import pytest

import paged_oracle as P

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


@pytest.mark.parametrize("window,n_first,ctype", [(0, 0, torch.float16), (40, 4, torch.bfloat16)])
def test_serving(be, window, n_first, ctype):
    import paged_serving as S
    layer, pages = S.make(be, window=window, n_first=n_first, ctype=ctype)
    D = layer.D

    def step(todo, n_shared=0):
        x = torch.randn((sum(n for _, n in todo), 1024), device="cuda")
        b = pages.batch(todo)
        y, q, o = layer(x, b, n_shared=n_shared)
        T = x.shape[0]
        # q and the cache hold the projections, rotated
        for name, got, heads in (("q", q, layer.H), ("k", layer.kv.view(-1, layer.Hkv, 2 * D)[b["slots"], :, :D], layer.Hkv)):
            raw = be.mul_mat(layer.w[name], layer.ty, 1024, x).view(T, heads, D).cpu()
            want, mag = P.rope(raw, b["pos"].cpu().view(1, T), "neox", D, 500000.0)
            half = torch.finfo(got.dtype).eps / 2
            # (a product of three matrices in one launch may differ in its sum's last bits: 2^-20)
            assert ((got.cpu().double() - want).abs() <= mag * (2.0 ** -20 + 2.0 ** -21) + want.abs() * half * 1.01 + 1e-7).all()
        want, mag, wgt = P.attention(q.cpu(), layer.kv.cpu(), b["seqs"].tolist(), D ** -0.5, None, window, n_first)
        assert ((o.cpu().double() - want).abs() <= P.attention_tol(mag, wgt, D)).all()
        assert y.shape == (T, 1024) and torch.isfinite(y).all()

    pages.open("system")
    step([("system", 48)])
    for u in "abc":
        pages.open(u, like="system", shared=48)
    step([("a", 20), ("b", 1), ("c", 33)], n_shared=48)
    for _ in range(3):
        step([("c", 1), ("a", 1), ("b", 1)], n_shared=48)
    step([("a", 1), ("c", 5)])


def test_example_runs(be):
    import paged_serving as S
    S.main()


def test_workspace_of_the_caller(be):
    """With a workspace of the size asked for, attention allocates nothing and gives
    the same bits; with less it is refused with a status."""
    import ghip
    q = torch.randn((6, 8, 128), device="cuda")
    kv = torch.randn((300, 16, 2, 256), device="cuda").half()
    seqs = torch.zeros((6, 3 + 200), dtype=torch.int32)
    for b in range(6):
        seqs[b, :3] = torch.tensor([b, 1, 3000 - b])
        seqs[b, 3:] = torch.randperm(300)[:200]
    seqs = seqs.cuda()
    for kw in (dict(max_q=1), dict(max_q=1, window=1000), dict(max_q=1, n_shared=0), dict(max_q=3)):
        want = be.flash_attn_paged(q, kv, seqs, scale=0.09, **kw)
        need = be.flash_attn_paged_workspace(q, kv, seqs, **kw)
        if not need:
            continue
        own = ghip.Backend(0)
        own.set_workspace(torch.empty(need, dtype=torch.uint8, device="cuda"))
        assert torch.equal(own.flash_attn_paged(q, kv, seqs, scale=0.09, **kw), want)
        own.set_workspace(torch.empty(need - 1, dtype=torch.uint8, device="cuda"))
        with pytest.raises(ghip.GhipError, match="workspace"):
            own.flash_attn_paged(q, kv, seqs, scale=0.09, **kw)
        torch.cuda.synchronize()
        own.close()


def test_streams_take_turns_at_the_workspace(be):
    """Split calls on two streams in turn: the second waits for the first."""
    import ghip
    kv = torch.randn((700, 16, 2, 256), device="cuda").half()
    seqs = torch.cat([torch.tensor([0, 1, 11000]), torch.randperm(700)[:690]]).to(torch.int32).view(1, -1).cuda()
    qs = [torch.randn((1, 8, 128), device="cuda") for _ in range(6)]
    want = [be.flash_attn_paged(q, kv, seqs, scale=0.09) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(be.flash_attn_paged(q, kv, seqs, scale=0.09))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_ragged_batch_joins_by_rows(be):
    """One long chunk beside many single rows, split keys: the join goes by rows."""
    import ghip
    g = torch.Generator().manual_seed(4)
    lens = [(40, 700)] + [(1, 600 + 7 * i) for i in range(20)]
    T = sum(n for n, _ in lens)
    kv = torch.randn((1200, 16, 1, 128), generator=g).half()
    per = 48
    seqs, at = torch.zeros((21, 3 + per), dtype=torch.int32), 0
    shared = torch.arange(20)
    for b, (n, m) in enumerate(lens):
        seqs[b, :3] = torch.tensor([at, n, m])
        seqs[b, 3:23] = shared
        seqs[b, 23:] = 20 + b * 28 + torch.arange(28)
        at += n
    q = torch.randn((T, 2, 64), generator=g)
    want, mag, wgt = P.attention(q, kv, seqs.tolist(), 0.125)
    got = be.flash_attn_paged(q.cuda(), kv.cuda(), seqs.cuda(), scale=0.125, n_shared=320, max_q=40).cpu().double()
    assert ((got - want).abs() <= P.attention_tol(mag, wgt, 64)).all()
