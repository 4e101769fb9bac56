"""ghip_flash_attn_paged over a table with a row for every slot of a server, most
of them idle (no rows in this batch), against the formula in 64 bits.  The workspace
is the caller's and holds NaN, so that a partial nobody wrote shows."""
import pytest

import paged_oracle as P
from test_gpu_flash_attn_paged import compare, make, ways

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def be():
    import ghip
    b = ghip.Backend(0)
    yield b
    b.close()


def check(be, slots, H, Hkv, D, ctype, n_shared, change=None, **kw):
    """slots: (rows, keys) of each; change(table): what the idle slots' rows hold instead"""
    q, kv, table = make(slots, H, Hkv, D, ctype, 16, n_shared)
    want, mag, wgt = P.attention(q, kv, table.tolist(), D ** -0.5, **kw)
    if change:
        change(table)
    q, kvd, td = q.cuda(), kv.cuda(), table.cuda()
    max_q = max(n for n, _ in slots)
    print(f"slots {len(slots)} live {sum(n > 0 for n, _ in slots)} H={H}/{Hkv} D={D} {ctype} shared={n_shared} {kw}", flush=True)
    for how in ways(n_shared):
        need = be.flash_attn_paged_workspace(q, kvd, td, n_shared=n_shared, max_q=max_q, **kw)
        if need:
            be.set_workspace(torch.full((need // 4,), float("nan"), device="cuda").view(torch.uint8))
        got = be.flash_attn_paged(q, kvd, td, scale=D ** -0.5, n_shared=n_shared, max_q=max_q, **kw).cpu()
        torch.cuda.synchronize()
        compare(got, want, mag, wgt, D)


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("H,Hkv,D,ctype", [(16, 1, 64, "f16"), (16, 4, 128, "bf16"), (6, 2, 256, "f16")])
@pytest.mark.parametrize("live", [(30, 34), (39, 40), (0, 2)])
def test_live_slots_among_idle_ones(be, live, H, Hkv, D, ctype, rows):
    """More idle slots than a workgroup of rows holds, before and after the live ones."""
    n_shared = 96
    slots = [(rows if live[0] <= b < live[1] else 0, n_shared + 5 + b % 7) for b in range(40)]
    check(be, slots, H, Hkv, D, ctype, n_shared)


def test_many_idle_slots(be):
    """Hundreds of slots (the rows are found 256 sequences at a time), a window over the prefix."""
    slots = [(1 if b in (3, 255, 256, 290, 511, 599) else 0, 70 + b % 3) for b in range(600)]
    check(be, slots, 8, 1, 64, "f16", 64)
    check(be, slots, 8, 1, 64, "f16", 64, window=20, n_first=3)


@pytest.mark.parametrize("rows", [1, 3])
@pytest.mark.parametrize("live", [(1, 6), (35, 40)])
def test_idle_first_slots_hold_nothing(be, live, rows):
    """The prefix is read through the pages of a slot that has rows: those of idle ones
    before it are gone, or past the cache."""
    n_shared = 96
    slots = [(rows if live[0] <= b < live[1] else 0, n_shared + 5 + b % 7) for b in range(40)]
    for what in (-1, 0, 10 ** 9):
        def change(table):
            for b in range(40):
                if not live[0] <= b < live[1]:
                    table[b, :3], table[b, 3:] = 0, what
        check(be, slots, 16, 4, 64, "f16", n_shared, change)


@pytest.mark.parametrize("rows", [1, 9, 70])
def test_cache_without_pages(be, rows):
    """Nothing is read in the place of missing pages (q lies at no multiple of 16 bytes):
    rows that see a key are NaN, those before the first one 0."""
    be.set_workspace(None)
    for n_shared in (0, 20):
        flat = torch.randn(2 * rows * 4 * 64 + 3, device="cuda")
        q = flat[3:].view(2 * rows, 4, 64)
        kv = torch.empty((0, 16, 2, 128), dtype=torch.float16, device="cuda")
        seqs = torch.tensor([[0, rows, rows, 0, 1], [rows, rows, rows // 2, 5, -1]], dtype=torch.int32, device="cuda")
        for sinks in (None, torch.zeros(4, device="cuda")):
            got = be.flash_attn_paged(q, kv, seqs, sinks=sinks, n_shared=n_shared, max_q=rows).cpu()
            torch.cuda.synchronize()
            first = rows + rows - rows // 2
            assert torch.isnan(got[:rows]).all() and torch.isnan(got[first:]).all() and (got[rows:first] == 0).all()


@pytest.mark.parametrize("rows", [1, 3])
def test_first_sequence_ends_inside_the_prefix(be, rows):
    """A sequence that is shorter than the prefix holds pages for its own keys alone: the
    prefix is read through one that has all of it."""
    def zeros(table):  # (what a table that is cleared at first holds there)
        table[:, 3:][table[:, 3:] < 0] = 0

    for change in (None, zeros):
        check(be, [(rows, 30), (rows, 100), (rows, 150), (rows, 97)], 16, 4, 64, "f16", 96, change)
        check(be, [(0, 200), (rows, 30)] + [(rows, 100 + b) for b in range(80)], 8, 2, 64, "bf16", 96, change)
        check(be, [(rows, 30), (rows, 64), (rows, 95)], 16, 4, 64, "f16", 96, change)
