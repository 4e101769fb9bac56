"""The serving example forks a conversation after any number of tokens: within a page, at a page's
end (nothing to copy), before the first whole page."""
import os
import sys

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_fork_anywhere(bits):
    import ghip
    import paged_serving as S
    be = ghip.Backend(0)
    layer, pages = S.make(be, bits=bits)
    pages.open("a")
    layer(torch.randn((40, 1024), device="cuda"), pages.batch([("a", 40)]))
    rows = (lambda: layer.kv.flatten(0, 1)) if bits == 16 else lambda: be.kv_read(layer.kv, torch.arange(64 * 16).cuda(), layer.scales)
    for n in (5, 16, 32, 35, 40):
        name = f"b{n}"
        src, dst = pages.fork(name, "a", n)
        layer.copy(src, dst)
        assert len(src) == n % 16 and pages.length[name] == n
        now = rows()
        for p in range(n):
            i, j = (t[p // 16] * 16 + p % 16 for t in (pages.tables["a"], pages.tables[name]))
            assert torch.equal(now[i], now[j])
    # they go on, each by itself
    y, _, _ = layer(torch.randn((5, 1024), device="cuda"), pages.batch([(f"b{n}", 1) for n in (5, 16, 32, 35, 40)]))
    assert y.shape == (5, 1024) and torch.isfinite(y).all()
    be.close()
