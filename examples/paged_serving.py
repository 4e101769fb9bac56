"""Attention of one decoder layer as a server runs it: a paged KV cache, prompts
and generated tokens of several conversations in one batch, a system prompt that
they share, a sliding window.

    python examples/paged_serving.py

Each step is mul_mat (q, k, v) -> rope (q) -> kv_append (k rotated on the way, v)
-> flash_attn_paged -> mul_mat (o), all on the current stream; what changes between
steps is in three small tables (positions, slots, sequences)."""
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llama.rust_amd"))
import ghip  # noqa: E402


class Pages:
    """Which pages each conversation has (host side)."""

    def __init__(self, pages, page):
        self.page, self.free, self.tables, self.length = page, list(range(pages)), {}, {}

    def open(self, name, like=None, shared=0):
        """A new conversation; its first `shared` tokens (whole pages) are `like`'s."""
        assert shared % self.page == 0 and (like is not None or shared == 0)
        self.tables[name] = self.tables[like][:shared // self.page] if like is not None else []
        self.length[name] = shared

    def extend(self, name, n):
        """Room for n more tokens -> (their positions, their slots)"""
        first, t = self.length[name], self.tables[name]
        while len(t) * self.page < first + n:
            t.append(self.free.pop())
        self.length[name] = first + n
        pos = range(first, first + n)
        return list(pos), [t[p // self.page] * self.page + p % self.page for p in pos]

    def batch(self, todo):
        """todo: (conversation, new tokens) in the order of their rows -> device tables"""
        pos, slots, rows, q0 = [], [], [], 0
        for name, n in todo:
            p, s = self.extend(name, n)
            pos, slots = pos + p, slots + s
            rows.append([q0, n, self.length[name]] + self.tables[name])
            q0 += n
        per = max(len(r) for r in rows)
        as_dev = lambda v, ty: torch.tensor(v, dtype=ty).cuda()
        return {"pos": as_dev(pos, torch.int32), "slots": as_dev(slots, torch.int64),
                "seqs": as_dev([r + [-1] * (per - len(r)) for r in rows], torch.int32), "max_q": max(n for _, n in todo)}


class PagedAttention:
    def __init__(self, be, weights, n_heads, n_kv, head, pages, page, rope, wtype=ghip.Q4_K, ctype=torch.float16, window=0, n_first=0):
        """weights: {"q", "k", "v", "o"}: quantized blocks, rows by input"""
        self.be, self.w, self.ty, self.rope = be, weights, wtype, rope
        self.H, self.Hkv, self.D, self.window, self.n_first = n_heads, n_kv, head, window, n_first
        self.kv = torch.zeros((pages, page, n_kv, 2 * head), dtype=ctype, device="cuda")

    def __call__(self, x, b, n_shared=0):
        """x [T, hidden] f32 -> (attention's contribution to the residual, q, attention's output)"""
        be, T, D = self.be, x.shape[0], self.D
        hidden = x.shape[1]
        q, k, v = (torch.empty((T, n * D), device="cuda") for n in (self.H, self.Hkv, self.Hkv))
        be.graph_compute([ghip.mul_mat_node(self.w[n], self.ty, hidden, x, y) for n, y in (("q", q), ("k", k), ("v", v))])
        q, k, v = q.view(T, self.H, D), k.view(T, self.Hkv, D), v.view(T, self.Hkv, D)
        be.rope(q, b["pos"], self.rope, out=q)
        be.kv_append(k, v, b["slots"], self.kv, pos=b["pos"], rope=self.rope)
        o = be.flash_attn_paged(q, self.kv, b["seqs"], scale=D ** -0.5, window=self.window, n_first=self.n_first,
                                n_shared=n_shared, max_q=b["max_q"])
        return be.mul_mat(self.w["o"], self.ty, self.H * D, o.view(T, self.H * D)), q, o


def make(be, n_heads=8, n_kv=2, head=128, hidden=1024, pages=64, page=16, seed=0, **kw):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = lambda n, k: be.quantize(torch.randn((n, k), generator=g, device="cuda") * k ** -0.5, ghip.Q4_K)
    weights = {"q": w(n_heads * head, hidden), "k": w(n_kv * head, hidden), "v": w(n_kv * head, hidden), "o": w(hidden, n_heads * head)}
    return PagedAttention(be, weights, n_heads, n_kv, head, pages, page, ghip.Rope(head, ghip.ROPE_NEOX, freq_base=500000.0), **kw), Pages(pages, page)


def main():
    be = ghip.Backend(0)
    layer, pages = make(be)
    x = lambda n: torch.randn((n, 1024), device="cuda")
    pages.open("system")
    layer(x(48), pages.batch([("system", 48)]))
    users = ["a", "b", "c"]
    for u in users:
        pages.open(u, like="system", shared=48)
    # the users' first turns, of different length, then a few tokens each
    todo = list(zip(users, (20, 1, 33)))
    y, _, _ = layer(x(sum(n for _, n in todo)), pages.batch(todo), n_shared=48)
    print("prompts", tuple(y.shape), float(y.abs().mean()))
    for _ in range(4):
        y, _, _ = layer(x(3), pages.batch([(u, 1) for u in users]), n_shared=48)
    print("tokens", tuple(y.shape), float(y.abs().mean()))


if __name__ == "__main__":
    main()
