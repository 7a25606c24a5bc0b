"""A serving step as it is used: pages and rows planned on the device, K and V written through its slots, the pages attended
to, over steps in which sessions begin, decode, wait and finish.  And 4-bit pages at sizes and lengths that the
kernels' rules tell apart.

The bar against 64 bits is that of attention over 4-bit pages (3e-6 in the 2-norm: f32 sums of scores, q and weights as two
f16 parts, the exponentials).  Over f16 and 8-bit pages it is 1e-5: a code's scale is one more f32 product (2^-24), q
goes through three 8-bit parts (2^-23 of its largest element, of which a score of 128 products adds up to sqrt(128)
2^-23 of that element's share, 1.4e-6 of a typical score's scale, times |s| <= 6)."""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import _paged as P
import _step as S

pytestmark = pytest.mark.gpu

TOL = {"q4": 3e-6, "q8": 1e-5, "f16": 1e-5}


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _turned(x, w, pos, cs, eps):
    at = cs[np.clip(pos, 0, len(cs) - 1)]
    return P.rope(S.normed(x, w, eps), at)


def _values(fmt, x):
    """What pages of a format hold of vectors x, in 64 bits."""
    if fmt == "q4":
        return S.values4(*S.quantise4(x)).astype(np.float64)
    if fmt == "q8":
        c, s = P.quantise(x)
        return np.asarray(c, np.float64) * np.asarray(s, np.float64)[..., None]
    return np.asarray(x, np.float16).astype(np.float64)


class _Server:
    """Sessions over one paged cache, on the device and, token by token, on the host."""

    eps = 1e-6

    def __init__(self, seed, fmt="q4", n=5, per=9, tpb=16, spare=4, rows=48, nh=4, nkv=2, hd=64, window=0):
        self.rng = np.random.default_rng(seed)
        self.fmt, self.n, self.tpb, self.rows, self.nh, self.nkv, self.hd, self.window = fmt, n, tpb, rows, nh, nkv, hd, window
        self.total = n * per // 2 + spare  # fewer than all sessions at their longest need
        r, t = self.rng, self.total
        self.h = dict(ctx=np.zeros(n, int), bt=np.full((n, per), -1), free=r.permutation(t), count=t)
        self.seen = [([], []) for _ in range(n)]
        a = np.arange(per * tpb)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
        self.cs = np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)
        self.w = [(1 + 0.2 * r.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        f, d = torch.float32, "cuda"
        self.d = dict(ctx=_i32(self.h["ctx"]), new=_i32([0] * n), bt=_i32(self.h["bt"]), free=_i32(self.h["free"]),
                      count=_i32([t]), starts=_i32([0] * (n + 1)), pos=_i32([0] * rows), slots=_i32([0] * rows),
                      cs=torch.from_numpy(self.cs).cuda(), qw=torch.from_numpy(self.w[0]).cuda(),
                      kw=torch.from_numpy(self.w[1]).cuda(), q=torch.zeros(rows, nh, hd, device=d),
                      k=torch.zeros(rows, nkv, hd, device=d), v=torch.zeros(rows, nkv, hd, device=d),
                      qt=torch.zeros(rows, nh, hd, device=d), out=torch.zeros(rows, nh, hd, device=d))
        if fmt == "f16":
            self.cache = [torch.zeros(t, 1, tpb, nkv, hd, dtype=torch.float16, device=d), None] * 2
            self.cache[2] = torch.zeros_like(self.cache[0])
        else:
            codes = (torch.uint8, hd // 2) if fmt == "q4" else (torch.int8, hd)
            scale = (torch.float16, (hd // 32, 2)) if fmt == "q4" else (f, ())
            self.cache = []
            for _ in range(2):
                self.cache += [torch.zeros(t, 1, nkv, tpb, codes[1], dtype=codes[0], device=d),
                               torch.zeros(t, 1, nkv, tpb, *scale[1], dtype=scale[0], device=d)]

    def ask(self, mixed=True):
        """New inputs of a step, on the host."""
        r, ctx = self.rng, self.h["ctx"]
        if mixed:
            top = self.h["bt"].shape[1] * self.tpb
            new = np.where(ctx == 0, r.integers(1, self.rows // 2, self.n), 1)
            new = np.where((ctx > 0) & (r.random(self.n) < 0.15), -1, new)
            new = np.where(ctx + new > top, -1, new)
            new = np.where(r.random(self.n) < 0.1, 0, new)
        else:
            new = np.ones(self.n, int)
        x = [r.standard_normal((self.rows, n, self.hd)).astype(np.float32) for n in (self.nh, self.nkv, self.nkv)]
        return new, x

    def give(self, new, x):
        """The inputs to the device, on the current stream."""
        self.d["new"].copy_(torch.from_numpy(new.astype(np.int32)), non_blocking=False)
        for name, y in zip("qkv", x):
            self.d[name].copy_(torch.from_numpy(y))
        self.d["out"].fill_(7.0)

    def step(self, ops, stream=None):
        d, c = self.d, self.cache
        geo = (self.total, 1, self.tpb, 0)
        heads = (self.nh, self.nkv, self.hd)
        ops.encode_kv_plan(d["ctx"], d["new"], d["bt"], self.total, self.tpb, d["free"], d["count"], d["ctx"], d["count"],
                           d["starts"], d["pos"], d["slots"], stream=stream)
        ops.encode_norm_rope_kv_write(d["q"], d["k"], d["v"], d["qt"], *heads, d["qw"], d["kw"], self.eps, d["pos"], d["cs"],
                                      d["slots"], c[0], c[2], *geo, kscale=c[1], vscale=c[3], stream=stream)
        if self.fmt == "q4":
            ops.encode_attention_q4(d["qt"], c[0], c[1], c[2], c[3], d["bt"], d["pos"], d["out"], *heads, *geo,
                                    window=self.window, row_starts_i32=d["starts"], stream=stream)
        elif self.fmt == "q8":
            ops.encode_attention_q8(d["qt"], c[0], c[1], c[2], c[3], d["bt"], d["pos"], d["out"], *heads, *geo,
                                    window=self.window, stream=stream)
        else:
            ops.encode_attention(d["qt"], c[0], c[2], d["bt"], d["pos"], d["out"], *heads, *geo, stream=stream)

    def expect(self, new, x):
        """The step on the host: rows of no session are NaN."""
        h = self.h
        before = h["ctx"]
        h["bt"], h["free"], h["ctx"], h["count"], starts, pos, _ = S.plan(before, new, h["bt"], self.total, self.tpb, h["free"],
                                                                          h["count"], self.rows)
        q = _turned(x[0], self.w[0], pos, self.cs, self.eps)
        k, v = _values(self.fmt, _turned(x[1], self.w[1], pos, self.cs, self.eps)), _values(self.fmt, x[2])
        out = torch.full((self.rows, self.nh, self.hd), float("nan"), dtype=torch.float64)
        for t in range(self.n):
            if h["ctx"][t] == 0:
                self.seen[t] = ([], [])
            ks, vs = self.seen[t]
            a, b = starts[t], starts[t + 1]
            ks += list(k[a:b])
            vs += list(v[a:b])
            assert len(ks) == h["ctx"][t]
            if a == b:
                continue
            kt, vt = torch.from_numpy(np.stack(ks)), torch.from_numpy(np.stack(vs))
            at = torch.arange(len(ks))
            for r in range(a, b):
                sees = (at <= pos[r]) & (at > pos[r] - self.window if self.window else at >= 0)
                out[r] = P.attend(torch.from_numpy(q[r]), kt, vt, sees)
        return out

    def check(self, want):
        d, h = self.d, self.h
        assert d["ctx"].cpu().tolist() == h["ctx"].tolist() and int(d["count"]) == h["count"]
        got = d["out"].cpu()
        there = ~torch.isnan(want).flatten(1).all(1)
        assert bool((got[~there] == 7.0).all())
        assert not bool(there.any()) or P.rel(got[there], want[there]) <= TOL[self.fmt]


# query heads, kv heads, head_dim, tokens per page, window
SERVERS = [(4, 2, 64, 16, 0), (9, 3, 64, 5, 0), (8, 1, 128, 16, 40), (4, 4, 128, 7, 0), (4, 1, 256, 16, 0)]


@pytest.mark.parametrize("nh,nkv,hd,tpb,window", SERVERS)
def test_steps(ops, nh, nkv, hd, tpb, window):
    s = _Server(hd + nh, nh=nh, nkv=nkv, hd=hd, tpb=tpb, per=-(-144 // tpb), window=window)
    for _ in range(12):
        new, x = s.ask()
        s.give(new, x)
        s.step(ops)
        s.check(s.expect(new, x))


@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
def test_decoding_over_each_cache(ops, fmt):
    """Rows of one token each are the other caches' calls too."""
    s = _Server(3, fmt=fmt, n=6, rows=6, nh=8, nkv=2, hd=128, per=4, spare=20)
    for _ in range(20):
        new, x = s.ask(mixed=False)
        s.give(new, x)
        s.step(ops)
        s.check(s.expect(new, x))


@pytest.mark.parametrize("nh,nkv,hd,rows", [(4, 2, 64, 48), (8, 1, 128, 48), (4, 2, 64, 2100)])
def test_steps_in_one_graph(ops, nh, nkv, hd, rows):
    """A captured step, replayed with the lengths that the device has by then, eager calls of the same context between."""
    s, other = (_Server(i, nh=nh, nkv=nkv, hd=hd, rows=rows, per=9 * rows // 48, n=5 if rows < 100 else 3) for i in (11, 12))
    cap, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=cap):
        s.step(ops, stream=cap)
    for _ in range(10):
        new, x = s.ask()
        s.give(new, x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        s.check(s.expect(new, x))
        new, x = other.ask()
        other.give(new, x)
        other.step(ops)
        other.check(other.expect(new, x))


def test_two_graphs_and_eager_steps_at_once(ops):
    """Graphs of two streams replayed without a wait between them, beside eager steps."""
    servers = [_Server(i, nh=8, nkv=2, hd=128, n=4, per=40, rows=160, spare=100) for i in (21, 22, 23)]
    caps, graphs = [torch.cuda.Stream() for _ in range(2)], [torch.cuda.CUDAGraph() for _ in range(2)]
    torch.cuda.synchronize()
    for s, c, g in zip(servers, caps, graphs):
        with torch.cuda.graph(g, stream=c):
            s.step(ops, stream=c)
    for _ in range(4):
        asked = [s.ask() for s in servers]
        for s, a in zip(servers, asked):
            s.give(*a)
        torch.cuda.synchronize()
        for c, g in zip(caps, graphs):
            with torch.cuda.stream(c):
                g.replay()
        servers[2].step(ops)
        torch.cuda.synchronize()
        for s, a in zip(servers, asked):
            s.check(s.expect(*a))


def test_steps_of_two_threads(ops):
    """Two threads, each with sessions and a stream of its own, over one context."""
    servers = [_Server(i, nh=8, nkv=2, hd=128, n=4, per=40, rows=160, spare=100) for i in (31, 32)]
    asked = [[] for _ in servers]
    want = []
    for s, a in zip(servers, asked):
        w = []
        for _ in range(8):
            a.append(s.ask())
            w.append(s.expect(*a[-1]))
        want.append(w)
    wrong = []

    def work(s, a, w):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for inputs, expected in zip(a, w):
                    s.give(*inputs)
                    s.step(ops, stream)
                    stream.synchronize()
                    got = s.d["out"].cpu()
                    there = ~torch.isnan(expected).flatten(1).all(1)
                    if not bool((got[~there] == 7.0).all()) or P.rel(got[there], expected[there]) > TOL["q4"]:
                        wrong.append("results")
        except Exception as e:  # told below: a thread's own exception would be lost
            wrong.append(repr(e))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=args) for args in zip(servers, asked, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ---- attention: few columns, sessions of all lengths, arrays past 32-bit offsets ----------


def _reference(q, cache, bt, pos, layer, per, window=0, cap=0.0):
    """As attention of _step, with pages gathered at once."""
    k, _, v, _ = S.as_f16_pages(cache)
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    for r in range(len(pos)):
        p = int(pos[r])
        if p < 0:
            continue
        kt, vt = (x[bt[r // per], layer].flatten(0, 1)[:p + 1].double() for x in (k, v))
        sees = torch.arange(p + 1) > p - window if window else torch.ones(p + 1, dtype=torch.bool)
        out[r] = P.attend(q[r], kt, vt, sees, cap=cap)
    return out


def _attend(ops, q, cache, bt, pos, layer=0, per=1, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    ops.encode_attention_q4(q.cuda(), *[c.cuda() for c in cache], _i32(bt), _i32(pos), out, nh, nkv, hd, total, layers, tpb, layer,
                            rows_per_table=per, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _lens(what, n, top, rng):
    if what == "apart":
        return [int(x) for x in np.exp(rng.uniform(0, np.log(top), n))]
    if what == "one long":
        return [top] + [int(x) for x in rng.integers(1, 40, n - 1)]
    return [top - int(x) for x in rng.integers(0, 20, n)]


# sessions, rows of each, query heads, kv heads, head_dim, tokens per page, positions, window, cap: sets of up to 4 columns
# and of 5, whole, split, and in two blocks for each compute unit
SHARES = [(1, 4, 1, 1, 64, 16, 700, 0, 0.0), (2, 2, 4, 2, 128, 7, 1333, 100, 0.0), (3, 1, 4, 1, 256, 16, 2900, 0, 20.0),
          (1, 5, 1, 1, 64, 16, 1030, 0, 0.0), (17, 1, 8, 8, 64, 16, 9000, 0, 0.0), (40, 1, 4, 1, 256, 16, 3000, 0, 0.0),
          (250, 1, 2, 2, 64, 16, 1500, 0, 0.0), (1, 1, 3, 1, 64, 16, 70000, 0, 0.0), (24, 1, 16, 8, 128, 16, 4000, 0, 0.0),
          (7, 3, 3, 3, 128, 16, 5000, 0, 0.0), (30, 1, 32, 8, 64, 16, 2500, 700, 0.0)]


@pytest.mark.parametrize("what", ["apart", "one long", "alike"])
@pytest.mark.parametrize("tables,per,nh,nkv,hd,tpb,ctx,window,cap", SHARES)
def test_sessions_of_all_lengths(ops, what, tables, per, nh, nkv, hd, tpb, ctx, window, cap):
    rng = np.random.default_rng(tables)
    g = torch.Generator().manual_seed(tables + hd)
    pages = -(-ctx // tpb)
    total = 400  # fewer than the tables name: sessions share pages here
    cache = S.cache_q4(total, 1, nkv, tpb, hd, 5)
    bt = torch.randint(0, total, (tables, pages), generator=g)
    lens = _lens(what, tables, ctx, rng)
    pos = [max(n - per + i, -1) for n in lens for i in range(per)]
    q = 1.5 * torch.randn(tables * per, nh, hd, generator=g)
    ref = _reference(q, cache, bt, pos, 0, per, window, cap)
    got = _attend(ops, q, cache, bt, pos, per=per, window=window, soft_cap=cap)
    there = torch.tensor(pos) >= 0
    assert bool((got[~there] == 7.0).all())
    assert P.rel(got[there], ref[there]) <= TOL["q4"]


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("gib", [3, 5])
def test_arrays_past_32_bit_offsets(ops, hd, gib):
    """Pages at both ends of codes of 3 and 5 GiB: written, read back and attended to."""
    g = torch.Generator().manual_seed(hd)
    nkv, tpb, layers, nh = 8, 16, 32, 16
    page = nkv * tpb * hd // 2
    total = (gib << 30) // (page * layers)
    cache = []
    for _ in range(2):
        cache += [torch.empty(total, layers, nkv, tpb, hd // 2, dtype=torch.uint8, device="cuda"),
                  torch.empty(total, layers, nkv, tpb, hd // 32, 2, dtype=torch.float16, device="cuda")]
    ctx, layer = 200, layers - 1
    pages = -(-ctx // tpb)
    order = [0, total - 1, total // 2, total // 3] + [total - 2 - i for i in range(pages - 4)]
    bt = torch.tensor([order])
    k, v = (torch.randn(ctx, nkv, hd, generator=g) for _ in range(2))
    q = torch.randn(ctx, nh, hd, generator=g)
    slots = [order[p // tpb] * tpb + p % tpb for p in range(ctx)]
    geo = (total, layers, tpb, layer)
    dq = q.cuda()
    ops.encode_norm_rope_kv_write(dq, k.cuda(), v.cuda(), dq, nh, nkv, hd, None, None, 0.0, _i32(range(ctx)), None, _i32(slots),
                                  cache[0], cache[2], *geo, kscale=cache[1], vscale=cache[3])
    held = [torch.from_numpy(S.values4(*S.quantise4(x.numpy())).astype(np.float32)) for x in (k, v)]
    back = [torch.zeros(ctx, nkv, hd, device="cuda") for _ in range(2)]
    ops.encode_kv_read_q4(cache[0], cache[1], cache[2], cache[3], _i32(bt), _i32(range(ctx)), *back, nkv, hd, *geo,
                          rows_per_table=ctx)
    torch.cuda.synchronize()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(back, held))
    rows = [0, 7, 100, 101, 102, ctx - 2, ctx - 1]
    want = torch.stack([P.attend(q[r], held[0][:r + 1].double(), held[1][:r + 1].double(), torch.ones(r + 1, dtype=torch.bool))
                        for r in rows])
    for starts in (None, [0, len(rows)]):
        out = torch.zeros(len(rows), nh, hd, device="cuda")
        ops.encode_attention_q4(dq[rows].contiguous(), *cache, _i32(bt), _i32(rows), out, nh, nkv, hd, *geo,
                                rows_per_table=1 if starts else len(rows), row_starts_i32=None if starts is None else _i32(starts))
        torch.cuda.synchronize()
        assert P.rel(out.cpu(), want) <= TOL["q4"]
    out = torch.zeros(1, nh, hd, device="cuda")  # two columns
    ops.encode_attention_q4(dq[-1:], *cache, _i32(bt), _i32([ctx - 1]), out, nh, nkv, hd, *geo)
    torch.cuda.synchronize()
    assert P.rel(out.cpu(), want[-1:]) <= TOL["q4"]
