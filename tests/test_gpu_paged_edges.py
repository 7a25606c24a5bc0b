"""Attention over shared pages (attention_paged.hip) where a result hangs on few positions of a split, on numbers near
the ends of f32, or on what else runs on the stream: against plain 64-bit results.

The bar is 3e-6 in the 2-norm, as for ordinary inputs: a score of size |s| <= 10 from f32 sums is off by a few 2^-24 |s|
(6e-7 each), the exponentials by 2^-22, and the sums of weights and values by a few 2^-24.  Sizes of scores beyond that
are equal among the positions that weigh anything, so that their rounding leaves the quotient."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu

TOL = 3e-6


def _pages(f16, total, layers, nkv, tpb, hd, seed):
    if not f16:
        return P.cache_q8(total, layers, nkv, tpb, hd, seed)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(total, layers, tpb, nkv, hd, generator=g).half() for _ in range(2))
    return [k, None, v, None]


def _random_tree(g, tree):
    return P.tree_bits([-1 if j == 0 else int(torch.randint(-1, j, (1,), generator=g)) for j in range(tree)])


def _tree_call(ops, q, cache, bt, ctx, bits, f16, **kw):
    tables, tree, nh, hd = q.shape
    kc, ks, vc, vs = cache
    total, layers = kc.shape[:2]
    tpb, nkv = (kc.shape[2], kc.shape[3]) if f16 else (kc.shape[3], kc.shape[2])
    out = torch.full(q.shape, 7.0, device="cuda")
    ops.encode_attention_tree(q.cuda(), kc.cuda(), vc.cuda(), bt.to(torch.int32).cuda(), ctx.to(torch.int32).cuda(),
                              P.words_of(bits).cuda(), out, nh, nkv, hd, total, layers, tpb, 0,
                              kscale=None if f16 else ks.cuda(), vscale=None if f16 else vs.cuda(), **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _attention(ops, q, cache, bt, pos, per, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    ops.encode_attention_q8(q.cuda(), *[c.cuda() for c in cache], bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda(), out,
                            nh, nkv, hd, total, layers, tpb, 0, rows_per_table=per, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _same_where_finite(got, ref):
    """NaN in the same places, and the others near."""
    bad = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), bad)
    assert P.rel(got[~bad], ref[~bad]) <= TOL


# ---- keys alone that are not finite, in a split of their own --------------------------------
# ctx is a whole number of units (four waves of 64 or 32 positions), so that the drafted slots stand in a split of their
# own, of which a root node sees nothing but itself


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,ctx", [(64, 1024), (128, 1280), (256, 640)])
@pytest.mark.parametrize("what", ["own slot", "a unit of the context", "NaN beside -inf"])
def test_nan_keys_reach_every_node_that_sees_them(ops, f16, hd, ctx, what):
    g = torch.Generator().manual_seed(hd)
    tree, nh, nkv, tpb = 20, 6, 2, 16
    bt = torch.randperm(ctx // tpb + 4, generator=g)[None, :ctx // tpb + 2]
    cache = _pages(f16, ctx // tpb + 4, 1, nkv, tpb, hd, 37)
    q = torch.randn(1, tree, nh, hd, generator=g)
    q[..., 0] = q[..., 0].abs() + 0.1
    bits = _random_tree(g, tree)[None]
    bits[0, :, 7] = False
    bits[0, 7] = False
    bits[0, 7, 7] = True  # a root that no other node sees
    at = dict(zip(["own slot", "a unit of the context", "NaN beside -inf"],
                  [[ctx + 7], range(256, 512), [ctx + 7]]))[what]
    for p in at:
        blk, sl = int(bt[0, p // tpb]), p % tpb
        if f16:
            cache[0][blk, 0, sl] = math.nan
        else:
            cache[1][blk, 0, :, sl] = math.nan
    if what == "NaN beside -inf" and f16:  # the root sees -inf scores in its split too
        bits[0, 7, 8:12] = True
        for p in range(ctx + 8, ctx + 12):
            cache[0][int(bt[0, p // tpb]), 0, p % tpb, :, 0] = -math.inf
    ref = P.tree(q, *cache, bt, torch.tensor([ctx]), bits, 0)
    assert bool(torch.isnan(ref[0, 7]).all())
    got = _tree_call(ops, q, cache, bt, torch.tensor([ctx]), bits, f16)
    if what == "a unit of the context":
        assert bool(torch.isnan(got).all())
    else:
        _same_where_finite(got, ref)


@pytest.mark.parametrize("hd,ctx", [(64, 1024), (128, 1280), (256, 640)])
def test_keys_of_minus_infinity_weigh_nothing(ops, hd, ctx):
    """Units of the context and the drafted slots whose scores are all -inf, beside others; and nothing but those."""
    g = torch.Generator().manual_seed(hd + 1)
    tree, nh, nkv, tpb = 20, 6, 2, 16
    bt = torch.randperm(ctx // tpb + 4, generator=g)[None, :ctx // tpb + 2]
    cache = _pages(True, ctx // tpb + 4, 1, nkv, tpb, hd, 39)
    q = torch.randn(1, tree, nh, hd, generator=g)
    q[..., 0] = q[..., 0].abs() + 0.1
    bits = _random_tree(g, tree)[None]

    def spoil(positions):
        for p in positions:
            cache[0][int(bt[0, p // tpb]), 0, p % tpb, :, 0] = -math.inf

    spoil([*range(256, 512), *range(ctx, ctx + tree)])
    ref = P.tree(q, *cache, bt, torch.tensor([ctx]), bits, 0)
    assert bool(torch.isfinite(ref).all())
    _same_where_finite(_tree_call(ops, q, cache, bt, torch.tensor([ctx]), bits, True), ref)
    spoil(range(ctx))
    assert bool(torch.isnan(_tree_call(ops, q, cache, bt, torch.tensor([ctx]), bits, True)).all())


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,ctx", [(64, 60), (64, 1024), (256, 640)])
@pytest.mark.parametrize("some", [True, False])
def test_queries_that_are_not_finite_over_missing_pages(ops, f16, hd, ctx, some):
    """A missing page is zeros, so a q with an infinity or a NaN has the score NaN there: its row is NaN, where some
    pages are missing and its other scores are -inf, and where all are."""
    g = torch.Generator().manual_seed(hd + 2)
    tree, nh, nkv, tpb = 12, 4, 2, 16
    bt = torch.randperm(ctx // tpb + 4, generator=g)[None, :ctx // tpb + 2]
    bt[0, (1 if some else slice(None))] = -1
    cache = _pages(f16, ctx // tpb + 4, 1, nkv, tpb, hd, 41)
    cache[0][..., 3] = -cache[0][..., 3].abs().clamp(min=1)
    q = torch.randn(1, tree, nh, hd, generator=g)
    bits = _random_tree(g, tree)[None]
    clean = P.tree(q, *cache, bt, torch.tensor([ctx]), bits, 0)
    q[0, 2, 1, 3], q[0, 5, 2, 3] = math.inf, math.nan
    got = _tree_call(ops, q, cache, bt, torch.tensor([ctx]), bits, f16)
    bad = torch.zeros(1, tree, nh, dtype=torch.bool)
    bad[0, 2, 1] = bad[0, 5, 2] = True
    assert bool(torch.isnan(got[bad]).all())
    if some:
        assert P.rel(got[~bad], clean[~bad]) <= TOL
    else:
        assert bool((got[~bad] == 0).all())


# ---- numbers near the ends of f32 ---------------------------------------------------------


@pytest.mark.parametrize("hd,ctx", [(64, 701), (128, 2500), (256, 1300)])
@pytest.mark.parametrize("keys,queries", [(1e34, 1e-34), (1e-34, 1e34), (1e36, 1e-36), (1e-36, 1e36), (1e32, 1e-20)])
@pytest.mark.parametrize("kw", [{}, dict(soft_cap=5.0)])
def test_scores_in_range_of_keys_and_queries_that_are_not(ops, hd, ctx, keys, queries, kw):
    """Keys of 1e34 against queries of 1e-34 have ordinary scores, and so the other way round; scores of 1e12 are finite
    too, and the largest takes all the weight."""
    g = torch.Generator().manual_seed(ctx)
    nh, nkv, tpb = 6, 2, 16
    bt = torch.randperm(-(-ctx // tpb) + 1, generator=g)[None, :-(-ctx // tpb)]
    cache = P.cache_q8(bt.shape[1] + 1, 1, nkv, tpb, hd, 43)
    cache[1] *= keys
    q = torch.randn(1, nh, hd, generator=g) * 1.2
    q = (q / q.abs().max() * 3).mul(queries)
    assert bool(torch.isfinite(q).all())
    ref = P.causal(q, *cache, bt, torch.tensor([ctx - 1]), 0, 1, cap=kw.get("soft_cap", 0.0))
    got = _attention(ops, q, cache, bt, torch.tensor([ctx - 1]), 1, **kw)
    assert bool(torch.isfinite(got).all()) and P.rel(got, ref) <= TOL


@pytest.mark.parametrize("hd,nh,nkv,ctx,rows", [(64, 14, 2, 300, 1), (128, 8, 2, 2500, 1), (256, 4, 1, 600, 1),
                                                (64, 32, 8, 400, 300), (128, 32, 8, 400, 300)])
def test_a_loud_element_of_q_leaves_the_others_their_bits(ops, hd, nh, nkv, ctx, rows):
    """One element of q 300 times the others where the keys hold zeros: the scores come from the others alone.  They are
    integers of 2^-29 of the largest's power of two, some 1000: a rounding of 0.29 * 2^-29 * 1000 = 5.4e-7 (rms) each, and
    as much of a score of keys of size 1."""
    g = torch.Generator().manual_seed(hd)
    tpb = 16
    bt = torch.randperm(-(-ctx // tpb) + 1, generator=g)[None, :-(-ctx // tpb)]
    cache = P.cache_q8(bt.shape[1] + 1, 1, nkv, tpb, hd, 47)
    cache[0][..., 5] = 0
    q = torch.randn(rows, nh, hd, generator=g) * 1.2
    q[..., 5] *= 300.0
    pos = torch.arange(ctx - rows, ctx)
    some = sorted({0, rows // 2, rows - 1})
    ref = torch.cat([P.causal(q[r:r + 1], *cache, bt, pos[r:r + 1], 0, 1) for r in some])
    assert P.rel(_attention(ops, q, cache, bt, pos, rows)[some], ref) <= TOL


def _values_of_size(order, nv, tpb, hd, g):
    """One table of 8-bit pages whose keys are 127 s in their first element, zero elsewhere: a query of 1 there scores
    127 s / sqrt(hd).  order: (positions, score, size of the values) in turn; a size of 0: zero scales."""
    n = sum(o[0] for o in order)
    pages = -(-n // tpb)
    bt = torch.randperm(pages + 1, generator=g)[None, :pages]
    kc, ks, vc, vs = P.cache_q8(pages + 1, 1, nv, tpb, hd, 53)
    kc.zero_()
    kc[..., 0] = 127
    p = 0
    for count, score, size in order:
        for i in range(p, p + count):
            at = (int(bt[0, i // tpb]), 0, slice(None), i % tpb)
            ks[at] = score * math.sqrt(hd) / 127
            vs[at] *= size
        p += count
    return (kc, ks, vc, vs), bt, n


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("order", [
    [(700, 0.0, 1e-32)], [(1500, 0.0, 1e-36)], [(1, 0.0, 1e-34)],
    [(600, 0.0, 0.0), (600, 0.0, 1e-33)],                # zeros first
    [(900, 0.0, 1.0), (900, 80.0, 1e-32)],               # small values of a weight e^80 times that of the others
    [(900, 80.0, 1e-32), (900, 0.0, 1.0)],
    [(64, 80.0, 1e-32), (64, 0.0, 1.0)] * 12, [(64, 0.0, 1e-30), (64, 0.0, 1e-10), (64, 0.0, 1e5)] * 3,
    [(64, 0.0, 1e5), (64, 0.0, 0.0), (64, 0.0, 1e-34)] * 5, [(64, 0.0, 1e33), (64, 0.0, 1e-34)] * 4, [(300, 0.0, 1e33), (300, 0.0, 1e-34)],
    [(64, 0.0, 1e3), (64, 85.0, 1e-30)] * 5])
def test_small_values_keep_their_bits(ops, hd, order):
    """Values whose scales the cache holds exactly, down to the smallest: the quotient is as near as that of ordinary
    ones, with large values, zeros and other weights before and behind."""
    g = torch.Generator().manual_seed(len(order))
    cache, bt, n = _values_of_size(order, 1, 16, hd, g)
    q = torch.zeros(1, 2, hd)
    q[..., 0] = 1.0
    ref = P.causal(q, *cache, bt, torch.tensor([n - 1]), 0, 1)
    got = _attention(ops, q, cache, bt, torch.tensor([n - 1]), 1)
    assert P.rel(got, ref) <= TOL


# ---- a window behind a context that is longer than the table -------------------------------------


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("tables,hd", [(7, 64), (7, 256), (70, 128)])  # the last: 32 columns at a time
def test_windows_of_contexts_past_the_table(ops, f16, tables, hd):
    """A node sees the positions above context + nodes - 1 - window that the table has, which may be none."""
    g = torch.Generator().manual_seed(61)
    tree, nh, nkv, tpb, pages, window = 9, 8, 2, 16, 5, 40
    room = pages * tpb
    bt = torch.randperm(tables * pages + 1, generator=g)[:tables * pages].view(tables, pages)
    cache = _pages(f16, tables * pages + 1, 1, nkv, tpb, hd, 59)
    q = torch.randn(tables, tree, nh, hd, generator=g)
    ctx = torch.tensor([room - 4, room, room + 7, room + 29, room + 33, room + 200, 2**31 - 1] * (tables // 7))
    bits = np.stack([_random_tree(g, tree) for _ in range(tables)])
    got = _tree_call(ops, q, cache, bt, ctx, bits, f16, window=window)
    ref = torch.zeros(q.shape, dtype=torch.float64)
    at = torch.arange(room)
    for t in range(tables):
        k, v = (P.gather(c, s, bt[t], 0, range(room), cache[0].shape[0], tpb) for c, s in (cache[:2], cache[2:]))
        for j in range(tree):
            c = int(ctx[t])
            sees = (at < c) & (at > c + int(bits[t, j].sum()) - 1 - window)
            for i in range(tree):
                if bits[t, j, i] and c + i < room:
                    sees[c + i] = True
            ref[t, j] = P.attend(q[t, j], k, v, sees)
    none = (ref == 0).all(-1)
    assert bool(none.any()) and bool((got[none] == 0).all())
    assert P.rel(got, ref) <= TOL


# ---- both sides of the rule that plans splits: fewer than 256 blocks, over tables of more than three units -------------


@pytest.mark.parametrize("tables,nkv", [(255, 1), (256, 1), (257, 1), (85, 3), (86, 3)])
def test_sessions_on_both_sides_of_256_blocks(ops, tables, nkv):
    g = torch.Generator().manual_seed(tables)
    hd, tpb, pages = 64, 16, 57  # 912 positions: four units of 256
    bt = torch.randint(0, 200, (tables, pages), generator=g)
    cache = P.cache_q8(200, 1, nkv, tpb, hd, 71)
    q = torch.randn(tables, 2 * nkv, hd, generator=g)
    pos = torch.randint(-1, pages * tpb, (tables,), generator=g)
    pos[0], pos[-1] = pages * tpb - 1, 800
    got = _attention(ops, q, cache, bt, pos, 1)
    some = torch.unique(torch.cat([torch.tensor([0, 1, tables // 2, tables - 1]), torch.randperm(tables, generator=g)[:10]]))
    ref = P.causal(q[some], *cache, bt[some], pos[some], 0, 1)
    none = pos[some] < 0
    assert bool((got[some][none] == 7.0).all())
    assert P.rel(got[some][~none], ref[~none]) <= TOL


# ---- beside graphs of the f16 cache's attention -----------------------------------------------------


def _f16_set(seed, ctx=4000):
    """Four sessions of the f16 cache whose positions cellm_hip_attention_gqa_f16kv splits."""
    g = torch.Generator().manual_seed(seed)
    tables, nh, nkv, hd, tpb = 4, 8, 2, 64, 16
    pages = -(-ctx // tpb)
    kc, vc = (torch.randn(tables * pages, 1, tpb, nkv, hd, generator=g).half().cuda() for _ in range(2))
    bt = torch.randperm(tables * pages, generator=g).view(tables, pages).to(torch.int32).cuda()
    q = torch.randn(tables, nh, hd, generator=g).cuda()
    pos = torch.randint(ctx // 2, ctx, (tables,), generator=g).to(torch.int32).cuda()
    out = torch.zeros_like(q)
    return dict(args=(q, kc, vc, bt, pos, out, nh, nkv, hd, tables * pages, 1, tpb, 0), out=out)


def _q8_set(seed, ctx=3000, hd=64):
    g = torch.Generator().manual_seed(seed)
    tables, nh, nkv, tpb = 3, 4, 2, 16
    pages = -(-ctx // tpb)
    bt = torch.randperm(tables * pages + 1, generator=g)[:tables * pages].view(tables, pages)
    cache = [c.cuda() for c in P.cache_q8(tables * pages + 1, 1, nkv, tpb, hd, seed)]
    q = torch.randn(tables, nh, hd, generator=g).cuda()
    pos = torch.randint(ctx // 2, ctx, (tables,), generator=g).to(torch.int32).cuda()
    out = torch.zeros_like(q)
    return dict(args=(q, *cache, bt.to(torch.int32).cuda(), pos, out, nh, nkv, hd, tables * pages + 1, 1, tpb, 0), out=out)


def _results(calls):
    out = []
    for call, s in calls:
        call(*s["args"])
        torch.cuda.synchronize()
        out.append(s["out"].clone())
        s["out"].zero_()
    return out


def test_eager_calls_have_scratch_that_no_graph_of_the_f16_cache_holds():
    """The scratch that an f16 call left on a stream, and a graph of that stream may hold, is not what an 8-bit call there
    uses: the free memory tells."""
    from cellm_amd import HipOps

    side, f16, q8 = torch.cuda.Stream(), _f16_set(1, 30000), _q8_set(2, hd=256)
    with HipOps(0) as own:
        own.encode_attention_q8(*q8["args"])  # the kernel's module is loaded, another stream's scratch taken
        own.encode_attention(*f16["args"], stream=side)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        own.encode_attention_q8(*q8["args"], stream=side)  # 64 KiB and some 250 splits of 16 x 258 floats
        torch.cuda.synchronize()
        assert before - torch.cuda.mem_get_info()[0] >= 2**21


def test_scratch_of_captures_is_given_back():
    """A program that captures again and again: the context's memory stands where it was once the graphs are gone and it
    says so, graphs captured afterwards give the eager result, and so do eager calls on the capture's stream."""
    from cellm_amd import HipOps

    s, cap = _q8_set(6, hd=256), torch.cuda.Stream()
    with HipOps(0) as own:
        (want,) = _results([(own.encode_attention_q8, s)])

        def captured():
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=cap):
                own.encode_attention_q8(*s["args"], stream=cap)
            return graph

        captured().replay()
        torch.cuda.synchronize()
        own.release_graph_scratch()
        before = torch.cuda.mem_get_info()[0]
        for _ in range(3):
            graphs = [captured() for _ in range(30)]
            for graph in graphs:
                s["out"].zero_()
                graph.replay()
                torch.cuda.synchronize()
                assert torch.equal(s["out"], want)
            assert before - torch.cuda.mem_get_info()[0] >= 30 * 2**21  # each its own
            del graph, graphs
            own.release_graph_scratch()
            assert before - torch.cuda.mem_get_info()[0] <= 10 * 2**21  # what the runtime keeps of its own
            s["out"].zero_()
            own.encode_attention_q8(*s["args"], stream=cap)
            torch.cuda.synchronize()
            assert torch.equal(s["out"], want)


def test_graphs_of_the_f16_cache_run_beside_eager_calls_of_their_stream(ops):
    """A graph of the f16 cache's attention replayed on one stream while 8-bit calls and trees run on the stream that it
    was captured on: each has its own result."""
    f16, q8 = _f16_set(3), [_q8_set(s) for s in (4, 5)]
    want_f16, *want_q8 = _results([(ops.encode_attention, f16), *((ops.encode_attention_q8, s) for s in q8)])
    cap, other, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    ops.encode_attention(*f16["args"], stream=cap)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=cap):
        for _ in range(20):
            ops.encode_attention(*f16["args"], stream=cap)
    for _ in range(6):
        for s in (f16, *q8):
            s["out"].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(other):
            graph.replay()
        for _ in range(10):
            for s in q8:
                ops.encode_attention_q8(*s["args"], stream=cap)
        torch.cuda.synchronize()
        for s, w in zip((f16, *q8), (want_f16, *want_q8)):
            assert torch.equal(s["out"], w)


# ---- drafts over the f16 cache, as a serving loop runs them --------------------------------------------


def test_drafted_decode_over_the_f16_cache(ops):
    """A prompt enters the f16 cache, a tree of drafts is written behind it, checked in one call and its accepted path
    kept; the next token attends to it.  The pages are those of the path entered token by token, and every accepted
    node's attention and the next token's are near what encode_attention gives there."""
    g = torch.Generator().manual_seed(73)
    nh, nkv, hd, tpb, prompt, tree, pages = 6, 2, 64, 8, 45, 13, 9
    parents = [-1, -1, 0, 0, 1, 2, 2, 5, 5, 4, 8, 8, 10]
    path = [0, 2, 5, 8, 10, 12]
    bits = P.tree_bits(parents)
    depth = torch.from_numpy(bits.sum(1).astype(np.int32)) - 1
    bt = torch.randperm(pages, generator=g)[None].to(torch.int32).cuda()
    a = np.arange(80)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    cs = torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda()
    x = [torch.randn(prompt + tree + 1, n, hd, generator=g).cuda() for n in (nh, nkv, nkv)]
    geo = (pages, 1, tpb, 0)

    def ints(values):
        return torch.tensor(list(values), dtype=torch.int32).cuda()

    def enter(cache, rows, pos, slots):
        q, k, v = (t[list(rows)].contiguous() for t in x)
        ops.encode_rope_half(q, nh, hd, pos, cs)
        ops.encode_rope_half(k, nkv, hd, pos, cs)
        ops.encode_kv_write(k.view(k.shape[0], -1), v.view(v.shape[0], -1), slots, *cache,
                            bt.expand(k.shape[0], -1).contiguous(), *geo)
        return q

    def attend(cache, q, pos):
        out = torch.empty_like(q)
        ops.encode_attention(q, *cache, bt.expand(q.shape[0], -1).contiguous(), pos, out, nh, nkv, hd, *geo)
        return out

    def fresh():
        return [torch.zeros(pages, 1, tpb, nkv, hd, dtype=torch.float16, device="cuda") for _ in range(2)]

    one, outs = fresh(), []
    enter(one, range(prompt), ints(range(prompt)), ints(range(prompt)))
    for i, node in enumerate(path):
        at = ints([prompt + i])
        outs.append(attend(one, enter(one, [prompt + node], at, at), at))
    at = ints([prompt + len(path)])
    last = attend(one, enter(one, [prompt + tree], at, at), at)

    two = fresh()
    enter(two, range(prompt), ints(range(prompt)), ints(range(prompt)))
    q = enter(two, range(prompt, prompt + tree), (prompt + depth).cuda(), ints(range(prompt, prompt + tree)))
    out = torch.empty_like(q)
    ops.encode_attention_tree(q, *two, bt, ints([prompt]), P.words_of(bits[None]).cuda(), out, nh, nkv, hd, *geo)
    ops.encode_kv_accept(*two, bt, ints([prompt]), torch.tensor([path + [-1] * 3], dtype=torch.int32).cuda(), tree, nkv, hd,
                         pages, 1, tpb)
    for o, node in zip(outs, path):
        assert P.rel(out[node].cpu(), o[0].cpu().double()) <= 2 * TOL
    assert torch.equal(attend(two, enter(two, [prompt + tree], at, at), at), last)
    where = torch.arange(prompt + len(path) + 1)
    blocks = bt[0].long()[where.cuda() // tpb]
    for c1, c2 in zip(one, two):
        assert torch.equal(c1[blocks, 0, where.cuda() % tpb], c2[blocks, 0, where.cuda() % tpb])


def _loop(ops, cache, state, stream=None):
    """Write of a tree of drafts, its check, the accepted path, and what then stands in the pages."""
    nh, nkv, hd, geo, tree = state["nh"], state["nkv"], state["hd"], state["geo"], state["tree"]
    kw = dict(stream=stream)
    ops.encode_rope_kv_write_q8(state["q"], state["k"], state["v"], state["qr"], nh, nkv, hd, state["pos"], state["cs"], *cache,
                                state["bt"], *geo, slots_i32=state["slots"], rows_per_table=tree, **kw)
    ops.encode_attention_tree(state["qr"], cache[0], cache[2], state["bt"], state["ctx"], state["masks"], state["out"], nh, nkv,
                              hd, *geo, kscale=cache[1], vscale=cache[3], **kw)
    ops.encode_kv_accept(cache[0], cache[2], state["bt"], state["ctx"], state["acc"], tree, nkv, hd, *geo[:3], kscale=cache[1],
                         vscale=cache[3], **kw)
    ops.encode_kv_read_q8(*cache, state["bt"], state["where"], state["ko"], state["vo"], nkv, hd, *geo,
                          rows_per_table=state["where"].numel() // state["bt"].shape[0], **kw)


def _loop_state(seed, tables=3, tree=21, ctx=1300):
    g = torch.Generator().manual_seed(seed)
    nh, nkv, hd, tpb = 6, 2, 64, 16
    pages = -(-(ctx + tree) // tpb)
    total, n = tables * pages, tables * tree
    bits = np.stack([_random_tree(g, tree) for _ in range(tables)])
    lens = torch.randint(ctx // 2, ctx, (tables,), generator=g)
    a = np.arange(ctx + tree)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    acc = torch.full((tables, 8), -1)
    for t in range(tables):
        path = np.flatnonzero(bits[t, tree - 1 - t])[:8]
        acc[t, :len(path)] = torch.from_numpy(path)
    where = (lens[:, None] + torch.arange(-4, 8)).reshape(-1)
    depth = torch.from_numpy(bits.sum(2)) - 1

    def ints(t):
        return t.to(torch.int32).cuda()

    def rows(heads):
        return torch.randn(n, heads, hd, generator=g).cuda()

    st = dict(nh=nh, nkv=nkv, hd=hd, tree=tree, geo=(total, 1, tpb, 0), bt=ints(torch.randperm(total, generator=g).view(tables, pages)),
              q=rows(nh), k=rows(nkv), v=rows(nkv), pos=ints((lens[:, None] + depth).reshape(-1)),
              slots=ints((lens[:, None] + torch.arange(tree)).reshape(-1)), ctx=ints(lens), masks=P.words_of(bits).cuda(),
              acc=ints(acc), where=ints(where), cs=torch.from_numpy(np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)).cuda())
    st["qr"], st["out"] = torch.zeros_like(st["q"]), torch.zeros_like(st["q"])
    st["ko"], st["vo"] = (torch.zeros(where.numel(), nkv * hd, device="cuda") for _ in range(2))
    return st, [c.cuda() for c in P.cache_q8(total, 1, nkv, tpb, hd, seed)]


_RESULTS = ("qr", "out", "ko", "vo")


def test_the_loop_in_one_graph(ops):
    """Write, check, acceptance and read captured together and replayed with new tokens each time: the eager calls' bits."""
    st, first = _loop_state(79)
    cap, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    cache = [c.clone() for c in first]
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=cap):
        _loop(ops, cache, st, cap)
    g = torch.Generator().manual_seed(83)
    for turn in range(4):
        for name in "qkv":
            st[name].copy_(torch.randn(st[name].shape, generator=g))
        eager = [c.clone() for c in first]
        _loop(ops, eager, st)
        torch.cuda.synchronize()
        want = [st[n].clone() for n in _RESULTS]
        for n in _RESULTS:
            st[n].zero_()
        for c, f in zip(cache, first):
            c.copy_(f)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(st[n], w) for n, w in zip(_RESULTS, want))
        assert all(torch.equal(a, b) for a, b in zip(cache, eager))


def test_loops_of_two_threads(ops):
    """Two threads with one context, each on a stream of its own."""
    import threading

    both = [_loop_state(s, ctx=c) for s, c in ((89, 1300), (97, 4200))]
    want = []
    for st, first in both:
        _loop(ops, [c.clone() for c in first], st)
        torch.cuda.synchronize()
        want.append([st[n].clone() for n in _RESULTS])
    wrong = []

    def work(st, first, expected):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(10):
                    for n in _RESULTS:
                        st[n].zero_()
                    cache = [c.clone() for c in first]
                    _loop(ops, cache, st, stream)
                    stream.synchronize()
                    if not all(torch.equal(st[n], w) for n, w in zip(_RESULTS, expected)):
                        wrong.append("results")
        except Exception as e:  # told below: a thread's own exception would be lost
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(*b, w)) for b, w in zip(both, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
