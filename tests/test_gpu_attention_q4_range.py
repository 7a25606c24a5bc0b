"""Attention over 4-bit pages where scores are as far below zero as f32 holds, and further.

With q the same in every dim and keys of positive elements the scores are -|q| sum(k) scale, apart by far more than the
exponential resolves: the row is the value of the largest one, whose weight is 1.  That position is the same for f32 sums
where the two largest scores are apart by more than the sums' error, some 2^-20 of them (asserted on the inputs).  The bar of the
values is that of test_gpu_attention_q4.py."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _paged as P
import _step as S

pytestmark = pytest.mark.gpu

TOL = 3e-6
GAP = 1e-5


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _pages(keys, values, tpb, g):
    """4-bit pages that hold keys and values [positions][nkv][hd], and the table [1][pages]."""
    n, nkv, hd = keys.shape
    pages = -(-n // tpb)
    bt = torch.randperm(pages + 2, generator=g)[None, :pages]
    cache = []
    for x in (keys, values):
        padded = torch.cat([x, torch.ones(pages * tpb - n, nkv, hd)]).view(pages, tpb, nkv, hd).transpose(1, 2)
        full = torch.ones(pages + 2, 1, nkv, tpb, hd)
        full[bt[0], 0] = padded
        cache += [torch.from_numpy(y) for y in S.quantise4(full.numpy())]
    return cache, bt


def _attend(ops, q, cache, bt, pos, ragged=False, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    kw.update(dict(row_starts_i32=_i32([0, rows])) if ragged else dict(rows_per_table=rows))
    ops.encode_attention_q4(q.cuda(), *[c.cuda() for c in cache], _i32(bt), _i32(pos), out, nh, nkv, hd, total, layers, tpb, 0, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _dense(q, cache, bt, pos, window=0, cap=0.0):
    """In 64 bits: outputs, and how far apart the two largest scores of a row and head are, over the largest one's size."""
    k, _, v, _ = S.as_f16_pages(cache)
    k, v = (x[bt[0], 0].flatten(0, 1).double() for x in (k, v))  # [positions][nkv][hd]
    rows, nh, hd = q.shape
    group = nh // k.shape[1]
    at = torch.arange(len(k))
    out, gap = torch.zeros(rows, nh, hd, dtype=torch.float64), math.inf
    for h in range(nh):
        s = q[:, h].double() @ k[:, h // group].T / math.sqrt(hd)
        if cap:
            s = torch.tanh(s / cap) * cap
        p = torch.as_tensor(pos)[:, None]
        s = torch.where((at <= p) & ((at > p - window) if window else (at >= 0)), s, -math.inf)
        out[:, h] = torch.softmax(s, -1) @ v[:, h // group]
        if not cap and s.shape[1] > 1:
            top = s.topk(2, -1).values
            gap = min(gap, float(((top[:, 0] - top[:, 1]) / top[:, 0].abs())[top[:, 0] < -1e30].clamp(max=1).min(dim=0).values)
                      if bool((top[:, 0] < -1e30).any()) else math.inf)
    return out, gap


def _far_below(g, ctx, nkv, hd, rows, nh, size):
    """Keys, values and queries: every head but the last (where there are several) has scores far below zero."""
    k, v = (torch.randn(ctx, nkv, hd, generator=g) for _ in range(2))
    q = -size * (1 + torch.rand(rows, nh, 1, generator=g)) * torch.ones(hd)
    if nh > 1:
        q[:, -1] = torch.randn(rows, hd, generator=g)
    return k.abs() + 0.1, v, q


# query heads and kv heads, rows: sets of up to 4 columns and of 16
SETS = [(1, 1, 1), (4, 1, 1), (2, 1, 2), (8, 1, 1), (6, 2, 5)]


@pytest.mark.parametrize("size", [1e34, 1e36])
@pytest.mark.parametrize("ctx", [1, 50, 600, 3000])  # one chunk, one unit, some units of one block, and split
@pytest.mark.parametrize("nh,nkv,rows", SETS)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_all_scores_far_below_zero(ops, hd, nh, nkv, rows, ctx, size):
    g = torch.Generator().manual_seed(hd + nh + ctx)
    k, v, q = _far_below(g, ctx, nkv, hd, rows, nh, size)
    cache, bt = _pages(k, v, 16, g)
    pos = [ctx - 1] + [int(p) for p in torch.randint(0, ctx, (rows - 1,), generator=g)]
    for window in (0, ctx // 3 + 1):
        ref, gap = _dense(q, cache, bt, pos, window)
        assert gap > GAP
        for ragged in (False, True):
            got = _attend(ops, q, cache, bt, pos, ragged, window=window)
            for r in range(rows):
                assert P.rel(got[r], ref[r]) <= TOL
    ref, _ = _dense(q, cache, bt, pos, cap=20.0)
    assert P.rel(_attend(ops, q, cache, bt, pos, soft_cap=20.0), ref) <= TOL


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("ragged", [False, True])
def test_all_scores_far_below_zero_of_many_rows(ops, hd, ragged):
    """Sets of 32 columns: 260 rows of 32/8 heads are 33 sets for each of 8 kv heads."""
    g = torch.Generator().manual_seed(hd)
    rows, ctx = 260, 400
    k, v, q = _far_below(g, ctx, 8, hd, rows, 32, 1e36)
    cache, bt = _pages(k, v, 16, g)
    pos = range(ctx - rows, ctx)
    ref, gap = _dense(q, cache, bt, list(pos))
    assert gap > GAP
    got = _attend(ops, q, cache, bt, pos, ragged)
    for h in range(32):
        assert P.rel(got[:, h], ref[:, h]) <= TOL


@pytest.mark.parametrize("ctx", [60, 700, 3000, 9000])
@pytest.mark.parametrize("nh,per", [(1, 4), (4, 1), (4, 4)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("of", ["q . k", "its exponent"])
def test_scores_of_minus_infinity(ops, of, hd, nh, per, ctx):
    """Scores past f32 weigh nothing beside others, and are NaN where a row has no others: rows whose splits see nothing,
    nothing but -inf, or both."""
    g = torch.Generator().manual_seed(hd + ctx)
    k, v, q = _far_below(g, ctx, 1, hd, per, nh, 1e38)
    kw = {}
    if of == "q . k":
        q[:] = -3e38
    elif of == "its exponent":  # scores of -3e38, which log2(e) takes past f32
        k[:], q[:], kw["attn_scale"] = 1.0, -3e38 / hd, 1.0
    some = range(ctx * 3 // 4, ctx * 3 // 4 + 5)
    k[some] = 0.0  # the score 0
    cache, bt = _pages(k, v, 16, g)
    pos = [ctx - 1, ctx // 3, ctx // 10, some[2]][:per]
    held = S.as_f16_pages(cache)[2][bt[0], 0].flatten(0, 1)[:, 0].double()
    for ragged in (False, True):
        got = _attend(ops, q, cache, bt, pos, ragged, **kw)
        for r, p in enumerate(pos):
            seen = [x for x in some if x <= p]
            if seen:
                assert P.rel(got[r], held[seen].mean(0).expand(nh, hd)) <= TOL
            else:
                assert bool(torch.isnan(got[r]).all())
    assert bool(torch.isnan(_attend(ops, -q, cache, bt, pos, **kw)).all())  # above f32
    q[:, 0] = -math.inf  # of zero keys NaN
    got = _attend(ops, q, cache, bt, pos, **kw)
    assert bool(torch.isnan(got[:, 0]).all())


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("sign", [-1, 1])
def test_exponents_past_f32_of_trees_over_f16_pages(ops, hd, sign):
    """Scores of 3e38 are f32 numbers, and log2(e) times that is none: NaN, not the zeros of a row that sees nothing."""
    nh, nkv, tpb, ctx, tree = 4, 2, 16, 700, 5
    pages = -(-(ctx + tree) // tpb)
    k = torch.ones(pages, 1, tpb, nkv, hd, dtype=torch.float16)
    q = torch.full((1, tree, nh, hd), sign * 3e38 / hd)
    masks = P.words_of(np.tril(np.ones((1, tree, tree), bool)))
    out = torch.zeros(q.shape, device="cuda")
    ops.encode_attention_tree(q.cuda(), k.cuda(), k.cuda(), _i32(np.arange(pages)[None]), _i32([ctx]), masks.cuda(), out, nh, nkv, hd,
                              pages, 1, tpb, 0, attn_scale=1.0)
    torch.cuda.synchronize()
    assert bool(torch.isnan(out).all())
