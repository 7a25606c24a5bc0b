"""Attention over 4-bit pages (attention_paged.hip) against plain 64-bit results over the f16 values that the codes stand
for.

The bar, 3e-6 in the 2-norm, is that of the f16 pages' trees: a score of size |s| <= 10 from f32 sums is off by a few
2^-24 |s| (6e-7 each), q as two f16 parts by 2^-23 of an element, the exponentials by 2^-22, weights as two f16 parts by
2^-22, and the sums of weights and values by a few 2^-24; the values themselves are exact."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _paged as P
import _step as S

pytestmark = pytest.mark.gpu

TOL = 3e-6


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


def _attend(ops, q, cache, bt, pos, layer=0, per=1, starts=None, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    ops.encode_attention_q4(q.cuda(), *[c.cuda() for c in cache], _i32(bt), _i32(pos), out, nh, nkv, hd, total, layers, tpb,
                            layer, rows_per_table=per, row_starts_i32=None if starts is None else _i32(starts), **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _check(got, ref, tol=TOL):
    """Rows that are NaN in ref as a whole are left as they were; the others near, NaN where NaN."""
    there = ~torch.isnan(ref).flatten(1).all(1)
    assert bool((got[~there] == 7.0).all())
    assert P.rel(got[there], ref[there]) <= tol


def _table(g, tables, per, spare=2):
    total = tables * per + spare
    return torch.randperm(total, generator=g)[:tables * per].view(tables, per), total


# tables, rows of each, query heads, kv heads, head_dim, tokens per page, positions, window, cap
CASES = [(1, 1, 1, 1, 64, 16, 1, 0, 0.0), (1, 1, 14, 2, 64, 16, 300, 0, 0.0), (3, 1, 32, 8, 128, 16, 700, 0, 0.0),
         (2, 1, 4, 1, 256, 16, 1300, 512, 50.0), (1, 1, 8, 8, 128, 7, 2000, 0, 0.0), (5, 1, 9, 3, 64, 5, 90, 33, 0.0),
         (1, 37, 6, 2, 64, 16, 37, 0, 0.0), (2, 70, 4, 2, 128, 16, 150, 0, 30.0), (1, 20, 3, 1, 256, 3, 61, 17, 0.0),
         (1, 130, 40, 1, 128, 32, 140, 0, 0.0), (1, 1, 64, 1, 64, 16, 65, 0, 0.0), (1, 3, 2, 1, 256, 1, 515, 0, 0.0)]


@pytest.mark.parametrize("tables,per,nh,nkv,hd,tpb,ctx,window,cap", CASES)
def test_against_plain(ops, tables, per, nh, nkv, hd, tpb, ctx, window, cap):
    g = torch.Generator().manual_seed(ctx + hd)
    bt, total = _table(g, tables, -(-ctx // tpb))
    cache = S.cache_q4(total, 2, nkv, tpb, hd, 5)
    lens = [max(1, ctx - 29 * t) for t in range(tables)]
    pos = torch.tensor([max(n - per + i, -1) for n in lens for i in range(per)])
    q = 1.5 * torch.randn(tables * per, nh, hd, generator=g)
    ref = S.attention(q, cache, bt, pos, 1, range(0, tables * per + 1, per), window=window, cap=cap)
    _check(_attend(ops, q, cache, bt, pos, 1, per, window=window, soft_cap=cap), ref)


@pytest.mark.parametrize("scale", [0.05, 1.0])
def test_scale(ops, scale):
    g = torch.Generator().manual_seed(2)
    bt, total = _table(g, 1, 20)
    cache = S.cache_q4(total, 1, 2, 16, 64, 5)
    q = 0.3 * torch.randn(1, 4, 64, generator=g)
    ref = S.attention(q, cache, bt, torch.tensor([311]), 0, [0, 1], scale=scale)
    _check(_attend(ops, q, cache, bt, [311], attn_scale=scale), ref)


# rows of each table: decoding beside prompts, tables without rows, one alone
RAGGED = [[1], [0, 1], [1, 1, 1, 1, 1], [40, 1, 0, 3, 1], [0, 0, 65, 0], [1, 130, 1, 1, 17, 0, 1], [3] * 40, [1] * 300]


@pytest.mark.parametrize("new", RAGGED)
@pytest.mark.parametrize("nh,nkv,hd,window", [(4, 2, 64, 0), (8, 1, 128, 50), (5, 5, 256, 0)])
def test_rows_of_any_number(ops, new, nh, nkv, hd, window):
    g = torch.Generator().manual_seed(len(new))
    tables, tpb = len(new), 16
    ctx = [int(torch.randint(max(n, 1), max(n, 1) + 300, (1,), generator=g)) for n in new]
    if tables > 100:
        ctx = [min(c, 40) for c in ctx]
    bt, total = _table(g, tables, -(-max(ctx) // tpb))
    cache = S.cache_q4(total, 1, nkv, tpb, hd, 5)
    starts = np.concatenate([[0], np.cumsum(new)])
    rows = int(starts[-1]) + 4  # padding behind the last
    pos = torch.full((rows,), -1)
    for t in range(tables):
        pos[starts[t]:starts[t + 1]] = torch.arange(ctx[t] - new[t], ctx[t])
    pos[-1] = 3  # a row of no table is left as it was whatever its position
    q = 1.5 * torch.randn(rows, nh, hd, generator=g)
    ref = S.attention(q, cache, bt, pos, 0, starts, window=window)
    _check(_attend(ops, q, cache, bt, pos, starts=starts, window=window), ref)


def test_row_starts_as_uniform_rows(ops):
    """The same rows by row_starts and by rows_per_table."""
    g = torch.Generator().manual_seed(4)
    bt, total = _table(g, 6, 30)
    cache = S.cache_q4(total, 1, 2, 16, 128, 5)
    for per in (1, 5, 33):
        pos = torch.randint(0, 480, (6 * per,), generator=g)
        pos[2] = -1
        q = torch.randn(6 * per, 8, 128, generator=g)
        ref = S.attention(q, cache, bt, pos, 0, range(0, 6 * per + 1, per))
        _check(_attend(ops, q, cache, bt, pos, per=per), ref)
        _check(_attend(ops, q, cache, bt, pos, starts=range(0, 6 * per + 1, per)), ref)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ctx", [40, 1100])
def test_missing_pages_are_zeros(ops, hd, ctx):
    g = torch.Generator().manual_seed(hd)
    bt, total = _table(g, 2, -(-ctx // 16))
    cache = S.cache_q4(total, 1, 2, 16, hd, 5)
    cache[1][:], cache[3][:] = torch.nan_to_num(cache[1]), torch.nan_to_num(cache[3])
    bt[0, 1], bt[1, :] = -1, total
    pos = torch.tensor([ctx - 1, ctx - 1])
    q = torch.randn(2, 6, hd, generator=g)
    ref = S.attention(q, cache, bt, pos, 0, [0, 1, 2])
    got = _attend(ops, q, cache, bt, pos)
    assert P.rel(got[:1], ref[:1]) <= TOL and bool((got[1] == 0).all())
    q[0, 1, 3], q[1, 2, 5] = math.inf, math.nan  # of zeros these make NaN
    got = _attend(ops, q, cache, bt, pos)
    assert bool(torch.isnan(got[0, 1]).all()) and bool(torch.isnan(got[1, 2]).all())
    assert bool((got[1, 3:] == 0).all()) and P.rel(got[0, 2:], ref[0, 2:]) <= TOL


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ctx", [70, 1500])
@pytest.mark.parametrize("where", ["k", "v"])
def test_nan_groups_reach_who_sees_them(ops, hd, ctx, where):
    """A group of scale NaN makes NaN of a row's dims that it reaches, and nothing of rows that do not see it, which
    share its tile; nor does a NaN behind every row's position."""
    g = torch.Generator().manual_seed(hd)
    bt, total = _table(g, 1, -(-(ctx + 3) // 16))
    cache = S.cache_q4(total, 1, 1, 16, hd, 5)
    per = 20
    pos = torch.arange(ctx - per, ctx)
    q = torch.randn(per, 3, hd, generator=g)
    clean = S.attention(q, cache, bt, pos, 0, [0, per])
    for p in (ctx - 5, ctx + 1):
        cache[1 if where == "k" else 3][int(bt[0, p // 16]), 0, :, p % 16, hd // 32 - 1] = math.nan
    got = _attend(ops, q, cache, bt, pos, per=per)
    assert P.rel(got[:per - 5], clean[:per - 5]) <= TOL
    seen = got[per - 5:]
    if where == "k":
        assert bool(torch.isnan(seen).all())
    else:
        assert bool(torch.isnan(seen[..., hd - 32:]).all()) and P.rel(seen[..., :hd - 32], clean[per - 5:, :, :hd - 32]) <= TOL


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_large_and_small_numbers(ops, hd):
    """Keys and values near f16's ends and among its subnormal numbers, and q that makes up for them."""
    g = torch.Generator().manual_seed(hd)
    bt, total = _table(g, 1, 50)
    for ksize, vsize in ((2e4, 2e4), (1e-6, 1e-6), (1.0, 6e4), (3e-3, 1.0)):
        x = [torch.randn(total, 1, 2, 16, hd, generator=g) * n / 4 for n in (ksize, vsize)]
        cache = []
        for y in x:
            cache += [torch.from_numpy(z) for z in S.quantise4(y.numpy())]
        q = torch.randn(1, 4, hd, generator=g) * 4 / ksize
        ref = S.attention(q, cache, bt, torch.tensor([799]), 0, [0, 1])
        _check(_attend(ops, q, cache, bt, [799]), ref)


def test_scores_far_apart(ops):
    """One score far above the others, at the beginning and at the end of a long context."""
    g = torch.Generator().manual_seed(6)
    bt, total = _table(g, 1, 200)
    for at in (3, 3100):
        cache = S.cache_q4(total, 1, 1, 16, 128, 5)
        q = torch.randn(1, 2, 128, generator=g)
        k = 30 * q[0, 0]
        c, s = S.quantise4(k.numpy())
        cache[0][int(bt[0, at // 16]), 0, 0, at % 16], cache[1][int(bt[0, at // 16]), 0, 0, at % 16] = (
            torch.from_numpy(c), torch.from_numpy(s))
        ref = S.attention(q, cache, bt, torch.tensor([3199]), 0, [0, 1])
        _check(_attend(ops, q, cache, bt, [3199]), ref)


def test_the_same_bits_every_time(ops):
    g = torch.Generator().manual_seed(8)
    bt, total = _table(g, 3, 120)
    cache = S.cache_q4(total, 1, 2, 16, 128, 5)
    pos = torch.tensor([1900, 1000, 77])
    q = torch.randn(3, 8, 128, generator=g)
    first = _attend(ops, q, cache, bt, pos)
    for _ in range(5):
        assert torch.equal(_attend(ops, q, cache, bt, pos), first)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("ctx", [70, 1500, 6000])
@pytest.mark.parametrize("per,nh,ragged", [(1, 1, False), (1, 4, False), (2, 2, False), (4, 1, False), (1, 4, True)])
def test_nan_groups_of_few_columns(ops, hd, ctx, per, nh, ragged):
    """As above for sets of up to 4 columns: NaN where it is seen, in K of all dims, in V of its own 32, and none from
    positions behind the row's own or before its window."""
    g = torch.Generator().manual_seed(hd + ctx)
    bt, total = _table(g, 1, -(-(ctx + 3) // 16))
    cache = S.cache_q4(total, 1, 1, 16, hd, 5)
    window = ctx // 2
    pos = torch.arange(ctx - per, ctx)
    q = torch.randn(per, nh, hd, generator=g)
    clean = S.attention(q, cache, bt, pos, 0, [0, per], window=window)
    for i in (1, 3):
        for p in (0, ctx - window - per - 1, ctx, ctx + 2):
            cache[i][int(bt[0, p // 16]), 0, :, p % 16] = math.nan
    kw = dict(starts=[0, per]) if ragged else dict(per=per)
    _check(_attend(ops, q, cache, bt, pos, window=window, **kw), clean)
    at = ctx - window // 2
    cache[3][int(bt[0, at // 16]), 0, :, at % 16, 1] = math.nan
    got = _attend(ops, q, cache, bt, pos, window=window, **kw)
    rest = torch.arange(hd) // 32 != 1
    assert bool(torch.isnan(got[..., ~rest]).all()) and P.rel(got[..., rest], clean[..., rest]) <= TOL
    cache[1][int(bt[0, at // 16]), 0, :, at % 16, 0] = math.nan
    assert bool(torch.isnan(_attend(ops, q, cache, bt, pos, window=window, **kw)).all())


def test_queries_of_any_size(ops):
    """Queries whose scores are far past 1, up to what f32 holds, and rows with an infinity or a NaN beside others."""
    g = torch.Generator().manual_seed(3)
    bt, total = _table(g, 4, 80)
    cache = S.cache_q4(total, 1, 1, 16, 128, 5)
    pos = torch.tensor([1200, 900, 40, 1100])
    q = torch.randn(4, 4, 128, generator=g)
    q[0] *= 1e-30
    q[1, 0] *= 3e4
    q[2, 1, 7], q[3, 2, 100] = math.inf, math.nan
    ref = S.attention(q, cache, bt, pos, 0, range(5))
    got = _attend(ops, q, cache, bt, pos)
    bad = torch.zeros(4, 4, dtype=torch.bool)
    bad[2, 1] = bad[3, 2] = True
    assert bool(torch.isnan(got[bad]).all())
    # the scores of row 1, head 0 reach 8e4, off by 5e-3 each, and the largest stands 370 above the next: its weight is 1
    assert P.rel(got[~bad], ref[~bad]) <= TOL


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("per,nh", [(2, 2), (3, 6), (20, 4)])
@pytest.mark.parametrize("tiny_first", [True, False])
def test_tiny_pages_beside_others(ops, hd, per, nh, tiny_first):
    """Pages of subnormal f16 values and of ordinary ones in one context; row 0 sees the tiny ones alone and has queries
    that make up for them, the last row sees all, and the others what their window leaves."""
    g = torch.Generator().manual_seed(hd + per)
    bt, total = _table(g, 1, 96)
    size = torch.ones(96)
    size[slice(0, 48) if tiny_first else slice(48, 96)] = 1e-6
    x = [torch.randn(total, 1, 1, 16, hd, generator=g) for _ in range(2)]
    cache = []
    for y in x:
        y[bt[0]] *= size.view(-1, 1, 1, 1, 1)
        cache += [torch.from_numpy(z) for z in S.quantise4(y.numpy())]
    pos = torch.randint(0, 1536, (per,), generator=g)
    pos[0], pos[-1], window = (700, 1535, 0) if tiny_first else (1535, 1530, 700)
    q = torch.randn(per, nh, hd, generator=g)
    q[0] *= 1e6
    ref = S.attention(q, cache, bt, pos, 0, [0, per], window=window)
    for kw in (dict(per=per), dict(starts=[0, per])):
        got = _attend(ops, q, cache, bt, pos, window=window, **kw)
        for r in range(per):
            assert P.rel(got[r], ref[r]) <= TOL


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("end", [1, 20, 31])
def test_tiny_values_among_others_of_a_chunk(ops, hd, end):
    """A row that sees subnormal f16 values alone, in 64 positions of which other rows see ordinary ones: products of
    the matrix unit keep 2^-24 of 2^-14 each, so the mean's error is 2^-38 for each of the two sums of 32 positions."""
    g = torch.Generator().manual_seed(hd + end)
    bt, total = _table(g, 1, 4)
    x = [torch.randn(total, 1, 2, 16, hd, generator=g) for _ in range(2)]
    x[1][bt[0, :2]] *= 2e-6
    cache = []
    for y in x:
        cache += [torch.from_numpy(z) for z in S.quantise4(y.numpy())]
    pos = torch.tensor([end - 1, 63, 40])
    q = torch.randn(3, 6, hd, generator=g)
    ref = S.attention(q, cache, bt, pos, 0, [0, 3])
    got = _attend(ops, q, cache, bt, pos, per=3)
    assert float((got[0] - ref[0]).abs().max()) <= 2.0 ** -37
    _check(got[1:], ref[1:])
