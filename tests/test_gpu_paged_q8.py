"""The 8-bit paged cache (kv_cache.hip) and attention over shared pages
(attention_paged.hip) against plain 64-bit results.

Codes, scales, rotated q and the values read back are defined operation by operation in
f32, so they are compared for equality.  Attention's bar, 3e-6 in the 2-norm: a score of
size |s| <= 10 from f32 sums is off by a few 2^-24 |s| (6e-7 each), q held to 2^-23 of
its head's largest moves it by 2^-23 * 4.5 * 0.29 * sqrt(hd) / sqrt(hd) = 1.6e-7 (rms),
the exponentials by 2^-22, and the sums of weights and values by a few 2^-24."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu

TOL = 3e-6


def _table(g, tables, per, spare=2):
    total = tables * per + spare
    return torch.randperm(total, generator=g)[:tables * per].view(tables, per), total


def _cos_sin(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def _expect_written(cache, bt, slots, per, layer, tpb, vectors):
    """Codes and scales that a write leaves, from those before; vectors [rows][nkv][hd] f32."""
    c, s = P.quantise(vectors)
    code, scale = (x.clone() for x in cache)
    for r, slot in enumerate(slots):
        if slot < 0 or slot // tpb >= bt.shape[1]:
            continue
        blk = int(bt[r // per, slot // tpb])
        if 0 <= blk < code.shape[0]:
            code[blk, layer, :, slot % tpb] = torch.from_numpy(c[r])
            scale[blk, layer, :, slot % tpb] = torch.from_numpy(s[r])
    return code, scale


def _same(a, b):
    """Equal, NaN where NaN."""
    return torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


# tables, rows of each, query heads, kv heads, head_dim, tokens per page, positions before: single tokens, prompts, odd counts
WRITES = [(1, 1, 9, 3, 64, 16, 0), (5, 1, 14, 2, 64, 16, 33), (2, 37, 8, 8, 128, 5, 11), (1, 130, 4, 1, 256, 16, 3),
          (3, 19, 5, 5, 128, 1, 2)]


@pytest.mark.parametrize("tables,per,nh,nkv,hd,tpb,past", WRITES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("drafted", [False, True])
def test_rope_write_and_read(ops, tables, per, nh, nkv, hd, tpb, past, interleaved, drafted):
    g = torch.Generator().manual_seed(hd + per)
    rows, room = tables * per, past + per
    bt, total = _table(g, tables, -(-room // tpb))
    q, k, v = (torch.randn(rows, n, hd, generator=g) for n in (nh, nkv, nkv))
    k = k * torch.exp(4 * torch.randn(rows, nkv, 1, generator=g))
    slots = past + torch.arange(per).repeat(tables)
    pos = torch.randint(0, room, (rows,), generator=g) if drafted else slots.clone()
    if per > 2:
        pos[1] = -1  # padding
    cs = _cos_sin(room - 1 if past else room, hd)  # the last position is past the table: clamped
    cache = P.cache_q8(total, 2, nkv, tpb, hd, 7)
    dev = [x.cuda() for x in cache]
    dq, dk, dv, dcs = q.cuda(), k.cuda(), v.cuda(), torch.from_numpy(cs).cuda()
    out = torch.full_like(dq, 7.0)
    btd, posd = bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda()
    ops.set_rope_interleaved(interleaved)
    try:
        ops.encode_rope_kv_write_q8(dq, dk, dv, out, nh, nkv, hd, posd, dcs, *dev, btd, total, 2, tpb, 1,
                                    slots_i32=slots.to(torch.int32).cuda() if drafted else None, rows_per_table=per)
    finally:
        ops.set_rope_interleaved(False)
    at = cs[np.clip(pos.numpy(), 0, cs.shape[0] - 1)]
    there = pos >= 0
    want_q = torch.from_numpy(P.rope(q.numpy(), at, interleaved))
    assert torch.equal(out.cpu()[there], want_q[there]) and bool((out.cpu()[~there] == 7.0).all())
    assert torch.equal(dk.cpu(), k) and torch.equal(dq.cpu(), q)
    went = torch.where(there, slots, -1).tolist()
    kw = _expect_written(cache[:2], bt, went, per, 1, tpb, P.rope(k.numpy(), at, interleaved))
    vw = _expect_written(cache[2:], bt, went, per, 1, tpb, v.numpy())
    for got, want in zip(dev, (*kw, *vw)):
        assert torch.equal(got.cpu(), want)
    # read back: the f32 product, rounded once more
    at = torch.where(there, slots, -1).to(torch.int32).cuda()
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        ko, vo = (torch.full((rows, nkv * hd), 5.0, dtype=dt, device="cuda") for _ in range(2))
        ops.encode_kv_read_q8(*dev, btd, at, ko, vo, nkv, hd, total, 2, tpb, 1, rows_per_table=per)
        for got, (c, s) in ((ko, kw), (vo, vw)):
            got = got.cpu().view(rows, nkv, hd)
            for r in range(rows):
                if not there[r]:
                    assert bool((got[r] == 5.0).all())
                    continue
                blk, sl = int(bt[r // per, int(slots[r]) // tpb]), int(slots[r]) % tpb
                want = (c[blk, 1, :, sl].float() * s[blk, 1, :, sl][:, None]).to(dt)
                assert torch.equal(got[r], want)


def test_rotated_q_in_place(ops):
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(6, n, 64, generator=g).cuda() for n in (4, 2, 2))
    dev = [x.cuda() for x in P.cache_q8(3, 1, 2, 4, 64, 1)]
    bt, pos = torch.tensor([[1, 0]], dtype=torch.int32).cuda(), torch.arange(6, dtype=torch.int32).cuda()
    cs, out = torch.from_numpy(_cos_sin(6, 64)).cuda(), torch.empty_like(q)
    for dst in (out, q):
        ops.encode_rope_kv_write_q8(q, k, v, dst, 4, 2, 64, pos, cs, *dev, bt, 3, 1, 4, 0, rows_per_table=6)
    assert torch.equal(out, q)


def test_vectors_at_the_ends_of_f32(ops):
    """Zeros, signed zeros, numbers below the smallest normal, the largest number, a lone outlier, infinities and NaN."""
    hd, tpb = 64, 16
    g = torch.Generator().manual_seed(3)
    x = torch.randn(16, 1, hd, generator=g)
    x[0] = 0.0
    x[1] = -0.0
    x[2] *= 1e-38
    x[3] *= 1e-42
    x[4, 0, 5] = 3.4028234663852886e38
    x[5] *= 1e30
    x[6, 0, 9] = math.inf
    x[7, 0, 63] = -math.inf
    x[8, 0, 0] = math.nan
    x[9] = 1.0
    x[10] = 0.5 * 127 / 127
    x[11] *= 127 * 1.1754943508222875e-38 * torch.ones(hd)
    x[12, 0] = torch.arange(hd) - 31.5  # halves: codes at the middle go to the even one
    x[13, 0] = torch.linspace(-127, 127, hd)
    cache = P.cache_q8(2, 1, 1, tpb, hd, 2)
    dev = [t.cuda() for t in cache]
    bt, pos = torch.tensor([[1]]), torch.arange(16)
    ops.encode_kv_write_q8(x.cuda(), x.flip(0).contiguous().cuda(), 1, hd, pos.to(torch.int32).cuda(), *dev,
                           bt.to(torch.int32).cuda(), 2, 1, tpb, 0, rows_per_table=16)
    want = (*_expect_written(cache[:2], bt, pos.tolist(), 16, 0, tpb, x.numpy()),
            *_expect_written(cache[2:], bt, pos.tolist(), 16, 0, tpb, x.flip(0).numpy()))
    for got, w in zip(dev, want):
        assert _same(got.cpu(), w)
    ko, vo = (torch.empty(16, hd, device="cuda") for _ in range(2))
    ops.encode_kv_read_q8(*dev, bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda(), ko, vo, 1, hd, 2, 1, tpb, 0,
                          rows_per_table=16)
    ko = ko.cpu()
    assert bool(torch.isnan(ko[6:9]).all()) and bool((ko[:4] == 0).all())  # 2 and 3: max / 127 < 2^-126
    fine = [i for i in range(16) if i not in (2, 3, 6, 7, 8)]
    err = (ko[fine] - x[fine, 0]).abs() / x[fine, 0].abs().amax(-1, keepdim=True).clamp(min=1e-45)
    # half a step, 1 / 254, and the roundings of the scale (127 times 2^-24), the quotient and the product
    assert float(err.max()) <= 1 / 254 + 130 * 2.0 ** -24


def test_missing_pages_and_slots_past_the_table(ops):
    hd, tpb, nkv = 128, 4, 2
    g = torch.Generator().manual_seed(5)
    cache = P.cache_q8(6, 2, nkv, tpb, hd, 4)
    dev = [t.cuda() for t in cache]
    bt = torch.tensor([[2, 6, 0], [-1, 5, 2**31 - 1]])  # 6, -1 and 2^31 - 1 are no pages
    pos = torch.tensor([0, 3, 4, 7, 9, 11, 12, 2**31 - 1, 0, 1, 5, 6, 8, 9, -1, -2**31])
    k, v = (torch.randn(16, nkv, hd, generator=g) for _ in range(2))
    btd, posd = bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda()
    ops.encode_kv_write_q8(k.cuda(), v.cuda(), nkv, hd, posd, *dev, btd, 6, 2, tpb, 0, rows_per_table=8)
    want = (*_expect_written(cache[:2], bt, pos.tolist(), 8, 0, tpb, k.numpy()),
            *_expect_written(cache[2:], bt, pos.tolist(), 8, 0, tpb, v.numpy()))
    for got, w in zip(dev, want):
        assert torch.equal(got.cpu(), w)
    ko, vo = (torch.full((16, nkv, hd), 3.0, device="cuda") for _ in range(2))
    ops.encode_kv_read_q8(*dev, btd, posd, ko, vo, nkv, hd, 6, 2, tpb, 0, rows_per_table=8)
    for r, p in enumerate(pos.tolist()):
        if p < 0:
            assert bool((ko[r] == 3.0).all()) and bool((vo[r] == 3.0).all())
            continue
        blk = int(bt[r // 8, p // tpb]) if p // tpb < 3 else -1
        for got, c, s in ((ko, want[0], want[1]), (vo, want[2], want[3])):
            w = c[blk, 0, :, p % tpb].float() * s[blk, 0, :, p % tpb][:, None] if 0 <= blk < 6 else torch.zeros(nkv, hd)
            assert torch.equal(got[r].cpu(), w)


# ---- attention ---------------------------------------------------------------------


def _attention(ops, q, cache, bt, pos, layer, per, stream=None, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    ops.encode_attention_q8(q.cuda(), *[c.cuda() for c in cache], bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda(), out,
                            nh, nkv, hd, total, layers, tpb, layer, rows_per_table=per, stream=stream, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _check(got, ref, tol=TOL):
    none = torch.isnan(ref).all(-1).all(-1)
    assert bool((got[none] == 7.0).all())
    if bool((~none).any()):
        assert P.rel(got[~none], ref[~none]) <= tol


# sessions, query heads, kv heads, head_dim, tokens per page, longest context: every length from one token on
@pytest.mark.parametrize("tables,nh,nkv,hd,tpb,ctx", [
    (7, 9, 3, 64, 16, 7), (3, 14, 2, 64, 16, 701), (5, 32, 8, 128, 16, 300), (2, 4, 1, 256, 7, 513), (1, 7, 7, 128, 1, 65),
    (4, 20, 1, 64, 32, 260), (70, 2, 2, 128, 16, 40), (1, 3, 1, 256, 64, 2100), (2, 8, 2, 128, 16, 4500),
    (300, 1, 1, 64, 3, 9)])
@pytest.mark.parametrize("kw", [{}, dict(window=33), dict(soft_cap=5.0, attn_scale=0.2)])
def test_last_token_of_every_session(ops, tables, nh, nkv, hd, tpb, ctx, kw):
    g = torch.Generator().manual_seed(ctx)
    bt, total = _table(g, tables, -(-ctx // tpb))
    cache = P.cache_q8(total, 2, nkv, tpb, hd, ctx)
    q = torch.randn(tables, nh, hd, generator=g) * 1.5
    pos = torch.randint(0, ctx, (tables,), generator=g)
    pos[0] = ctx - 1
    if tables > 2:
        pos[1], pos[2] = 0, -1
    ref = P.causal(q, *cache, bt, pos, 1, 1, kw.get("attn_scale"), kw.get("soft_cap", 0.0), kw.get("window", 0))
    _check(_attention(ops, q, cache, bt, pos, 1, 1, **kw), ref)


# sessions, rows of each, positions before them, heads, kv heads, head_dim, page: prompts whole, in parts and padded
@pytest.mark.parametrize("tables,per,past,nh,nkv,hd,tpb", [
    (1, 33, 0, 14, 2, 64, 16), (2, 50, 70, 8, 8, 128, 5), (1, 70, 200, 5, 1, 256, 16), (3, 17, 1, 6, 3, 128, 16),
    (1, 300, 0, 2, 2, 64, 32), (2, 5, 900, 16, 1, 64, 16), (1, 130, 30, 33, 1, 64, 16)])
@pytest.mark.parametrize("kw", [{}, dict(window=40), dict(soft_cap=5.0)])
def test_prompts(ops, tables, per, past, nh, nkv, hd, tpb, kw):
    g = torch.Generator().manual_seed(per + past)
    n = past + per
    bt, total = _table(g, tables, -(-n // tpb))
    cache = P.cache_q8(total, 1, nkv, tpb, hd, per)
    q = torch.randn(tables * per, nh, hd, generator=g) * 1.5
    pos = (past + torch.arange(per)).repeat(tables).view(tables, per)
    for t in range(1, tables):  # shorter ones padded in front or behind
        pos[t] = torch.where(torch.arange(per) < per // 3, -1, pos[t]) if t == 1 else \
            torch.where(torch.arange(per) > per // 2, -1, pos[t])
    pos = pos.reshape(-1)
    ref = P.causal(q, *cache, bt, pos, 0, per, None, kw.get("soft_cap", 0.0), kw.get("window", 0))
    _check(_attention(ops, q, cache, bt, pos, 0, per, **kw), ref)


# enough sets of 32 columns for the kernel to take them so (tables * kv heads * ceil(rows * heads / kv heads / 32) >= 256),
# whole ones and short ones, with more sets than are planned (512) and fewer
@pytest.mark.parametrize("tables,per,past,nh,nkv,hd,tpb", [
    (8, 21, 90, 16, 8, 64, 16), (5, 65, 7, 24, 8, 128, 16), (2, 160, 30, 32, 8, 64, 7), (1, 700, 0, 12, 3, 64, 16),
    (64, 9, 50, 8, 2, 128, 32)])
@pytest.mark.parametrize("kw", [{}, dict(window=45), dict(soft_cap=5.0)])
def test_many_columns(ops, tables, per, past, nh, nkv, hd, tpb, kw):
    g = torch.Generator().manual_seed(per + past)
    n = past + per
    bt, total = _table(g, tables, -(-n // tpb))
    bt[-1, 1] = total  # a missing page
    cache = P.cache_q8(total, 1, nkv, tpb, hd, per)
    q = torch.randn(tables * per, nh, hd, generator=g) * 1.5
    pos = (past + torch.arange(per)).repeat(tables)
    pos[per // 2] = -1
    got = _attention(ops, q, cache, bt, pos, 0, per, **kw)
    some = torch.randperm(tables * per, generator=g)[:90]
    some = torch.unique(torch.cat([some, torch.tensor([0, per // 2, tables * per - 1])]))
    ref = torch.cat([P.causal(q[r:r + 1], *cache, bt[r // per:r // per + 1], pos[r:r + 1], 0, 1, None, kw.get("soft_cap", 0.0),
                              kw.get("window", 0)) for r in some.tolist()])
    _check(got[some], ref)


def test_more_sets_than_a_grid_dimension_holds(ops):
    g = torch.Generator().manual_seed(3)
    tables, hd, tpb = 33000, 64, 16
    cache = P.cache_q8(50, 1, 1, tpb, hd, 8)
    bt = torch.randint(0, 50, (tables, 1), generator=g)
    pos = torch.randint(-1, tpb, (tables,), generator=g)
    q = torch.randn(tables, 1, hd, generator=g)
    got = _attention(ops, q, cache, bt, pos, 0, 1)
    some = torch.cat([torch.arange(20), torch.arange(tables - 20, tables), torch.randperm(tables, generator=g)[:60]])
    _check(got[some], P.causal(q[some], *cache, bt[some], pos[some], 0, 1))


def test_rows_of_a_table_in_any_order(ops):
    """Positions that jump, repeat, pass the table and are missing, with missing pages among the table's."""
    g = torch.Generator().manual_seed(11)
    bt, total = _table(g, 3, 21)
    bt[0, 3], bt[1, 0], bt[2, 20] = total, -1, total + 7
    cache = P.cache_q8(total, 1, 2, 4, 64, 9)
    q = torch.randn(3 * 40, 6, 64, generator=g)
    pos = torch.randint(-1, 21 * 4, (120,), generator=g)
    pos[3], pos[50], pos[119] = 21 * 4, 10**9, 2**31 - 1
    for window in (0, 9, 2**30):
        ref = P.causal(q, *cache, bt, pos, 0, 40, window=window)
        _check(_attention(ops, q, cache, bt, pos, 0, 40, window=window), ref)


def test_what_is_not_attended_to_never_arrives(ops):
    """NaN scales outside a row's positions leave it as it is; inside they reach exactly the rows that see them, and a
    q vector with an infinity or a NaN reaches exactly its own head."""
    g = torch.Generator().manual_seed(13)
    hd, nh, nkv, tpb, per, past = 64, 4, 2, 16, 24, 100
    bt, total = _table(g, 1, 8)
    cache = P.cache_q8(total, 1, nkv, tpb, hd, 5)
    q = torch.randn(per, nh, hd, generator=g)
    pos = past + torch.arange(per)
    clean = P.causal(q, *cache, bt, pos, 0, per, window=30)
    for p in (past + 10, 60):  # one that the rows from the tenth on see, one before the windows
        cache[1][int(bt[0, p // tpb]), 0, 1, p % tpb] = math.nan
    cache[3][int(bt[0, 127 // tpb]), 0, :, 127 % tpb] = math.nan  # behind every row
    q[3, 1, 7], q[5, 0, 0] = math.inf, math.nan
    got = _attention(ops, q, cache, bt, pos, 0, per, window=30)
    bad = torch.zeros(per, nh, dtype=torch.bool)
    bad[10:, 2:] = True  # kv head 1
    bad[3, 1] = bad[5, 0] = True
    assert bool(torch.isnan(got[bad]).all())
    assert P.rel(got[~bad], clean[~bad]) <= TOL


def test_scores_far_apart(ops):
    """Keys so large that one position takes all the weight, and queries near the ends of f32."""
    g = torch.Generator().manual_seed(17)
    bt, total = _table(g, 2, 40)
    cache = P.cache_q8(total, 1, 1, 16, 128, 3)
    cache[1] *= 1e3
    q = torch.randn(2, 2, 128, generator=g)
    q[0, 1] *= 1e-30
    q[1, 0] *= 1e25
    cache[1][int(bt[1, 0]):int(bt[1, 0]) + 1] *= 1e-3
    pos = torch.tensor([639, 500])
    got, ref = _attention(ops, q, cache, bt, pos, 0, 1), P.causal(q, *cache, bt, pos, 0, 1)
    # scores of 1e4 rounded to 2^-24 of themselves: weights off by up to 1e-3 where two of them are that near; here the
    # largest is alone, so the outputs are its values
    assert bool(torch.isfinite(got).all())
    assert P.rel(got[0, 1], ref[0, 1]) <= TOL and P.rel(got[1, 0], ref[1, 0]) <= TOL


# ---- drafted trees -----------------------------------------------------------------


def _tree_call(ops, q, cache, bt, ctx, masks, layer, f16, stream=None, **kw):
    tables, tree, nh, hd = q.shape
    kc, ks, vc, vs = cache
    total, layers = kc.shape[:2]
    tpb, nkv = (kc.shape[2], kc.shape[3]) if f16 else (kc.shape[3], kc.shape[2])
    out = torch.full(q.shape, 7.0, device="cuda")
    ops.encode_attention_tree(q.cuda(), kc.cuda(), vc.cuda(), bt.to(torch.int32).cuda(), ctx.to(torch.int32).cuda(),
                              masks.cuda(), out, nh, nkv, hd, total, layers, tpb, layer, kscale=None if f16 else ks.cuda(),
                              vscale=None if f16 else vs.cuda(), stream=stream, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _pages(f16, total, layers, nkv, tpb, hd, seed):
    if not f16:
        return P.cache_q8(total, layers, nkv, tpb, hd, seed)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(total, layers, tpb, nkv, hd, generator=g).half() for _ in range(2))
    return [k, None, v, None]


def _random_tree(g, tree):
    return P.tree_bits([-1 if j == 0 else int(torch.randint(-1, j, (1,), generator=g)) for j in range(tree)])


TREES = [(1, 26, 14, 2, 64, 16, 1000), (3, 1, 4, 4, 128, 16, 40), (2, 63, 8, 1, 128, 5, 130), (2, 64, 3, 3, 256, 16, 70),
         (1, 65, 6, 2, 64, 1, 5), (1, 200, 2, 1, 64, 32, 300), (4, 7, 20, 2, 128, 16, 0), (1, 256, 1, 1, 128, 16, 33),
         (2, 12, 4, 2, 256, 16, 2500), (6, 61, 16, 8, 64, 16, 60), (11, 37, 24, 8, 128, 16, 30)]


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("tables,tree,nh,nkv,hd,tpb,ctx", TREES)
@pytest.mark.parametrize("kw", [{}, dict(window=256), dict(soft_cap=5.0, attn_scale=0.15)])
def test_trees(ops, f16, tables, tree, nh, nkv, hd, tpb, ctx, kw):
    g = torch.Generator().manual_seed(tree + ctx)
    bt, total = _table(g, tables, -(-(ctx + tree) // tpb))
    cache = _pages(f16, total, 2, nkv, tpb, hd, tree)
    q = torch.randn(tables, tree, nh, hd, generator=g) * 1.5
    lens = torch.full((tables,), ctx)
    bits = np.stack([_random_tree(g, tree) for _ in range(tables)])
    if tables > 1:
        lens[1] = ctx // 2
        bits[1, tree // 2] = False  # a node that is not there
    if tables > 2:
        lens[2] = -1
    ref = P.tree(q, *cache, bt, lens, bits, 1, kw.get("attn_scale"), kw.get("soft_cap", 0.0), kw.get("window", 0))
    got = _tree_call(ops, q, cache, bt, lens, P.words_of(bits), 1, f16, **kw)
    _check(got.view(-1, nh, hd), ref.view(-1, nh, hd))


@pytest.mark.parametrize("f16", [True, False])
def test_trees_at_the_ends_of_their_tables(ops, f16):
    """Slots past the table, a context past it, missing pages, bits past the tree, masks that leave out the node itself,
    and no context at all."""
    g = torch.Generator().manual_seed(23)
    tables, tree, nh, nkv, hd, tpb = 6, 9, 4, 2, 64, 4
    bt, total = _table(g, tables, 5)
    bt[1, 2], bt[2, 0] = total + 1, -1
    cache = _pages(f16, total, 1, nkv, tpb, hd, 3)
    q = torch.randn(tables, tree, nh, hd, generator=g)
    ctx = torch.tensor([14, 8, 3, 0, 20, 2**31 - 1])
    bits = np.random.RandomState(4).rand(tables, tree, tree) < 0.3
    bits[:, 0, 0] = True
    bits[3, 4] = False
    bits[3, 4, 8] = True
    ref = P.tree(q, *cache, bt, ctx, bits, 0)
    words = P.words_of(bits)
    words |= torch.tensor(-1 << tree)  # bits past the tree mean nothing
    got = _tree_call(ops, q, cache, bt, ctx, words, 0, f16)
    _check(got.view(-1, nh, hd), ref.view(-1, nh, hd))


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("hd,ctx,tables", [(64, 10, 1), (128, 70, 1), (256, 700, 1), (64, 900, 1), (64, 10, 64), (128, 70, 64)])
def test_garbage_in_slots_that_a_node_does_not_see(ops, f16, hd, ctx, tables):
    """NaN, infinities and the largest numbers in other nodes' slots, behind the tree and before the window: a node that
    does not see them keeps its result, one that does has theirs.  64 tables that are all the same take 32 columns at a
    time."""
    g = torch.Generator().manual_seed(29)
    tree, nh, nkv, tpb = 20, 6, 2, 16
    bt, total = _table(g, 1, -(-(ctx + tree) // tpb) + 1)
    cache = _pages(f16, total, 1, nkv, tpb, hd, 31)
    q = torch.randn(1, tree, nh, hd, generator=g)
    bits = _random_tree(g, tree)[None]
    bits[0, :, 5] = False  # only node 5 sees itself
    bits[0, 5, 5] = True
    clean = P.tree(q, *cache, bt, torch.tensor([ctx]), bits, 0)

    def spoil(p, what):
        blk, sl = int(bt[0, p // tpb]), p % tpb
        if f16:
            for c in (cache[0], cache[2]):
                c[blk, 0, sl] = torch.tensor(what, dtype=torch.float16)
        else:
            for s in (cache[1], cache[3]):
                s[blk, 0, :, sl] = math.nan

    for what in ([math.nan], [math.inf], [-math.inf, math.inf] * (hd // 2)):
        spoil(ctx + 5, what)
        for p in range(ctx + tree, bt.shape[1] * tpb):
            spoil(p, what)
        got = _tree_call(ops, q.repeat(tables, 1, 1, 1), cache, bt.repeat(tables, 1), torch.tensor([ctx] * tables),
                         P.words_of(bits).repeat(tables, 1, 1), 0, f16)
        assert tables == 1 or torch.equal(torch.nan_to_num(got[0], nan=1e9), torch.nan_to_num(got[-1], nan=1e9))
        got = got[-1]
        others = [j for j in range(tree) if j != 5]
        assert P.rel(got[others], clean[0, others]) <= TOL
        assert bool(torch.isnan(got[5]).all())


# ---- the accepted path ------------------------------------------------------------------


@pytest.mark.parametrize("f16", [True, False])
@pytest.mark.parametrize("nkv,hd,tpb,layers", [(2, 64, 16, 3), (3, 128, 5, 2), (1, 256, 1, 1)])
def test_accepted_paths_move(ops, f16, nkv, hd, tpb, layers):
    g = torch.Generator().manual_seed(hd)
    tree, tables = 40, 7
    bt, total = _table(g, tables, -(-80 // tpb))
    bt[5, 0] = -1  # the first page is missing
    cache = _pages(f16, total, layers, nkv, tpb, hd, 3)
    if not f16:
        cache[1][3], cache[3][2] = math.nan, math.nan
    ctx = torch.tensor([7, 0, 39, -1, 33, 2, 70])  # the last: slots past the table
    acc = torch.full((tables, 24), -1)
    acc[0, :5] = torch.tensor([0, 1, 2, 3, 4])  # nothing moves
    acc[1, :20] = torch.sort(torch.randperm(tree, generator=g)[:20]).values
    acc[2, 0] = 39
    acc[3, :3] = torch.tensor([1, 2, 3])
    acc[4, :6] = torch.tensor([2, 5, 4, 6, 7, 8])  # ends after 5
    acc[5, :3] = torch.tensor([1, 40, 5])          # ends after 1
    acc[6, :4] = torch.tensor([3, 6, 9, 12])
    want = [None if c is None else c.clone() for c in cache]
    room = bt.shape[1] * tpb
    for t in range(tables):
        last = -1
        for i in range(24):
            n = int(acc[t, i])
            if ctx[t] < 0 or n <= last or n >= tree:
                break
            last = n
            a, b = int(ctx[t]) + n, int(ctx[t]) + i
            if max(a, b) >= room:
                continue
            ba, bb = int(bt[t, a // tpb]), int(bt[t, b // tpb])
            if ba < 0 or bb < 0:
                continue
            for c in want:
                if c is None:
                    continue
                if f16:
                    c[bb, :, b % tpb] = c[ba, :, a % tpb].clone()
                else:
                    c[bb, :, :, b % tpb] = c[ba, :, :, a % tpb].clone()
    dev = [None if c is None else c.cuda() for c in cache]
    ops.encode_kv_accept(dev[0], dev[2], bt.to(torch.int32).cuda(), ctx.to(torch.int32).cuda(), acc.to(torch.int32).cuda(),
                         tree, nkv, hd, total, layers, tpb, kscale=dev[1], vscale=dev[3])
    for got, w in zip(dev, want):
        assert w is None or _same(got.cpu(), w)


# ---- together, on streams and in graphs ----------------------------------------------------


def test_drafted_decode_equals_decode_token_by_token(ops):
    """A prompt enters the 8-bit cache, a tree of drafts is checked against it in one call, its accepted path is kept, and
    the next token attends to it: every accepted node's attention, and the pages, are those of the path entered token by
    token."""
    g = torch.Generator().manual_seed(41)
    nh, nkv, hd, tpb, prompt, tree = 6, 2, 64, 8, 45, 13
    parents = [-1, -1, 0, 0, 1, 2, 2, 5, 5, 4, 8, 8, 10]
    path = [0, 2, 5, 8, 10, 12]
    bits = P.tree_bits(parents)
    depth = torch.from_numpy(bits.sum(1).astype(np.int32)) - 1
    bt = torch.randperm(9, generator=g)[None].to(torch.int32).cuda()
    cs = torch.from_numpy(_cos_sin(80, hd)).cuda()
    x = [torch.randn(prompt + tree + 1, n, hd, generator=g).cuda() for n in (nh, nkv, nkv)]
    geo = (9, 1, tpb, 0)

    def fresh():
        return [c.cuda() for c in P.cache_q8(9, 1, nkv, tpb, hd, 2)]

    def enter(cache, rows, pos, slots=None):
        q, k, v = (t[rows].contiguous() for t in x)
        n = q.shape[0]
        ops.encode_rope_kv_write_q8(q, k, v, q, nh, nkv, hd, pos, cs, *cache, bt, *geo,
                                    slots_i32=slots, rows_per_table=n)
        return q

    def attend(cache, q, pos):
        out = torch.empty_like(q)
        ops.encode_attention_q8(q, *cache, bt, pos, out, nh, nkv, hd, *geo, rows_per_table=q.shape[0])
        return out

    def at(*p):
        return torch.tensor(p, dtype=torch.int32).cuda()

    one, outs = fresh(), []
    pos = torch.arange(prompt, dtype=torch.int32).cuda()
    first = attend(one, enter(one, range(prompt), pos), pos)
    for i, node in enumerate(path):
        outs.append(attend(one, enter(one, [prompt + node], at(prompt + i)), at(prompt + i)))
    last = attend(one, enter(one, [prompt + tree], at(prompt + len(path))), at(prompt + len(path)))

    two = fresh()
    assert torch.equal(attend(two, enter(two, range(prompt), pos), pos), first)
    nodes = range(prompt, prompt + tree)
    q = enter(two, nodes, (prompt + depth).cuda(), slots=torch.tensor(nodes, dtype=torch.int32).cuda())
    out = torch.empty_like(q)
    ops.encode_attention_tree(q, two[0], two[2], bt, at(prompt), P.words_of(bits[None]).cuda(), out, nh, nkv, hd, *geo,
                              kscale=two[1], vscale=two[3])
    acc = torch.tensor([path + [-1] * 3], dtype=torch.int32).cuda()
    ops.encode_kv_accept(two[0], two[2], bt, at(prompt), acc, tree, nkv, hd, 9, 1, tpb, kscale=two[1], vscale=two[3])
    for o, node in zip(outs, path):
        assert P.rel(out[node].cpu(), o[0].cpu().double()) <= 2 * TOL
    again = attend(two, enter(two, [prompt + tree], at(prompt + len(path))), at(prompt + len(path)))
    assert torch.equal(again, last)
    where = torch.arange(prompt + len(path) + 1, dtype=torch.int32).cuda()
    reads = []
    for c in (one, two):
        ko, vo = (torch.empty(where.numel(), nkv * hd, device="cuda") for _ in range(2))
        ops.encode_kv_read_q8(*c, bt, where, ko, vo, nkv, hd, *geo, rows_per_table=where.numel())
        reads.append((ko, vo))
    assert all(torch.equal(a, b) for a, b in zip(*reads))


def _decode_set(seed, tables=3, ctx=1500, hd=64, nh=4, nkv=2, tpb=16):
    g = torch.Generator().manual_seed(seed)
    bt, total = _table(g, tables, -(-ctx // tpb))
    cache = [c.cuda() for c in P.cache_q8(total, 1, nkv, tpb, hd, seed)]
    q = torch.randn(tables, nh, hd, generator=g).cuda()
    pos = torch.randint(ctx // 2, ctx, (tables,), generator=g).to(torch.int32).cuda()
    out = torch.zeros_like(q)
    return dict(args=(q, *cache, bt.to(torch.int32).cuda(), pos, out, nh, nkv, hd, total, 1, tpb, 0), out=out, q=q)


def test_graphs_of_one_stream_run_at_once(ops):
    """Two graphs captured on one stream, the first before any eager call there, replayed on two streams at once and with
    eager calls between: each replay has its own inputs' result."""
    sets = [_decode_set(s) for s in (1, 2)]
    want = []
    for s in sets:
        ops.encode_attention_q8(*s["args"])
        torch.cuda.synchronize()
        want.append(s["out"].clone())
    cap = torch.cuda.Stream()
    graphs = []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=cap):
            ops.encode_attention_q8(*s["args"], stream=cap)
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in sets]
    for turn in range(6):
        for s in sets:
            s["out"].zero_()
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        if turn % 2:
            extra = _decode_set(9 + turn)
            ops.encode_attention_q8(*extra["args"], stream=cap)
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            assert torch.equal(s["out"], w)


def test_calls_of_one_graph_that_need_more_and_more(ops):
    """A short context, then longer ones, captured one after the other: their scratch grows within the graph, whose earlier
    nodes keep what they were given."""
    sets = [_decode_set(s, ctx=c) for s, c in ((1, 900), (2, 4100), (3, 9000), (4, 900))]
    want = []
    for s in sets:
        ops.encode_attention_q8(*s["args"])
        torch.cuda.synchronize()
        want.append(s["out"].clone())
    cap, gr = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=cap):
        for s in sets:
            ops.encode_attention_q8(*s["args"], stream=cap)
    for _ in range(4):
        for s in sets:
            s["out"].zero_()
        gr.replay()
        torch.cuda.synchronize()
        for s, w in zip(sets, want):
            assert torch.equal(s["out"], w)
        ops.encode_attention_q8(*sets[2]["args"])
        torch.cuda.synchronize()


def test_calls_on_many_streams(ops):
    sets = [_decode_set(s, ctx=900 + 700 * s) for s in range(4)]
    want = []
    for s in sets:
        ops.encode_attention_q8(*s["args"])
        torch.cuda.synchronize()
        want.append(s["out"].clone())
        s["out"].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for s, st in zip(sets, streams):
            ops.encode_attention_q8(*s["args"], stream=st)
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert torch.equal(s["out"], w)


def test_offsets_past_32_bits(ops):
    """Pages whose codes lie more than 2^32 bytes, and whose f16 elements more than 2^32 elements, into their arrays."""
    nkv, hd, tpb, layers = 8, 128, 64, 8
    total = 2**32 // (nkv * hd * tpb * layers) + 40  # codes: 4.3 GB an array
    kc, vc = (torch.zeros(total, layers, nkv, tpb, hd, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(total, layers, nkv, tpb, device="cuda") for _ in range(2))
    g = torch.Generator().manual_seed(2)
    rows = 150
    bt = torch.tensor([[total - 1, 0, total - 3]])
    k, v, q = (torch.randn(rows, n, hd, generator=g) for n in (nkv, nkv, 8))
    pos = torch.arange(rows)
    btd, posd = bt.to(torch.int32).cuda(), pos.to(torch.int32).cuda()
    geo = (total, layers, tpb, layers - 1)
    ops.encode_kv_write_q8(k.cuda(), v.cuda(), nkv, hd, posd, kc, ks, vc, vs, btd, *geo, rows_per_table=rows)
    out = torch.full((rows, 8, hd), 7.0, device="cuda")
    ops.encode_attention_q8(q.cuda(), kc, ks, vc, vs, btd, posd, out, 8, nkv, hd, *geo, rows_per_table=rows)
    small = [c[[total - 1, 0, total - 3]][:, -1:].cpu() for c in (kc, ks, vc, vs)]
    ref = P.causal(q, *small, torch.tensor([[0, 1, 2]]), pos, 0, rows)
    _check(out.cpu(), ref)
    want = P.quantise(k.numpy())[0]
    assert torch.equal(small[0][2, 0, :, 1], torch.from_numpy(want[129]))
    del kc, vc, ks, vs
    torch.cuda.empty_cache()
    kc, vc = (torch.zeros(total, layers, tpb, nkv, hd, dtype=torch.float16, device="cuda") for _ in range(2))
    for i, b in enumerate(bt[0].tolist()):
        n = min(tpb, rows - i * tpb)
        kc[b, -1, :n] = k[i * tpb:i * tpb + n].half().cuda()
        vc[b, -1, :n] = v[i * tpb:i * tpb + n].half().cuda()
    tree, ctx = 20, rows - 20
    bits = _random_tree(g, tree)[None]
    small = [kc[bt[0].tolist()][:, -1:].cpu(), None, vc[bt[0].tolist()][:, -1:].cpu(), None]
    ref = P.tree(q[:tree][None], *small, torch.tensor([[0, 1, 2]]), torch.tensor([ctx]), bits, 0)
    out = torch.full((1, tree, 8, hd), 7.0, device="cuda")
    ops.encode_attention_tree(q[:tree].cuda(), kc, vc, btd, torch.tensor([ctx], dtype=torch.int32).cuda(),
                              P.words_of(bits).cuda(), out, 8, nkv, hd, *geo)
    _check(out.cpu()[0], ref[0])
