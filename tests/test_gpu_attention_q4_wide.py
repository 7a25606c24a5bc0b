"""Attention over 4-bit pages in sets of 32 columns, which calls take that have more than 16 columns a table and 256 sets of 32
and more: plain rows, windows and caps, last sets of a few columns, missing pages, groups of NaN, tiny pages beside others,
rows that wait, and codes past 32-bit offsets.  The bar is that of test_gpu_attention_q4.py."""
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


def _attend(ops, q, cache, bt, pos, starts, ragged, layer=0, **kw):
    rows, nh, hd = q.shape
    total, layers, nkv, tpb, _ = cache[0].shape
    out = torch.full((rows, nh, hd), 7.0, device="cuda")
    kw.update(dict(row_starts_i32=_i32(starts)) if ragged else dict(rows_per_table=starts[1]))
    ops.encode_attention_q4(q.cuda(), *[c.cuda() for c in cache], _i32(bt), _i32(pos), out, nh, nkv, hd, total, layers, tpb,
                            layer, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def _dense(q, cache, bt, pos, starts, window=0, cap=0.0, layer=0):
    """In 64 bits; rows of no position or table are NaN, and so are sums that a NaN reaches."""
    k, _, v, _ = S.as_f16_pages(cache)
    total, nh = len(k), q.shape[1]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    for t in range(len(starts) - 1):
        a, b = int(starts[t]), int(starts[t + 1])
        if a == b:
            continue
        there = ((bt[t] >= 0) & (bt[t] < total))[:, None, None, None]
        kt, vt = (torch.where(there, x[bt[t].clamp(0, total - 1), layer], torch.zeros((), dtype=x.dtype)).flatten(0, 1).double()
                  for x in (k, v))
        at, p = torch.arange(len(kt)), torch.as_tensor(pos)[a:b, None].clamp(max=len(kt) - 1)
        sees = (at <= p) & ((at > p - window) if window else (at >= 0))
        hurts = torch.isnan(vt)
        vt = torch.nan_to_num(vt)
        for h in range(nh):
            g = h // (nh // kt.shape[1])
            s = q[a:b, h].double() @ kt[:, g].T / math.sqrt(q.shape[2])
            if cap:
                s = torch.tanh(s / cap) * cap
            w = torch.softmax(torch.where(sees, s, -math.inf), -1)
            w = torch.where((sees & torch.isnan(s)).any(-1, keepdim=True), torch.nan, torch.nan_to_num(w))
            o = w @ vt[:, g]
            reached = sees.double() @ hurts[:, g].double() > 0
            out[a:b, h] = torch.where((p < 0) | reached, torch.nan, o)
    return out


def _check(got, ref, pos, rows=None):
    """Rows of no position left as they were, NaN where ref is, else near."""
    rows = len(pos) if rows is None else rows
    there = torch.zeros(len(pos), dtype=torch.bool)
    there[:rows] = torch.as_tensor(pos)[:rows] >= 0
    assert bool((got[~there] == 7.0).all())
    got, ref = got[there], ref[there]
    nan = torch.isnan(ref)
    assert torch.equal(torch.isnan(got), nan)
    for h in range(ref.shape[1]):
        at = ~nan[:, h]
        assert not bool(at.any()) or P.rel(got[:, h][at], ref[:, h][at]) <= TOL


def _sets(rows, nh, nkv):
    return nkv * -(-rows * (nh // nkv) // 32)


# rows of each table, query heads, kv heads, head_dim, tokens per page, positions: last sets of 16, 2, 10, 32 and 17 columns
SHAPES = [([260], 32, 8, 128, 16, 300), ([130], 64, 64, 64, 7, 200), ([590], 14, 2, 64, 16, 700), ([40] * 16, 16, 4, 128, 16, 90),
          ([272] * 2, 15, 5, 128, 5, 400), ([2067], 4, 1, 128, 64, 2100), ([340], 24, 8, 64, 16, 900)]


def _case(new, nh, nkv, hd, tpb, ctx, seed=5):
    g = torch.Generator().manual_seed(hd + nh)
    tables, pages = len(new), -(-ctx // tpb)
    total = tables * pages + 2
    bt = torch.randperm(total, generator=g)[:tables * pages].view(tables, pages)
    cache = S.cache_q4(total, 1, nkv, tpb, hd, seed)
    starts = [int(x) for x in np.concatenate([[0], np.cumsum(new)])]
    pos = np.concatenate([np.arange(ctx - 3 * t - n, ctx - 3 * t) for t, n in enumerate(new)]).clip(-1)
    q = 1.5 * torch.randn(len(pos), nh, hd, generator=g)
    return q, cache, bt, pos, starts


@pytest.mark.parametrize("window,cap", [(0, 0.0), (100, 0.0), (0, 5.0), (37, 50.0)])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_rows_of_tables(ops, shape, ragged, window, cap):
    new, nh, nkv, hd, *_ = shape
    assert len(new) * _sets(new[0], nh, nkv) >= 256
    q, cache, bt, pos, starts = _case(*shape)
    pos[3], pos[len(pos) // 2] = -1, 0
    ref = _dense(q, cache, bt, pos, starts, window, cap)
    _check(_attend(ops, q, cache, bt, pos, starts, ragged, window=window, soft_cap=cap), ref, pos)


@pytest.mark.parametrize("window,cap", [(0, 0.0), (60, 30.0)])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts_beside_decoding_sessions(ops, hd, window, cap):
    """Tables of any rows and none, and rows behind the last, which stay as they were."""
    new = [1, 0, 150, 1, 1, 17, 1, 0, 97, 1]
    q, cache, bt, pos, starts = _case(new, 32, 8, hd, 16, 333)
    assert 8 * (len(pos) * 4 // 32 + len(new)) >= 256
    q, pos = torch.cat([q, q[:5]]), np.concatenate([pos, [-1, 3, -1, 9, -1]])
    ref = _dense(q, cache, bt, pos, starts, window, cap)
    _check(_attend(ops, q, cache, bt, pos, starts, True, window=window, soft_cap=cap), ref, pos, starts[-1])


@pytest.mark.parametrize("cap", [0.0, 10.0])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_missing_pages_are_zeros(ops, hd, ragged, cap):
    q, cache, bt, pos, starts = _case([260], 32, 8, hd, 16, 420)
    bt[0, 1], bt[0, 7], bt[0, 20] = -1, len(cache[0]), -5
    ref = _dense(q, cache, bt, pos, starts, cap=cap)
    _check(_attend(ops, q, cache, bt, pos, starts, ragged, soft_cap=cap), ref, pos)
    bt[:] = -1
    assert bool((_attend(ops, q, cache, bt, pos, starts, ragged, soft_cap=cap) == 0).all())
    q[9, 5, 3], q[200, 31, 0] = math.inf, math.nan  # of zeros these make NaN
    got = _attend(ops, q, cache, bt, pos, starts, ragged, soft_cap=cap)
    bad = torch.zeros(260, 32, dtype=torch.bool)
    bad[9, 5] = bad[200, 31] = True
    assert bool(torch.isnan(got[bad]).all()) and bool((got[~bad] == 0).all())


@pytest.mark.parametrize("window", [0, 90])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_nan_groups_reach_who_sees_them(ops, hd, ragged, where, window):
    """NaN in the rows and dims that see it, in all 32 columns of a set or some of them; none in the others."""
    q, cache, bt, pos, starts = _case([264], 32, 8, hd, 16, 400)
    for p, heads in ((395, slice(2, 5)), (300, slice(3, 4)), (170, slice(7, 8)), (0, slice(0, 1))):
        cache[1 if where == "k" else 3][int(bt[0, p // 16]), 0, heads, p % 16, hd // 32 - 1] = math.nan
    ref = _dense(q, cache, bt, pos, starts, window)
    assert bool(torch.isnan(ref).any()) and bool(torch.isfinite(ref[:, 4:8]).any())
    _check(_attend(ops, q, cache, bt, pos, starts, ragged, window=window), ref, pos)


@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("tiny_first", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_tiny_pages_beside_others(ops, hd, tiny_first, ragged):
    """A context of which every other 64 positions, and of each wave's every other, hold subnormal f16 values."""
    q, cache, bt, pos, starts = _case([260], 32, 8, hd, 16, 640)
    small = torch.tensor([((p // 4 + p // 16) % 2 == 0) == tiny_first for p in range(bt.shape[1])])
    for i in (0, 2):
        x = torch.from_numpy(S.values4(cache[i].numpy(), cache[i + 1].numpy()).astype(np.float32))
        x[bt[0, small]] *= 1e-6
        cache[i], cache[i + 1] = (torch.from_numpy(y) for y in S.quantise4(x.numpy()))
    ref = _dense(q, cache, bt, pos, starts)
    _check(_attend(ops, q, cache, bt, pos, starts, ragged), ref, pos)


@pytest.mark.parametrize("hd", [64, 128])
def test_all_pages_tiny(ops, hd):
    q, cache, bt, pos, starts = _case([260], 32, 8, hd, 16, 300)
    for i in (0, 2):
        x = S.values4(cache[i].numpy(), cache[i + 1].numpy()).astype(np.float32) * np.float32(1e-6)
        cache[i], cache[i + 1] = (torch.from_numpy(y) for y in S.quantise4(x))
    q = q * 1e6
    ref = _dense(q, cache, bt, pos, starts)
    for ragged in (False, True):
        _check(_attend(ops, q, cache, bt, pos, starts, ragged), ref, pos)


@pytest.mark.parametrize("hd", [64, 128])
def test_codes_past_32_bit_offsets(ops, hd):
    """Pages at both ends of codes of 5 GiB."""
    g = torch.Generator().manual_seed(hd)
    nkv, nh, tpb, layers, rows, ctx = 8, 32, 16, 32, 260, 300
    page = nkv * tpb * hd // 2
    total = (5 << 30) // (page * layers)
    pages = -(-ctx // tpb)
    bt = torch.tensor([[0, total - 1, total // 2, total - 2] + [total - 3 - 7 * i for i in range(pages - 4)]])
    small = S.cache_q4(pages, 1, nkv, tpb, hd, 9)
    cache = []
    for x in small:
        big = torch.empty((total, layers) + x.shape[2:], dtype=x.dtype, device="cuda")
        big[bt[0].cuda(), layers - 1] = x[:, 0].cuda()
        cache.append(big)
    q, pos, starts = torch.randn(rows, nh, hd, generator=g), np.arange(ctx - rows, ctx), [0, rows]
    ref = _dense(q, small, torch.arange(pages)[None], pos, starts)
    for ragged in (False, True):
        _check(_attend(ops, q, cache, bt, pos, starts, ragged, layers - 1), ref, pos)


def test_they_take_no_scratch():
    """Sets of 32 columns are not split: no call of theirs takes scratch, on a stream or in a graph."""
    from cellm_amd import HipOps

    q, cache, bt, pos, starts = _case([40] * 16, 16, 4, 128, 16, 1500)
    q, cache, bt, pos, out = q.cuda(), [c.cuda() for c in cache], _i32(bt), _i32(pos), torch.zeros(640, 16, 128, device="cuda")
    starts = _i32(starts)
    total = len(cache[0])

    def call(ops, stream, ragged):
        kw = dict(row_starts_i32=starts) if ragged else dict(rows_per_table=40)
        ops.encode_attention_q4(q, *cache, bt, pos, out, 16, 4, 128, total, 1, 16, 0, stream=stream, **kw)

    def held(f):
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        f()
        torch.cuda.synchronize()
        return before - torch.cuda.mem_get_info()[0]

    stream = torch.cuda.Stream()
    for ops in (HipOps(0), HipOps(0)):  # what the runtime loads with the kernels comes with the first
        most = 0
        for ragged in (False, True):
            eager = held(lambda: call(ops, stream, ragged))
            graph = torch.cuda.CUDAGraph()

            def capture():
                with torch.cuda.graph(graph, stream=stream):
                    call(ops, stream, ragged)

            captured = held(capture)
            graph.replay()
            torch.cuda.synchronize()
            del graph
            most = max(most, eager, captured)
        ops.close()
    assert most <= 2**22  # scratch of splits would be 8 MiB
