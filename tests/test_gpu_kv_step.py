"""Pages and rows of a step, head norms with rotation and write, and 4-bit pages read back (kv_step.hip), against plain
results.

Everything here is defined operation by operation: whole numbers, and f32 or f16 operations rounded once each (the sum of
squares and the root of the norm in 64 bits, whose order moves the f32 quotient only where it stands within 2^-50 of a
border), so all is compared for equality."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import _paged as P
import _step as S

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.as_tensor(np.asarray(x, np.int32)).cuda()


# ---- the plan -----------------------------------------------------------------------------


def _sessions(rng, n, per, tpb, spare, what):
    """Random sessions: (ctx, new, bt, total, free, count)."""
    room = per * tpb
    ctx = rng.integers(0, max(1, room - tpb), n)
    new = np.ones(n, np.int64)
    kind = rng.random(n)
    if what == "mixed":
        new[kind < 0.2] = 0
        new[(kind >= 0.2) & (kind < 0.35)] = -1 - rng.integers(0, 5)
        prompts = (kind >= 0.35) & (kind < 0.6)
        new[prompts] = rng.integers(1, room // 2 + 2, int(prompts.sum()))  # some past the table
        ctx[kind > 0.95] = -1
        ctx[(kind > 0.9) & (kind <= 0.95)] = room  # full tables
    elif what == "prompts":
        ctx[:] = 0
        new = rng.integers(1, room + 1, n)
    total = n * per + spare
    perm = rng.permutation(total)
    bt = perm[:n * per].reshape(n, per).copy()
    held = -(-np.maximum(ctx, 0) // tpb)
    mine = np.arange(per) < held[:, None]
    free = rng.permutation(np.concatenate([bt[~mine], perm[n * per:]]))
    bt[~mine] = -1
    return ctx, new, bt, total, np.concatenate([free, np.full(total - len(free), -7)]), len(free)


def _plan(ops, ctx, new, bt, total, tpb, free, count, rows, in_place=False):
    n = len(ctx)
    d = dict(ctx=_i32(ctx), new=_i32(new), bt=_i32(bt), free=_i32(free), count=_i32([count]))
    lens, left = (d["ctx"], d["count"]) if in_place else (_i32([99] * n), _i32([99]))
    starts, pos, slots = _i32([99] * (n + 1)), _i32([99] * rows), _i32([99] * rows)
    ops.encode_kv_plan(d["ctx"], d["new"], d["bt"], total, tpb, d["free"], d["count"], lens, left, starts, pos, slots)
    torch.cuda.synchronize()
    if not in_place:
        assert d["ctx"].tolist() == list(ctx) and d["count"].tolist() == [count]
    return d["bt"], d["free"], lens, left, starts, pos, slots


def _check_plan(got, want):
    for name, g, w in zip(("tables", "free", "lens", "left", "starts", "positions", "slots"), got, want):
        assert np.array_equal(g.cpu().numpy(), np.asarray(w).reshape(g.shape)), name


# sessions, pages of a table, tokens of a page: one session, one page, more than a wave, than a block's threads
PLANS = [(1, 1, 16), (1, 40, 16), (7, 5, 1), (63, 9, 7), (200, 12, 16), (1024, 3, 4), (1025, 4, 16), (2500, 3, 2)]


@pytest.mark.parametrize("n,per,tpb", PLANS)
@pytest.mark.parametrize("what", ["decode", "mixed", "prompts"])
@pytest.mark.parametrize("scarce", ["", "pages", "rows"])
def test_plan(ops, n, per, tpb, what, scarce):
    rng = np.random.default_rng(n * 31 + per)
    ctx, new, bt, total, free, count = _sessions(rng, n, per, tpb, 5, what)
    if scarce == "pages":
        count = count // 3
    asked = int(np.maximum(new, 0).sum())
    rows = min(asked // 2 + 1 if scarce == "rows" else asked + 9, 1 << 20)
    want = S.plan(ctx, new, bt, total, tpb, free, count, rows)
    _check_plan(_plan(ops, ctx, new, bt, total, tpb, free, count, rows), want)
    _check_plan(_plan(ops, ctx, new, bt, total, tpb, free, count, rows, in_place=True), want)


@pytest.mark.parametrize("n,per,tpb,what", [(5000, 2, 16, "mixed"), (4096, 3, 8, "prompts"), (4097, 3, 8, "prompts"),
                                            (20000, 1, 4, "decode"), (3, 1 << 16, 8, "prompts"), (2, 1 << 20, 1, "prompts")])
def test_plan_of_many(ops, n, per, tpb, what):
    """More sessions than the row starts in LDS, and more rows and pages than a block deals with at once."""
    rng = np.random.default_rng(n)
    ctx, new, bt, total, free, count = _sessions(rng, n, per, tpb, 5, what)
    rows = min(int(np.maximum(new, 0).sum()) + 9, 1 << 20)
    want = S.plan(ctx, new, bt, total, tpb, free, count, rows)
    _check_plan(_plan(ops, ctx, new, bt, total, tpb, free, count, rows), want)


def test_plan_at_its_limits(ops):
    """A first session that does not fit lets nobody pass, one that no table holds does; all pages gone to the last; no
    rows, no sessions; entries that are no page; a free list too short for what comes back, a count out of its range."""
    bt = np.full((4, 4), -1)
    free = np.arange(16)
    one = lambda ctx, new, count, rows, bt=bt, free=free: (  # noqa: E731
        np.array(ctx), np.array(new), bt, 16, 4, free, count, rows)
    held = np.array([[0, 1, -1, 3], [4, 99, 6, 7], [8, 9, 10, 11], [-1, -1, -1, -1]])
    for case in (one([0] * 4, [9, 1, 1, 1], 2, 20), one([0] * 4, [17, 1, 1, 1], 2, 20), one([0] * 4, [4] * 4, 4, 16),
                 one([0] * 4, [4] * 4, 4, 15), one([0] * 4, [4] * 4, 16, 0), one([0] * 4, [0] * 4, 16, 5),
                 one([16, 16, 12, 0], [-1, -3, -1, -1], 0, 3, held, np.full(16, -7)),
                 one([16, 16, 3, 5], [-1, -3, 13, 3], 0, 30, held, np.full(16, -7)),
                 one([16, 16, 12, 0], [-1, -3, -1, -1], 1, 3, held, np.array([12, -7, -7])),
                 one([2**31 - 1, 0, 0, 0], [2**31 - 1, 1, 1, 1], 16, 5), one([0] * 4, [1] * 4, -3, 5),
                 one([0] * 4, [1] * 4, 1000, 5), one([2] * 4, [1] * 4, 0, 5)):
        want = S.plan(*case)
        _check_plan(_plan(ops, *case), want)
        _check_plan(_plan(ops, *case, in_place=True), want)
    none = np.zeros((0, 4), int)
    got = _plan(ops, np.zeros(0, int), np.zeros(0, int), none, 16, 4, free, 5, 3)
    assert got[3].tolist() == [5] and got[4].tolist() == [0] and got[5].tolist() == [-1] * 3 == got[6].tolist()


def test_plan_as_a_loop(ops):
    """Forty steps of the same sessions, lengths and free pages in place, some finished and begun again: no page is ever
    held twice, none is lost."""
    rng = np.random.default_rng(3)
    n, per, tpb, rows = 50, 12, 4, 300
    total = 260
    ctx, bt, free, count = np.zeros(n, int), np.full((n, per), -1), rng.permutation(total), total
    d = dict(ctx=_i32(ctx), bt=_i32(bt), free=_i32(free), count=_i32([count]))
    starts, pos, slots = _i32([0] * (n + 1)), _i32([0] * rows), _i32([0] * rows)
    for _ in range(40):
        new = np.where(ctx == 0, rng.integers(0, 30, n), np.where(rng.random(n) < 0.08, -1, rng.integers(0, 3, n)))
        bt, free, ctx, count, *rest = S.plan(ctx, new, bt, total, tpb, free, count, rows)
        ops.encode_kv_plan(d["ctx"], _i32(new), d["bt"], total, tpb, d["free"], d["count"], d["ctx"], d["count"], starts, pos,
                           slots)
        _check_plan((d["bt"], d["free"], d["ctx"], d["count"], starts, pos, slots), (bt, free, ctx, count, *rest))
        held = [bt[t, j] for t in range(n) for j in range(-(-ctx[t] // tpb))]
        assert sorted([*held, *free[:count]]) == list(range(total))


# ---- norm, rotation and write -------------------------------------------------------------


def _cos_sin(n, hd):
    a = np.arange(n)[:, None] * 10000.0 ** (-2.0 * np.arange(hd // 2) / hd)
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def _pages(fmt, total, layers, nkv, tpb, hd, seed):
    if fmt == "q4":
        return S.cache_q4(total, layers, nkv, tpb, hd, seed)
    if fmt == "q8":
        return P.cache_q8(total, layers, nkv, tpb, hd, seed)
    g = torch.Generator().manual_seed(seed)
    k, v = (torch.randn(total, layers, tpb, nkv, hd, generator=g).half() for _ in range(2))
    return [k, None, v, None]


def _held(fmt, x):
    """Codes and scales, or f16 numbers, of vectors x [..., hd]."""
    if fmt == "q4":
        return [torch.from_numpy(y) for y in S.quantise4(x)]
    if fmt == "q8":
        return [torch.from_numpy(np.ascontiguousarray(y)) for y in P.quantise(x)]
    return [torch.from_numpy(np.asarray(x, np.float32)).half(), None]


def _expect(fmt, cache, slots, layer, tpb, k, v):
    """The pages after rows k, v [rows][nkv][hd] went to their slots."""
    out = [None if x is None else x.clone() for x in cache]
    total = cache[0].shape[0]
    for i, x in ((0, k), (2, v)):
        codes, scales = _held(fmt, x)
        for r, s in enumerate(slots):
            if not 0 <= s < total * tpb:
                continue
            b, o = s // tpb, s % tpb
            if fmt == "f16":
                out[i][b, layer, o] = codes[r]
            else:
                out[i][b, layer, :, o] = codes[r]
                out[i + 1][b, layer, :, o] = scales[r]
    return out


def _same(a, b):
    """Equal, NaN where NaN."""
    return a is None or torch.equal(torch.nan_to_num(a.float(), nan=12345.0), torch.nan_to_num(b.float(), nan=12345.0))


def _write(ops, q, k, v, out, qw, kw, eps, pos, cs, slots, cache, fmt, layer, **kw_):
    total, layers = cache[0].shape[:2]
    nkv, hd = k.shape[1:]
    tpb = cache[0].shape[2] if fmt == "f16" else cache[0].shape[3]
    dev = [None if x is None else x.cuda() for x in cache]
    c = lambda x: None if x is None else x.cuda()  # noqa: E731
    ops.encode_norm_rope_kv_write(q, c(k), c(v), out, q.shape[1], nkv, hd, c(qw), c(kw), eps, _i32(pos), c(cs), _i32(slots),
                                  dev[0], dev[2], total, layers, tpb, layer, kscale=dev[1], vscale=dev[3], **kw_)
    torch.cuda.synchronize()
    return [None if x is None else x.cpu() for x in dev]


# rows, query heads, kv heads, head_dim, tokens per page
WRITES = [(1, 9, 3, 64, 16), (1, 1, 1, 256, 16), (37, 14, 2, 64, 5), (64, 8, 8, 128, 16), (130, 4, 1, 256, 3), (19, 5, 5, 128, 1)]


@pytest.mark.parametrize("rows,nh,nkv,hd,tpb", WRITES)
@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("weight", [torch.float32, torch.float16, torch.bfloat16, None])
def test_norm_rope_write(ops, rows, nh, nkv, hd, tpb, fmt, interleaved, weight):
    g = torch.Generator().manual_seed(hd + rows)
    total = -(-rows // tpb) + 3
    q, k, v = (torch.randn(rows, n, hd, generator=g) for n in (nh, nkv, nkv))
    k = k * torch.exp(3 * torch.randn(rows, nkv, 1, generator=g))
    v = v * torch.exp(3 * torch.randn(rows, nkv, 1, generator=g))
    qw, kw = ((None, None) if weight is None else [(1 + 0.3 * torch.randn(hd, generator=g)).to(weight) for _ in range(2)])
    if weight is torch.float16:
        kw = None  # one of the two
    slots = torch.randperm(total * tpb, generator=g)[:rows].tolist()
    pos = torch.randint(0, 50, (rows,), generator=g).tolist()
    if rows > 5:
        pos[1], slots[2], slots[3], pos[4] = -1, -1, total * tpb, 10**6  # padding, no slot, past the pages, past the table
    cs = torch.from_numpy(_cos_sin(40, hd))
    cache = _pages(fmt, total, 2, nkv, tpb, hd, 7)
    dq = q.cuda()
    out = torch.full_like(dq, 7.0)
    ops.set_rope_interleaved(interleaved)
    try:
        got = _write(ops, dq, k, v, out, qw, kw, 1e-6, pos, cs, slots, cache, fmt, 1)
        _write(ops, dq, k, v, dq, qw, kw, 1e-6, pos, cs, slots, cache, fmt, 1)  # in place
    finally:
        ops.set_rope_interleaved(False)
    at = cs.numpy()[np.clip(np.array(pos), 0, 39)]
    there = torch.tensor(pos) >= 0
    turned = lambda x, w: P.rope(S.normed(x.numpy(), None if w is None else w.float().numpy(), 1e-6), at, interleaved)  # noqa: E731
    want = torch.from_numpy(turned(q, qw))
    out, dq = out.cpu(), dq.cpu()
    assert torch.equal(out[there], want[there]) and bool((out[~there] == 7.0).all())
    assert torch.equal(dq[there], want[there]) and torch.equal(dq[~there], q[~there])
    went = [s if p >= 0 else -1 for s, p in zip(slots, pos)]
    for a, b in zip(got, _expect(fmt, cache, went, 1, tpb, turned(k, kw), v.numpy())):
        assert _same(a, b)


def test_no_rotation(ops):
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(6, n, 64, generator=g) for n in (4, 2, 2))
    w = 1 + 0.3 * torch.randn(64, generator=g)
    cache = _pages("q4", 3, 1, 2, 4, 64, 7)
    out = torch.empty_like(q).cuda()
    got = _write(ops, q.cuda(), k, v, out, w, w, 1e-5, range(6), None, range(6), cache, "q4", 0)
    assert torch.equal(out.cpu(), torch.from_numpy(S.normed(q.numpy(), w.numpy(), 1e-5)))
    for a, b in zip(got, _expect("q4", cache, range(6), 0, 4, S.normed(k.numpy(), w.numpy(), 1e-5), v.numpy())):
        assert _same(a, b)


def _loud_vectors(hd):
    """Vectors at the ends of f32 and f16: zeros, one value, tiny, huge, beyond f16, with infinities and NaN."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(16, 1, hd, generator=g)
    x[0] = 0.0
    x[1] = 3.1415926
    x[2] *= 1e-42
    x[3] *= 1e-7      # scales of f16's subnormal numbers
    x[4] *= 3e-9      # scales of 0
    x[5] *= 4e4
    x[6] *= 1e38
    x[7] = torch.where(x[7] > 0, 65504.0, -65504.0)
    x[8, 0, 5], x[8, 0, 40] = math.inf, -1e9
    x[9, 0, 33] = math.nan
    x[10] = -2.0**-24
    x[11] = 65503.0 + x[11]
    x[12] = -65000.0 + 400 * x[12]
    x[13] = 100.0 + 1e-4 * x[13]
    x[14, 0, 3] = -math.inf
    x[15] = torch.linspace(-1, 1, hd)
    return x


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("fmt", ["f16", "q8", "q4"])
def test_vectors_at_the_ends(ops, hd, fmt):
    x = _loud_vectors(hd)
    cache = _pages(fmt, 4, 1, 1, 4, hd, 3)
    q, w = torch.randn(16, 1, hd), torch.ones(hd)
    out = torch.empty_like(q).cuda()
    for weight in (None, w):
        got = _write(ops, x.cuda(), x, x, out, weight, weight, 1e-6, range(16), None, range(16), cache, fmt, 0)
        y = S.normed(x.numpy(), None if weight is None else w.numpy(), 1e-6)
        assert _same(out.cpu(), torch.from_numpy(y))
        for a, b in zip(got, _expect(fmt, cache, range(16), 0, 4, y, x.numpy())):
            assert _same(a, b)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_values_of_four_bits(hd):
    """The reference itself: every element within its bound of what its code stands for."""
    x = np.clip(_loud_vectors(hd).numpy(), -65504, 65504)
    ok = np.isfinite(x).all((1, 2))
    x = x[ok]
    codes, scales = S.quantise4(x)
    v = S.values4(codes, scales).astype(np.float64)
    assert np.isfinite(v).all()
    s = np.repeat(scales[..., 0].astype(np.float64), 32, -1)
    # half a step, the ends moved by the scale's and the base's rounding, one f16 step of scale where an end stands at
    # f16's, and the value's own rounding
    step = np.maximum(np.abs(x) * 2.0**-11, 2.0**-25)
    bound = s / 2 + 15 * np.maximum(s * 2.0**-10, 2.0**-25) + step + np.maximum(np.abs(v) * 2.0**-11, 2.0**-25)
    assert (np.abs(v - x) <= bound).all()


@pytest.mark.parametrize("tables,per,nkv,hd,tpb", [(1, 1, 1, 64, 16), (3, 17, 2, 128, 5), (2, 40, 3, 256, 16), (4, 9, 5, 64, 7)])
def test_read_four_bits(ops, tables, per, nkv, hd, tpb):
    g = torch.Generator().manual_seed(per)
    need = -(-per // tpb)
    total = tables * need + 2
    bt = torch.randperm(total, generator=g)[:tables * need].view(tables, need)
    cache = S.cache_q4(total, 2, nkv, tpb, hd, 9)
    cache[1][0, 1] = math.nan
    if tables > 1:
        bt[1, 0] = total + 3  # a missing page
    pos = torch.arange(per).repeat(tables)
    if per > 2:
        pos[2], pos[1] = -1, need * tpb
    dev = [c.cuda() for c in cache]
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        ko, vo = (torch.full((tables * per, nkv * hd), 5.0, dtype=dt, device="cuda") for _ in range(2))
        ops.encode_kv_read_q4(*dev, _i32(bt), _i32(pos), ko, vo, nkv, hd, total, 2, tpb, 1, rows_per_table=per)
        for got, (c, s) in ((ko, cache[:2]), (vo, cache[2:])):
            got = got.cpu().view(-1, nkv, hd)
            x = torch.from_numpy(S.values4(c[:, 1].numpy(), s[:, 1].numpy()))  # [block][nkv][tpb][hd]
            for r, p in enumerate(pos.tolist()):
                if p < 0:
                    assert bool((got[r] == 5.0).all())
                    continue
                blk = int(bt[r // per, p // tpb]) if p // tpb < need else total
                want = x[blk, :, p % tpb] if blk < total else torch.zeros(nkv, hd)
                assert _same(got[r], want.float().to(dt))


# ---- codes half way between two, and heads whose norm is out of the ordinary ---------------


def _halfway(steps, s, rng):
    """f32 numbers at and next to (k + 1 / 2) s, k below `steps`, by up to 300 steps of f32."""
    k = rng.integers(0, steps, 4096) + 0.5
    x = (k * np.float64(s)).astype(np.float32)
    d = rng.choice([0, 0, 1, 1, 2, 3, 10, 40, 100, 300], x.size) * rng.choice([-1, 1], x.size)
    return (x.view(np.int32) + d).astype(np.int32).view(np.float32)


@pytest.mark.parametrize("fmt", ["q8", "q4"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_codes_between_two(ops, fmt, hd):
    """Codes are the rounded quotient's, however near it lies to a tie."""
    rng = np.random.default_rng(hd)
    rows, nkv = 40, 4
    x = []
    for _ in range(2 * rows * nkv):
        if fmt == "q8":  # the scale is the largest over 127
            top = np.float32(np.exp(rng.uniform(-20, 20)))
            v = rng.choice(_halfway(126, top / np.float32(127), rng), hd) * rng.choice([-1, 1], hd).astype(np.float32)
            v[rng.integers(hd)] = top
        else:  # base 0 or one that f16 holds, and the scale one too
            s, v = np.float16(np.exp(rng.uniform(-6, 4))).astype(np.float32), np.zeros(hd, np.float32)
            for g in range(0, hd, 32):
                base = rng.choice([np.float32(0), np.float32(-8) * s])
                v[g:g + 32] = base + rng.choice(_halfway(14, s, rng), 32)
                v[g], v[g + 1] = base, base + np.float32(15) * s
        x.append(np.clip(v, -top, top) if fmt == "q8" else v)
    k, v = (torch.from_numpy(np.stack(y).reshape(rows, nkv, hd)) for y in (x[:rows * nkv], x[rows * nkv:]))
    q = torch.zeros(rows, nkv, hd, device="cuda")
    cache = _pages(fmt, 6, 1, nkv, 8, hd, 3)
    slots = list(range(rows))
    got = _write(ops, q, k, v, q, None, None, 0.0, [0] * rows, None, slots, cache, fmt, 0)
    for a, b in zip(got, _expect(fmt, cache, slots, 0, 8, k.numpy(), v.numpy())):
        assert _same(a, b)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("eps", [0.0, 1e-6, 1e30])
def test_norms_of_every_size(ops, hd, eps):
    """Heads of zeros, of f32's smallest and largest numbers, and with infinities and NaN, to f16 pages and to q_out."""
    g = torch.Generator().manual_seed(hd)
    sizes = [0.0, 1e-45, 1e-42, 1e-38, 1e-20, 1.0, 1e18, 1e30, 3e37]
    q = torch.stack([torch.randn(2, hd, generator=g).clamp(-4, 4) * n for n in sizes] * 2)
    for r, bad in ((-1, float("inf")), (-2, float("-inf")), (-3, float("nan"))):
        q[r, 0, 5] = bad
    k = q.flip(0).contiguous()
    rows = q.shape[0]
    w = 1 + 0.3 * torch.randn(hd, generator=g)
    cache = _pages("f16", 3, 1, 2, 16, hd, 3)
    slots = list(range(rows))
    out = torch.zeros_like(q).cuda()
    got = _write(ops, q.cuda(), k, k, out, w, w, eps, [0] * rows, None, slots, cache, "f16", 0)
    assert _same(out.cpu(), torch.from_numpy(S.normed(q.numpy(), w.numpy(), eps)))
    with np.errstate(over="ignore"):
        for a, b in zip(got, _expect("f16", cache, slots, 0, 16, S.normed(k.numpy(), w.numpy(), eps), k.numpy())):
            assert _same(a, b)
