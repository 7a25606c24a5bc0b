"""Operators of one serving step over a paged cache whose lengths only the device knows, as
cases for timing and for checking outputs.

Pages are handed out and rows laid out from the sessions' lengths, q and k are normed per
head, rotated and written to f16, 8-bit or 4-bit pages through the slot map, and the step's
rows attend to 4-bit pages.  Where `own` is false, `run` computes them with elementary torch
operations; where it is true, through HipOps.  The kinds:

  plan     block tables, free pages, row starts, positions and slots of a step from the
           sessions' lengths: decoding, prompting, idle and finished ones
  write    norm of each head of q and k, RoPE, K and V into the pages by slot; of 8-bit and
           4-bit pages the written tokens read back (what their codes stand for)
  attend   attention over 4-bit pages: the last token of every session, prompts, or a step's
           rows with prompts and decoding sessions side by side

A 4-bit vector is held in groups of 32 dims: a base z = f16(min), a scale s = f16((max - z) /
15) and codes c = rint((x - z) / s) in 0..15, which stand for f16(c * s + z).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False
_ops = None


def _hip():
    """The program's one context."""
    global _ops
    if _ops is None:
        from cellm_amd import HipOps

        _ops = HipOps(0)
    return _ops


_TINY = 1.1754943508222875e-38  # the smallest normal f32: 8-bit scales below it are 0
_EPS = float(np.float32(1e-6))


def listed():
    return [
        # The smallest calls: eight decoding sessions take a token each, now and then a page.
        dict(name="plan_decode_8", kind="plan", tables=8, ctx=700, prompt=0, prompts=0, tpb=16, spare=64, rows=8,
             short=False),
        # A busy server's step: 256 sessions, most decoding, some prompts of up to 500 tokens, some idle or finished.
        dict(name="plan_mixed_256", kind="plan", tables=256, ctx=4000, prompt=500, prompts=24, tpb=16, spare=4096,
             rows=8192, short=False),
        # Prompts alone, more than there are pages for: the last sessions wait.
        dict(name="plan_prompts_64", kind="plan", tables=64, ctx=100, prompt=2000, prompts=64, tpb=32, spare=8192,
             rows=65536, short=True),
        # The one new token of a session of a small model (hidden 576), f16 pages: latency alone.
        dict(name="write_f16_1", kind="write", cache="f16", tables=1, rows=1, past=300, pad=0, n_heads=9, n_kv_heads=3,
             head_dim=64, tpb=16, weight="f16", out="f32"),
        # 64 decoding sessions of a model with 32 query heads over 8 kv heads, 4-bit pages; 7 rows of the step are padding.
        dict(name="write_q4_64", kind="write", cache="q4", tables=64, rows=1, past=900, pad=7, n_heads=32, n_kv_heads=8,
             head_dim=128, tpb=16, weight="f32", out="f16"),
        # A 2048-token prompt of that model enters an 8-bit cache.
        dict(name="write_q8_2048", kind="write", cache="q8", tables=1, rows=2048, past=0, pad=0, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=16, weight="f16", out="f32"),
        # Four prompts of 1999 tokens with the Gemma-3-1B shape (4 query heads of 256 over one kv head), 4-bit pages.
        dict(name="write_q4_7996", kind="write", cache="q4", tables=4, rows=1999, past=11, pad=5, n_heads=4,
             n_kv_heads=1, head_dim=256, tpb=16, weight="bf16", out="f32"),
        # One session of the Qwen2.5-0.5B shape some 700 tokens into an answer: a few microseconds.
        dict(name="attend_1_session", kind="attend", tables=1, rows=1, prompts=1, mixed=False, ctx=701, ragged=False,
             n_heads=14, n_kv_heads=2, head_dim=64, tpb=16, window=0, cap=0.0),
        # Eight sessions between 4096 and 8192 positions, 32 query heads over 8 kv heads.
        dict(name="attend_8_sessions_8k", kind="attend", tables=8, rows=1, prompts=8, mixed=False, ctx=8192, ragged=True,
             n_heads=32, n_kv_heads=8, head_dim=128, tpb=16, window=0, cap=0.0),
        # One very long context: 131072 positions, the largest read.
        dict(name="attend_131072", kind="attend", tables=1, rows=1, prompts=1, mixed=False, ctx=131072, ragged=False,
             n_heads=32, n_kv_heads=8, head_dim=128, tpb=32, window=0, cap=0.0),
        # The second 1024 tokens of a prompt that is read in parts: the largest products.
        dict(name="attend_prompt_1024", kind="attend", tables=1, rows=1024, prompts=1, mixed=False, ctx=2048,
             ragged=False, n_heads=32, n_kv_heads=8, head_dim=128, tpb=16, window=0, cap=0.0),
        # A step of 20 sessions: parts of 200 tokens of three prompts beside 17 decoding sessions, sliding window and
        # capped scores.
        dict(name="attend_mixed_20", kind="attend", tables=20, rows=200, prompts=3, mixed=True, ctx=4000, ragged=True,
             n_heads=16, n_kv_heads=4, head_dim=128, tpb=16, window=1024, cap=50.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    kind = rng.choice(["plan", "plan", "write", "write", "write", "attend", "attend", "attend", "attend"])
    tpb = rng.choice([16, 16, 32, 7, 64])
    if kind == "plan":
        tables = _log_int(rng, 1, 700)
        prompts = rng.choice([0, rng.randint(0, tables)])
        prompt = _log_int(rng, 2, 1000) if prompts else 0
        rows = tables + prompts * prompt
        return dict(kind=kind, tables=tables, ctx=_log_int(rng, 1, 5000), prompt=prompt, prompts=prompts, tpb=tpb,
                    spare=rng.randint(1, 4096), rows=rng.choice([rows, max(1, rows * 2 // 3)]), short=rng.random() < 0.3)
    nkv, group, hd = rng.randint(1, 8), rng.randint(1, 8), rng.choice([64, 128, 128, 256])
    heads = dict(n_heads=nkv * group, n_kv_heads=nkv, head_dim=hd, tpb=tpb)
    if kind == "write":
        rows = _log_int(rng, 1, 900)
        return dict(kind=kind, cache=rng.choice(["f16", "q8", "q4", "q4"]), tables=rng.randint(1, 8), rows=rows,
                    past=rng.randint(0, 2000), pad=rng.randint(0, rows - 1) if rng.random() < 0.4 else 0, **heads,
                    weight=rng.choice(["f32", "f16", "bf16"]), out=rng.choice(["f16", "f32"]))
    window, cap = rng.choice([0, 0, 512, 1024]), rng.choice([0.0, 0.0, 0.0, 50.0])
    if rng.random() < 0.3:  # a step with prompts and decoding sessions
        tables, ctx = _log_int(rng, 2, 40), _log_int(rng, 16, 5000)
        return dict(kind=kind, tables=tables, rows=rng.randint(2, min(ctx, 300)), prompts=rng.randint(0, min(tables, 4)),
                    mixed=True, ctx=ctx, ragged=rng.random() < 0.7, window=window, cap=cap, **heads)
    if rng.random() < 0.35:  # prompts, some of them padded to the longest
        ctx, tables = _log_int(rng, 8, 2048), rng.randint(1, 3)
        return dict(kind=kind, tables=tables, rows=rng.randint(max(1, ctx // 3), ctx), prompts=tables, mixed=False,
                    ctx=ctx, ragged=rng.random() < 0.5, window=window, cap=cap, **heads)
    tables = _log_int(rng, 1, 64)
    return dict(kind=kind, tables=tables, rows=1, prompts=tables, mixed=False, ctx=_log_int(rng, 1, 40000),
                ragged=rng.random() < 0.7, window=window, cap=cap, **heads)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw_one(rng)
        scores = pool = 0
        if c["kind"] == "attend":
            scores = c["tables"] * c["rows"] * c["n_heads"] * c["ctx"]
            pool = c["tables"] * c["ctx"] * c["n_kv_heads"] * c["head_dim"]
        if _cost(c) <= most and scores <= 4e8 and pool <= 2e8:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---- inputs ---------------------------------------------------------------------


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _contexts(case):
    """Positions held by each table: all the same, or spread from half of ctx to ctx."""
    n, ctx = case["tables"], case["ctx"]
    if not case.get("ragged") or n == 1:
        return [ctx] * n
    return [ctx - (ctx // 2) * i // (n - 1) for i in range(n)]


def _new_tokens(case):
    """Rows of each table of an attend case, in the order of _contexts."""
    new = case["rows"]
    if not case["mixed"]:
        return [new] * case["tables"]
    return [min(new if t < case["prompts"] else 1, n) for t, n in enumerate(_contexts(case))]


def _tables(g, tables, per, spare=3):
    """Shuffled pages, a few of them of other sessions."""
    total = tables * per + spare
    return torch.randperm(total, generator=g, device="cuda")[:tables * per].to(torch.int32).view(tables, per), total


def _quantise8(x):
    """Codes and scales of the vectors x[..., hd]: s = max|x| / 127, c = round-half-even(x / s)."""
    a = x.abs().amax(-1, keepdim=True)
    s = a / torch.full_like(a, 127.0)  # a tensor divides; a number would multiply by its reciprocal
    s = torch.where(s >= _TINY, s, torch.zeros_like(s))
    c = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))).clamp(-127, 127)
    c = torch.where(s > 0, c, torch.zeros_like(c))
    return c.to(torch.int8), s.squeeze(-1)


def _quantise4(x):
    """Codes [..., hd / 2] (the even dim of a byte in its low half) and (scale, base) [..., hd / 32, 2] of x[..., hd]."""
    g = x.clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    base = g.amin(-1, keepdim=True).half()
    b = base.float()
    r = g.amax(-1, keepdim=True) - b
    s = (r / torch.full_like(r, 15.0)).clamp(min=0.0).half()
    over = 15.0 * s.float() + b >= 65520.0  # the last code would stand for an infinity
    s = torch.where(over, (s.view(torch.int16) - 1).view(torch.float16), s)
    f = s.float()
    c = torch.round((g - b) / torch.where(f > 0, f, torch.ones_like(f))).clamp(0, 15)
    c = torch.where(f > 0, c, torch.zeros_like(c)).to(torch.uint8).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), torch.cat([s, base], -1)


def _keys(g, shape):
    """Keys have a few loud channels, values differ in size from token to token."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = torch.rand(shape[-1], generator=g, device="cuda") < 0.03
    return x * torch.where(loud, 6.0, 1.0)


def _values(g, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))


def _cache(g, case, total, layers, kind):
    """K and V pages: [block][layer][kv head][slot] vectors of codes with their scales, or f16 [block][layer][slot][kv
    head][dim]."""
    nkv, hd, tpb = case["n_kv_heads"], case["head_dim"], case["tpb"]
    if kind == "f16":
        shape = (total, layers, tpb, nkv, hd)
        return dict(k=_keys(g, shape).half(), v=_values(g, shape).half(), ks=None, vs=None)
    shape = (total, layers, nkv, tpb, hd)
    k, ks = (_quantise4 if kind == "q4" else _quantise8)(_keys(g, shape))
    v, vs = (_quantise4 if kind == "q4" else _quantise8)(_values(g, shape))
    return dict(k=k, ks=ks, v=v, vs=vs)


def _rope_table(positions, head_dim):
    half = head_dim // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / head_dim)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


_LAYERS, _LAYER = 2, 1  # caches of one layer's operators hold two, the second is used
_TYPES = dict(f32=torch.float32, f16=torch.float16, bf16=torch.bfloat16)


def _prepare_plan(case, g):
    n, tpb = case["tables"], case["tpb"]
    per = -(-(case["ctx"] + case["prompt"] + 1) // tpb)
    ctx = torch.randint(0, case["ctx"] + 1, (n,), generator=g, device="cuda", dtype=torch.int32)
    new = torch.ones(n, device="cuda", dtype=torch.int32)
    what = torch.rand(n, generator=g, device="cuda")
    new[what < 0.05] = 0    # idle
    new[what > 0.95] = -1   # finished
    if case["prompts"]:
        at = torch.randperm(n, generator=g, device="cuda")[:case["prompts"]]
        new[at] = torch.randint(1, case["prompt"] + 1, (case["prompts"],), generator=g, device="cuda", dtype=torch.int32)
    bt, total = _tables(g, n, per, case["spare"])
    held = (ctx + tpb - 1) // tpb
    j = torch.arange(per, device="cuda")
    bt = torch.where(j < held[:, None], bt, -1).contiguous()
    used = torch.zeros(total + 1, device="cuda", dtype=torch.int32)
    used[bt.long().reshape(-1)] = 1  # -1: the entry past the last page
    order = torch.randperm(total, generator=g, device="cuda")
    free = order[torch.argsort(used[:total][order], stable=True)].to(torch.int32)
    count = total - used[:total].sum(dtype=torch.int32).view(1)
    if case["short"]:  # pages for about two thirds of what is asked
        count = torch.minimum(count, (new.clamp(min=0).sum(dtype=torch.int32) * 2 // (3 * tpb) + 1).view(1)).to(torch.int32)
    rows = case["rows"]
    made = lambda k: torch.zeros(k, device="cuda", dtype=torch.int32)  # noqa: E731
    return dict(kind="plan", case=case, ctx=ctx, new=new, bt=bt, total=total, free=free, count=count, lens=made(n),
                left=made(1), starts=made(n + 1), pos=made(rows), slots=made(rows))


def _prepare_write(case, g):
    nkv, hd, tpb, tables, rows = case["n_kv_heads"], case["head_dim"], case["tpb"], case["tables"], case["rows"]
    st = dict(kind="write", case=case)
    st["bt"], st["total"] = _tables(g, tables, -(-(case["past"] + rows) // tpb))
    at = case["past"] + torch.arange(rows, device="cuda")
    st["slots"] = (st["bt"][:, at // tpb] * tpb + at % tpb).view(-1).to(torch.int32)
    st["pos"] = at.to(torch.int32).repeat(tables)
    n = tables * rows
    if case["pad"]:  # rows behind the step's last
        st["pos"][n - case["pad"]:] = -1
        st["slots"][n - case["pad"]:] = -1
    st.update(_cache(g, case, st["total"], _LAYERS, case["cache"]))
    st["q"] = torch.randn(n, case["n_heads"] * hd, generator=g, device="cuda") * 3.0
    st["kx"], st["vx"] = _keys(g, (n, nkv, hd)).view(n, -1), _values(g, (n, nkv, hd)).view(n, -1)
    st["qw"], st["kw"] = ((1.0 + 0.2 * torch.randn(hd, generator=g, device="cuda")).to(_TYPES[case["weight"]])
                          for _ in range(2))
    st["q_out"] = torch.zeros_like(st["q"])
    st["k_out"], st["v_out"] = (torch.zeros(n, nkv * hd, device="cuda", dtype=_TYPES[case["out"]]) for _ in range(2))
    st["cos_sin"] = _rope_table(case["past"] + rows, hd)
    return st


def _prepare_attend(case, g):
    tables, rows = case["tables"], case["rows"]
    st = dict(kind="attend", case=case)
    order = torch.randperm(tables, generator=g, device="cuda")
    lens = torch.tensor(_contexts(case), device="cuda", dtype=torch.int32)[order]
    st["bt"], st["total"] = _tables(g, tables, -(-case["ctx"] // case["tpb"]))
    if case["mixed"]:  # packed rows, a few of padding behind them
        new = torch.tensor(_new_tokens(case), device="cuda")[order]
        st["starts"] = torch.cat([new.new_zeros(1), new.cumsum(0)]).to(torch.int32)
        n = sum(_new_tokens(case)) + 3
        r = torch.arange(n, device="cuda")
        t = torch.searchsorted(st["starts"][1:].long(), r, right=True).clamp(max=tables - 1)
        pos = lens[t] - new[t] + r - st["starts"].long()[t]
        st["pos"] = torch.where(r < n - 3, pos, -1).to(torch.int32)
    else:  # the rows of a table are its last tokens; a shorter prompt is padded in front with rows of no position
        st["starts"] = None
        pos = (lens[:, None] - rows + torch.arange(rows, device="cuda", dtype=torch.int32)).clamp(min=-1)
        st["pos"] = pos.reshape(-1).contiguous()
        n = tables * rows
    st.update(_cache(g, case, st["total"], _LAYERS, "q4"))
    st["q"] = torch.randn(n, case["n_heads"] * case["head_dim"], generator=g, device="cuda") * 1.5
    st["out"] = torch.zeros_like(st["q"])
    return st


def prepare(case, seed):
    g = _gen(seed)
    return {"plan": _prepare_plan, "write": _prepare_write, "attend": _prepare_attend}[case["kind"]](case, g)


# ---- the plain forms ----------------------------------------------------------------


def _plain_plan(st):
    c = st["case"]
    n, tpb, total, rows = c["tables"], c["tpb"], st["total"], c["rows"]
    bt, ctx, new = st["bt"], st["ctx"].long(), st["new"].long()
    per = bt.shape[1]
    j = torch.arange(per, device="cuda")
    held = (ctx.clamp(min=0) + tpb - 1) // tpb
    there = (bt >= 0) & (bt < total)
    # the pages of finished sessions go onto the free ones
    back = ((new < 0) & (ctx >= 0))[:, None] & (j < held[:, None]) & there
    rank = back.reshape(-1).long().cumsum(0) - 1
    count = st["count"].long()
    free = torch.cat([st["free"], st["free"].new_zeros(1)])  # the last takes what is none
    at = torch.where(back.reshape(-1), count + rank, free.numel() - 1).clamp(max=free.numel() - 1)
    free = free.scatter(0, at, bt.reshape(-1))
    count = count + back.sum()
    # sessions in order, up to the first whose pages or rows are not there
    valid = (ctx >= 0) & (new > 0) & (ctx + new <= per * tpb)
    asked = torch.where(valid, new, 0)
    need = torch.where(valid, (ctx + new + tpb - 1) // tpb - held, 0)
    pages, taken = need.cumsum(0), asked.cumsum(0)
    got = valid & (pages <= count) & (taken <= rows)
    page = count - 1 - ((pages - need)[:, None] + j - held[:, None])
    mine = got[:, None] & (j >= held[:, None]) & (j < (held + need)[:, None])
    bt = torch.where(mine, free[page.clamp(0, free.numel() - 2)], bt)
    st["bt"].copy_(bt)
    st["free"].copy_(free[:-1])
    granted = torch.where(got, new, 0)
    starts = torch.cat([granted.new_zeros(1), granted.cumsum(0)])
    r = torch.arange(rows, device="cuda")
    t = torch.searchsorted(starts[1:], r, right=True).clamp(max=n - 1)
    p = ctx[t] + r - starts[t]
    some = r < starts[n]
    block = bt[t, (p // tpb).clamp(0, per - 1)].long()
    slot = torch.where(some & (block >= 0) & (block < total), block * tpb + p % tpb, -1)
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return dict(tables=st["bt"], free=st["free"], lens=i32(torch.where(new < 0, torch.where(ctx < 0, ctx, 0), ctx + granted)),
                left=i32(count - torch.where(got, need, 0).sum()), starts=i32(starts), pos=i32(torch.where(some, p, -1)),
                slots=i32(slot))


def _normed(x, w):
    """Each head vector over its root mean square, times the weights; the sum of squares and the root in 64 bits."""
    inv = 1.0 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + _EPS)
    return x * inv.float() * w.float()


def _rotate(x, c):
    """Rotate-half of the heads x [rows, heads, hd] by (cos, sin) [rows, hd / 2, 2]."""
    half = x.shape[-1] // 2
    x0, x1, co, si = x[..., :half], x[..., half:], c[:, None, :, 0], c[:, None, :, 1]
    return torch.cat([x0 * co - x1 * si, x1 * co + x0 * si], -1)


def _values4(codes, scales):
    """What 4-bit codes [..., hd / 2] with (scale, base) [..., hd / 32, 2] stand for, as f32."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, 32)).float()
    s = scales.float()
    return (c * s[..., :1] + s[..., 1:]).half().float().flatten(-2)


def _plain_write(st):
    c = st["case"]
    n, nkv, hd, tpb = st["pos"].numel(), c["n_kv_heads"], c["head_dim"], c["tpb"]
    some = (st["pos"] >= 0)[:, None]
    cs = st["cos_sin"][st["pos"].long().clamp(0, st["cos_sin"].shape[0] - 1)]
    q = _rotate(_normed(st["q"].view(n, -1, hd), st["qw"]), cs).view(n, -1)
    q = torch.where(some, q, st["q_out"])
    k = _rotate(_normed(st["kx"].view(n, nkv, hd), st["kw"]), cs)
    v = st["vx"].view(n, nkv, hd)
    # rows of no slot come last: what they write goes to the slot of the first row, which then has its own again
    slot = torch.where(st["slots"] >= 0, st["slots"], st["slots"][0]).long()
    block, off = slot // tpb, slot % tpb
    first = torch.where(st["slots"] >= 0, torch.arange(n, device="cuda"), 0)
    if c["cache"] == "f16":
        for x, page in ((k, "k"), (v, "v")):
            st[page][block, _LAYER, off] = x[first].half()
        return dict(q=q, k=st["k"], v=st["v"])
    outs = []
    for x, page, scale in ((k, "k", "ks"), (v, "v", "vs")):
        codes, s = (_quantise4 if c["cache"] == "q4" else _quantise8)(x[first])
        st[page][block, _LAYER, :, off] = codes
        st[scale][block, _LAYER, :, off] = s
        codes, s = st[page][block, _LAYER, :, off], st[scale][block, _LAYER, :, off]
        x = _values4(codes, s) if c["cache"] == "q4" else codes.float() * s[..., None]
        outs.append(torch.where(some, x.to(st["k_out"].dtype).view(n, -1), st["k_out"]))
    return dict(q=q, k=outs[0], v=outs[1])


def _plain_attend(st):
    c = st["case"]
    tables, nkv, nh, hd = c["tables"], c["n_kv_heads"], c["n_heads"], c["head_dim"]
    n = st["pos"].numel()
    r = torch.arange(n, device="cuda")
    most = c["rows"]
    if st["starts"] is None:
        t, i = r // most, r % most
        at = r.view(tables, most)
        real = at >= 0
    else:
        starts = st["starts"].long()
        t = torch.searchsorted(starts[1:], r, right=True).clamp(max=tables - 1)
        i = (r - starts[t]).clamp(max=most - 1)
        at = starts[:-1, None] + torch.arange(most, device="cuda")
        real = at < starts[1:, None]
        at = at.clamp(max=n - 1)
    bt = st["bt"].long()
    k, v = (_values4(st[x][:, _LAYER][bt], st[x + "s"][:, _LAYER][bt]).permute(0, 2, 1, 3, 4).reshape(tables, nkv, -1, hd)
            for x in ("k", "v"))
    q = st["q"].view(n, nkv, nh // nkv, hd)[at].transpose(1, 2).reshape(tables, nkv, -1, hd)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    pos = torch.where(real, st["pos"][at].long(), -1)[..., None]
    p = torch.arange(k.shape[2], device="cuda")
    seen = (p <= pos) & (p > pos - c["window"]) if c["window"] else p <= pos
    s = s.view(tables, nkv, most, nh // nkv, -1)
    s = torch.where(seen[:, None, :, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = w.sum(-1, keepdim=True)
    o = torch.matmul(w.view(tables, nkv, -1, w.shape[-1]), v).view(tables, nkv, most, nh // nkv, hd)
    o = (o / torch.where(l > 0, l, torch.ones_like(l))).transpose(1, 2).reshape(tables, most, nh * hd)
    return torch.where((st["pos"] >= 0)[:, None], o[t, i], st["out"])


# ---- the framework's operators ----------------------------------------------------------


def _own_plan(st):
    _hip().encode_kv_plan(st["ctx"], st["new"], st["bt"], st["total"], st["case"]["tpb"], st["free"], st["count"],
                          st["lens"], st["left"], st["starts"], st["pos"], st["slots"])
    return dict(tables=st["bt"], free=st["free"], lens=st["lens"], left=st["left"], starts=st["starts"], pos=st["pos"],
                slots=st["slots"])


def _own_write(st):
    ops, c = _hip(), st["case"]
    nkv, hd, tpb, total = c["n_kv_heads"], c["head_dim"], c["tpb"], st["total"]
    ops.encode_norm_rope_kv_write(st["q"], st["kx"], st["vx"], st["q_out"], c["n_heads"], nkv, hd, st["qw"], st["kw"], _EPS,
                                  st["pos"], st["cos_sin"], st["slots"], st["k"], st["v"], total, _LAYERS, tpb, _LAYER,
                                  kscale=st["ks"], vscale=st["vs"])
    if c["cache"] == "f16":
        return dict(q=st["q_out"], k=st["k"], v=st["v"])
    read = ops.encode_kv_read_q4 if c["cache"] == "q4" else ops.encode_kv_read_q8
    read(st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["pos"], st["k_out"], st["v_out"], nkv, hd, total, _LAYERS, tpb,
         _LAYER, rows_per_table=c["rows"])
    return dict(q=st["q_out"], k=st["k_out"], v=st["v_out"])


def _own_attend(st):
    c = st["case"]
    _hip().encode_attention_q4(st["q"], st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["pos"], st["out"], c["n_heads"],
                               c["n_kv_heads"], c["head_dim"], st["total"], _LAYERS, c["tpb"], _LAYER, soft_cap=c["cap"],
                               window=c["window"], rows_per_table=c["rows"] if st["starts"] is None else 1,
                               row_starts_i32=st["starts"])
    return st["out"]


def run(state):
    if own:
        return {"plan": _own_plan, "write": _own_write, "attend": _own_attend}[state["kind"]](state)
    return {"plan": _plain_plan, "write": _plain_write, "attend": _plain_attend}[state["kind"]](state)


# ---- what a pass cannot do without --------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "plan":  # lengths in and out, a page entry read and written for each page taken, positions and slots
        new = case["tables"] + case["prompts"] * case["prompt"] // 2
        return dict(bytes=16 * case["tables"] + 8 * (new // case["tpb"]) + 8 * case["rows"] + 16, flops=0)
    nkv, nh, hd, tables = case["n_kv_heads"], case["n_heads"], case["head_dim"], case["tables"]
    if kind == "write":
        n = tables * case["rows"] - case["pad"]
        vec = {"f16": 2 * hd, "q8": hd + 4, "q4": hd // 2 + hd // 8}[case["cache"]]
        back = 0 if case["cache"] == "f16" else vec + hd * (2 if case["out"] == "f16" else 4)
        return dict(bytes=n * (8 * nh * hd + 2 * nkv * (4 * hd + vec + back) + 4 * hd + 8),
                    flops=n * hd * (6 * (nh + nkv) + 6 * nkv))
    vec, window = hd // 2 + hd // 8, case["window"]
    read = seen = rows = 0
    for n, new in zip(_contexts(case), _new_tokens(case)):
        lens = [p + 1 for p in range(max(0, n - new), n)]
        lens = [min(x, window) if window else x for x in lens]
        read += min(n, window + len(lens) - 1) if window else n
        seen += sum(lens)
        rows += len(lens)
    return dict(bytes=2 * vec * nkv * read + 8 * rows * nh * hd, flops=4 * hd * nh * seen)


# ---- results in 64 bits -----------------------------------------------------------------


def _f16(x):
    """f64 numbers rounded to the nearest f16, halves to even, at once, as f64 (finite ones below 65520)."""
    _, e = torch.frexp(x)
    step = ((e - 11).clamp(min=-24).long() + 1023 << 52).view(torch.float64)  # the power of two itself
    return torch.round(x / step) * step


def _exact_turned(x, w, cs, wide):
    """Norm, weights and rotation of x [rows, heads, hd] as numpy arrays: all in 64 bits, or (the vectors that are
    quantised, whose codes are defined in 32 bits) each product and sum rounded once."""
    t = np.float64 if wide else np.float32
    inv = 1.0 / np.sqrt(np.square(x.astype(np.float64)).sum(-1, keepdims=True) / x.shape[-1] + _EPS)
    y = x.astype(t) * inv.astype(t) * w.astype(t)
    lo, hi = np.split(y, 2, axis=-1)
    co, si = cs[:, None, :, 0].astype(t), cs[:, None, :, 1].astype(t)
    return np.concatenate([lo * co - hi * si, hi * co + lo * si], axis=-1)


def _exact_held(x, kind):
    """The values that the pages hold for f32 vectors, in 64 bits."""
    if kind == "q8":
        a = np.abs(x).max(-1, keepdims=True)
        s = (a / np.float32(127)).astype(np.float32)
        s[s < np.float32(_TINY)] = 0
        with np.errstate(divide="ignore", invalid="ignore"):
            code = np.where(s > 0, np.clip(np.rint((x / s).astype(np.float32)), -127, 127), 0)
        return code.astype(np.float64) * s.astype(np.float64)
    y = np.clip(x, np.float32(-65504), np.float32(65504)).reshape(x.shape[:-1] + (-1, 32))
    z = y.min(-1, keepdims=True).astype(np.float16).astype(np.float32)
    s = np.maximum((y.max(-1, keepdims=True) - z) / np.float32(15), np.float32(0)).astype(np.float16)
    s = np.where(s.astype(np.float64) * 15 + z >= 65520, np.nextafter(s, np.float16(0)), s).astype(np.float32)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(s > 0, np.clip(np.rint((y - z) / s), 0, 15), 0)
    return (code.astype(np.float64) * s + z).astype(np.float16).astype(np.float64).reshape(x.shape)


def _exact_write(st):
    c = st["case"]
    n, hd, tpb = st["pos"].numel(), c["head_dim"], c["tpb"]
    live = st["pos"].cpu().numpy() >= 0
    cs = st["cos_sin"].cpu().numpy()[st["pos"].cpu().numpy() * live]
    host = lambda name: st[name].cpu().numpy().reshape(n, -1, hd)  # noqa: E731
    qw, kw = st["qw"].float().cpu().numpy(), st["kw"].float().cpu().numpy()
    q = _exact_turned(host("q"), qw, cs, True) * live[:, None, None]
    k = _exact_turned(host("kx"), kw, cs, c["cache"] == "f16")
    found = dict(q=torch.from_numpy(q.reshape(n, -1)))
    for name, x in (("k", k), ("v", host("vx"))):
        if c["cache"] == "f16":
            pages = st[name].double().cpu()
            slot = st["slots"].cpu().numpy()
            for row in np.flatnonzero(slot >= 0):
                pages[slot[row] // tpb, _LAYER, slot[row] % tpb] = torch.from_numpy(x[row].astype(np.float64))
            found[name] = pages
        else:
            found[name] = torch.from_numpy((_exact_held(x, c["cache"]) * live[:, None, None]).reshape(n, -1))
    return found


def _exact_tokens(st, t, positions, page, scale):
    """K or V of a table's positions in 64 bits: [positions, kv heads, hd]."""
    tpb = st["case"]["tpb"]
    block, off = st["bt"][t, positions // tpb].long(), positions % tpb
    codes, s = st[page][block, _LAYER, :, off], st[scale][block, _LAYER, :, off].double()
    c = torch.empty(codes.shape[:2] + (codes.shape[2] * 2,), dtype=torch.float64, device="cuda")
    c[..., 0::2], c[..., 1::2] = codes % 16, codes // 16
    return _f16(c * s[..., 0].repeat_interleave(32, -1) + s[..., 1].repeat_interleave(32, -1))


def _exact_attend(st):
    c = st["case"]
    nkv, nh, hd = c["n_kv_heads"], c["n_heads"], c["head_dim"]
    n = st["pos"].numel()
    q = st["q"].double().view(n, nh, hd)
    out = torch.zeros_like(q)
    starts = [c["rows"] * t for t in range(c["tables"] + 1)] if st["starts"] is None else st["starts"].tolist()
    for t in range(c["tables"]):
        a, b = starts[t], starts[t + 1]
        pos = st["pos"][a:b].long()
        at = torch.arange(int(pos.max()) + 1, device="cuda")
        sees = at[None] <= pos[:, None]
        if c["window"]:
            sees &= at[None] + c["window"] > pos[:, None]
        k, v = _exact_tokens(st, t, at, "k", "ks"), _exact_tokens(st, t, at, "v", "vs")
        some = sees.any(1)
        for h in range(nh):
            s = q[a:b, h] @ k[:, h * nkv // nh].T / math.sqrt(hd)
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            s.masked_fill_(~sees, -math.inf)
            s[~some] = 0.0
            out[a:b, h] = torch.softmax(s, 1) @ v[:, h * nkv // nh] * some[:, None]
    return out.view(n, nh * hd)


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    return _exact_write(st) if case["kind"] == "write" else _exact_attend(st)
