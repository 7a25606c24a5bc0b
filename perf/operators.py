"""Operators over a paged K/V cache, as cases for timing and for checking outputs.

The cache holds 8-bit codes with one f32 scale per (token, kv head), or f16; the
operators write it, read it back, attend to it (one row per session, prompts, and trees
of drafted tokens) and keep the accepted path of a tree.  Where `own` is false, `run`
computes them with elementary torch operations in 32 bits; where it is true, through
HipOps.  The kinds:

  write    RoPE on q and k, K and V quantised into the pages, and the written tokens read
           back as f32 (what the 8-bit codes stand for)
  read     a session's K and V read back from 8-bit pages, as f16 or f32
  attend   attention over 8-bit pages: the last token of every session, or the new tokens
           of prompts, whose rows share one table
  tree     attention of the nodes of drafted trees over f16 or 8-bit pages
  accept   the accepted path's K and V moved behind the context, in every layer
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


_TINY = 1.1754943508222875e-38  # the smallest normal f32: scales below it are 0


def listed():
    return [
        # The smallest calls: the one new token of one session of a small model (hidden 576), latency alone.
        dict(name="write_decode_1", kind="write", tables=1, rows=1, past=300, tree=False, n_heads=9, n_kv_heads=3,
             head_dim=64, tpb=16),
        # A 2048-token prompt of a model with 32 query heads over 8 kv heads enters the cache.
        dict(name="write_prompt_2048", kind="write", tables=1, rows=2048, past=0, tree=False, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=16),
        # A session's 8000 tokens leave the cache (to be moved, or for a consumer of f16): an odd count.
        dict(name="read_8000", kind="read", tables=1, rows=8000, past=0, n_kv_heads=8, head_dim=128, tpb=16,
             dtype="f16"),
        # One session of the Qwen2.5-0.5B shape some 700 tokens into an answer: a few microseconds.
        dict(name="attend_1_session", kind="attend", tables=1, rows=1, ctx=701, ragged=False, n_heads=14,
             n_kv_heads=2, head_dim=64, tpb=16, window=0, cap=0.0),
        # Eight sessions between 4096 and 8192 positions, 32 query heads over 8 kv heads.
        dict(name="attend_8_sessions_8k", kind="attend", tables=8, rows=1, ctx=8192, ragged=True, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=16, window=0, cap=0.0),
        # One very long context: 131072 positions, the largest read.
        dict(name="attend_131072", kind="attend", tables=1, rows=1, ctx=131072, ragged=False, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=32, window=0, cap=0.0),
        # The second 1024 tokens of a prompt that is read in parts: the largest products.
        dict(name="attend_prompt_1024", kind="attend", tables=1, rows=1024, ctx=2048, ragged=False, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=16, window=0, cap=0.0),
        # A sliding layer of the Gemma-3-1B shape (4 query heads of 256 over one kv head, window 512) with capped
        # scores, sixteen sessions.
        dict(name="attend_window_16", kind="attend", tables=16, rows=1, ctx=4096, ragged=True, n_heads=4,
             n_kv_heads=1, head_dim=256, tpb=16, window=512, cap=50.0),
        # One session's tree of 26 drafted tokens over the f16 cache, Qwen2.5-0.5B shape.
        dict(name="tree_f16_26", kind="tree", cache="f16", tables=1, tree=26, ctx=1000, ragged=False, n_heads=14,
             n_kv_heads=2, head_dim=64, tpb=16, window=0, cap=0.0),
        # Eight sessions' trees of 63 tokens over 8-bit pages, contexts of 2048 to 4096.
        dict(name="tree_q8_8x63", kind="tree", cache="q8", tables=8, tree=63, ctx=4096, ragged=True, n_heads=32,
             n_kv_heads=8, head_dim=128, tpb=16, window=0, cap=0.0),
        # After the check of one drafted tree: the accepted tokens' K and V move, 24 layers of the f16 cache.
        dict(name="accept_f16_4", kind="accept", cache="f16", tables=4, tree=26, ctx=300, n_layers=24, n_kv_heads=2,
             head_dim=64, tpb=16),
        # The same for 8 sessions of a 32-layer model over 8-bit pages.
        dict(name="accept_q8_8", kind="accept", cache="q8", tables=8, tree=63, ctx=200, n_layers=32, n_kv_heads=8,
             head_dim=128, tpb=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    kind = rng.choice(["write", "read", "attend", "attend", "attend", "tree", "tree", "accept"])
    nkv, group, hd, tpb = rng.randint(1, 8), rng.randint(1, 8), rng.choice([64, 128, 128, 256]), rng.choice([16, 16, 32, 7, 64])
    heads = dict(n_heads=nkv * group, n_kv_heads=nkv, head_dim=hd, tpb=tpb)
    if kind == "write":
        return dict(kind=kind, tables=rng.randint(1, 8), rows=_log_int(rng, 1, 700), past=rng.randint(0, 2000),
                    tree=rng.random() < 0.3, **heads)
    if kind == "read":
        del heads["n_heads"]
        return dict(kind=kind, tables=rng.randint(1, 4), rows=_log_int(rng, 1, 8000), past=rng.randint(0, 500),
                    dtype=rng.choice(["f16", "f32"]), **heads)
    window, cap = rng.choice([0, 0, 512, 1024]), rng.choice([0.0, 0.0, 0.0, 50.0])
    if kind == "attend":
        if rng.random() < 0.35:  # prompts, some of them padded to the longest
            ctx = _log_int(rng, 8, 2048)
            return dict(kind=kind, tables=rng.randint(1, 3), rows=rng.randint(max(1, ctx // 3), ctx), ctx=ctx,
                        ragged=rng.random() < 0.5, window=window, cap=cap, **heads)
        return dict(kind=kind, tables=_log_int(rng, 1, 64), rows=1, ctx=_log_int(rng, 1, 40000),
                    ragged=rng.random() < 0.7, window=window, cap=cap, **heads)
    if kind == "tree":
        return dict(kind=kind, cache=rng.choice(["f16", "q8"]), tables=_log_int(rng, 1, 16),
                    tree=_log_int(rng, 2, 100), ctx=_log_int(rng, 1, 16000), ragged=rng.random() < 0.7,
                    window=window, cap=cap, **heads)
    del heads["n_heads"]
    return dict(kind=kind, cache=rng.choice(["f16", "q8"]), tables=_log_int(rng, 1, 16), tree=_log_int(rng, 2, 100),
                ctx=_log_int(rng, 1, 600), n_layers=rng.randint(1, 32), **heads)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw_one(rng)
        pool = c.get("n_layers", 1) * c["tables"] * (c.get("ctx", 0) + c.get("tree", 0)) * c["n_kv_heads"] * c["head_dim"]
        if _cost(c) <= most and (c["kind"] != "accept" or pool <= 64e6):
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


def _tables(g, tables, per, spare=3):
    """Shuffled pages, a few of them of other sessions."""
    total = tables * per + spare
    return torch.randperm(total, generator=g, device="cuda")[:tables * per].to(torch.int32).view(tables, per), total


def _quantise(x):
    """Codes and scales of the vectors x[..., hd]: s = max|x| / 127, c = round-half-even(x / s)."""
    a = x.abs().amax(-1, keepdim=True)
    s = a / torch.full_like(a, 127.0)  # a tensor divides; a number would multiply by its reciprocal
    s = torch.where(s >= _TINY, s, torch.zeros_like(s))
    c = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))).clamp(-127, 127)
    c = torch.where(s > 0, c, torch.zeros_like(c))
    return c.to(torch.int8), s.squeeze(-1)


def _keys(g, shape):
    """Keys have a few loud channels, values differ in size from token to token."""
    x = torch.randn(shape, generator=g, device="cuda")
    loud = torch.rand(shape[-1], generator=g, device="cuda") < 0.03
    return x * torch.where(loud, 6.0, 1.0)


def _values(g, shape):
    x = torch.randn(shape, generator=g, device="cuda")
    return x * torch.exp(0.5 * torch.randn(shape[:-1] + (1,), generator=g, device="cuda"))


def _cache(g, case, total, layers):
    """K and V pages: [block][layer][kv head][slot][dim] codes with [block][layer][kv head][slot] scales, or f16
    [block][layer][slot][kv head][dim]."""
    nkv, hd, tpb = case["n_kv_heads"], case["head_dim"], case["tpb"]
    if case.get("cache") == "f16":
        shape = (total, layers, tpb, nkv, hd)
        return dict(k=_keys(g, shape).half(), v=_values(g, shape).half(), ks=None, vs=None)
    shape = (total, layers, nkv, tpb, hd)
    k, ks = _quantise(_keys(g, shape))
    v, vs = _quantise(_values(g, shape))
    return dict(k=k, ks=ks, v=v, vs=vs)


def _rope_table(positions, head_dim):
    half = head_dim // 2
    inv = 10000.0 ** (-2.0 * torch.arange(half, device="cuda", dtype=torch.float64) / head_dim)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _tree_parents(g, tables, tree):
    """Parents of every node (-1: the context's last token), always of a lower number; drafts are bushy near the root."""
    r = torch.rand(tables, tree, generator=g, device="cuda", dtype=torch.float64).cpu().numpy()
    return np.array([[-1 if j < min(3, tree) else int(j * r[t, j] * 0.7) for j in range(tree)] for t in range(tables)])


def _tree_masks(parents):
    """int64 words of 64 nodes: bit i of node j's words is set where j descends from i or is i."""
    tables, tree = parents.shape
    words = (tree + 63) // 64
    bits = np.zeros((tables, tree, words * 64), bool)
    for j in range(tree):
        for t in range(tables):
            if parents[t, j] >= 0:
                bits[t, j] = bits[t, parents[t, j]]
        bits[:, j, j] = True
    return np.packbits(bits, axis=-1, bitorder="little").view("<i8").reshape(tables, tree, words)


_LAYERS, _LAYER = 2, 1  # caches of one layer's operators hold two, the second is used


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    nkv, hd, tpb, tables = case["n_kv_heads"], case["head_dim"], case["tpb"], case["tables"]
    st = dict(kind=kind, case=case)
    if kind in ("write", "read"):
        rows = case["rows"]
        st["bt"], st["total"] = _tables(g, tables, -(-(case["past"] + rows) // tpb))
        at = case["past"] + torch.arange(rows, device="cuda", dtype=torch.int32)
        st["pos"] = at.repeat(tables)
        st.update(_cache(g, case, st["total"], _LAYERS))
        n = tables * rows
        out = torch.float16 if case.get("dtype") == "f16" else torch.float32
        st["k_out"], st["v_out"] = (torch.zeros(n, nkv * hd, device="cuda", dtype=out) for _ in range(2))
        if kind == "write":
            st["q"] = torch.randn(n, case["n_heads"] * hd, generator=g, device="cuda") * 1.5
            st["kx"], st["vx"] = _keys(g, (n, nkv, hd)).view(n, -1), _values(g, (n, nkv, hd)).view(n, -1)
            st["q_out"] = torch.zeros_like(st["q"])
            st["cos_sin"] = _rope_table(case["past"] + rows, hd)
            st["slots"] = None
            if case["tree"]:  # drafted tokens: slots in a row, positions by their depth
                depth = _tree_masks(_tree_parents(g, tables, rows))
                depth = np.unpackbits(depth.view(np.uint8), axis=-1).reshape(tables, rows, -1).sum(-1) - 1
                st["slots"] = st["pos"]
                st["pos"] = (case["past"] + torch.from_numpy(depth.astype(np.int32)).cuda()).view(-1).contiguous()
        return st
    if kind == "attend":
        rows, lens = case["rows"], torch.tensor(_contexts(case), device="cuda", dtype=torch.int32)
        lens = lens[torch.randperm(tables, generator=g, device="cuda")]
        st["bt"], st["total"] = _tables(g, tables, -(-case["ctx"] // tpb))
        # the rows of a table are its last tokens; a shorter prompt is padded in front with rows of no position
        st["pos"] = (lens[:, None] - rows + torch.arange(rows, device="cuda", dtype=torch.int32)).clamp(min=-1)
        st["pos"] = st["pos"].reshape(-1).contiguous()
        n = tables * rows
    elif kind == "tree":
        lens = torch.tensor(_contexts(case), device="cuda", dtype=torch.int32)
        st["ctx"] = lens[torch.randperm(tables, generator=g, device="cuda")]
        st["bt"], st["total"] = _tables(g, tables, -(-(case["ctx"] + case["tree"]) // tpb))
        st["masks"] = torch.from_numpy(_tree_masks(_tree_parents(g, tables, case["tree"]))).cuda()
        n = tables * case["tree"]
    else:
        tree = case["tree"]
        st["ctx"] = torch.tensor(_contexts(case), device="cuda", dtype=torch.int32)
        st["bt"], st["total"] = _tables(g, tables, -(-(case["ctx"] + tree) // tpb))
        parents, most = _tree_parents(g, tables, tree), min(tree, 8)
        acc = np.full((tables, most), -1, np.int32)
        for t in range(tables):  # the path to some node, its root first
            j, path = int(torch.randint(tree // 2, tree, (1,), generator=g, device="cuda")), []
            while j >= 0:
                path.append(j)
                j = parents[t, j]
            path = path[::-1][:most]
            acc[t, :len(path)] = path
        st["accepted"] = torch.from_numpy(acc).cuda()
        st.update(_cache(g, case, st["total"], case["n_layers"]))
        return st
    st.update(_cache(g, case, st["total"], _LAYERS))
    st["q"] = torch.randn(n, case["n_heads"] * hd, generator=g, device="cuda") * 1.5
    st["out"] = torch.zeros_like(st["q"])
    return st


# ---- the plain forms ----------------------------------------------------------------


def _rotate(x, c):
    """Rotate-half of the heads x [rows, heads, hd] by (cos, sin) [rows, hd / 2, 2]."""
    half = x.shape[-1] // 2
    x0, x1, co, si = x[..., :half], x[..., half:], c[:, None, :, 0], c[:, None, :, 1]
    return torch.cat([x0 * co - x1 * si, x1 * co + x0 * si], -1)


def _plain_write(st):
    c = st["case"]
    n, nkv, hd, tpb = st["pos"].numel(), c["n_kv_heads"], c["head_dim"], c["tpb"]
    cs = st["cos_sin"][st["pos"].long().clamp(0, st["cos_sin"].shape[0] - 1)]
    slot = (st["pos"] if st["slots"] is None else st["slots"]).long()
    table = torch.arange(n, device="cuda") // c["rows"]
    block, off = st["bt"][table, slot // tpb].long(), slot % tpb
    q = _rotate(st["q"].view(n, -1, hd), cs).view(n, -1)
    for x, code, scale in ((_rotate(st["kx"].view(n, nkv, hd), cs), "k", "ks"), (st["vx"].view(n, nkv, hd), "v", "vs")):
        codes, s = _quantise(x)
        st[code][block, _LAYER, :, off] = codes
        st[scale][block, _LAYER, :, off] = s
    k, v = _plain_read(st, slot)
    return dict(q=q, k=k, v=v)


def _plain_read(st, slot):
    c = st["case"]
    table = torch.arange(slot.numel(), device="cuda") // c["rows"]
    block, off = st["bt"][table, slot // c["tpb"]].long(), slot % c["tpb"]
    return [(st[code][block, _LAYER, :, off].float() * st[scale][block, _LAYER, :, off][..., None])
            .to(st["k_out"].dtype).view(slot.numel(), -1) for code, scale in (("k", "ks"), ("v", "vs"))]


def _plain_gather(st, code, scale):
    """The tables' K or V as f32 [tables, kv heads, positions, hd]."""
    x = st[code][:, _LAYER][st["bt"].long()]
    if st[scale] is None:
        x = x.permute(0, 3, 1, 2, 4).float()  # [tables, pages, slots, kv heads, hd]
    else:
        x = (x.float() * st[scale][:, _LAYER][st["bt"].long()][..., None]).permute(0, 2, 1, 3, 4)
    return x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])


def _plain_attention(st, seen):
    """seen [tables, rows, positions]: which positions each row attends to."""
    c = st["case"]
    tables, rows, _ = seen.shape
    nkv, hd, nh = c["n_kv_heads"], c["head_dim"], c["n_heads"]
    k, v = _plain_gather(st, "k", "ks"), _plain_gather(st, "v", "vs")
    q = st["q"].view(tables, rows, nkv, nh // nkv, hd).transpose(1, 2).reshape(tables, nkv, -1, hd)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    if c["cap"]:
        s = torch.tanh(s / c["cap"]) * c["cap"]
    s = s.view(tables, nkv, rows, nh // nkv, -1)
    s = torch.where(seen[:, None, :, None, :], s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(tables, nkv, -1, p.shape[-1]), v).view(tables, nkv, rows, nh // nkv, hd)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    return o.transpose(1, 2).reshape(tables * rows, nh * hd)


def _seen_causal(st):
    c = st["case"]
    pos = st["pos"].view(c["tables"], c["rows"], 1)
    p = torch.arange(st["bt"].shape[1] * c["tpb"], device="cuda")
    return (p <= pos) & (p > pos - c["window"]) if c["window"] else p <= pos


def _seen_tree(st):
    c = st["case"]
    p = torch.arange(st["bt"].shape[1] * c["tpb"], device="cuda")
    ctx, masks, tree = st["ctx"].view(-1, 1, 1).long(), st["masks"], c["tree"]
    bit = (p - ctx).clamp(0, tree - 1).expand(-1, tree, -1)
    drafted = (torch.gather(masks, 2, bit // 64) >> (bit % 64)) & 1
    context = p < ctx
    if c["window"]:
        depth = torch.zeros_like(ctx)
        for w in range(masks.shape[2]):
            depth = depth + ((masks[:, :, w:w + 1, None] >> torch.arange(64, device="cuda")) & 1).sum(-1)
        context = context & (p > ctx + depth - 1 - c["window"])
    return context | ((p >= ctx) & (p < ctx + tree) & (drafted > 0))


def _plain_accept(st):
    c = st["case"]
    most, tpb = st["accepted"].shape[1], c["tpb"]
    at = torch.arange(most, device="cuda")
    src = st["ctx"][:, None] + torch.where(st["accepted"] >= 0, st["accepted"], at)  # past the path: onto itself
    dst = (st["ctx"][:, None] + at).reshape(-1).long()
    src = src.reshape(-1).long()
    table = torch.arange(c["tables"], device="cuda").repeat_interleave(most)
    bs, bd = st["bt"][table, src // tpb].long(), st["bt"][table, dst // tpb].long()
    if c["cache"] == "f16":
        for x in (st["k"], st["v"]):
            x[bd, :, dst % tpb] = x[bs, :, src % tpb]
        return dict(k=st["k"], v=st["v"])
    for x in (st["k"], st["v"], st["ks"], st["vs"]):
        x[bd, :, :, dst % tpb] = x[bs, :, :, src % tpb]
    return {n: st[n] for n in ("k", "v", "ks", "vs")}  # bytes are moved, none is computed: the codes as they are


def _run_plain(st):
    kind, c = st["kind"], st["case"]
    if kind == "write":
        return _plain_write(st)
    if kind == "read":
        return _plain_read(st, st["pos"].long())
    if kind == "attend":
        return _plain_attention(st, _seen_causal(st))
    if kind == "tree":
        return _plain_attention(st, _seen_tree(st))
    return _plain_accept(st)


# ---- the framework's operators ----------------------------------------------------------


def _run_own(st):
    ops, kind, c = _hip(), st["kind"], st["case"]
    nkv, hd, tpb, total = c["n_kv_heads"], c["head_dim"], c["tpb"], st["total"]
    if kind in ("write", "read"):
        slots = st["pos"]
        if kind == "write":
            slots = st["pos"] if st["slots"] is None else st["slots"]
            ops.encode_rope_kv_write_q8(st["q"], st["kx"], st["vx"], st["q_out"], c["n_heads"], nkv, hd, st["pos"],
                                        st["cos_sin"], st["k"], st["ks"], st["v"], st["vs"], st["bt"], total, _LAYERS,
                                        tpb, _LAYER, slots_i32=st["slots"], rows_per_table=c["rows"])
        ops.encode_kv_read_q8(st["k"], st["ks"], st["v"], st["vs"], st["bt"], slots, st["k_out"], st["v_out"], nkv, hd,
                              total, _LAYERS, tpb, _LAYER, rows_per_table=c["rows"])
        return [st["k_out"], st["v_out"]] if kind == "read" else dict(q=st["q_out"], k=st["k_out"], v=st["v_out"])
    if kind == "attend":
        ops.encode_attention_q8(st["q"], st["k"], st["ks"], st["v"], st["vs"], st["bt"], st["pos"], st["out"],
                                c["n_heads"], nkv, hd, total, _LAYERS, tpb, _LAYER, soft_cap=c["cap"],
                                window=c["window"], rows_per_table=c["rows"])
        return st["out"]
    if kind == "tree":
        ops.encode_attention_tree(st["q"], st["k"], st["v"], st["bt"], st["ctx"], st["masks"], st["out"], c["n_heads"],
                                  nkv, hd, total, _LAYERS, tpb, _LAYER, kscale=st["ks"], vscale=st["vs"],
                                  soft_cap=c["cap"], window=c["window"])
        return st["out"]
    ops.encode_kv_accept(st["k"], st["v"], st["bt"], st["ctx"], st["accepted"], c["tree"], nkv, hd, total,
                         c["n_layers"], tpb, kscale=st["ks"], vscale=st["vs"])
    return {n: st[n] for n in ("k", "v", "ks", "vs") if st[n] is not None}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------


def work(case):
    kind, nkv, hd, tables = case["kind"], case["n_kv_heads"], case["head_dim"], case["tables"]
    q8 = hd + 4  # bytes of a vector's codes and scale
    if kind in ("write", "read"):
        n = tables * case["rows"]
        if kind == "read":
            return dict(bytes=2 * n * nkv * (q8 + hd * (2 if case["dtype"] == "f16" else 4)) + 8 * n, flops=2 * n * nkv * hd)
        # q, k, v in, q out, codes and scales written and read, K and V out again
        return dict(bytes=n * (8 * case["n_heads"] * hd + 2 * nkv * (8 * hd + 2 * q8) + 4 * hd + 8),
                    flops=n * hd * (3 * (case["n_heads"] + nkv) + 6 * nkv))
    if kind == "accept":
        path = min(case["tree"], 5) * tables * case["n_layers"] * 2 * nkv  # vectors of a path of about five nodes
        return dict(bytes=2 * path * (2 * hd if case["cache"] == "f16" else q8) + 4 * tables * 8, flops=0)
    nh, window, vec = case["n_heads"], case["window"], 2 * hd if case.get("cache") == "f16" else q8
    read = seen = rows = 0
    for n in _contexts(case):
        if kind == "tree":
            lens = [(min(n, window) if window else n) + min(4, case["tree"])] * case["tree"]
            read += (min(n, window) if window else n) + case["tree"]
        else:
            lens = [p + 1 for p in range(max(0, n - case["rows"]), n)]
            lens = [min(x, window) if window else x for x in lens]
            read += min(n, window + len(lens) - 1) if window else n
        seen += sum(lens)
        rows += len(lens)
    return dict(bytes=2 * vec * nkv * read + 8 * rows * nh * hd, flops=4 * hd * nh * seen)


# ---- results in 64 bits -----------------------------------------------------------------


def _exact_quantised(x):
    """The values that a vector's codes stand for.  The code of an element is defined in 32 bits (one division for the
    scale, one for the quotient), so these are rounded here too; the value, code times scale, is not."""
    a = np.abs(x).max(-1, keepdims=True)
    s = (a / np.float32(127)).astype(np.float32)
    s[s < np.float32(_TINY)] = 0
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint((x / s).astype(np.float32)), -127, 127), 0)
    return c.astype(np.float64) * s.astype(np.float64)


def _exact_write(st):
    c = st["case"]
    n, hd = st["pos"].numel(), c["head_dim"]
    cs = st["cos_sin"].cpu().numpy()[st["pos"].cpu().numpy()][:, None]  # [rows, 1, half, 2]

    def turned(x, t):  # in x's and t's precision, each product and sum rounded once
        lo, hi = np.split(x, 2, axis=-1)
        return np.concatenate([lo * t[..., 0] - hi * t[..., 1], hi * t[..., 0] + lo * t[..., 1]], axis=-1)

    q = turned(st["q"].double().cpu().numpy().reshape(n, -1, hd), cs.astype(np.float64))
    k = _exact_quantised(turned(st["kx"].cpu().numpy().reshape(n, -1, hd), cs))  # what is quantised is the f32 vector
    v = _exact_quantised(st["vx"].cpu().numpy().reshape(n, -1, hd))
    return {name: torch.from_numpy(x.reshape(n, -1)) for name, x in (("q", q), ("k", k), ("v", v))}


def _exact_tokens(st, t, positions, code, scale):
    """K or V of a table's positions in 64 bits: [positions, kv heads, hd]."""
    tpb = st["case"]["tpb"]
    block, off = st["bt"][t, positions // tpb].long(), positions % tpb
    if st[scale] is None:
        return st[code][block, _LAYER, off].double()
    return st[code][block, _LAYER, :, off].double() * st[scale][block, _LAYER, :, off].double()[..., None]


def _exact_attention(st):
    c = st["case"]
    nkv, nh, hd = c["n_kv_heads"], c["n_heads"], c["head_dim"]
    per = c["tree"] if c["kind"] == "tree" else c["rows"]
    q, out = st["q"].double().view(c["tables"], per, nh, hd), torch.zeros_like(st["q"], dtype=torch.float64)
    out = out.view(c["tables"], per, nh, hd)
    for t in range(c["tables"]):
        if c["kind"] == "tree":
            ctx = int(st["ctx"][t])
            at = torch.arange(ctx + c["tree"], device="cuda")
            words = st["masks"][t].cpu().numpy().view(np.uint8)
            bits = torch.from_numpy(np.unpackbits(words, axis=-1, bitorder="little")[:, :c["tree"]].astype(bool)).cuda()
            sees = torch.cat([torch.ones(c["tree"], ctx, dtype=torch.bool, device="cuda"), bits], 1)
            if c["window"]:
                own_pos = ctx + bits.sum(1) - 1
                sees[:, :ctx] &= at[None, :ctx] + c["window"] > own_pos[:, None]
        else:
            pos = st["pos"].view(c["tables"], -1)[t].long()
            at = torch.arange(int(pos.max()) + 1, device="cuda")
            sees = at[None] <= pos[:, None]
            if c["window"]:
                sees &= at[None] + c["window"] > pos[:, None]
        k, v = _exact_tokens(st, t, at, "k", "ks"), _exact_tokens(st, t, at, "v", "vs")
        some = sees.any(1)
        for h in range(nh):
            s = q[t, :, h] @ k[:, h * nkv // nh].T / math.sqrt(hd)
            if c["cap"]:
                s = c["cap"] * torch.tanh(s / c["cap"])
            s.masked_fill_(~sees, -math.inf)
            s[~some] = 0.0
            out[t, :, h] = torch.softmax(s, 1) @ v[:, h * nkv // nh] * some[:, None]
    return out.view(c["tables"] * per, nh * hd)


def _exact_accept(st):
    c, tpb = st["case"], st["case"]["tpb"]
    names = ("k", "v") if c["cache"] == "f16" else ("ks", "vs")
    new = {n: st[n].double() for n in names}
    bt, ctx = st["bt"].cpu().numpy(), st["ctx"].cpu().numpy()
    for t, path in enumerate(st["accepted"].cpu().numpy()):
        for i, node in enumerate(path[path >= 0]):
            a, b = int(ctx[t]) + int(node), int(ctx[t]) + i
            for n in names:  # slots are the third axis of f16 pages and the fourth of the scales
                src, dst = new[n][bt[t, a // tpb]], new[n][bt[t, b // tpb]]
                if n in ("k", "v"):
                    dst[:, b % tpb] = src[:, a % tpb].clone()
                else:
                    dst[:, :, b % tpb] = src[:, :, a % tpb].clone()
    return new if c["cache"] == "f16" else dict(new, k=None, v=None)


def exact(case, seed):
    st = prepare(case, seed)
    if st["kind"] == "write":
        return _exact_write(st)
    if st["kind"] == "read":
        return [torch.cat([_exact_tokens(st, t, p.long(), code, scale).reshape(p.numel(), -1)
                           for t, p in enumerate(st["pos"].view(case["tables"], -1))])
                for code, scale in (("k", "ks"), ("v", "vs"))]
    return _exact_accept(st) if st["kind"] == "accept" else _exact_attention(st)
