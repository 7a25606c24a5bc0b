"""Plain references of a step over a paged cache (kv_step.hip) and of 4-bit pages, on the CPU."""
from __future__ import annotations

import numpy as np
import torch

import _paged as P


def plan(ctx, new, bt, total, tpb, free, count, rows):
    """One session after the other; arrays are numpy int64, changed copies are returned:
    (tables, free, lens, left, starts, positions, slots)."""
    bt, free = bt.copy(), free.copy()
    n, per = bt.shape
    lens, starts, at = ctx.copy(), [0], []
    count = max(0, min(count, len(free)))
    for t in range(n):
        if ctx[t] >= 0 and new[t] < 0:
            lens[t] = 0
            for j in range(min(-(-int(ctx[t]) // tpb), per)):
                if 0 <= bt[t, j] < total and count < len(free):
                    free[count] = bt[t, j]
                    count += 1
    full = False
    for t in range(n):
        c, a = int(ctx[t]), int(new[t])
        if c >= 0 and a > 0 and c + a <= per * tpb and not full:
            held = -(-c // tpb)
            need = -(-(c + a) // tpb) - held
            if need <= count and len(at) + a <= rows:
                for j in range(held, held + need):
                    count -= 1
                    bt[t, j] = free[count]
                lens[t] = c + a
                at += [(t, c + i) for i in range(a)]
            else:
                full = True
        starts.append(len(at))
    pos, slots = np.full(rows, -1), np.full(rows, -1)
    for r, (t, p) in enumerate(at):
        pos[r] = p
        blk = bt[t, p // tpb]
        if 0 <= blk < total:
            slots[r] = blk * tpb + p % tpb
    return bt, free, lens, count, np.array(starts), pos, slots


def f16(x):
    """f64 to f16, rounded once (numpy's cast of f64 rounds once)."""
    return np.asarray(x, np.float64).astype(np.float16)


def quantise4(x):
    """Codes [..., hd / 2] and (scale, base) f16 [..., hd / 32, 2] of f32 vectors, each operation rounded once."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (-1, 32))
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(bad[..., None], np.float32(0), g), np.float32(-65504), np.float32(65504))
    z = g.min(-1).astype(np.float16)
    r = g.max(-1) - z.astype(np.float32)
    s = np.maximum(r / np.float32(15), np.float32(0)).astype(np.float16)
    over = 15 * s.astype(np.float64) + z >= 65520
    s = np.where(over, np.nextafter(s, np.float16(0)), s)
    sf = s.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(sf > 0, np.clip(np.rint((g - z.astype(np.float32)[..., None]) / sf), 0, 15), 0)
    c[bad] = 0
    s, z = np.where(bad, np.float16(np.nan), s), np.where(bad, np.float16(np.nan), z)
    c = c.astype(np.uint8).reshape(x.shape)
    return c[..., 0::2] | c[..., 1::2] << 4, np.stack([s, z], -1).astype(np.float16)


def values4(codes, scales):
    """What codes and scales (numpy or torch) stand for, as f16 (numpy)."""
    codes, scales = np.asarray(codes), np.asarray(scales)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(codes.shape[:-1] + (-1, 32)).astype(np.float64)
    s = scales.astype(np.float64)
    with np.errstate(invalid="ignore", over="ignore"):
        v = f16(c * s[..., :1] + s[..., 1:])
    return v.reshape(codes.shape[:-1] + (-1,))


def normed(x, w, eps):
    """Heads x [..., hd] f32 over their root mean square, times w: the sum and the root in 64 bits, then f32."""
    if w is None:
        return np.asarray(x, np.float32)
    x = np.asarray(x, np.float32)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        d = x.astype(np.float64)
        inv = (1.0 / np.sqrt((d * d).sum(-1, keepdims=True) / x.shape[-1] + float(np.float32(eps)))).astype(np.float32)
        return (x * inv) * np.asarray(w, np.float32)


def cache_q4(total, layers, nkv, tpb, hd, seed):
    """Random 4-bit pages: codes [total][layers][nkv][tpb][hd / 2] and scales [..., hd / 32, 2], for K and V."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        c, s = quantise4(torch.randn(total, layers, nkv, tpb, hd, generator=g).numpy())
        out += [torch.from_numpy(c), torch.from_numpy(s)]
    return out


def as_f16_pages(cache):
    """The f16 pages [total][layers][tpb][nkv][hd] that 4-bit ones stand for: (k, None, v, None)."""
    kc, ks, vc, vs = cache
    k, v = (torch.from_numpy(values4(c.numpy(), s.numpy())).permute(0, 1, 3, 2, 4).contiguous()
            for c, s in ((kc, ks), (vc, vs)))
    return k, None, v, None


def attention(q, cache, bt, pos, layer, starts, **kw):
    """Attention over 4-bit pages in 64 bits, q [rows][nh][hd]; rows of no position or table are NaN."""
    k, _, v, _ = as_f16_pages(cache)
    out = torch.full(q.shape, float("nan"), dtype=torch.float64)
    for t in range(len(starts) - 1):
        a, b = int(starts[t]), int(starts[t + 1])
        if a < b:
            out[a:b] = P.causal(q[a:b], k, None, v, None, bt[t:t + 1], pos[a:b], layer, b - a, **kw)
    return out
