"""Plain 64-bit references of the paged 8-bit cache and of attention over shared pages, on the CPU."""
from __future__ import annotations

import math

import numpy as np
import torch

MOST = np.float32(float.fromhex("0x1.0204060000000p+121"))  # the largest scale of which 127 are finite
TINY = np.float32(1.1754943508222875e-38)


def quantise(x):
    """Codes and scales of f32 vectors x[..., hd], each f32 operation rounded once: s = max|x| / 127 (0 below the
    smallest normal number, NaN with a non-finite element), c = rint(x / s)."""
    x = np.asarray(x, np.float32)
    bad = ~np.isfinite(x).all(-1, keepdims=True)
    a = np.where(bad, np.float32(0), np.abs(np.where(bad, 0, x)).max(-1, keepdims=True)).astype(np.float32)
    s = (a / np.float32(127)).astype(np.float32)
    s[s < TINY] = 0
    s = np.minimum(s, MOST)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        c = np.where(s > 0, np.clip(np.rint((x / s).astype(np.float32)), -127, 127), 0)
    c[np.broadcast_to(bad, c.shape)] = 0
    return c.astype(np.int8), np.where(bad, np.float32(np.nan), s)[..., 0]


def rope(x, cs, interleaved=False):
    """x [rows, heads, hd] f32 turned by cs [rows, hd / 2, 2], every product and sum rounded to f32."""
    x0, x1 = (x[..., 0::2], x[..., 1::2]) if interleaved else np.split(x, 2, axis=-1)
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    lo, hi = x0 * c - x1 * s, x1 * c + x0 * s
    if not interleaved:
        return np.concatenate([lo, hi], -1)
    return np.stack([lo, hi], -1).reshape(x.shape)


def cache_q8(total, layers, nkv, tpb, hd, seed):
    """Random 8-bit pages: codes [total][layers][nkv][tpb][hd] and scales, for K and V."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        c, s = quantise(torch.randn(total, layers, nkv, tpb, hd, generator=g).numpy())
        out += [torch.from_numpy(c), torch.from_numpy(np.ascontiguousarray(s))]
    return out


def token(cache, scale, block, layer, slot):
    """K or V of one token in 64 bits, [nkv][hd]."""
    if scale is None:
        return cache[block, layer, slot].double()
    return cache[block, layer, :, slot].double() * scale[block, layer, :, slot].double()[:, None]


def gather(cache, scale, bt, layer, positions, total, tpb):
    """K or V [positions][nkv][hd] of one table's positions in 64 bits; a missing page is zeros."""
    rows = []
    for p in positions:
        blk = int(bt[p // tpb])
        t = token(cache, scale, blk if 0 <= blk < total else 0, layer, p % tpb)
        rows.append(t if 0 <= blk < total else torch.zeros_like(t))
    return torch.stack(rows)


def attend(q, k, v, sees, scale=None, cap=0.0):
    """One row: q [nh][hd], k and v [positions][nkv][hd], sees [positions]; 64 bits. Nothing seen: zeros."""
    nh, hd = q.shape
    g = nh // k.shape[1]
    out = torch.zeros(nh, hd, dtype=torch.float64)
    at = torch.nonzero(sees).flatten()
    if at.numel() == 0:
        return out
    for h in range(nh):
        s = (k[at, h // g] @ q[h].double()) * (scale or 1 / math.sqrt(hd))
        if cap:
            s = torch.tanh(s / cap) * cap
        out[h] = torch.softmax(s, 0) @ v[at, h // g]
    return out


def causal(q, kc, ks, vc, vs, bt, pos, layer, per, scale=None, cap=0.0, window=0):
    """q [rows][nh][hd]; 64 bits; rows of no position are NaN (nothing is to be written there)."""
    total = kc.shape[0]
    tpb = kc.shape[3] if ks is not None else kc.shape[2]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    for t in range(q.shape[0] // per):
        rows = range(t * per, (t + 1) * per)
        top = min(max(int(pos[r]) for r in rows) + 1, bt.shape[1] * tpb)
        if top <= 0:
            continue
        k, v = (gather(c, s, bt[t], layer, range(top), total, tpb) for c, s in ((kc, ks), (vc, vs)))
        at = torch.arange(top)
        for r in rows:
            if pos[r] >= 0:
                end = min(int(pos[r]) + 1, top)
                out[r] = attend(q[r], k, v, (at < end) & ((at >= end - window) if window else (at >= 0)), scale, cap)
    return out


def bits_of(words, tree):
    return np.unpackbits(np.ascontiguousarray(words).view(np.uint8), axis=-1, bitorder="little")[..., :tree].astype(bool)


def words_of(bits):
    """[tables][tree][tree] truth values as int64 words [tables][tree][ceil(tree / 64)]."""
    pad = -bits.shape[-1] % 64
    b = np.concatenate([bits, np.zeros(bits.shape[:-1] + (pad,), bool)], -1)
    return torch.from_numpy(np.packbits(b, axis=-1, bitorder="little").view("<i8").copy())


def tree_bits(parents):
    """Ancestors and itself, from parents [tree] (-1: none)."""
    n = len(parents)
    b = np.zeros((n, n), bool)
    for j, p in enumerate(parents):
        if p >= 0:
            b[j] = b[p]
        b[j, j] = True
    return b


def tree(q, kc, ks, vc, vs, bt, ctx, bits, layer, scale=None, cap=0.0, window=0):
    """q [tables][tree][nh][hd], bits [tables][tree][tree]; rows that are skipped are NaN."""
    total = kc.shape[0]
    tpb = kc.shape[3] if ks is not None else kc.shape[2]
    out = torch.full(q.shape, math.nan, dtype=torch.float64)
    n = q.shape[1]
    for t in range(q.shape[0]):
        if ctx[t] < 0:
            continue
        room = bt.shape[1] * tpb
        c = min(int(ctx[t]), room)
        end = min(c + n, room)
        k, v = (gather(x, s, bt[t], layer, range(end), total, tpb) for x, s in ((kc, ks), (vc, vs)))
        for j in range(n):
            if not bits[t, j].any():
                continue
            sees = torch.zeros(end, dtype=torch.bool)
            start = max(c + int(bits[t, j].sum()) - window, 0) if window else 0
            sees[start:c] = True
            sees[c:end] = torch.from_numpy(bits[t, j, :end - c])
            out[t, j] = attend(q[t, j], k, v, sees, scale, cap)
    return out


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())
