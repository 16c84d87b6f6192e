"""The operators for several requests at once, from their definitions in 64 bits: pages and slots, rotary positions, the cache
in 4 bits, attention, sampling."""
import math

import numpy as np

PAGE = 64
DTYPES = {"bf16": 1, "f16": 3, "f32": 2}
EPS = {"bf16": 2.0 ** -7, "f16": 2.0 ** -10, "f32": 2.0 ** -23}


def pages(n):
    return -(-n // PAGE)


def nearest(x, dtype):
    """the numbers of a 16-bit type nearest to x, even ones of two"""
    x = np.asarray(x, np.float64)
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore"):
        m, e = np.frexp(x)
        e = np.maximum(e, -125)
        return np.ldexp(np.rint(np.ldexp(x, 8 - e)), e - 8)


def plan(cached, fresh, table, stack, n_pages, max_tokens):
    """(table, the free list, its whole buffer's new entries, lengths, starts, key_starts, positions, slots, left)"""
    table, stack = table.copy(), list(stack)
    n, width = table.shape
    for i in range(n):
        if fresh[i] < 0:
            stack += table[i, :pages(cached[i])].tolist()
    given = list(stack)
    available, asked, taken = len(stack), 0, 0
    lengths, starts, keys, positions, slots, left = [], [0], [0], [], [], 0
    for i in range(n):
        a, f = int(cached[i]), int(fresh[i])
        need = pages(a + f) - pages(a) if f > 0 and a + f <= width * PAGE else 0
        asked += need
        served = a + max(f, 0) <= width * PAGE and (need == 0 or asked <= available)
        for j in range(need if served else 0):
            table[i, pages(a) + j] = stack[available - 1 - taken]
            taken += 1
        left += not served
        lengths.append(0 if f < 0 else a + f if served else a)
        starts.append(starts[-1] + max(f, 0))
        keys.append(keys[-1] + lengths[-1])
        for p in range(a, a + max(f, 0)):
            positions.append(p)
            page = int(table[i, p // PAGE]) if served else -1
            slots.append(page * PAGE + p % PAGE if 0 <= page < n_pages else -1)
    rest = max_tokens - len(positions)
    return table, given, available - taken, lengths, starts, keys, (positions + [0] * rest)[:max_tokens], (slots + [-1] * rest)[:max_tokens], left


def turned(x, cos, sin, rot, interleaved):
    """x [tokens][heads][dim], cos and sin [tokens][rot / 2]"""
    y = x.copy()
    if rot:
        a, b = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
        c, s = cos[:, None], sin[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def quantised(x):
    """x [..., dim]: nibbles [..., dim], scale and offset [..., dim / 64]"""
    g = x.reshape(*x.shape[:-1], -1, 64)
    bad = ~np.isfinite(g).all(-1)
    g = np.where(bad[..., None], 0.0, g)
    lo, hi = g.min(-1), g.max(-1)
    offset = nearest(np.clip(lo, -65504.0, 65504.0), "f16") + 0.0  # one zero
    scale = nearest(np.minimum((hi - lo) / 15.0, 65504.0), "f16")
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(scale[..., None] > 0, np.clip(np.rint((g - offset[..., None]) / scale[..., None]), 0, 15), 0)
    scale[bad] = offset[bad] = np.nan
    return n.reshape(x.shape), scale, offset


def value_of(n, scale, offset):
    return n * np.repeat(scale, 64, -1) + np.repeat(offset, 64, -1)


def key_order(dim):
    i = np.arange(dim)
    return (i % 64 // 16) * (dim // 4) + 16 * (i // 64) + i % 16


def value_order(dim):
    i = np.arange(dim)
    return (i % 64 // 4) * (dim // 16) + 4 * (i // 64) + i % 4


def packed_pages(k, v):
    """cache bytes [pages][heads][72 dim] of keys and values, each (nibbles, scale, offset) with leading [pages][heads][64]"""
    P, H, _, dim = k[0].shape
    out = np.zeros((P, H, 72 * dim), np.uint8)
    for which, (x, order) in enumerate(((k, key_order(dim)), (v, value_order(dim)))):
        n = np.zeros(x[0].shape, np.uint8)
        n[..., order] = x[0].astype(np.uint8)
        out[:, :, 32 * dim * which:32 * dim * (which + 1)] = (n[..., 0::2] | n[..., 1::2] << 4).reshape(P, H, -1)
        par = np.stack([x[1], x[2]], -1).transpose(0, 1, 3, 4, 2).astype(np.float16)  # [P][H][group][scale, offset][64]
        at = 64 * dim + 4 * dim * which
        out[:, :, at:at + 4 * dim] = np.ascontiguousarray(par).reshape(P, H, -1).view(np.uint8)
    return out


def attention(q, k, v, scale, seen, spread=None):
    """q [n][H][d], k and v [L][KV][d], seen [n][L]; the result, and the weighted sum of `spread` [L][KV][d]"""
    H, KV = q.shape[1], k.shape[1]
    k, v, spread = (np.repeat(x, H // KV, 1) for x in (k, v, np.abs(v) if spread is None else spread))
    s = np.einsum("nhd,lhd->hnl", q, np.where(seen.any(0)[:, None, None], k, 0.0)) * scale
    s = np.where(seen[None], s, -np.inf)
    top = s.max(-1, keepdims=True, initial=-np.inf)
    p = np.where(seen[None], np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
    p = p / np.maximum(p.sum(-1, keepdims=True), 1e-300)
    return np.einsum("hnl,lhd->nhd", p, v), np.einsum("hnl,lhd->nhd", p, spread)


def sample(x, temperature, top_k, top_p, min_p, u):
    """a token of one row of logits"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return 0
    if not temperature > 0:
        return int(order[0])
    if top == np.inf:
        x, top = np.where(x == np.inf, 0.0, -np.inf), 0.0
    w = np.exp((x[order] - top) / temperature)
    n = len(x)
    if top_k > 0:
        n = min(n, top_k)
    if top_p < 1:
        sums = np.cumsum(w[:n])
        n = min(n, int(np.searchsorted(sums, top_p * sums[-1])) + 1) if top_p > 0 else 1
    if min_p > 0:
        n = min(n, max(1, int(np.count_nonzero(w >= min(min_p, 1.0)))))
    kept = np.sort(order[:n])
    sums = np.cumsum(np.exp((x[kept] - top) / temperature))
    return int(kept[min(len(kept) - 1, int(np.searchsorted(sums, u * sums[-1], side="right")))])


def rotary(kind, rot, max_pos, base, factor=1.0, original=0.0, slow=0.0, fast=0.0):
    """cosines and sines by the definitions of include/awq_infer.h"""
    i = np.arange(rot // 2)
    b = base * factor ** (rot / (rot - 2)) if kind == 2 else base
    f = b ** (-2.0 * i / rot)
    amplitude = 1.0
    if kind == 1:
        f = f / factor
    if kind == 3:
        index = [rot * math.log(original / (2 * math.pi * turns)) / (2 * math.log(base)) for turns in (fast, slow)]
        share = np.clip((i - index[0]) / (index[1] - index[0]), 0, 1)
        f = f * (1 - share) + f / factor * share
        amplitude = 0.1 * math.log(factor) + 1.0
    angle = np.arange(max_pos)[:, None] * f
    return amplitude * np.cos(angle), amplitude * np.sin(angle)
