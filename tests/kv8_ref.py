"""Plain forms of the paged 8-bit cache of keys and values for tests: appending in float32 exactly as it is defined (numpy, one
rounding an operation), attention in 64 bits with a bound on what the kernels may differ by.

The bound is derived from what they round, for one output of one row (p the softmax weights, v the values):
  half an ulp of the output's type                              2^-8 |o| (bf16), 2^-11 |o| (f16)
  weights rounded to f16, 11 bits                               2^-11 sum p |v|
  weights under f16's normal range, relative to the largest     n 2^-25 127 max(v_scale)
  a score: fp32 sums of dim products, its factor, the exponent  (dim + 8) 2^-24 max_j sum |q k_j| scale + 2^-22 max |s|,
  which moves the output by at most twice that times sum p |v|
  the rest: sums and quotients in fp32                          2^-18 sum p |v|
"""
import math

import numpy as np
import torch

BLOCK = 64
HALF_ULP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Cache:
    """Codes as [blocks, heads, 64, dim] of keys and values on the host (numpy), with the kernels' layout on request."""

    def __init__(self, blocks, heads, dim, seed=0, std=34.0):
        rng = np.random.default_rng(seed)
        self.codes = [np.clip(np.rint(rng.standard_normal((blocks, heads, BLOCK, dim)) * std), -127, 127).astype(np.int64) + 128 for _ in range(2)]
        self.scale = [np.exp(0.2 * rng.standard_normal((blocks, heads))).astype(np.float32) / np.float32(34) for _ in range(2)]

    def tensors(self, device="cuda"):
        k, v = (torch.from_numpy(c.astype(np.uint8)) for c in self.codes)
        n, h, _, d = k.shape
        v = v.view(n, h, BLOCK // 4, 4, d).transpose(-1, -2).contiguous()
        return k.to(device), v.to(device), torch.from_numpy(self.scale[0].copy()).to(device), torch.from_numpy(self.scale[1].copy()).to(device)

    def values(self, which):
        return (self.codes[which] - 128).astype(np.float64) * self.scale[which].astype(np.float64)[:, :, None, None]


def from_layout(k_codes, v_codes):
    """(key codes, value codes) as int64 numpy [blocks, heads, 64, dim]."""
    n, h, _, d = k_codes.shape
    return k_codes.cpu().numpy().astype(np.int64), v_codes.cpu().transpose(-1, -2).reshape(n, h, BLOCK, d).numpy().astype(np.int64)


def rotated(x, cos, sin):
    """float32 rows x [tokens, heads, dim] rotated by rows of the tables, one rounding an operation."""
    half = cos.shape[1]
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    c, s = cos[:, None, :], sin[:, None, :]
    return np.concatenate([a * c - b * s, b * c + a * s, rest], -1).astype(np.float32)


def append(cache, k, v, table, lens, news, cos=None, sin=None):
    """The definition of lq_kv8_append on a Cache; k, v float32 numpy [tokens, heads, dim]. Returns the rows' positions."""
    f32 = np.float32
    start, positions = 0, []
    for i, (n, new) in enumerate(zip(lens, news)):
        for t in range(new):
            positions.append(n - new + t)
        rows = np.arange(start, start + new)
        start += new
        pos = np.arange(n - new, n)
        for which, x in ((0, k[rows]), (1, v[rows])):
            if which == 0 and cos is not None and new:
                at = np.clip(pos, 0, cos.shape[0] - 1)
                x = rotated(x, cos[at], sin[at])
            for place in sorted(set((pos[pos >= 0] // BLOCK).tolist())):
                if place >= table.shape[1]:
                    continue
                block = int(table[i, place])
                if not 0 <= block < cache.codes[0].shape[0]:
                    continue
                here = (pos // BLOCK == place) & (pos >= 0)
                kept = int(pos[here][0]) % BLOCK
                y = x[here]
                most = np.where(np.isfinite(y), np.abs(y), f32(0)).max((0, 2))
                scale = np.maximum(most, f32(2.0 ** -90)) * f32(f32(1) / f32(127))
                held = cache.scale[which][block].copy()
                codes = cache.codes[which][block]
                if kept:
                    scale = np.maximum(scale, held)
                    grows = scale > held
                    ratio = held / scale
                    again = np.rint((codes[:, :kept] - 128).astype(f32) * ratio[:, None, None]).astype(np.int64) + 128
                    codes[:, :kept] = np.where(grows[:, None, None], again, codes[:, :kept])
                with np.errstate(invalid="ignore", over="ignore"):
                    c = np.clip(np.rint(y * (f32(1) / scale)[None, :, None]), -127, 127)
                c = np.where(np.isnan(c), 0, c).astype(np.int64) + 128
                codes[:, kept:kept + y.shape[0]] = c.transpose(1, 0, 2)
                cache.scale[which][block] = scale
    return np.array(positions, dtype=np.int64)


def attention(cache, q, table, lens, news, scale=None, causal=True, window=0):
    """(out, (lse, its bound), bound) in float64: q a CPU tensor [tokens, heads, dim]; bound: what each output may be off."""
    dim, heads = q.shape[2], q.shape[1]
    kv_heads = cache.codes[0].shape[1]
    group = heads // kv_heads
    scale = dim ** -0.5 if scale is None else scale
    x = q.double().numpy()
    out, lse, bound, lse_bound = np.zeros(x.shape), np.full(x.shape[:2], -np.inf), np.zeros(x.shape), np.zeros(x.shape[:2])
    ulp = HALF_ULP[q.dtype]
    start = 0
    for i, (n, new) in enumerate(zip(lens, news)):
        rows, pos = np.arange(start, start + new), np.arange(n - new, n)
        start += new
        if not new:
            continue
        blocks = [int(b) for b in table[i, :-(-n // BLOCK)]]
        for h in range(heads):
            kv = h // group
            if n > 0:
                k, v = ((cache.codes[w][blocks, kv] - 128).astype(np.float64) * cache.scale[w][blocks, kv].astype(np.float64)[:, None, None] for w in (0, 1))
                k, v = k.reshape(-1, dim)[:n], v.reshape(-1, dim)[:n]
                v_scale = np.repeat(cache.scale[1][blocks, kv].astype(np.float64), BLOCK)[:n]
            else:
                k = v = np.zeros((0, dim))
            key = np.arange(n)
            for r, p in zip(rows, pos):
                seen = np.ones(n, bool)
                if causal:
                    seen &= key <= p
                if window:
                    seen &= key > p - window
                if not seen.any():
                    continue
                ks, vs, sq = k[seen], v[seen], x[r, h]
                with np.errstate(invalid="ignore", over="ignore"):
                    s = ks @ sq * scale
                    m = s.max()
                    w = np.exp(s - m)
                    total = w.sum()
                    w /= total
                    out[r, h] = w @ vs
                lse[r, h] = m + math.log(total) if np.isfinite(total) else np.nan
                size = w @ np.abs(vs)
                score = (dim + 8) * 2.0 ** -24 * (np.abs(ks) @ np.abs(sq)).max() * scale + 2.0 ** -22 * np.abs(s).max()
                lse_bound[r, h] = score + 2.0 ** -20 * (1 + abs(lse[r, h]))
                bound[r, h] = ulp * np.abs(out[r, h]) + (2.0 ** -11 + 2 * score + 2.0 ** -18) * size + seen.sum() * 2.0 ** -25 * 127 * v_scale[seen].max()
    return out, (lse, lse_bound), bound


def blocks_of(lens, pool, seed=0, spare=-1, width=None):
    """A block table for sequences of these lengths, blocks of a pool of `pool` in random order, unused entries `spare`."""
    per = [-(-n // BLOCK) for n in lens]
    order = np.random.default_rng(seed).permutation(pool)
    table = np.full((len(lens), width or max(1, max(per, default=1))), spare, dtype=np.int32)
    at = 0
    for i, n in enumerate(per):
        table[i, :n] = order[at:at + n]
        at += n
    assert at <= pool
    return table


def tables(positions, rot):
    rate = 10000.0 ** (-np.arange(rot // 2) / (rot // 2))
    angle = np.arange(positions)[:, None] * rate
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
