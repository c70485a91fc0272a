"""Paged 8-bit KV cache restatement in 64 bits.  TEST INFRASTRUCTURE.

The format (include/megakernel.h, megakernel_kv8_cache): a pool of blocks of
B positions, e4m3 codes k [n_blocks][n_kv][B][D] and v [n_blocks][n_kv][D][B],
one power-of-two scale per block, head and K / V.  The codes are those of
oracle/fp8.py.  Written position by position, from the definitions alone.
"""
from __future__ import annotations

import math

import numpy as np

from . import fp8

MIN_EXP, MAX_EXP = -126, 119  # 448 * 2^119 is fp32's last such value


def scale_exp(amax: float) -> int:
    """The smallest e >= -126 with amax <= 448 * 2^e (-126 for zero), at most 119."""
    if amax <= 0:
        return MIN_EXP
    m, e = math.frexp(amax)
    return min(max(MIN_EXP, e - 9 + (m > 0.875)), MAX_EXP)


def encode(x: np.ndarray, e: int) -> np.ndarray:
    """Codes of x / 2^e: what is beyond 448 saturates, NaN is the NaN code."""
    with np.errstate(invalid="ignore"):
        y = np.clip(np.ldexp(np.asarray(x, np.float64), -e), -448.0, 448.0)
    c = fp8.e4m3_encode(np.nan_to_num(y, nan=0.0).astype(np.float32))
    return np.where(np.isnan(x), np.uint8(0x7F), c).astype(np.uint8)


def decode(c: np.ndarray) -> np.ndarray:
    return fp8.e4m3_decode_table().astype(np.float64)[c]


class Pool:
    """The cache as arrays; k and v codes, scales in float64."""

    def __init__(self, k, v, k_scale, v_scale):
        self.k, self.v = np.array(k, np.uint8), np.array(v, np.uint8)
        self.ks, self.vs = np.array(k_scale, np.float64), np.array(v_scale, np.float64)
        self.n_blocks, self.n_kv, self.block, self.dim = self.k.shape

    def place(self, table_row, p: int):
        """(block, row) of position p, or None where it has none."""
        if p < 0 or p // self.block >= len(table_row):
            return None
        b = int(table_row[p // self.block])
        return (b, p % self.block) if 0 <= b < self.n_blocks else None

    def append(self, table, start, length, k_new, v_new):
        for i in range(len(length)):
            groups: dict[int, list[tuple[int, int]]] = {}
            for t in range(start[i], start[i + 1]):
                at = self.place(table[i], int(length[i]) - int(start[i + 1]) + t)
                if at:
                    groups.setdefault(at[0], []).append((at[1], t))
            for b, rows in groups.items():
                r0 = rows[0][0]
                for codes, scale, new in ((self.k, self.ks, k_new), (self.v.transpose(0, 1, 3, 2), self.vs, v_new)):
                    for h in range(self.n_kv):
                        x = np.stack([new[t, h] for _, t in rows]).astype(np.float64)
                        fin = np.abs(x[np.isfinite(x)])
                        e = scale_exp(float(fin.max()) if fin.size else 0.0)
                        if r0 > 0:
                            eo = int(math.log2(scale[b, h]))
                            if eo < e:
                                old = decode(codes[b, h, :r0]) * 2.0 ** eo
                                codes[b, h, :r0] = encode(old, e)
                            e = max(e, eo)
                        scale[b, h] = 2.0 ** e
                        for (r, _), row in zip(rows, x):
                            codes[b, h, r] = encode(row, e)

    def values(self, b: int, r: int):
        """K and V [n_kv][D] at row r of block b."""
        return (decode(self.k[b, :, r]) * self.ks[b][:, None], decode(self.v[b, :, :, r]) * self.vs[b][:, None])

    def read(self, table, start, length, k_out, v_out):
        for i in range(len(length)):
            for t in range(start[i], start[i + 1]):
                p = int(length[i]) - int(start[i + 1]) + t
                at = self.place(table[i], p) if p < length[i] else None
                k_out[t], v_out[t] = self.values(*at) if at else (0.0, 0.0)

    def attention(self, table, start, length, q, out, scale: float):
        """out, and sum_j p_j |v_j| and max_j sum_d |q_d k_jd| * scale per row, which bound rounding."""
        group = q.shape[1] // self.n_kv
        size, reach = np.zeros(out.shape), np.zeros(out.shape[:2])
        for i in range(len(length)):
            at = [(j, self.place(table[i], j)) for j in range(max(0, int(length[i])))]
            there = [(j, *self.values(*a)) for j, a in at if a]
            pos = np.array([x[0] for x in there])
            keys, vals = (np.stack([x[k] for x in there]) if there else None for k in (1, 2))
            for t in range(start[i], start[i + 1]):
                n = int((pos <= int(length[i]) - int(start[i + 1]) + t).sum()) if there else 0
                if n == 0:
                    out[t] = 0.0
                    continue
                for h in range(q.shape[1]):
                    k, v = keys[:n, h // group], vals[:n, h // group]
                    s = k @ q[t, h] * scale
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t, h] = w @ v
                    size[t, h] = w @ np.abs(v)
                    reach[t, h] = (np.abs(k) @ np.abs(q[t, h])).max() * scale
        return size, reach


def norm_rope(x, gain, inv_freq, pos, eps: float):
    """RMSNorm per head, then the rotate-half rotation; float64 [T][H][D]."""
    x, h = np.asarray(x, np.float64), x.shape[-1] // 2
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gain, np.float64)
    a = np.asarray(pos, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(a), np.sin(a)
    return np.concatenate([y[..., :h] * c - y[..., h:] * s, y[..., h:] * c + y[..., :h] * s], -1), np.concatenate([np.abs(y[..., :h]) + np.abs(y[..., h:])] * 2, -1)


class Scores:
    """What scores are and what rows see (include/megakernel.h, megakernel_kv8_scores)."""

    def __init__(self, softcap=0.0, slopes=None, window=0, first=None, prefix=None):
        self.softcap, self.slopes, self.window, self.first, self.prefix = softcap, slopes, window, first, prefix

    def span(self, i: int, t: int, p: int, length: int):
        """[lo, hi) of row t at position p of sequence i."""
        lo, hi = 0, p + 1
        if self.window:
            lo = max(lo, p + 1 - self.window)
        if self.first is not None:
            lo = max(lo, int(self.first[t]))
        if self.prefix is not None and p >= 0:
            hi = max(hi, int(self.prefix[i]))
        return lo, min(hi, length)


def scored_rows(pool: Pool, table, start, length, q, scale: float, x: Scores, tokens=None):
    """Yields (sequence, row, head, positions, scores, weights, values, reach, bias) of
    every row that sees something, or None for the last six: reach is
    max_j sum_d |q_d k_jd| * scale and bias the largest |slope * distance|."""
    group = q.shape[1] // pool.n_kv
    for i in range(len(length)):
        n = min(max(0, int(length[i])), len(table[i]) * pool.block)
        at = [(j, pool.place(table[i], j)) for j in range(n)]
        there = [(j, *pool.values(*a)) for j, a in at if a]
        pos = np.array([y[0] for y in there], np.int64)
        keys, vals = (np.stack([y[k] for y in there]) if there else None for k in (1, 2))
        for t in range(start[i], start[i + 1]):
            if tokens is not None and t not in tokens:
                continue
            p = int(length[i]) - int(start[i + 1]) + t
            lo, hi = x.span(i, t, p, n)
            seen = (pos >= lo) & (pos < hi) if there else np.zeros(0, bool)
            for h in range(q.shape[1]):
                if not seen.any():
                    yield i, t, h, None, None, None, None, 0.0, 0.0
                    continue
                k, v, j = keys[seen, h // group], vals[seen, h // group], pos[seen]
                s = k @ q[t, h] * scale
                if x.softcap:
                    s = x.softcap * np.tanh(s / x.softcap)
                far = np.abs(j - p) * float(x.slopes[h]) if x.slopes is not None else np.zeros(len(j))
                s = s - far
                w = np.exp(s - s.max())
                yield i, t, h, j, s, w / w.sum(), v, (np.abs(k) @ np.abs(q[t, h])).max() * scale, np.abs(far).max()


def select(mass, length: int, keep: int, recent: int, sinks: int):
    """The positions that stay of one sequence and head, in rising order."""
    if length <= keep:
        return list(range(length))
    fixed = list(range(sinks)) + list(range(length - recent, length))
    rest = range(sinks, length - recent)
    # by falling weight, NaN last, then by rising position
    order = sorted(rest, key=lambda j: (math.isnan(mass[j]), -mass[j] if not math.isnan(mass[j]) else 0.0, j))
    return sorted(fixed + order[: keep - recent - sinks])


def compact(pool: Pool, table, kept, kept_len, new_table):
    """Rows moved to the blocks of new_table: read, then appended to blocks that start anew."""
    n_seq, _, keep = kept.shape
    rows = [max(0, min(int(n), keep, len(new_table[i]) * pool.block)) for i, n in enumerate(kept_len)]
    got = []
    for i in range(n_seq):
        k, v = np.zeros((2, rows[i], pool.n_kv, pool.dim))
        for h in range(pool.n_kv):
            for r in range(rows[i]):
                at = pool.place(table[i], int(kept[i, h, r]))
                if at:
                    kk, vv = pool.values(*at)
                    k[r, h], v[r, h] = kk[h], vv[h]
        got.append((k, v))
    for i, (k, v) in enumerate(got):
        pool.append([new_table[i]], [0, rows[i]], [rows[i]], k, v)


def rotary(x, inv_freq, pos, interleaved: bool, amplitude: float):
    """The rotation of the first 2 * len(inv_freq) dimensions; float64 [T][H][D], and |a| + |b| of each value's pair."""
    x = np.asarray(x, np.float64)
    n = 2 * len(inv_freq)
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., : n // 2], x[..., n // 2 : n])
    t = np.asarray(pos, np.float64)[:, None, None] * np.asarray(inv_freq, np.float64)
    c, s = np.cos(t) * amplitude, np.sin(t) * amplitude
    y, size = x.copy(), np.abs(x)
    both = np.abs(a) + np.abs(b)
    for out, first, second in ((y, a * c - b * s, b * c + a * s), (size, both, both)):
        if interleaved:
            out[..., 0:n:2], out[..., 1:n:2] = first, second
        else:
            out[..., : n // 2], out[..., n // 2 : n] = first, second
    return y, size
