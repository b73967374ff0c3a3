"""The rotary and 4-bit cache forms in plain numpy, in 64 bits, for the tests: positions, rotation, quantisation,
the cache's bytes, and attention over them."""
from __future__ import annotations

import math

import numpy as np

HALF_STEP = {"F32": 2.0 ** -24, "F16": 2.0 ** -11, "Bf16": 2.0 ** -8}  # of a rounding, relative to the value
INDEX = {"I32": np.int32, "I64": np.int64}


def rounded(x: np.ndarray, dtype: str) -> np.ndarray:
    """f32 values rounded to the type (nearest, ties to even), as f64."""
    f = np.asarray(x, dtype=np.float32)
    if dtype == "F32":
        return f.astype(np.float64)
    if dtype == "F16":
        return f.astype(np.float16).astype(np.float64)
    bits = f.view(np.uint32).astype(np.uint64)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000
    out = bits.astype(np.uint32).view(np.float32).astype(np.float64)
    return np.where(np.isnan(f), np.nan, out)


def stored(x: np.ndarray, dtype: str) -> np.ndarray:
    """Values of the type as the device holds them."""
    f = np.ascontiguousarray(x, dtype=np.float32)
    if dtype == "F32":
        return f
    if dtype == "F16":
        return f.astype(np.float16).view(np.uint16)
    return (rounded(f, "Bf16").astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


def loaded(a: np.ndarray, dtype: str) -> np.ndarray:
    """The f64 values of what the device holds."""
    if dtype == "F32":
        return a.view(np.float32).astype(np.float64)
    if dtype == "F16":
        return a.view(np.float16).astype(np.float64)
    return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def frequencies(rot, base=10000.0, scaling="none", factor=1.0, low=1.0, high=4.0, original=8192):
    f = np.array([math.pow(base, -2.0 * i / rot) for i in range(rot // 2)])
    if scaling == "linear":
        return f / factor
    if scaling == "ramp":
        keep = np.clip((original * f / (2 * math.pi) - low) / (high - low), 0.0, 1.0)
        return f * (keep + (1 - keep) / factor)
    return f


def table(rot, first, count, amplitude=1.0, **how) -> np.ndarray:
    """[count][rot / 2][cos, sin] in f64."""
    a = (first + np.arange(count, dtype=np.float64))[:, None] * frequencies(rot, **how)[None, :]
    return np.stack([np.cos(a), np.sin(a)], -1) * amplitude


def pairs_of(rot, layout):
    i = np.arange(rot // 2)
    return (i, i + rot // 2) if layout == "halves" else (2 * i, 2 * i + 1)


def rotate(x, rows, rot, layout, inverse=False):
    """x [tokens, heads, head_dim], rows [tokens, rot / 2, 2] (the table's, as f64): f64."""
    y = np.array(x, dtype=np.float64)
    i0, i1 = pairs_of(rot, layout)
    c, s = rows[:, None, :, 0], rows[:, None, :, 1] * (-1.0 if inverse else 1.0)
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def quantise(y, group):
    """y [..., head_dim] (values of a 16-bit type): codes, f16 scales and zero points of the groups."""
    g = np.asarray(y, np.float64).reshape(*y.shape[:-1], -1, group)
    with np.errstate(all="ignore"):
        lo = np.minimum(g.min(-1), 0).astype(np.float32)
        hi = np.maximum(g.max(-1), 0).astype(np.float32)
        scale = ((hi - lo) / np.float32(15)).astype(np.float16)
        bad = ~np.isfinite(g).all(-1) | ~np.isfinite(scale)
        scale = np.where(bad, np.float16(np.nan), scale)
        unit = np.where(bad | (scale == 0), 1.0, scale.astype(np.float64))
        zero = np.where(bad, 0, np.clip(np.rint(-lo.astype(np.float64) / unit), 0, 15))
        code = np.clip(np.rint(g / unit[..., None]) + zero[..., None], 0, 15)
        code = np.where(bad[..., None], 0, code)
    return code.reshape(y.shape).astype(np.uint8), scale, zero.astype(np.uint32)


class Cache:
    """A cache's bytes and where its parts lie."""

    def __init__(self, pages, heads, dim, group, page, fill=0):
        self.heads, self.dim, self.group, self.page = heads, dim, group, page
        self.record = page * (dim + 8 * (dim // group))
        self.bytes = np.full((pages, heads, self.record), fill, np.uint8)

    def code_at(self, t, d, value):
        word, half = d // 8, self.page * self.dim // 2
        if value:
            w = half // 4 + ((t // 4) * (self.dim // 8) + word) * 4 + t % 4
        else:
            w = t * (self.dim // 8) + (word % 4) * (self.dim // 32) + word // 4
        return w * 4 + d % 8 // 2, d % 2 * 4

    def word_at(self, t, g, value):
        groups = self.dim // self.group
        return self.page * self.dim + 4 * ((groups if value else 0) * self.page + g * self.page + t)

    def put(self, slot, head, y, value):
        code, scale, zero = quantise(y, self.group)
        rec, t = self.bytes[slot // self.page, head], slot % self.page
        for d in range(self.dim):
            at, shift = self.code_at(t, d, value)
            rec[at] = (rec[at] & (0xF0 >> shift)) | (int(code[d]) << shift)
        for g in range(self.dim // self.group):
            at = self.word_at(t, g, value)
            word = int(np.float16(scale[g]).view(np.uint16)) | int(zero[g]) << 16
            if np.isnan(scale[g]):
                word = 0x7E00
            rec[at:at + 4] = np.frombuffer(np.uint32(word).tobytes(), np.uint8)

    def get(self, slot, value):
        """The f64 values of a slot: [heads, head_dim]."""
        rec, t = self.bytes[slot // self.page], slot % self.page
        d = np.arange(self.dim)
        at, shift = self.code_at(t, d, value)
        code = (rec[:, at] >> shift) & 15
        out = np.empty((self.heads, self.dim))
        for g in range(self.dim // self.group):
            w = self.word_at(t, g, value)
            word = np.ascontiguousarray(rec[:, w:w + 4]).view(np.uint16).reshape(-1, 2)
            part = slice(g * self.group, (g + 1) * self.group)
            scale = np.ascontiguousarray(word[:, 0]).view(np.float16).astype(np.float64)
            with np.errstate(invalid="ignore"):
                out[:, part] = (code[:, part].astype(np.float64) - word[:, 1:2]) * scale[:, None]
        return out


def attend(q, cache, tables, starts, lengths, causal=True, window=0, scale=None, pages=None):
    """q [tokens, heads, head_dim] in f64.  Gives the outputs (NaN where no sequence has the row), their log-sum-exp
    and, for a tolerance, sum p |v|, the largest |v| a row sees, and sum |q| times the largest scale of its keys."""
    t, heads, dim = q.shape
    gqa = heads // cache.heads
    pages = cache.bytes.shape[0] if pages is None else pages
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, lse = np.full(q.shape, np.nan), np.full((t, heads), np.nan)
    mass, top, reach = np.zeros(q.shape), np.zeros((t, heads)), np.zeros((t, heads))
    for b in range(len(lengths)):
        n, end = starts[b + 1] - starts[b], min(int(lengths[b]), tables.shape[1] * cache.page)
        there = [j for j in range(end) if 0 <= tables[b, j // cache.page] < pages]
        slots = [int(tables[b, j // cache.page]) * cache.page + j % cache.page for j in there]
        k = np.array([cache.get(s, False) for s in slots]).reshape(len(slots), cache.heads, dim)
        v = np.array([cache.get(s, True) for s in slots]).reshape(len(slots), cache.heads, dim)
        for i in range(n):
            row, place = starts[b] + i, int(lengths[b]) - n + i
            seen = np.array([(not causal or j <= place) and (window == 0 or j > place - window) for j in there], bool)
            for h in range(heads):
                if not seen.any():
                    out[row, h], lse[row, h] = 0.0, -np.inf
                    continue
                kk, vv = k[seen, h // gqa], v[seen, h // gqa]
                s = kk @ q[row, h] * scale
                m = s.max()
                p = np.exp(s - m)
                out[row, h], lse[row, h] = p @ vv / p.sum(), m + math.log(p.sum())
                mass[row, h], top[row, h] = p @ np.abs(vv) / p.sum(), np.abs(vv).max()
                reach[row, h] = np.abs(q[row, h]).sum() * np.abs(kk).max() * scale
    return out, lse, mass, top, reach


def attention_tolerance(out, mass, top, reach, keys, dim, dtype):
    """What rounding may do to an output, per element.

    * A probability and a value may each be rounded once to 11 bits: 2^-11 of each product, of sum p |v|.
    * A score's products are added in f32 as sum q n - zero sum q, codes and zeros of at most 15 steps.  A group's
      range is 15 steps wide, so some element of it is at least 7 from its zero: a step is at most a seventh of the largest
      |k|, and both sums together take at most 2 (dim + 4) roundings of sum |q| 15 / 7 |k|, each of 2^-23 (the matrix unit's
      additions need not round to nearest).  A score off by e moves the probability, and the sum, by e each.
    * exp, the sum of the probabilities and the products' sum: (keys + 8) roundings of 2^-23.
    * Values are added as sum p s n - sum p s zero in f32, codes and zeros of at most 15 steps of at most a seventh of the
      largest |v| (as above), and sum p is 1: (keys + 8) roundings of 2^-23 of 15 / 7 of it in each of the two sums.  So
      an output whose values are all 0 may come out as that much.
    * A probability p is held as the f16 number 2^11 p: below 2^-25 of the row's largest these are subnormal, a step
      2^-24 apart, so off by at most 2^-36 of the largest.  With the products that they go into, keys * 2^-35 of the
      largest |v|.
    * The output is rounded once to its type.
    """
    score = reach[..., None] * (30.0 / 7.0) * (dim + 4) * 2.0 ** -23
    off = mass * (2 * 2.0 ** -11 + 2 * score + (keys + 8) * 2.0 ** -23) + top[..., None] * (
        keys * 2.0 ** -35 + 2 * 15.0 / 7.0 * (keys + 8) * 2.0 ** -23)
    return off + (np.abs(out) + off) * HALF_STEP[dtype]
