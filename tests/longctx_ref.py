"""Plain numpy statements, in 64 bits, of the long-context operators: stretched rotary positions,
bounds of the keys of a block, block selection, attention over selected blocks.  Written from the
definitions in include/drk_kv.h; they share no code with the library or the C oracle."""
import math

import numpy as np

from deusridet_amd import cabi
from tests import util as U

HALF_STEP = {cabi.BF16: 2.0 ** -8, cabi.F16: 2.0 ** -11}


# ---- rotary positions -------------------------------------------------------------------------
def rope_turns(r):
    """Turns per position of every pair of a cabi.Rope."""
    i = np.arange(r.rotary_dim // 2)
    f = np.float64(r.theta) ** (-2.0 * i / r.rotary_dim) / (2 * math.pi)
    if r.factor == 1.0:
        return f
    g = np.clip((r.original_positions * f - r.low_turns) / (np.float64(r.high_turns) - r.low_turns), 0.0, 1.0)
    return f * (g + (1 - g) / r.factor)


def rope(r, x, pos, inverse=False):
    """x [T, H, D] float64 -> (rotated, |a| + |b| of every element's pair: what an error of cos / sin scales with)"""
    x = np.asarray(x, np.float64)
    half = r.rotary_dim // 2
    w = 2 * math.pi * np.asarray(pos, np.float64)[:, None] * rope_turns(r)[None]
    co, si = r.magnitude * np.cos(w)[:, None], r.magnitude * np.sin(w)[:, None] * (-1 if inverse else 1)
    ia, ib = (np.arange(half) * 2, np.arange(half) * 2 + 1) if r.interleaved else (np.arange(half), np.arange(half) + half)
    y, mag = x.copy(), np.zeros_like(x)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * co - b * si, b * co + a * si
    mag[..., ia] = mag[..., ib] = abs(r.magnitude) * (np.abs(a) + np.abs(b))
    return y, mag


# ---- pools ------------------------------------------------------------------------------------
class Pool:
    """Random pages on the host: float64 values k, v [L, NB, KVH, bs, D] and the bytes that hold them."""

    def __init__(self, rng, L, KVH, QH, D, bs, NB, dtype, mul=1.0):
        self.L, self.KVH, self.QH, self.D, self.bs, self.NB, self.dtype = L, KVH, QH, D, bs, NB, dtype
        self.g = cabi.layout(L, KVH, QH, D, bs, NB, dtype)
        shape = (L, NB, 2, KVH, bs, D)
        scales = np.zeros((L, NB, 2, KVH, bs, 0), np.uint8)
        if dtype in (cabi.F16, cabi.BF16):
            bits = U.normal_bits(rng, shape, dtype, mul)
            vals = U.from_bits(bits, dtype).astype(np.float64)
            raw = bits.view(np.uint8).reshape(L, NB, -1)
        elif dtype == cabi.INT8:
            codes = rng.integers(-127, 128, shape).astype(np.int8)
            sc = (rng.random((L, NB, 2, KVH, bs)) * 0.02 + 0.004).astype(np.float16)
            vals = codes.astype(np.float64) * sc.astype(np.float64)[..., None]
            raw = np.concatenate([codes.view(np.uint8).reshape(L, NB, -1), sc.view(np.uint8).reshape(L, NB, -1)], 2)
        else:
            import torch
            t = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * np.float32(mul)).to(torch.float8_e4m3fn)
            vals = t.float().numpy().astype(np.float64)
            raw = t.view(torch.uint8).numpy().reshape(L, NB, -1)
        del scales
        self.raw, self.k, self.v = np.ascontiguousarray(raw), vals[:, :, 0], vals[:, :, 1]

    def poison(self, layer, blk, first):
        """NaN (int8: the largest code with a NaN scale) into tokens first.. of a block, in the bytes only."""
        n = self.KVH * self.bs * self.D
        b = self.raw[layer, blk]
        if self.dtype in (cabi.F16, cabi.BF16):
            b.view(np.uint16)[:2 * n].reshape(2, self.KVH, self.bs, self.D)[:, :, first:] = 0x7FFF
        elif self.dtype == cabi.FP8_E4M3:
            b[:2 * n].reshape(2, self.KVH, self.bs, self.D)[:, :, first:] = 0x7F
        else:
            b[2 * n:].view(np.uint16).reshape(2, self.KVH, self.bs)[:, :, first:] = 0x7FFF


# ---- bounds -----------------------------------------------------------------------------------
def exponent(amax):
    for e in range(-40, 41):
        if amax <= 127 * 2.0 ** e:
            return e
    return 40


def bounds(keys):
    """keys [n, D] float64 -> (low codes, high codes, e); NaN passed over"""
    with np.errstate(all="ignore"):
        lo = np.where(np.isnan(keys), np.inf, keys).min(0)
        hi = np.where(np.isnan(keys), -np.inf, keys).max(0)
    lo, hi = np.where(lo > hi, 0.0, lo), np.where(lo > hi, 0.0, hi)
    e = exponent(max(np.abs(lo).max(), np.abs(hi).max()))
    return (np.floor(np.clip(lo / 2.0 ** e, -127, 127)).astype(np.int8),
            np.ceil(np.clip(hi / 2.0 ** e, -127, 127)).astype(np.int8), e)


def bounds_buffers(L, NB, KVH, D, rng):
    """Random (codes [L, NB, KVH, 2, D], exponents [L, NB, KVH]) with low <= high."""
    c = rng.integers(-127, 128, (L, NB, KVH, 2, D)).astype(np.int8)
    c.sort(axis=3)
    return c, rng.integers(-9, -3, (L, NB, KVH)).astype(np.int8)


def bounds_bytes(codes, exps):
    raw = np.concatenate([codes.reshape(-1).view(np.uint8), exps.reshape(-1).view(np.uint8)])
    return np.concatenate([raw, np.zeros(-len(raw) % 16, np.uint8)])


# ---- selection --------------------------------------------------------------------------------
def query_codes(q):
    """q [D] float64 -> (codes int64, e)"""
    q = np.where(np.isnan(q), 0.0, q)
    e = exponent(np.abs(q).max())
    return np.rint(np.clip(q / 2.0 ** e, -127, 127)).astype(np.int64), e


def select(q, codes, exps, table, length, bs, keep, sink, recent):
    """One row: q [QH, D] float64, codes [NB, KVH, 2, D], exps [NB, KVH], table 1-d -> int32 [KVH, keep]"""
    QH, KVH, NB = q.shape[0], codes.shape[1], codes.shape[0]
    nb = max(0, -(-length // bs))
    out = np.full((KVH, keep), -1, np.int32)
    qc = [query_codes(x) for x in q]
    for h in range(KVH):
        forced, scored = [], []
        for b in range(nb):
            blk = table[b]
            if blk < 0 or blk >= NB:
                continue
            if b < sink or b >= nb - recent:
                forced.append(b)
                continue
            lo, hi = codes[blk, h].astype(np.int64)
            s = max(math.ldexp(float(np.maximum(c * lo, c * hi).sum()), int(exps[blk, h]) + e)
                    for c, e in qc[h * (QH // KVH):(h + 1) * (QH // KVH)])
            scored.append((-s, b))
        best = sorted(forced + [b for _, b in sorted(scored)[:keep - len(forced)]])
        out[h, :len(best)] = best
    return out


# ---- attention --------------------------------------------------------------------------------
def attend(pool, layer, q, table, length, sel, scale, gate=None):
    """One row: q [QH, D] float64, sel [KVH, n] -> (out [QH, D] float64, bound on what a kernel may be off by before its
    last rounding, or None for a row without a token).

    The bound counts: each weight rounded to 16 bits in the second product and -- with the 16-bit storage types -- in
    the denominator, which moves the mean of the values by at most u sum p |v - out| / sum p <= u (A + |out|), A = sum p |v| /
    sum p, u half a step of the weights' type (8-bit pages: fp16); the score's fp32 sums, (D + 8) 2^-24 of sum |q k|, twice, since numerator and denominator carry
    it; the output's fp32 sums over the tokens, n 2^-24 A; and for weights below fp16's normal range 2^-25 each.  int8
    codes travel as 1152 + code, so their sums and the weights' roundings count with 1279 times the scale instead of
    |v|."""
    QH, D, bs, KVH = pool.QH, pool.D, pool.bs, pool.KVH
    G = QH // KVH
    out, tol = np.zeros((QH, D)), np.zeros((QH, D))
    u = HALF_STEP[cabi.BF16] if pool.dtype == cabi.BF16 else HALF_STEP[cabi.F16]
    seen = False
    for h in range(KVH):
        ks, vs = [], []
        for b in map(int, sel[h]):
            if b < 0 or b * bs >= length or not 0 <= table[b] < pool.NB:
                continue
            n = min(bs, length - b * bs)
            ks.append(pool.k[layer, table[b], h, :n])
            vs.append(pool.v[layer, table[b], h, :n])
        if not ks:
            continue
        seen = True
        k, v = np.concatenate(ks), np.concatenate(vs)
        for i in range(h * G, (h + 1) * G):
            s = (k @ q[i]) * scale
            p = np.exp(s - s.max())
            o = p @ v / p.sum()
            vmag = np.abs(v)
            if pool.dtype == cabi.INT8:
                vmag = np.broadcast_to(np.abs(v).max(1, keepdims=True) / 127 * 1279 * 1.5, v.shape)   # the codes' maximum may be below 127
            A = p @ np.abs(v) / p.sum()
            wide = p @ vmag / p.sum()
            ds = (D + 8) * 2.0 ** -24 * (np.abs(k) @ np.abs(q[i])).max() * scale
            if pool.dtype == cabi.INT8:
                ds *= 20                                         # 1152 sum q comes off again: |1152 + code| <= 1279 against codes spread over +-127
            e = 1.1 * u * (A + np.abs(o)) + 2 * (ds + 2.0 ** -20) * A + (len(k) + 8) * 2.0 ** -24 * wide
            if pool.dtype != cabi.BF16:
                e = e + 2.0 ** -25 * (len(k) if pool.dtype != cabi.INT8 else 200 * len(k)) * np.abs(v).max() / p.sum() + 2.0 ** -24 * D * np.abs(k).max() * scale * A
            if gate is not None:
                sg = 1 / (1 + np.exp(-gate[i]))
                o, e = o * sg, e * sg + np.abs(o) * sg * 2.0 ** -20
            out[i], tol[i] = o, e
    return (out, tol) if seen else (None, None)


def attend_ok(got, want, tol, io):
    """Elementwise: the bound, and half a step of the output's type."""
    lim = tol + HALF_STEP[io] * (np.abs(want) + tol) + (2.0 ** -25 if io == cabi.F16 else 0.0)
    err = np.abs(np.asarray(got, np.float64) - want)
    return bool((err <= lim).all()), float((err / lim).max())
