"""The attention cache's operators from their definitions, in 64 bits on the CPU, for the tests.

Everything is numpy and written row by row; inputs are what the calls get (already rounded to the
call's type). The error bounds beside the values are derived here from the kernels' roundings, before
any comparison: see attend_bounds.
"""
from __future__ import annotations

import math

import numpy as np

GROUP = 64


def bf16(x):
    """f32 array rounded to bf16 (nearest, ties to even), as f32."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    out = ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32).copy()
    nan = np.isnan(x)
    out[nan] = np.nan
    return out


def quantise(x):
    """Rows [..., dim] (f32) -> (values, low, step) as f64 [..., dim] each (low and step per element)."""
    x = np.asarray(x, np.float32)
    dim = x.shape[-1]
    val, low_e, step_e = (np.zeros(x.shape) for _ in range(3))
    for g in range(0, dim, GROUP):
        part = x[..., g:g + GROUP]
        hi, lo = part.max(axis=-1, keepdims=True), part.min(axis=-1, keepdims=True)
        with np.errstate(all="ignore"):
            step = bf16((hi - lo) * (np.float32(1.0) / np.float32(15.0))).astype(np.float64)
            low = bf16(lo).astype(np.float64)
            at = (part.astype(np.float64) - low) / np.where(step == 0, 1.0, step)
            code = np.where(step == 0, 0.0, np.clip(np.rint(at), 0, 15))
            v = (low + step * code).astype(np.float32).astype(np.float64)
        bad = np.broadcast_to(~np.isfinite(part.astype(np.float64)).all(axis=-1, keepdims=True) | ~np.isfinite(step),
                              v.shape)
        val[..., g:g + GROUP] = np.where(bad, np.nan, v)
        low_e[..., g:g + GROUP] = np.where(bad, np.nan, np.broadcast_to(low, v.shape))
        step_e[..., g:g + GROUP] = np.where(bad, np.nan, np.broadcast_to(step, v.shape))
    return val, low_e, step_e


UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}  # half a step, relative
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}  # half a step of the subnormals


class Rows:
    """The quantised rows of one head: keys and values with their low and step."""

    def __init__(self, keys, values):
        self.k, self.k_low, self.k_step = quantise(keys)
        self.v, self.v_low, self.v_step = quantise(values)


def attend_head(q, rows, which, scale, dtype):
    """One query of one head over the rows `which` (a list, repeats count): out, lse, p and bounds on
    the kernels' error in each.

    z = scale * q . k is summed in f32 over dim products and their low terms (at most dim + 16
    roundings of 2^-23 relative to the sum of magnitudes; the tensor core's additions truncate). The
    query itself is exact in f16 for 16-bit types, and 2^-22 off for f32 (two halves). ex2 is off by
    2^-22 relative, its argument by 2^-24 of |z - max| (in log2). p * step is rounded to f16 (2^-12
    relative) in 16-bit calls, to two halves (2^-22) in f32 ones; half a subnormal step of f16 in units
    where the largest step is 4096 adds 2^-37 of it per row, times the code. Sums over n rows add n
    roundings of 2^-23. The result is rounded to the call's type. With many columns (16-bit types), the
    values themselves are rounded to f16 as well (2^-12 more), in units of their row's power of two (at
    most twice its largest level), whose subnormals add 2^-25 of it.
    """
    d = len(q)
    n = len(which)
    if n == 0:
        return np.zeros(d), -math.inf, np.zeros(0), np.zeros(d), 0.0, np.zeros(0)
    q = np.asarray(q, np.float64)
    k, v = rows.k[which], rows.v[which]
    z = scale * (k @ q)
    mag = abs(scale) * ((np.abs(rows.k_low[which]) + 15 * rows.k_step[which]) @ np.abs(q))
    dz = ((d + 16) * 2.0 ** -23 + (2.0 ** -22 if dtype == "f32" else 2.0 ** -30)) * mag.max()
    top = z.max()
    e = np.exp(z - top)
    total = e.sum()
    p = e / total
    lse = top + math.log(total)
    # relative error of one p: exponent's argument, ex2, sum and division
    spread = min((top - z).max() / math.log(2.0), 160.0)
    dp = 2.0 * dz + (spread + 8) * 2.0 ** -23 + (n + 32) * 2.0 ** -23
    out = p @ v
    level = 15 * rows.v_step[which] + np.abs(rows.v_low[which])
    a = p @ level
    round_p = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    # a subnormal p * level: half of 2^-24 in units of (the level's power of two) / 4096, times 2^3 of lag
    tiny = (n * 2.0 ** -25 / 4096 * 8 + 2.0 ** -25) * 2 * np.nanmax(level) if dtype != "f32" else 0.0
    err = a * (round_p + dp + (n + 64) * 2.0 ** -23) + tiny
    err = err + UNIT[dtype] * (np.abs(out) + err) + TINY[dtype]
    return out, lse, p, err, dz + (n + 32) * 2.0 ** -23 + abs(lse) * 2.0 ** -22, p * dp + 2.0 ** -126


def attend_head_tight(q, rows, which, scale, dtype, wide=False):
    """out, lse, p and the error of each, as attend_head, with every row's error by its own magnitude.

    A score's error is that of its own sum, (dim + 16) roundings of 2^-23 of scale * sum |key| |q| with |key| at most
    |low| + 15 step, and the query's (2^-22 in f32 calls). p's relative error dp is its score's, the normaliser's (their mean),
    and the exponential's. p * step is rounded to f16 (2^-12) in bf16 calls and to two halves (2^-22) else, in units where
    2^11 is at most the largest p * step of the column and group when it was set: half of f16's 2^-24 adds
    2^-36 of that per row, times a code of 15. Sums over n rows add n roundings of 2^-23.

    wide: blocks of 128 columns. A query's sum meets low and 8 step as two halves, and a key lies up to 2^8 below its
    tile's unit (2^-20 of the score's magnitudes for both). Values are rounded to f16 as p is (2^-12 each), p in units
    of the largest p * level, which may be taken 2^9 too large (rows up to 2^8 apart share a unit): 2^-25 / 2^12 * 2^9
    = 2^-28 of it per row.
    """
    n, d = len(which), len(q)
    q = np.asarray(q, np.float64)
    k, v = rows.k[which], rows.v[which]
    z = scale * (k @ q)
    mag = abs(scale) * ((np.abs(rows.k_low[which]) + 15 * rows.k_step[which]) @ np.abs(q))
    dz = ((d + 16) * 2.0 ** -23 + (2.0 ** -22 if dtype == "f32" else 2.0 ** -30) + (2.0 ** -20 if wide else 0)) * mag
    top = z.max()
    e = np.exp(z - top)
    p = e / e.sum()
    lse = top + math.log(e.sum())
    spread = np.minimum((top - z) / math.log(2.0), 160.0)
    dp = dz + (spread + 8) * 2.0 ** -23
    dp = dp + p @ dp + (n + 32) * 2.0 ** -23
    out = p @ v
    level = 15 * rows.v_step[which] + np.abs(rows.v_low[which])
    round_p = 2.0 ** -11 if wide else 2.0 ** -12 if dtype == "bf16" else 2.0 ** -22
    tiny = 15 * n * (2.0 ** -36 * (p[:, None] * rows.v_step[which]).max(axis=0) + 2.0 ** -136)
    if wide:
        tiny = tiny + n * 2.0 ** -28 * (p[:, None] * level).max()
    err = (p * (dp + round_p + (n + 64) * 2.0 ** -23)) @ level + tiny
    err = err + UNIT[dtype] * (np.abs(out) + err) + TINY[dtype]
    return out, lse, p, err, p @ dz + (n + 32) * 2.0 ** -23 + abs(lse) * 2.0 ** -22, p * dp + 2.0 ** -126


def evict(length, keep, w, ids=None, protect=None):
    """(new length, source row of every new row, rows that leave)."""
    rank = []
    for r in range(length):
        x = float(w[r])
        top = x != x or (protect is not None and int(ids[r]) >= int(protect))
        rank.append(math.inf if top else x)
    order = sorted(range(length), key=lambda r: (-rank[r], r))
    m = min(length, keep)
    kept = set(order[:m])
    movers = iter(sorted(r for r in kept if r >= m))
    src = [r if r in kept else next(movers) for r in range(m)]
    return m, src, [r for r in range(length) if r not in kept]
