"""What the attention kernels over the 8-bit cache may be off by, from each
rounding that they make (test infrastructure beside kv8_ref.py, whose bound is
one for all of them and wider).

For one row and head: s_t = scale * sum_d q k, p = softmax(s), out = sum p v,
v = code * 2^e. A kernel has

* the query as it enters the products, q': exact in f16 (decode rows, f16), in
  f16 after a power-of-two scale (decode rows, bf16), or the sum of two (bf16)
  or three (f16) e4m3 parts (more packed rows); `entering` restates it, and
  |q - q'| moves s_t by at most scale * sum |q - q'| |k|;
* sums of n products in fp32: exact products, n additions of which each loses
  at most a unit in the last place of the running magnitudes: n 2^-23 sum |q' k|
  with n = dim times the parts, and (keys) 2^-23 sum w |code| for the output;
* the exponent in base 2, three fp32 roundings of terms no larger than
  |s| + max |s + e| + 80: 2^-22 of that, and ex2's own 2^-22;
* the weight as a half: 2^-11 of it, and where it is subnormal 2^-25 of the
  stored unit, which is at most 2^-15 (decode) or 2^-7 (rows) of the largest
  p 2^e of the row; the weights' sum is fp32 over the unrounded weights:
  (keys) 2^-24 of it;
* the result: half a unit in the last place, and 2^-22 for the quotient.
"""
from __future__ import annotations

import math

import numpy as np

import kv8_ref as ref

DECODE_ROWS = 16  # packed rows (query rows x group) that the decode kernel takes


def query_exponents(q: np.ndarray, top: int, low: int, high: int) -> np.ndarray:
    """Scale exponents of rows: the largest magnitude in (.., 2^top] of e4m3's
    448-rule for top = None; limits as in the kernels."""
    amax = np.where(np.isfinite(q), np.abs(q), 0.0).max(-1)
    f, x = np.frexp(np.where(amax == 0, 2.0 ** -200, amax))  # amax = f 2^x, f in [0.5, 1)
    if top is None:
        e = np.where(f > 0.875, x - 8, x - 9)                # smallest e with amax <= 448 2^e
    else:
        e = x - 1 - top
    return np.clip(e, low, high)


def parts_of(q: np.ndarray, parts: int) -> np.ndarray:
    """The sum of the first `parts` e4m3 parts of rows [.., dim] (float64)."""
    up = np.exp2(-query_exponents(q, None, -60, 120).astype(np.float64))[..., None]
    left, total = q * up, np.zeros_like(q)
    for _ in range(parts):
        c = ref.decode_e4m3(ref.encode_e4m3(left))
        total, left = total + c, left - c
    return total / up


def entering(q: np.ndarray, rows: int, bf16: bool):
    """(q', products a score sums, a stored weight's smallest unit) of a
    sequence with `rows` packed rows; q float64 [.., dim]."""
    dim = q.shape[-1]
    if rows > DECODE_ROWS:
        parts = 2 if bf16 else 3
        return parts_of(q, parts), dim * parts, 2.0 ** -7
    if not bf16:
        return q, dim, 2.0 ** -15
    up = np.exp2(-query_exponents(q, 14, -60, 113).astype(np.float64))[..., None]
    return (q * up).astype(np.float16).astype(np.float64) / up, dim, 2.0 ** -15


def head(q, q1, products, unit, k, v, vexp, seen, scale, bf16):
    """(out, bound) for rows q [n, dim] of one KV head: q1 = q'; k, v [keys,
    dim]; vexp [keys] the V scales' exponents; seen [n, keys]."""
    s = np.where(seen, q @ k.T * scale, -np.inf)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - m)
    p /= p.sum(-1, keepdims=True)
    out = p @ v
    s2 = s / math.log(2.0)
    top = np.where(seen, np.abs(s2 + vexp), 0.0).max(-1, keepdims=True) + 80
    delta = (np.abs(q - q1) + products * 2.0 ** -23 * np.abs(q1)) @ np.abs(k).T * scale
    delta += math.log(2.0) * 2.0 ** -22 * (np.where(seen, np.abs(s2), 0.0) + top) + 2.0 ** -22
    grow = np.expm1(np.where(seen, delta, 0.0))
    keys = k.shape[0]
    # the sum of weights: their own growth and the rounding of the sum
    total = (p * grow).sum(-1, keepdims=True) + keys * 2.0 ** -24
    rel = (1 + grow) * (1 + total) * (1 + 2.0 ** -11) * (1 + keys * 2.0 ** -23 + 2.0 ** -22) - 1
    bound = (p * rel) @ np.abs(v)
    code = np.abs(v) * np.exp2(-vexp)[:, None]
    largest = (p * np.exp2(vexp)).max(-1, keepdims=True)
    bound += 2.0 ** -25 * unit * largest * (seen @ code)
    mant, low = (7, -126) if bf16 else (10, -14)
    return out, bound + 0.5 * np.exp2(
        np.floor(np.log2(np.maximum(np.abs(out) + bound, 2.0 ** low))) - mant)


def attention(q, kpool, vpool, md, hq, hkv, page, causal, bf16):
    """(out, bound) of a step: q [rows, hq, dim]; kpool, vpool (codes, exps)."""
    rows, _, dim = q.shape
    G = hq // hkv
    q = np.asarray(q, np.float64)
    kval, vval = ref.values(*kpool), ref.values(*vpool)
    vexp = np.clip(vpool[1].astype(np.float64) - 127, ref.MIN_E, ref.MAX_E)
    out, bound = np.zeros((rows, hq, dim)), np.zeros((rows, hq, dim))
    for b in range(md.batch):
        p0, p1 = int(md.kv[b]), int(md.kv[b + 1])
        n = (p1 - p0 - 1) * page + int(md.last[b])
        t = np.arange(n)
        slots = np.asarray(md.pages[p0:p1], np.int64)[t // page] * page + t % page
        q0, q1 = int(md.qo[b]), int(md.qo[b + 1])
        r = q1 - q0
        if r == 0:
            continue
        see = t[None, :] <= (n - r + np.arange(r)[:, None] if causal else n)
        see = np.repeat(see * np.ones((r, 1), bool), G, 0)
        qin, products, unit = entering(q[q0:q1], r * G, bf16)
        for h in range(hkv):
            at = (slice(q0, q1), slice(h * G, (h + 1) * G))
            flat = lambda x: x[:, h * G:(h + 1) * G].reshape(r * G, dim)  # noqa: E731
            o, e = head(flat(q[q0:q1]), flat(qin), products, unit, kval[slots, h], vval[slots, h],
                        vexp[slots // ref.BLOCK, h], see, 1.0 / math.sqrt(dim), bf16)
            out[at], bound[at] = o.reshape(r, G, dim), e.reshape(r, G, dim)
    return out, bound


def cancelling_queries(rng, rows, hq, dim, bf16):
    """Rows whose halves cancel but for what the last part holds: half of the
    dims +X + t, half -X + t, with X the earlier parts' and t the last part's
    (in units where e4m3's largest is 448: X = 300, t = 1/4 in f16; 288 and 2
    in bf16). A query without its last part scores 0 against any key whose dims
    are equal."""
    x, t = (288.0, 2.0) if bf16 else (300.0, 0.25)
    sign = np.where(np.arange(dim) % 2 == 0, 1.0, -1.0)
    q = np.empty((rows, hq, dim))
    for r in range(rows):
        for h in range(hq):
            q[r, h] = (rng.permutation(sign) * x + t) * 2.0 ** -8
    return q.astype(np.float32)


def even_keys(rng, kcodes, kexps, dim, bf16):
    """Sets every key's dims equal, of either sign: against cancelling_queries
    the scores are of the order of one."""
    slots, hkv, _ = kcodes.shape
    t = (2.0 if bf16 else 0.25) * 2.0 ** -8
    size = 1.0 / (t * dim * dim ** -0.5)  # a score of 1
    e = math.floor(math.log2(size)) - 3
    val = np.round(size / 2.0 ** e) * np.where(rng.random((slots, hkv)) < 0.5, 1.0, -1.0)
    kcodes[:] = ref.encode_e4m3(val)[..., None]
    kexps[:] = 127 + e
