"""The 8-bit KV cache restated in 64 bits (test infrastructure): quantisation,
append, and attention with the error bound its kernels are held to."""
from __future__ import annotations

import math

import numpy as np

BLOCK = 16
MIN_E, MAX_E = -32, 64


def decode_e4m3(codes: np.ndarray) -> np.ndarray:
    """uint8 e4m3 codes as float64."""
    c = codes.astype(np.int64)
    sign = np.where(c & 0x80, -1.0, 1.0)
    e, m = (c >> 3) & 15, c & 7
    x = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    return np.where((c & 0x7F) == 0x7F, np.nan, sign * x)


_GRID = decode_e4m3(np.arange(127, dtype=np.uint8))  # 0 .. 448, ascending


def encode_e4m3(x: np.ndarray) -> np.ndarray:
    """float64 to e4m3 codes: nearest, ties to the even code, saturating."""
    a = np.abs(x)
    hi = np.clip(np.searchsorted(_GRID, a, side="left"), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - _GRID[lo], _GRID[hi] - a
    pick = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    pick = np.where(a >= 448.0, 126, pick)
    code = np.where(np.isnan(x), 0x7F, pick | np.where(np.signbit(x), 0x80, 0))
    return code.astype(np.uint8)


def needed(amax: float) -> int:
    """Smallest e with amax <= 448 * 2^e, within the limits."""
    if amax == 0:
        return MIN_E
    f, x = math.frexp(amax / 448.0)  # f in [0.5, 1)
    return min(max(x - 1 if f == 0.5 else x, MIN_E), MAX_E)


def values(codes: np.ndarray, exps: np.ndarray) -> np.ndarray:
    """[slots, hkv, dim] float64 values; exponent bytes outside the limits read
    as the nearest within."""
    e = np.clip(exps.astype(np.float64) - 127, MIN_E, MAX_E)
    return decode_e4m3(codes) * np.repeat(np.exp2(e), BLOCK, axis=0)[..., None]


def append(x: np.ndarray, codes: np.ndarray, exps: np.ndarray, slots, skip=()):
    """Append fp32 rows x [rows, hkv, dim] in place; rows in `skip` are not
    appended."""
    slots = [int(s) for s in slots]
    rows = len(slots)
    good = [0 <= s < codes.shape[0] and i not in skip for i, s in enumerate(slots)]
    runs = []  # adjacent rows of one block, skipped rows aside
    for i in range(rows):
        if not good[i]:
            continue
        if runs and slots[i] // BLOCK == slots[runs[-1][-1]] // BLOCK and \
                slots[i] > slots[runs[-1][-1]]:
            runs[-1].append(i)
        else:
            runs.append([i])
    for run in runs:
        at = [slots[i] for i in run]
        blk, kept = divmod(at[0], BLOCK)
        for h in range(codes.shape[1]):
            v = x[run, h].astype(np.float64)
            fin = np.abs(v[np.isfinite(v)])
            e = needed(float(fin.max()) if fin.size else 0.0)
            if kept:
                old = int(exps[blk, h]) - 127
                e = max(e, old)
                if e > old:
                    k = slice(blk * BLOCK, blk * BLOCK + kept)
                    codes[k, h] = encode_e4m3(decode_e4m3(codes[k, h]) * 2.0 ** (old - e))
            codes[at, h] = encode_e4m3(v * 2.0 ** -e)
            exps[blk, h] = e + 127


def rotate(x: np.ndarray, pos, cache: np.ndarray) -> np.ndarray:
    """fp32 rotation of [rows, heads, dim], each product and sum rounded."""
    r = cache.shape[1] // 2
    c, s = cache[pos][:, None, :r], cache[pos][:, None, r:]
    out = x.astype(np.float32).copy()
    a, b = out[..., :r].copy(), out[..., r:2 * r].copy()
    out[..., :r] = a * c - b * s
    out[..., r:2 * r] = b * c + a * s
    return out


def attention(q: np.ndarray, kval: np.ndarray, vval: np.ndarray, md, hq, hkv, page, causal, bf16):
    """float64 attention over pool values (rows of NaN outside the sequences
    are never touched). Returns (out, bound): the elementwise bound on the
    kernels' error, from their roundings:
      * a query element: 2^-9 of it for f16, nothing for bf16, and 2^-19 of the
        row's largest (the last part's subnormals; no kernel rounds more); the score moves by at
        most eps = scale * sum |dq k|, the weights by e^(+-eps), so the output
        by (e^(2 eps) - 1) sum p |v|;
      * a weight: 2^-9 + 2^-12 of it (no kernel rounds more: halves), its
        exponential 2^-14 (score up to some hundreds in fp32, exp2 in
        hardware) on the weight and again on the sum, and 2^-31 of the
        largest weight per key (underflow);
      * the result: half a unit in the last place."""
    rows, _, dim = q.shape
    G = hq // hkv
    scale = 1.0 / math.sqrt(dim)
    out = np.zeros((rows, hq, dim))
    bound = np.zeros((rows, hq, dim))
    qerr = 0.0 if bf16 else 2.0 ** -9
    for b in range(md.batch):
        p0, p1 = int(md.kv[b]), int(md.kv[b + 1])
        n = (p1 - p0 - 1) * page + int(md.last[b])
        t = np.arange(n)
        slots = np.asarray(md.pages[p0:p1], np.int64)[t // page] * page + t % page
        q0, q1 = int(md.qo[b]), int(md.qo[b + 1])
        r = q1 - q0
        if r == 0:
            continue
        K, V = kval[slots], vval[slots]
        for h in range(hkv):
            k, v = K[:, h], V[:, h]
            qq = q[q0:q1, h * G:(h + 1) * G]
            s = np.einsum("rgd,nd->rgn", qq, k) * scale
            dq = qerr * np.abs(qq) + 2.0 ** -19 * np.abs(qq).max(-1, keepdims=True)
            eps = np.einsum("rgd,nd->rgn", dq, np.abs(k)) * scale
            if causal:
                seen = t[None, :] <= n - r + np.arange(r)[:, None]
                s = np.where(seen[:, None, :], s, -np.inf)
            m = s.max(-1, keepdims=True)
            w = np.exp(s - m)
            l = w.sum(-1, keepdims=True)
            w = w / l
            o = np.einsum("rgn,nd->rgd", w, v)
            mass = np.einsum("rgn,nd->rgd", w, np.abs(v))
            e = np.where(np.isfinite(s), eps, 0.0).max(-1)[..., None]
            tail = n * 2.0 ** -31 * np.abs(v).max() / l[..., 0][..., None]
            rel = np.expm1(2 * e) + 2.0 ** -9 + 2.0 ** -12 + 2 * 2.0 ** -14
            mant, low = (7, -126) if bf16 else (10, -14)
            ulp = np.exp2(np.floor(np.log2(np.maximum(np.abs(o) + rel * mass, 2.0 ** low))) - mant)
            out[q0:q1, h * G:(h + 1) * G] = o
            bound[q0:q1, h * G:(h + 1) * G] = rel * mass + tail + 0.5 * ulp
    return out, bound
