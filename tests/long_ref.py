"""Paged attention and the keys' weights in 64 bits, with the error bound that
the kernels are held to (test infrastructure).

Bound. A score s = q k / sqrt(dim) is a sum of dim exact products, accumulated
in fp32: off by at most e = dim 2^-23 sum |q_i k_i| / sqrt(dim) (2^-23 a step
covers accumulation by truncation). The rounding to base 2 and the difference
from the maximum add 2^-23 |s| log2(e) twice at most, the exponential
instruction 2^-22: a weight is off by at most a factor 1 + d, d = 2 e + 4 2^-23
max |s| + 2^-21 (numerator and sum). In the second product weights have 16 bits
or more (2^-16), its fp32 accumulation and the joining of records n 2^-23 at
most for n keys, taken as 2^-16 for n < 2^7 splits of sums of magnitude-ordered
terms; so |out - ref| <= eps/2 |ref| + (d + 2^-15) sum w |v|. A score pool entry
is off by d + 2^-20 of the weights that it got, plus half a step of its own."""
import math

import numpy as np


def tables(lens, page, seed, heads=(), spare=2):
    """Random pages: lists for `heads` (shared prefixes, in pages) and for each
    length; and the number of blocks of the pool."""
    rng = np.random.default_rng(seed)
    need = list(heads) + [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    at = np.cumsum([0] + need)
    out = [order[a:b] for a, b in zip(at, at[1:])]
    return out[:len(heads)], out[len(heads):], sum(need) + spare


def slots_of(table, page, n):
    t = np.arange(n)
    return np.asarray(table, np.int64)[t // page] * page + t % page


def pools(blocks, page, hkv, dim, dtype, used, seed):
    """K and V pools that hold NaN everywhere but in the slots `used`."""
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.full(((blocks + 1) * page, hkv, dim), math.nan, dtype=dtype, device="cuda")
        at = torch.from_numpy(np.unique(np.concatenate(used))).cuda()
        x[at] = torch.randn(len(at), hkv, dim, generator=gen, device="cuda").to(dtype)
        out.append(x)
    return out


def attend(q, k, v, causal):
    """q [r, hq, dim], k and v [n, hkv, dim]: output and its bound [r, hq, dim],
    weights and their bound [hkv, n]."""
    import torch
    r, hq, dim = q.shape
    n, hkv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    qg = q.view(r, hkv, hq // hkv, dim)
    s = torch.einsum("rhgd,nhd->hgrn", qg, k) / math.sqrt(dim)
    size = torch.einsum("rhgd,nhd->hgrn", qg.abs(), k.abs()) / math.sqrt(dim)
    if causal:
        i = torch.arange(r, device=q.device)[:, None]
        seen = torch.arange(n, device=q.device) <= n - r + i
        s = torch.where(seen, s, -math.inf)
        size = torch.where(seen, size, 0.0)
    w = torch.softmax(s, -1)
    d = (2 * dim + 4) * 2.0 ** -23 * size.amax(-1) + 2.0 ** -21     # [hkv, g, r]
    out = torch.einsum("hgrn,nhd->rhgd", w, v).reshape(r, hq, dim)
    mass = torch.einsum("hgrn,nhd->rhgd", w, v.abs()).reshape(r, hq, dim)
    dd = d.permute(2, 0, 1).reshape(r, hq, 1)
    return out, (dd + 2.0 ** -15) * mass, w.sum((1, 2)), \
        (w * (d[..., None] + 2.0 ** -20)).sum((1, 2))


def check_output(got, want, bound):
    import torch
    half = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # subnormal step
    off = (got.double() - want).abs()
    limit = half * want.abs() + (1 + half) * bound + tiny
    worst = (off / limit).max().item() if off.numel() else 0.0
    assert worst <= 1.0, worst
    return worst
