"""The error bound of the 8-bit cache's attention (kv8_bounds.py) without a
GPU: it takes the kernels' arithmetic as restated here, and refuses it with one
part of the queries left out, or with weights of 8 bits."""
import numpy as np
import pytest

import kv8_bounds as bounds
import kv8_ref as ref
from fekv.metadata import build_step_metadata


def emulate(q, pools, n, G, scale, bf16, parts, weight_bits=11):
    """One sequence, no mask, head by head: queries as `parts` parts, weights
    2^(s + e - max) rounded to `weight_bits`, the result to the 16-bit type."""
    (kc, ke), (vc, ve) = pools
    K, V = ref.values(kc, ke), ref.decode_e4m3(vc)
    rows, hq, _ = q.shape
    out = np.zeros(q.shape)
    qin = bounds.parts_of(q.astype(np.float64), parts)
    for h in range(hq):
        e = np.repeat(ve[:, h // G].astype(float) - 127, 16)[:n]
        s2 = qin[:, h] @ K[:n, h // G].T * scale / np.log(2.0) + e
        w = np.exp2(s2 - s2.max(-1, keepdims=True))
        m, x = np.frexp(w)
        stored = np.ldexp(np.round(m * 2.0 ** weight_bits) / 2.0 ** weight_bits, x)
        out[:, h] = stored @ V[:n, h // G] / (w * np.exp2(-e)).sum(-1, keepdims=True)
    if bf16:
        m, x = np.frexp(out)
        return np.ldexp(np.round(m * 256) / 256, x)
    return out.astype(np.float16).astype(np.float64)


def case(seed, bf16, dim, cancel):
    rng = np.random.default_rng(seed)
    hq, hkv, n, rows = 8, 4, 48, 17
    pools = []
    for _ in range(2):
        codes = ref.encode_e4m3(rng.standard_normal((n, hkv, dim)) * 60)
        pools.append((codes, rng.integers(117, 125, (n // 16, hkv)).astype(np.uint8)))
    if cancel:
        q = bounds.cancelling_queries(rng, rows, hq, dim, bf16)
        bounds.even_keys(rng, *pools[0], dim, bf16)
    else:
        q = rng.standard_normal((rows, hq, dim))
        m, x = np.frexp(q)
        bits = 2.0 ** (8 if bf16 else 11)
        q = np.ldexp(np.round(m * bits) / bits, x)
    md = build_step_metadata([np.arange(n // 16)], [n - rows], [rows], 16)
    want, bound = bounds.attention(q, *pools, md, hq, hkv, 16, False, bf16)
    run = lambda parts, bits=11: np.abs(emulate(  # noqa: E731
        q, pools, n, hq // hkv, dim ** -0.5, bf16, parts, bits) - want) <= bound
    return run, want, bound


@pytest.mark.parametrize("dim", [128, 256])
@pytest.mark.parametrize("bf16", [True, False])
def test_bound_takes_all_parts_and_refuses_one_less(bf16, dim):
    parts = 2 if bf16 else 3
    run, want, bound = case(dim, bf16, dim, True)
    assert run(parts).all()
    assert not run(parts - 1).all(-1).any()  # every row and head shows it
    run, want, bound = case(dim + 1, bf16, dim, False)
    assert run(parts).all()


def test_bound_refuses_weights_of_fewer_bits():
    """Outputs in f16 show weights rounded to 8 bits (bf16's) where the kernels
    keep 11."""
    run, want, bound = case(5, False, 128, False)
    assert run(3).all()
    assert not run(3, 8).all()


@pytest.mark.parametrize("bf16,parts,exact_to,absolute", [(True, 2, 9, -17.8), (False, 3, 6, -17.8)])
def test_what_the_parts_of_a_query_hold(bf16, parts, exact_to, absolute):
    """Elements down to 2^-exact_to of a row's largest enter exactly (9 and 6
    octaves whatever the largest is), smaller ones to 2^absolute of it."""
    bits = 8 if bf16 else 11
    rng = np.random.default_rng(1)
    m = np.arange(2 ** (bits - 1), 2 ** bits) / 2.0 ** (bits - 1)  # every significand, 1 .. 2
    worst = 0.0
    for top in [1.0, 1.25, 1.75, 1.75 + 2.0 ** (1 - bits), 2 - 2.0 ** (1 - bits)]:
        for octave in range(0, 24):
            x = m * 2.0 ** -octave
            x = x[x <= top]
            row = np.concatenate([[top], x, -x, rng.permutation(x)])
            off = np.abs(bounds.parts_of(row[None], parts)[0] - row)
            if octave < exact_to:
                assert off.max() == 0, (top, octave)
            worst = max(worst, off.max() / top)
    assert 2.0 ** (absolute - 1) < worst <= 2.0 ** absolute, np.log2(worst)
