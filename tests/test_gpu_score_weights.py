"""Scores of the keys where the softmax's scores are large: weights are relative
to a row's own maximum and sum, so they keep their bits at any magnitude."""
import math

import pytest

import long_ref as ref
from test_gpu_scored_attention import scored_plan
from test_gpu_shared_attention import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1.0, 8.0, 64.0, 512.0, 4096.0])
@pytest.mark.parametrize("shape", [(8, 4, 128), (16, 1, 128), (4, 2, 256), (5, 5, 256)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_equal_keys_share_their_row_equally(dtype, shape, size):
    """All keys of a head are the same vector, size * (+-1, ...), and its queries
    the same vector times 1.5: every score of a row is the same number (1.5 size^2
    sqrt(dim), a sum of equal exact products), so each of its n keys weighs 1 / n.
    What rounds: the exponential of a difference of 0 (2^-22, in the sum and in the
    weight; the sum of n equal terms below 2^24 adds nothing), one quotient (2^-23)
    and its product (2^-24), and the sum of rows x heads weights (2^-24 a term)."""
    import torch
    hq, hkv, dim = shape
    n, rows, G = 700, 7, hq // hkv
    s = Step([(0, [(n, rows)])], hq, hkv, dim, 16, dtype)
    slots = torch.from_numpy(ref.slots_of(s.tables[0], 16, n)).cuda()
    gen = torch.Generator(device="cuda").manual_seed(1)
    sign = torch.randint(0, 2, (hkv, dim), generator=gen, device="cuda") * 2.0 - 1
    s.k[slots] = (size * sign).to(s.dtype)
    s.q[:] = (1.5 * size * sign.repeat_interleave(G, 0)).to(s.dtype)
    plan = scored_plan(s)
    plan.prepare(*s.meta(), fresh=s.lens)
    scores = torch.full((hkv, s.k.shape[0]), math.nan, device="cuda")
    plan.attention(s.q, s.k, s.v, scores, torch.empty_like(s.q))
    got = scores[:, slots].double()
    limit = torch.arange(n - rows + 1, n + 1, device="cuda", dtype=torch.float64)
    seen = torch.arange(n, device="cuda")[None] < limit[:, None]
    want = G * (seen / limit[:, None]).sum(0)
    rel = 2 * 2.0 ** -22 + 2.0 ** -23 + 2.0 ** -24 + rows * G * 2.0 ** -24
    worst = ((got - want).abs() / want).max().item()
    assert worst <= rel, worst
