"""Rotary embedding with several position axes, alone and fused with the
append: bit-exact against the rotation written out in float32 (products and
sums rounded one by one), and against rope() where all axes agree."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

SECTIONS = {128: [((16, 24, 24), False), ((24, 20, 20), True), ((64,), False), ((0, 31, 33), False)],
            64: [((11, 11, 10), True), ((8, 24), False)],
            256: [((44, 42, 42), True), ((32, 32, 32, 32), False)],
            20: [((4, 3, 3), True)], 0: [((0, 0), False)]}


def rotated(x, pos, cache, pairs):
    """float32 [rows, heads, dim] turned pair by pair; each operation rounds."""
    r = len(pairs)
    x = x.copy()
    if r:
        at = np.stack([pos[a] for a in pairs], 1)  # [rows, pairs]
        j = np.arange(r)
        c, s = cache[at, j][:, None], cache[at, j + r][:, None]
        a, b = x[..., :r].copy(), x[..., r:2 * r].copy()
        x[..., :r] = a * c - b * s
        x[..., r:2 * r] = b * c + a * s
    return x


def make(rows, hq, hkv, dim, rot, axes, dtype, seed, most=700, slots=None):
    import torch
    rng = np.random.default_rng(seed)
    t = {n: torch.from_numpy(rng.standard_normal((rows, h, dim)).astype(np.float32) * 2).to(dtype)
         for n, h in (("q", hq), ("k", hkv), ("v", hkv))}
    t["pos"] = torch.from_numpy(rng.integers(0, most, (axes, rows)))
    ang = rng.uniform(0, 7, (most, rot // 2))
    t["cache"] = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)], 1).astype(np.float32))
    slots = rows + 48 if slots is None else slots
    slots = (slots + 15) // 16 * 16
    for n in ("kc", "vc"):
        t[n] = torch.from_numpy(rng.standard_normal((slots, hkv, dim)).astype(np.float32)).to(dtype)
    t["slots"] = torch.from_numpy(rng.permutation(slots)[:rows])
    return t


def same(got, want):
    import torch
    assert got.shape == want.shape
    assert torch.equal(got.cpu().contiguous().view(torch.int16), want.contiguous().view(torch.int16))


CASES = [(1, 16, 8, 128, 128), (64, 32, 8, 128, 128), (37, 6, 3, 128, 64), (5, 40, 8, 128, 128),
         (3, 16, 2, 256, 256), (9, 5, 5, 256, 128), (130, 8, 1, 128, 128), (7, 3, 1, 44, 20),
         (6, 2, 2, 128, 0), (1500, 12, 4, 128, 128),
         (2500, 12, 4, 128, 128), (4097, 0, 8, 128, 64), (4100, 20, 4, 256, 128),
         (4500, 32, 8, 128, 128),
         (4099, 4, 1, 128, 128), (4097, 64, 8, 128, 128)]


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("shape", CASES)
def test_rotation_and_append(shape, dtype):
    import fekv
    import torch
    rows, hq, hkv, dim, rot = shape
    for i, (sections, turns) in enumerate(SECTIONS[rot]):
        pairs = fekv.rope_sections(sections, turns)
        t = make(rows, hq, hkv, dim, rot, len(sections), getattr(torch, dtype), rows + i)
        t["slots"][::3] = -1
        pos, cache = t["pos"].numpy(), t["cache"].numpy()
        q, k = (torch.from_numpy(rotated(t[n].float().numpy(), pos, cache, pairs)).to(t[n].dtype)
                for n in "qk")
        d = {n: x.cuda() for n, x in t.items()}
        fekv.rope_axes_append(d["q"], d["k"], d["v"], d["kc"], d["vc"], d["slots"], d["pos"],
                              d["cache"], pairs)
        kc, vc = t["kc"].clone(), t["vc"].clone()
        live = t["slots"] >= 0
        kc[t["slots"][live]] = k[live]
        vc[t["slots"][live]] = t["v"][live]
        same(d["q"], q)
        same(d["k"], t["k"])  # read only without k_out
        same(d["kc"], kc)
        same(d["vc"], vc)
        # into k_out, in place, and without pools
        e = {n: x.cuda() for n, x in t.items()}
        fekv.rope_axes_append(e["q"], e["k"], e["v"], e["kc"], e["vc"], e["slots"], e["pos"],
                              e["cache"], pairs, k_out=e["k"])
        same(e["k"], k)
        same(e["kc"], kc)
        f = {n: x.cuda() for n, x in t.items()}
        out = torch.zeros_like(f["k"])
        fekv.rope_axes_append(None, f["k"], f["v"], f["kc"], f["vc"], f["slots"], f["pos"],
                              f["cache"], pairs, k_out=out)
        same(out, k)
        same(f["q"], t["q"])
        fekv.rope_axes(f["q"], f["k"], f["pos"], f["cache"], pairs)
        same(f["q"], q)
        same(f["k"], k)
        assert fekv.device_errors() == 0


@pytest.mark.parametrize("turns", [False, True])
def test_one_position_gives_rope(turns):
    import fekv
    import torch
    t = {n: x.cuda() for n, x in make(33, 8, 4, 128, 128, 3, torch.bfloat16, 5).items()}
    t["pos"][:] = t["pos"][0].clone()
    q, k = t["q"].clone(), t["k"].clone()
    fekv.rope(q, k, t["pos"][0].contiguous(), t["cache"])
    fekv.rope_axes(t["q"], t["k"], t["pos"], t["cache"],
                   fekv.rope_sections((24, 20, 20), turns))
    same(t["q"], q.cpu())
    same(t["k"], k.cpu())


@pytest.mark.parametrize("rows", [20, 4200])
def test_rows_out_of_range_are_skipped_and_flagged(rows):
    import fekv
    import torch
    from fekv import _lib
    pairs = fekv.rope_sections((24, 20, 20), True)
    t = make(rows, 8, 4, 128, 128, 3, torch.float16, 9)
    t["pos"][1, 4] = 700
    t["pos"][2, 7] = -1
    t["slots"][11] = t["kc"].shape[0]
    d = {n: x.cuda() for n, x in t.items()}
    fekv.rope_axes_append(d["q"], d["k"], d["v"], d["kc"], d["vc"], d["slots"], d["pos"],
                          d["cache"], pairs)
    assert fekv.device_errors() == _lib.FE_DEVERR_POS_RANGE | _lib.FE_DEVERR_SLOT_RANGE
    ok = t["pos"].clamp(0, 699).numpy()
    q, k = (torch.from_numpy(rotated(t[n].float().numpy(), ok, t["cache"].numpy(), pairs))
            .to(t[n].dtype) for n in "qk")
    bad = [4, 7]
    q[bad] = t["q"][bad]
    kc, vc = t["kc"].clone(), t["vc"].clone()
    live = [i for i in range(rows) if i not in (4, 7, 11)]
    kc[t["slots"][live]] = k[live]
    vc[t["slots"][live]] = t["v"][live]
    same(d["q"], q)
    same(d["kc"], kc)
    same(d["vc"], vc)


def test_unaligned_buffers():
    """Views that start 8 bytes into an allocation take the plain form."""
    import fekv
    import torch
    t = make(6, 4, 2, 128, 128, 2, torch.bfloat16, 3)
    pairs = fekv.rope_sections((40, 24))
    pos, cache = t["pos"].numpy(), t["cache"].numpy()

    def shifted(x):
        y = torch.zeros(x.numel() + 4, dtype=x.dtype, device="cuda")[4:].view(x.shape)
        y.copy_(x)
        return y

    q, k = shifted(t["q"]), shifted(t["k"])
    fekv.rope_axes(q, k, t["pos"].cuda(), t["cache"].cuda(), pairs)
    for got, n in ((q, "q"), (k, "k")):
        same(got, torch.from_numpy(rotated(t[n].float().numpy(), pos, cache, pairs)).to(t[n].dtype))


def test_other_stream_and_replay():
    import fekv
    import torch
    t = make(40, 8, 4, 128, 128, 3, torch.bfloat16, 21)
    pairs = fekv.rope_sections((24, 20, 20), True)
    d = {n: x.cuda() for n, x in t.items()}
    base = d["q"].clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    args = [d[n] for n in ("k", "v", "kc", "vc", "slots", "pos", "cache")]
    fekv.rope_axes_append(d["q"], *args, pairs, stream=side)
    side.synchronize()
    want, kc = d["q"].clone(), d["kc"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        fekv.rope_axes_append(d["q"], *args, pairs)
    for shift in (0, 1):
        d["q"].copy_(base)
        d["pos"].copy_((t["pos"] + shift) % 700)
        d["kc"].zero_()
        g.replay()
        torch.cuda.synchronize()
        if shift == 0:
            same(d["q"], want.cpu())
            same(d["kc"][t["slots"]], kc[t["slots"]].cpu())
        else:
            pos = ((t["pos"] + 1) % 700).numpy()
            same(d["q"], torch.from_numpy(rotated(t["q"].float().numpy(), pos, t["cache"].numpy(),
                                                  pairs)).to(t["q"].dtype))
