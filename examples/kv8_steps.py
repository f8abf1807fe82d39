"""A few serving steps over the 8-bit KV cache, beside the 16-bit one.

Random queries, keys and values stand for a model's projections: prompts in
chunks, decode steps for the batch, a fork of one sequence (its shared pages by
reference, its partial tail copied), decode steps of parent and child, and a
prefix read back to 16 bits. Each step goes through both caches; the script
prints how far the 8-bit outputs are from the 16-bit ones and what a token
costs in either.

    python examples/kv8_steps.py [--layers 4 --batch 8 --prompt 700 --steps 20]
"""
import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..",
                                "flashengine.cpp_b200"))
import fekv  # noqa: E402
from fekv.metadata import build_step_metadata  # noqa: E402


class Cache:
    """Block tables and both caches of `layers` layers."""

    def __init__(self, layers, hq, hkv, dim, page, blocks, batch, max_pages, dtype):
        self.hq, self.hkv, self.dim, self.page, self.dtype = hq, hkv, dim, page, dtype
        slots = (blocks + 1) * page
        shape = (slots, hkv, dim)
        self.wide = [[torch.zeros(shape, dtype=dtype, device="cuda") for _ in range(2)]
                     for _ in range(layers)]
        self.kv8 = [[fekv.Kv8Pool.empty(blocks, page, hkv, dim) for _ in range(2)]
                    for _ in range(layers)]
        bf16 = dtype is torch.bfloat16
        args = (hq, hkv, dim, page, batch, max_pages, bf16, blocks)
        self.plan, self.plan8 = fekv.AttentionPlan(*args), fekv.Kv8Plan(*args)
        self.free = list(range(blocks))
        self.tables, self.lengths = [], []
        f = 1e6 ** (-torch.arange(dim // 2, device="cuda", dtype=torch.float64) / (dim // 2))
        a = torch.arange(max_pages * page, device="cuda", dtype=torch.float64)[:, None] * f
        self.rope = torch.cat([a.cos(), a.sin()], 1).float()

    def fork(self, parent):
        """A child of `parent`: shares its full pages, copies its partial tail."""
        n = self.lengths[parent]
        full = n // self.page
        child = self.tables[parent][:full] + [self.free.pop() for _ in range(n % self.page > 0)]
        lists = fekv.fork_copies([self.tables[parent]], [child], [n], self.page)
        src, dst, ntok = (torch.from_numpy(x).cuda() for x in lists)
        if len(lists[0]):
            blocks = self.wide[0][0].shape[0] // self.page
            fekv.copy_blocks([k for k, _ in self.wide], [v for _, v in self.wide], src, dst, ntok,
                             self.page, self.hkv * self.dim, blocks)
            fekv.copy_blocks_kv8([k for k, _ in self.kv8], [v for _, v in self.kv8], src, dst, ntok,
                                 self.page)
        self.tables.append(child)
        self.lengths.append(n)
        return len(self.tables) - 1

    def step(self, who, rows):
        """One step that adds rows[i] tokens to sequence who[i], through every
        layer and both caches. Returns the relative error of the 8-bit
        outputs."""
        for b, r in zip(who, rows):
            need = -(-(self.lengths[b] + r) // self.page)
            self.tables[b] += [self.free.pop() for _ in range(need - len(self.tables[b]))]
        md = build_step_metadata([self.tables[b] for b in who], [self.lengths[b] for b in who],
                                 rows, self.page)
        for p in (self.plan, self.plan8):
            p.prepare(md.qo, md.kv, md.pages, md.last)
        slots, pos = torch.from_numpy(md.slots).cuda(), torch.from_numpy(md.positions).cuda()
        off = total = 0.0
        for (kc, vc), (k8, v8) in zip(self.wide, self.kv8):
            draw = lambda h: torch.randn(md.rows, h, self.dim, device="cuda").to(self.dtype)  # noqa: E731
            q, k, v = draw(self.hq), draw(self.hkv), draw(self.hkv)
            q8 = torch.empty_like(q)
            fekv.append_kv8(q, k, v, k8, v8, slots, pos, self.rope, q_out=q8)
            fekv.rope_append(q, k, v, kc, vc, slots, pos, self.rope)
            assert torch.equal(q, q8)
            out, out8 = torch.empty_like(q), torch.empty_like(q)
            self.plan.attention(q, kc, vc, out, True)
            self.plan8.attention(q, k8, v8, out8, True)
            off += float((out8.float() - out.float()).square().sum())
            total += float(out.float().square().sum())
        for b, r in zip(who, rows):
            self.lengths[b] += r
        return (off / total) ** 0.5

    def prefix(self, b, tokens):
        """The first tokens' keys of sequence b in layer 0, from the 8-bit cache."""
        t = self.tables[b][:-(-tokens // self.page)]
        i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        out = torch.empty(tokens, self.hkv, self.dim, dtype=self.dtype, device="cuda")
        fekv.gather_kv8(self.kv8[0][0], out, i32(0, len(t)), i32(*t),
                        i32((tokens - 1) % self.page + 1), i32(0), tokens, self.page)
        slots = torch.tensor(t, device="cuda").repeat_interleave(self.page)[:tokens] * self.page + \
            torch.arange(tokens, device="cuda") % self.page
        return out, self.wide[0][0][slots]


def main(argv=None):
    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args(argv)
    torch.manual_seed(0)
    hq, hkv, dim, page = 32, 8, 128, 16
    most = -(-(a.prompt + 2 * a.steps + 1) // page) + 1
    c = Cache(a.layers, hq, hkv, dim, page, (a.batch + 1) * most, a.batch + 1, most,
              torch.bfloat16)
    c.tables, c.lengths = [[] for _ in range(a.batch)], [0] * a.batch
    who = list(range(a.batch))
    errors = {"prompt": [], "decode": [], "forked": []}
    lens = [max(1, a.prompt - 37 * b % a.prompt) for b in who]
    for chunk in range(0, max(lens), 256):  # prompts in chunks of 256
        live = [b for b in who if lens[b] > chunk]
        errors["prompt"].append(c.step(live, [min(256, lens[b] - chunk) for b in live]))
    for _ in range(a.steps):
        errors["decode"].append(c.step(who, [1] * len(who)))
    who.append(c.fork(0))
    for _ in range(a.steps):
        errors["forked"].append(c.step(who, [1] * len(who)))
    got, want = c.prefix(0, c.lengths[0])
    keys = float((got.float() - want.float()).norm() / want.float().norm())
    assert fekv.device_errors() == 0
    for name, e in errors.items():
        print(f"{name:7s} {len(e):3d} steps, outputs off by {np.mean(e):.3f} (largest {max(e):.3f})")
    print(f"keys of a sequence of {c.lengths[0]} off by {keys:.3f}")
    print(f"bytes a token and layer: 16-bit {2 * hkv * dim * 2}, 8-bit "
          f"{2 * hkv * dim + 2 * hkv / fekv.KV8_BLOCK:.0f}")
    return errors, keys


if __name__ == "__main__":
    main()
