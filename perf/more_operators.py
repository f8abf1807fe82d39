"""Cases for the operators that long shared prompts need around the paged KV cache: rotary
positions with several axes on the way into it, attention for sequences that share a prefix,
attention that keeps a score of every cached key, and the eviction of keys by that score.

 * axes: pair j of a head (x[j], x[j + rot / 2]) is turned by the angle of position
   pos[axis(j), row]; queries in place, keys into the pool with their values.
 * shared: out = softmax(q k^T / sqrt(dim)) v per query head, GQA; the sequences of a group
   have the same first pages, `prefix` tokens, then pages of their own.
 * scored: the same attention without groups; scores[h, slot] of each visible key grows by its
   softmax weights, summed over the sequence's rows and the heads of KV head h; the newest
   `fresh` keys have no score yet: theirs is set.
 * select: per sequence and KV head the first `sink` tokens, the last `recent` and the best of
   the others by score, `budget` in all, in order; ties go to the lowest index, -1 fills up.
 * compact: the selected tokens' keys, values and scores move to the front of their sequence.

Where `own` is false the operators run in plain torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

own = False

HEADS = [(16, 8, 128), (32, 8, 128), (32, 4, 128), (64, 8, 128), (8, 8, 128), (40, 8, 128),
         (6, 3, 128), (16, 1, 128), (16, 2, 256), (8, 4, 256), (5, 5, 256)]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------

def listed():
    ax = dict(op="axes", page=16, shape=1, dim=128, rot=128)
    sh = dict(op="shared", page=16, shape=2, dim=128, groups=1, causal=True)
    sc = dict(op="scored", page=16, shape=3, dim=128, rows=1, fresh=1)
    ev = dict(page=16, shape=4, hkv=8)
    return [
        # a decode step of 64 sequences behind image prompts, one row each: latency counts
        dict(ax, name="axes step 64", dtype="bf16", hq=32, hkv=8, s0=16, s1=24, s2=24,
             interleaved=False, seqs=64, rows=1, ctx1=4096),
        # prompts of images and video: 16 chunks of about 4096 rows, axes taking turns pair by pair
        dict(ax, name="axes prompt 64k", dtype="bf16", hq=32, hkv=8, s0=24, s1=20, s2=20,
             interleaved=True, seqs=16, rows=4093, ctx1=64),
        # a few short requests over one instruction: the smallest step
        dict(sh, name="shared 4", dtype="f16", hq=16, hkv=8, seqs=4, rows=1, prefix=512, own0=1,
             own1=64),
        # a serving batch of 128 over a 2048-token prompt, up to 256 tokens of its own each
        dict(sh, name="shared 128", dtype="bf16", hq=32, hkv=4, seqs=128, rows=1, prefix=2048,
             own0=1, own1=257),
        # one long document, 64 questions about it
        dict(sh, name="shared 64 long", dtype="bf16", hq=64, hkv=8, seqs=64, rows=1, prefix=16384,
             own0=16, own1=2048),
        # speculative verification over the shared prompt: 16-row blocks, full mask
        dict(sh, name="shared verify 128x16", dtype="bf16", hq=32, hkv=4, seqs=128, rows=16,
             prefix=2048, own0=17, own1=272, causal=False),
        # four short sequences: the latency of a single user's step
        dict(sc, name="scored 4", dtype="f16", hq=16, hkv=8, seqs=4, ctx0=17, ctx1=1000),
        # the serving batch of an 8-billion-parameter model
        dict(sc, name="scored 64", dtype="bf16", hq=32, hkv=8, seqs=64, ctx0=512, ctx1=4096),
        # four sequences of up to 1000 tokens, half of them kept
        dict(ev, name="select 4", op="select", seqs=4, ctx0=511, ctx1=1000, budget=384, sink=4,
             recent=64),
        # long contexts cut to 4096 tokens
        dict(ev, name="select 64 long", op="select", seqs=64, ctx0=4096, ctx1=32768, budget=4096,
             sink=4, recent=512),
        # one sequence that grew by a few pages over its budget
        dict(ev, name="compact 1", op="compact", dtype="f16", dim=128, seqs=1, ctx0=575, ctx1=575,
             budget=512, sink=4, recent=64),
        # 64 sequences cut to half of their contexts and less
        dict(ev, name="compact 64", op="compact", dtype="bf16", dim=128, seqs=64, ctx0=2048,
             ctx1=8192, budget=1024, sink=4, recent=128),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["axes", "shared", "shared", "scored", "scored", "select", "compact"])
    hq, hkv, dim = rng.choice(HEADS)
    c = dict(op=op, shape=rng.randrange(1 << 20), page=rng.choice([16, 16, 32, 48, 64]), hkv=hkv)
    seqs = _log(rng, 1, 128)
    if op == "axes":
        rows = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 4096)])
        rot = rng.choice([dim, dim, dim // 2])
        turns = rng.random() < 0.5
        # two axes share what the first leaves; taking turns, none is longer than the first
        s1 = rng.randint(0, rot // 6)
        s2 = s1 if turns else rng.randint(0, rot // 6)
        return dict(c, dtype=rng.choice(["bf16", "f16"]), hq=hq, dim=dim, rot=rot,
                    s0=rot // 2 - s1 - s2, s1=s1, s2=s2, interleaved=turns, seqs=seqs,
                    rows=max(1, min(rows, 32768 // seqs)), ctx1=_log(rng, 2, 4096))
    c["dtype"] = rng.choice(["bf16", "f16"])
    if op == "shared":
        groups = rng.choice([1, 1, 2, 5])
        seqs = max(1, seqs // groups)
        rows = rng.choice([1, 1, 1, rng.randint(2, 8), rng.randint(9, 33)])
        prefix = _log(rng, 16, 16384)
        own1 = _log(rng, 2, 1024)
        # within the largest listed case's work
        while groups * seqs * rows * hq * (prefix + own1) > (1 << 26):
            prefix, own1, seqs = max(16, prefix // 2), max(2, own1 // 2), max(1, seqs - seqs // 4)
            rows = max(1, rows - 1)
        prefix = -(-prefix // c["page"]) * c["page"]
        return dict(c, hq=hq, dim=dim, groups=groups, seqs=seqs, rows=rows, prefix=prefix,
                    own0=rows, own1=rows + own1, causal=rng.random() < 0.7)
    if op == "scored":
        rows = rng.choice([1, 1, 1, rng.randint(2, 16), rng.randint(17, 40)])
        seqs = max(1, seqs // rows)
        ctx1 = max(2, min(_log(rng, 2, 16384), (1 << 17) // (seqs * rows)))
        fresh = rng.choice([rows, rows, 1 << 20])
        return dict(c, hq=hq, dim=dim, seqs=seqs, rows=rows, fresh=fresh,
                    ctx0=rows + rng.randint(0, 1) * ctx1 // 2, ctx1=rows + ctx1)
    ctx1 = max(2, min(_log(rng, 2, 32768), (1 << 18) // seqs))
    budget = max(1, _log(rng, max(1, ctx1 // 16), ctx1))
    recent = rng.randint(0, budget // 2)
    c.update(seqs=seqs, ctx0=max(1, ctx1 // rng.choice([1, 2, 8])), ctx1=ctx1, budget=budget,
             sink=min(budget - recent, rng.choice([0, 4])), recent=recent)
    if op == "select":
        c.pop("dtype")
        return c
    return dict(c, dim=dim)


def _lens(case):
    """Tokens of each sequence (of its own, where it shares), a matter of the case."""
    rng = random.Random(case["shape"])
    a, b = ("own0", "own1") if case["op"] == "shared" else ("ctx0", "ctx1")
    if case["op"] == "axes":
        return [rng.randint(0, case["ctx1"]) + case["rows"] for _ in range(case["seqs"])]
    return [_log(rng, case[a], case[b]) for _ in range(case["seqs"] * case.get("groups", 1))]


def work(case):
    op, hkv = case["op"], case["hkv"]
    lens = _lens(case)
    if op == "select":
        return {"bytes": 4 * hkv * (sum(lens) + len(lens) * case["budget"]),
                "flops": hkv * sum(lens)}
    kv = hkv * case["dim"]
    if op == "compact":
        moved = sum(max(0, case["budget"] - case["sink"]) for n in lens if n > case["budget"])
        return {"bytes": moved * (8 * kv + 8 * hkv) + 4 * hkv * case["budget"] * len(lens),
                "flops": 0}
    n = case["seqs"] * case["rows"] * case.get("groups", 1)
    q = case["hq"] * case["dim"]
    if op == "axes":
        # q in and out, k and v in and into the pools, a cos / sin row, three positions, a slot
        return {"bytes": n * (4 * q + 8 * kv + 4 * case["rot"] + 32), "flops": n * 3 * (q + kv)}
    r = case["rows"]
    hidden = r * (r - 1) // 2 if case.get("causal", True) else 0
    if op == "shared":
        pairs = sum(r * (case["prefix"] + m) - hidden for m in lens)
        keys = case["groups"] * case["prefix"] + sum(lens)
        return {"bytes": 4 * keys * kv + 4 * n * q, "flops": 4 * pairs * q}
    pairs = sum(r * m - hidden for m in lens)
    read = sum(max(0, m - case["fresh"]) for m in lens)
    return {"bytes": 4 * sum(lens) * kv + 4 * hkv * (sum(lens) + read) + 4 * n * q,
            "flops": 4 * pairs * q}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _tables(case, seed, lens, spare=3):
    """A block table of random pages for each length, and the number of pages in the pool."""
    need = [-(-n // case["page"]) for n in lens]
    total = sum(need) + spare
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for n in need:
        out.append(order[at:at + n])
        at += n
    return out, total


def _slots(table, page, a, b):
    t = torch.arange(a, b)
    return torch.tensor(table, dtype=torch.int64)[t // page] * page + t % page


def _padded(tables, page, lens):
    """Slots [len(lens), max(lens)] of whole sequences, 0 past their ends."""
    index = torch.zeros(len(lens), max(lens), dtype=torch.int64)
    for i, (t, n) in enumerate(zip(tables, lens)):
        index[i, :n] = _slots(t, page, 0, n)
    return index.cuda()


def _sums(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _fekv():
    path = os.path.join(os.getcwd(), "flashengine.cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fekv

    return fekv


def _pools(gen, slots, hkv, dim, dtype):
    return [torch.randn(slots, hkv, dim, generator=gen, device="cuda", dtype=torch.float32)
            .to(dtype) for _ in range(2)]


def _score_pool(gen, hkv, slots):
    """Accumulated weights: most keys have little, a few much."""
    u = torch.rand(hkv, slots, generator=gen, device="cuda")
    return torch.exp(3.0 * torch.randn(hkv, slots, generator=gen, device="cuda") - 4.0) + 1e-4 * u


def _axis_of(case):
    """The axis of each pair: sections one after the other, or taking turns while they last."""
    sizes = (case["s0"], case["s1"], case["s2"])
    if not case["interleaved"]:
        return [a for a, n in enumerate(sizes) for _ in range(n)]
    return [j % 3 if j // 3 < sizes[j % 3] else 0 for j in range(sum(sizes))]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"axes": _prepare_axes, "shared": _prepare_shared, "scored": _prepare_scored,
            "select": _prepare_evict, "compact": _prepare_evict}[case["op"]](case, seed, gen)


def _prepare_axes(case, seed, gen):
    lens, rows, dtype = _lens(case), case["rows"], DTYPES[case["dtype"]]
    hq, hkv, dim, rot = case["hq"], case["hkv"], case["dim"], case["rot"]
    tables, pages = _tables(case, seed, lens)
    n = case["seqs"] * rows
    s = {"case": case}
    s["q"] = torch.randn(n, hq, dim, generator=gen, device="cuda").to(dtype)
    s["k"] = torch.randn(n, hkv, dim, generator=gen, device="cuda").to(dtype)
    s["v"] = torch.randn(n, hkv, dim, generator=gen, device="cuda").to(dtype)
    s["kc"], s["vc"] = _pools(gen, (pages + 1) * case["page"], hkv, dim, dtype)
    s["slots"] = torch.cat([_slots(t, case["page"], m - rows, m)
                            for t, m in zip(tables, lens)]).cuda()
    # time runs on; a row's height and width are those of a patch of an image
    t = torch.cat([torch.arange(m - rows, m) for m in lens]).cuda()
    side = torch.randint(1, 64, (2, n), generator=gen, device="cuda")
    s["pos"] = torch.stack([t, t // 4 + side[0], t // 4 + side[1]]).contiguous()
    half = rot // 2
    freq = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    most = int(s["pos"].max()) + 1
    ang = torch.arange(most, device="cuda", dtype=torch.float64)[:, None] * freq
    s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
    s["axis"] = torch.tensor(_axis_of(case), device="cuda")
    if own:
        s["pairs"] = _fekv().rope_sections((case["s0"], case["s1"], case["s2"]),
                                           case["interleaved"])
    return s


def _prepare_shared(case, seed, gen):
    lens, rows, page, n = _lens(case), case["rows"], case["page"], case["seqs"]
    hq, hkv, dim, groups = case["hq"], case["hkv"], case["dim"], case["groups"]
    tables, pages = _tables(case, seed, [case["prefix"]] * groups + lens)
    heads, tables = tables[:groups], tables[groups:]
    s = {"case": case}
    dtype = DTYPES[case["dtype"]]
    s["kc"], s["vc"] = _pools(gen, (pages + 1) * page, hkv, dim, dtype)
    s["q"] = (torch.randn(len(lens) * rows, hq, dim, generator=gen, device="cuda") * 1.5).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    s["prefix"] = _padded(heads, page, [case["prefix"]] * groups)
    s["index"] = _padded(tables, page, lens)
    s["lens"] = torch.tensor(lens, device="cuda")
    if own:
        full = [heads[b // n] + t for b, t in enumerate(tables)]
        s["plan"] = _fekv().SharedPlan(hq, hkv, dim, page, len(lens), max(map(len, full)),
                                       case["dtype"] == "bf16", pages)
        s["plan"].prepare([i * rows for i in range(len(lens) + 1)], _sums(map(len, full)),
                          [p for t in full for p in t], [(m - 1) % page + 1 for m in lens])
    return s


def _prepare_scored(case, seed, gen):
    lens, rows, page = _lens(case), case["rows"], case["page"]
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    tables, pages = _tables(case, seed, lens)
    s = {"case": case}
    dtype = DTYPES[case["dtype"]]
    s["kc"], s["vc"] = _pools(gen, (pages + 1) * page, hkv, dim, dtype)
    s["q"] = (torch.randn(len(lens) * rows, hq, dim, generator=gen, device="cuda") * 1.5).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    s["scores"] = _score_pool(gen, hkv, (pages + 1) * page)
    s["index"] = _padded(tables, page, lens)
    s["lens"] = torch.tensor(lens, device="cuda")
    s["valid"] = torch.cat([torch.arange(n) + i * max(lens) for i, n in enumerate(lens)]).cuda()
    if own:
        s["plan"] = _fekv().ScoredPlan(hq, hkv, dim, page, len(lens), max(map(len, tables)),
                                       case["dtype"] == "bf16", pages,
                                       max_keys=rows * sum(n + 15 for n in lens))
        s["plan"].prepare([i * rows for i in range(len(lens) + 1)], _sums(map(len, tables)),
                          [p for t in tables for p in t], [(n - 1) % page + 1 for n in lens],
                          fresh=[min(case["fresh"], n) for n in lens])
    return s


def _prepare_evict(case, seed, gen):
    lens, page, hkv = _lens(case), case["page"], case["hkv"]
    tables, pages = _tables(case, seed, lens)
    s = {"case": case, "scores": _score_pool(gen, hkv, (pages + 1) * page)}
    s["index"] = _padded(tables, page, lens)
    s["lens"] = torch.tensor(lens, device="cuda")
    s["kept"] = torch.empty(len(lens), hkv, case["budget"], dtype=torch.int32, device="cuda")
    s["kv"] = _i32(_sums(map(len, tables)))
    s["pages"] = _i32([p for t in tables for p in t])
    s["last"] = _i32([(n - 1) % page + 1 for n in lens])
    s["most"] = max(lens)
    if case["op"] == "compact":
        s["kc"], s["vc"] = _pools(gen, (pages + 1) * page, hkv, case["dim"], DTYPES[case["dtype"]])
        s["kept"].copy_(_select(s))
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    return {"axes": _run_axes, "shared": _run_shared, "scored": _run_scored,
            "select": _run_select, "compact": _run_compact}[s["case"]["op"]](s)


def _turn(x, pos, rope, axis):
    r = rope.shape[1] // 2
    at = pos[axis].t()                                              # [rows, pairs]
    j = torch.arange(r, device=x.device)
    c, sn = rope[at, j][:, None], rope[at, j + r][:, None]
    x = x.float()
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * c - b * sn, b * c + a * sn, x[..., 2 * r:]], -1)


def _run_axes(s):
    if own:
        _fekv().rope_axes_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["slots"], s["pos"],
                                 s["rope"], s["pairs"])
    else:
        dtype = s["q"].dtype
        k = _turn(s["k"], s["pos"], s["rope"], s["axis"])
        s["q"].copy_(_turn(s["q"], s["pos"], s["rope"], s["axis"]).to(dtype))
        s["kc"][s["slots"]] = k.to(dtype)
        s["vc"][s["slots"]] = s["v"]
    return s["q"], s["kc"], s["vc"]


def _grouped(q, batch, rows, hkv):
    """[batch * rows, hq, dim] -> [batch, hkv, rows * (hq / hkv), dim] in 32 bits."""
    q = q.float().view(batch, rows, hkv, -1, q.shape[-1]).permute(0, 2, 1, 3, 4)
    return q.reshape(batch, hkv, -1, q.shape[-1])


def _ungrouped(o, rows, hq):
    batch, hkv, _, dim = o.shape
    return o.view(batch, hkv, rows, -1, dim).permute(0, 2, 1, 3, 4).reshape(-1, hq, dim)


def _hidden(lens, most, rows, causal, per):
    """Keys that a packed row does not see, [batch, 1, rows * per, most]."""
    t = torch.arange(most, device="cuda")
    ahead = torch.arange(rows, device="cuda") - rows + 1 if causal \
        else torch.zeros(rows, dtype=torch.int64, device="cuda")
    limit = (lens[:, None] + ahead).repeat_interleave(per, 1)
    return (t >= limit[..., None])[:, None]


def _run_shared(s):
    case = s["case"]
    if own:
        s["plan"].attention(s["q"], s["kc"], s["vc"], s["out"], case["causal"])
        return s["out"]
    hq, hkv, dim, rows, groups = (case[x] for x in ("hq", "hkv", "dim", "rows", "groups"))
    per = hq // hkv
    q = _grouped(s["q"], len(s["lens"]), rows, hkv) / math.sqrt(dim)     # [b, hkv, r, dim]
    # the rows of a group, one after the other, against the group's prefix
    wide = q.view(groups, -1, hkv, rows * per, dim).transpose(1, 2)
    wide = wide.reshape(groups, hkv, -1, dim)
    a = torch.matmul(wide, s["kc"][s["prefix"]].float().permute(0, 2, 3, 1))
    b = torch.matmul(q, s["kc"][s["index"]].float().permute(0, 2, 3, 1))
    b = b.masked_fill_(_hidden(s["lens"], b.shape[-1], rows, case["causal"], per), -math.inf)

    def narrow(x):  # [groups, hkv, seqs * r, n] -> [b, hkv, r, n]
        x = x.view(groups, hkv, -1, rows * per, x.shape[-1]).transpose(1, 2)
        return x.reshape(-1, hkv, rows * per, x.shape[-1])

    top = torch.maximum(narrow(a.amax(-1, keepdim=True)), b.amax(-1, keepdim=True))
    b = b.sub_(top).exp_()
    top = top.view(groups, -1, hkv, rows * per, 1).transpose(1, 2).reshape(groups, hkv, -1, 1)
    a = a.sub_(top).exp_()
    total = narrow(a.sum(-1, keepdim=True)) + b.sum(-1, keepdim=True)
    o = narrow(torch.matmul(a, s["vc"][s["prefix"]].float().transpose(1, 2)))
    o = o + torch.matmul(b, s["vc"][s["index"]].float().transpose(1, 2))
    s["out"].copy_(_ungrouped(o / total, rows, hq).to(s["out"].dtype))
    return s["out"]


def _run_scored(s):
    case = s["case"]
    if own:
        s["plan"].attention(s["q"], s["kc"], s["vc"], s["scores"], s["out"])
        return s["out"], s["scores"]
    hq, hkv, dim, rows = (case[x] for x in ("hq", "hkv", "dim", "rows"))
    q = _grouped(s["q"], len(s["lens"]), rows, hkv)
    p = torch.matmul(q, s["kc"][s["index"]].float().permute(0, 2, 3, 1)).div_(math.sqrt(dim))
    p = p.masked_fill_(_hidden(s["lens"], p.shape[-1], rows, True, hq // hkv), -math.inf)
    p = p.sub_(p.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    o = torch.matmul(p, s["vc"][s["index"]].float().transpose(1, 2))
    s["out"].copy_(_ungrouped(o, rows, hq).to(s["out"].dtype))
    weight = p.sum(2).transpose(0, 1).reshape(hkv, -1)[:, s["valid"]]
    at = s["index"].reshape(-1)[s["valid"]]
    t = torch.arange(p.shape[-1], device="cuda")
    old = (t < (s["lens"] - case["fresh"])[:, None]).reshape(-1)[s["valid"]]
    s["scores"][:, at] = torch.where(old, s["scores"][:, at], 0.0) + weight
    return s["out"], s["scores"]


def _select(s):
    """Kept tokens [batch, hkv, budget], ascending, -1 past the last."""
    case, lens = s["case"], s["lens"][:, None, None]
    t = torch.arange(s["most"], device="cuda")
    x = s["scores"][:, s["index"]].transpose(0, 1)                       # [batch, hkv, keys]
    x = torch.where((t < case["sink"]) | (t >= lens - case["recent"]), math.inf, x)
    x = torch.where(t < lens, x, -math.inf)
    order = torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :case["budget"]]
    order = torch.where(order < lens, order, s["most"]).sort(-1)[0]
    kept = torch.full_like(s["kept"], -1)
    kept[..., :order.shape[-1]] = torch.where(order < s["most"], order, -1)
    return kept


def _run_select(s):
    if own:
        _fekv().select_tokens(s["scores"], s["kv"], s["pages"], s["last"], s["kept"],
                              s["case"]["page"], s["most"], sink=s["case"]["sink"],
                              recent=s["case"]["recent"])
    else:
        s["kept"].copy_(_select(s))
    return s["kept"]


def _run_compact(s):
    if own:
        _fekv().compact_tokens(s["kc"], s["vc"], s["scores"], s["kept"], s["kv"], s["pages"],
                               s["last"], s["case"]["page"])
    else:
        hkv = s["case"]["hkv"]
        b, h, j = (s["kept"] >= 0).nonzero(as_tuple=True)
        src = s["index"][b, s["kept"][b, h, j].long()]
        dst = s["index"][b, j]
        for pool in (s["kc"], s["vc"]):
            rows = pool.view(-1, pool.shape[-1])
            rows[dst * hkv + h] = rows[src * hkv + h]
        s["scores"][h, dst] = s["scores"][h, src]
    return s["kc"], s["vc"], s["scores"]


# ---------------------------------------------------------------------------------------------
# the operators' definition in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "select":
        return None  # whole numbers
    return {"axes": _exact_axes, "shared": _exact_shared, "scored": _exact_scored,
            "compact": _exact_compact}[case["op"]](case, s)


def _exact_axes(case, s):
    r, axis = case["rot"] // 2, _axis_of(case)
    out = []
    for x in (s["q"], s["k"]):
        x = x.double()
        y = x.clone()
        for j in range(r):  # one pair at a time, as a complex number
            row = s["rope"][s["pos"][axis[j]]]
            turn = torch.complex(row[:, j].double(), row[:, j + r].double())[:, None]
            z = torch.complex(x[..., j], x[..., j + r]) * turn
            y[..., j], y[..., j + r] = z.real, z.imag
        out.append(y)
    pools = [s["kc"].double(), s["vc"].double()]
    pools[0][s["slots"]] = out[1]
    pools[1][s["slots"]] = s["v"].double()
    return out[0], pools[0], pools[1]


def _attend64(q, k, v, causal):
    """One sequence: q [r, hq, dim], k and v [n, hkv, dim]; output and weights [hkv, g, r, n]."""
    r, hq, dim = q.shape
    n, hkv = k.shape[:2]
    score = torch.einsum("rhgd,nhd->hgrn", q.double().view(r, hkv, -1, dim), k.double())
    score = score * dim ** -0.5
    if causal:
        i, t = torch.arange(r, device="cuda")[:, None], torch.arange(n, device="cuda")
        score = torch.where(t <= n - r + i, score, -math.inf)
    w = torch.softmax(score, -1)
    return torch.einsum("hgrn,nhd->rhgd", w, v.double()).reshape(r, hq, dim), w


def _exact_shared(case, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    r = case["rows"]
    for b, n in enumerate(s["lens"].tolist()):
        at = torch.cat([s["prefix"][b // case["seqs"]], s["index"][b, :n]])
        out[b * r:b * r + r] = _attend64(s["q"][b * r:b * r + r], s["kc"][at], s["vc"][at],
                                         case["causal"])[0]
    return out


def _exact_scored(case, s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    scores, r = s["scores"].double(), case["rows"]
    for b, n in enumerate(s["lens"].tolist()):
        at = s["index"][b, :n]
        out[b * r:b * r + r], w = _attend64(s["q"][b * r:b * r + r], s["kc"][at], s["vc"][at], True)
        scores[:, at[max(0, n - case["fresh"]):]] = 0.0
        scores[:, at] += w.sum((1, 2))
    return out, scores


def _exact_compact(case, s):
    pools = [s["kc"].double(), s["vc"].double(), s["scores"].double()]
    for b, n in enumerate(s["lens"].tolist()):
        for h in range(case["hkv"]):
            kept = s["kept"][b, h, :min(n, case["budget"])].long()
            src, dst = s["index"][b, kept], s["index"][b, :len(kept)]
            for p in pools[:2]:
                p[dst, h] = p[src, h]
            pools[2][h, dst] = pools[2][h, src]
    return pools
