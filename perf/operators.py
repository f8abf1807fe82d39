"""Cases for the operators of the 8-bit paged KV cache: append (rotation, quantisation and
scatter through the slot mapping), attention over it, gathering whole sequences back to 16
bits, and the block copies of forked sequences.

The cache. Keys and values are held as e4m3 codes, [cache_slots, hkv, dim], with one power-of-
two scale for each block of 16 consecutive slots and KV head, stored as its biased exponent
(uint8 [cache_slots / 16, hkv]): value = code * 2 ** (exponent - 127).
 * append: a run of rows with consecutive slots inside one block shares a new scale, the
   smallest power of two that keeps the run's largest finite magnitude within 448, no smaller
   than the block's old scale when tokens before the run are kept (their codes are then
   rounded to the new scale), exponents limited to [-32, 64]. Larger magnitudes saturate.
 * attention: out = softmax(q k^T / sqrt(dim)) v per query head, GQA, keys through the page
   table, causal rows see t <= length - rows + i.
 * gather: the values of whole sequences, rounded to the 16-bit type.
 * copy: the first ntok tokens of a page onto another page, codes and scales, in every layer.

Where `own` is false the operators run in plain torch operations in 32 bits.
"""
import math
import os
import random
import sys

import torch

own = False

BLOCK = 16
MIN_E, MAX_E = 95, 191  # biased exponents that an append writes: 2^-32 .. 2^64
HEADS = [(16, 8, 128), (32, 8, 128), (32, 4, 128), (64, 8, 128), (8, 8, 128), (40, 8, 128),
         (6, 3, 128), (16, 1, 128), (16, 2, 256), (8, 4, 256), (5, 5, 256)]
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------

def listed():
    at = dict(op="attention", page=16, causal=True, shape=1)
    ap = dict(op="append", page=16, shape=2)
    return [
        # one token each for four short sequences: the smallest step, where launches count
        dict(ap, name="append step 4", dtype="f16", hq=16, hkv=8, dim=128, rot=128, seqs=4,
             rows=1, ctx0=1, ctx1=1000),
        # a decode step of 64 sequences: most rows land inside a block that is partly full
        dict(ap, name="append step 64", dtype="bf16", hq=32, hkv=8, dim=128, rot=128, seqs=64,
             rows=1, ctx0=512, ctx1=4096),
        # long prompts: 16 chunks of about 4096 rows that start and end inside blocks; partial
        # rotation stays with the 256-wide heads that use it (draws)
        dict(ap, name="append prompt 64k", dtype="bf16", hq=32, hkv=8, dim=128, rot=128, seqs=16,
             rows=4093, ctx0=1, ctx1=64),
        # four short sequences, one query row each: the latency of a single user's decode step
        dict(at, name="decode 4", dtype="f16", hq=16, hkv=8, dim=128, seqs=4, rows=1, chunks=0,
             ctx0=17, ctx1=1000),
        # 64 sequences of ordinary lengths, the serving batch of an 8-billion-parameter model
        dict(at, name="decode 64", dtype="bf16", hq=32, hkv=8, dim=128, seqs=64, rows=1,
             chunks=0, ctx0=512, ctx1=4096),
        # long contexts: half of one GPU's share of the long-context batch
        dict(at, name="decode 64 long", dtype="bf16", hq=64, hkv=8, dim=128, seqs=64, rows=1,
             chunks=0, ctx0=2048, ctx1=32768),
        # speculative verification: a 16-row block for each of 128 sequences, full mask
        dict(at, name="verify 128x16", dtype="bf16", hq=32, hkv=4, dim=128, seqs=128, rows=16,
             chunks=128, causal=False, ctx0=2064, ctx1=2560),
        # chunked prefill beside decode rows: 4 chunks of 512 rows and 60 single rows
        dict(at, name="mixed 4x512+60", dtype="bf16", hq=32, hkv=8, dim=128, seqs=64, rows=512,
             chunks=4, ctx0=256, ctx1=2560),
        # prefixes of a few sequences read back: an odd number of tokens, f16
        dict(op="gather", name="gather 3", page=16, shape=3, dtype="f16", hkv=8, dim=128, seqs=3,
             ctx0=17, ctx1=511),
        # a whole batch moved out of the cache
        dict(op="gather", name="gather 64", page=16, shape=3, dtype="bf16", hkv=8, dim=128,
             seqs=64, ctx0=512, ctx1=4096),
        # one fork in a small model
        dict(op="copy", name="fork 1", page=16, shape=4, hkv=8, dim=128, layers=4, copies=1,
             pages=64),
        # 64 forks with partial tails in all 48 layers
        dict(op="copy", name="fork 64x48", page=16, shape=4, hkv=4, dim=128, layers=48,
             copies=64, pages=1500),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "gather", "copy"])
    hq, hkv, dim = rng.choice(HEADS)
    dtype = rng.choice(["bf16", "f16"])
    page = rng.choice([16, 16, 32, 48, 64])
    shape = rng.randrange(1 << 20)
    if op == "append":
        seqs = _log(rng, 1, 128)
        rows = rng.choice([1, 1, _log(rng, 2, 16), _log(rng, 2, 4096)])
        rows = max(1, min(rows, 32768 // seqs))
        rot = rng.choice([dim, dim, dim // 2, 0])
        return dict(op=op, shape=shape, dtype=dtype, hq=hq, hkv=hkv, dim=dim, rot=rot, page=page,
                    seqs=seqs, rows=rows, ctx0=1, ctx1=_log(rng, 2, 4096))
    if op == "attention":
        kind = rng.choice(["decode", "decode", "verify", "prefill", "mixed"])
        seqs = _log(rng, 1, 96)
        ctx1 = _log(rng, 2, 16384)
        rows, chunks = 1, 0
        if kind == "verify":
            rows, chunks = rng.randrange(2, 33), seqs
        elif kind in ("prefill", "mixed"):
            rows = _log(rng, 17, 1024)
            chunks = rng.randrange(1, 5)
            seqs = chunks if kind == "prefill" else chunks + seqs
        # within the plain form's memory and the listed cases' work
        ctx1 = max(2, min(ctx1, (1 << 20) // seqs))
        while chunks * rows * (ctx1 + rows) * hq > (1 << 29) and rows > 2:
            rows //= 2
        while chunks * rows * (ctx1 + rows) * hq > (1 << 29):
            ctx1 //= 2
        ctx0 = max(1, ctx1 // rng.choice([1, 2, 8, 1 << 14]))
        return dict(op=op, shape=shape, dtype=dtype, hq=hq, hkv=hkv, dim=dim, page=page, seqs=seqs,
                    rows=rows, chunks=chunks, causal=rng.random() < 0.7, ctx0=ctx0 + rows,
                    ctx1=ctx1 + rows)
    if op == "gather":
        seqs = _log(rng, 1, 96)
        ctx1 = max(1, min(_log(rng, 1, 16384), (1 << 17) // seqs))
        return dict(op=op, shape=shape, dtype=dtype, hkv=hkv, dim=dim, page=page, seqs=seqs,
                    ctx0=1, ctx1=ctx1)
    copies = _log(rng, 1, 64)
    layers = _log(rng, 1, 48)
    return dict(op=op, shape=shape, hkv=hkv, dim=dim, page=page, layers=layers, copies=copies,
                pages=2 * copies + rng.randrange(1, 64))


def _contexts(case):
    """Tokens of each sequence after the step (spread over the logarithm), a matter of the case."""
    rng = random.Random(case["shape"])
    lens = [_log(rng, case["ctx0"], case["ctx1"]) for _ in range(case["seqs"])]
    if case["op"] == "attention":
        lens = [max(n, r) for n, r in zip(lens, _rows(case))]
    return lens


def _rows(case):
    """Query rows of each sequence: `chunks` sequences bring case["rows"], the others one."""
    c = case["chunks"]
    return [case["rows"]] * c + [1] * (case["seqs"] - c)


def _copies(case):
    rng = random.Random(case["shape"])
    order = list(range(case["pages"]))
    rng.shuffle(order)
    n = case["copies"]
    return order[:n], order[n:2 * n], [rng.randint(1, case["page"]) for _ in range(n)]


def work(case):
    kv = case["hkv"] * case["dim"]
    if case["op"] == "append":
        n = case["seqs"] * case["rows"]
        q = case["hq"] * case["dim"]
        codes = 2 * n * kv
        blocks = n / BLOCK + case["seqs"]
        # q in and out, k and v in, codes and scales out, one cos / sin row a token
        return {"bytes": n * (4 * q + 4 * kv + 4 * case["rot"] + 16) + codes +
                2 * blocks * case["hkv"], "flops": n * (3 * (q + kv))}
    if case["op"] == "attention":
        lens, rows = _contexts(case), _rows(case)
        q = case["hq"] * case["dim"]
        pairs = 0
        for n, r in zip(lens, rows):
            pairs += r * n - (r * (r - 1) // 2 if case["causal"] else 0)
        keys = sum(lens)
        return {"bytes": keys * 2 * kv + keys / BLOCK * 2 * case["hkv"] + 4 * sum(rows) * q,
                "flops": 4 * pairs * q}
    if case["op"] == "gather":
        keys = sum(_contexts(case))
        return {"bytes": keys * 3 * kv + keys / BLOCK * case["hkv"], "flops": keys * kv}
    ntok = sum(_copies(case)[2])
    return {"bytes": case["layers"] * 2 * 2 * (ntok * kv + ntok / BLOCK * case["hkv"]),
            "flops": 0}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _pow2(e):
    """2 ** (e - 127) of biased exponents, in 32 bits."""
    return (e.to(torch.int32) << 23).view(torch.float32)


def _needed(amax):
    """Biased exponent of the smallest power of two s with amax <= 448 s, within its limits."""
    bits = amax.contiguous().view(torch.int32)
    return (((bits + 0x1FFFFF) >> 23) - 8).clamp(MIN_E, MAX_E)


def _codes(x):
    return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _cache(gen, slots, hkv, dim, outliers):
    """A pool as appends leave it: normal values, a few channels far larger where `outliers`,
    block scales that differ."""
    codes = torch.empty(slots, hkv, dim, dtype=torch.float8_e4m3fn, device="cuda")
    exps = torch.empty(slots // BLOCK, hkv, dtype=torch.uint8, device="cuda")
    wide = torch.ones(hkv, dim, device="cuda")
    if outliers:
        at = torch.randint(0, dim, (hkv, 4), generator=gen, device="cuda")
        wide.scatter_(1, at, 6.0)
    step = max(BLOCK, (1 << 26) // (hkv * dim) // BLOCK * BLOCK)
    for s in range(0, slots, step):
        n = min(step, slots - s)
        x = torch.randn(n, hkv, dim, generator=gen, device="cuda") * wide
        x = x.view(n // BLOCK, BLOCK, hkv, dim)
        if not outliers:
            x = x * (0.25 + torch.rand(n // BLOCK, 1, hkv, 1, generator=gen, device="cuda"))
        e = _needed(x.abs().amax(dim=(1, 3)))
        codes[s:s + n] = _codes(x / _pow2(e)[:, None, :, None]).view(n, hkv, dim)
        exps[s // BLOCK:(s + n) // BLOCK] = e.to(torch.uint8)
    return codes, exps


def _tables(case, seed, lens, spare=0):
    """A block table of random pages for each sequence, and the number of pages in the pool."""
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


def _flat(tables):
    return [p for t in tables for p in t]


def _sums(v):
    out = [0]
    for x in v:
        out.append(out[-1] + x)
    return out


def _fekv():
    path = os.path.join(os.getcwd(), "flashengine.cpp_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import fekv

    return fekv


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": case}
    page, hkv, dim = case["page"], case["hkv"], case["dim"]
    if case["op"] == "copy":
        shape = (case["layers"], (case["pages"] + 1) * page)
        s["pools"] = []
        for _ in range(2):
            codes = _codes(torch.randn(*shape, hkv, dim, generator=gen, device="cuda"))
            exps = torch.randint(110, 130, (case["layers"], shape[1] // BLOCK, hkv), generator=gen,
                                 device="cuda", dtype=torch.uint8)
            s["pools"].append((codes, exps))
        s["lists"] = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in _copies(case)]
        if own:
            f = _fekv()
            s["layers"] = [[f.Kv8Pool(c[i], e[i]) for i in range(case["layers"])]
                           for c, e in s["pools"]]
        return s

    lens = _contexts(case)
    if case["op"] == "append":  # tokens that are in the cache before the step
        lens = [n + case["rows"] - 1 for n in lens]
    tables, pages = _tables(case, seed, lens, spare=3)
    cache_slots = (pages + 1) * page
    pools = [_cache(gen, cache_slots, hkv, dim, outliers=i == 0) for i in range(2)]
    if own:
        f = _fekv()
        s["kpool"], s["vpool"] = (f.Kv8Pool(c, e) for c, e in pools)
    s["pools"] = pools
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "gather":
        s["out"] = torch.empty(sum(lens), hkv, dim, dtype=dtype, device="cuda")
        s["index"] = torch.cat([_slots(t, page, 0, n) for t, n in zip(tables, lens)]).cuda()
        i32 = dict(dtype=torch.int32, device="cuda")
        s["kv"] = torch.tensor(_sums([len(t) for t in tables]), **i32)
        s["pages"] = torch.tensor(_flat(tables), **i32)
        s["last"] = torch.tensor([(n - 1) % page + 1 for n in lens], **i32)
        s["offset"] = torch.tensor(_sums(lens)[:-1], **i32)
        s["most"] = max(lens)
        return s

    rows = [case["rows"]] * case["seqs"] if case["op"] == "append" else _rows(case)
    n = sum(rows)
    hq = case["hq"]
    s["q"] = (torch.randn(n, hq, dim, generator=gen, device="cuda") * 1.5).to(dtype)
    s["out"] = torch.empty_like(s["q"])
    if case["op"] == "append":
        # new keys have the cache's outlier channels now and then, so some blocks grow
        k = torch.randn(n, hkv, dim, generator=gen, device="cuda")
        far = torch.rand(n, hkv, 1, generator=gen, device="cuda") < 0.1
        s["k"] = torch.where(far, k * 8.0, k).to(dtype)
        s["v"] = torch.randn(n, hkv, dim, generator=gen, device="cuda").to(dtype)
        s["slots"] = torch.cat([_slots(t, page, m - r, m)
                                for t, m, r in zip(tables, lens, rows)]).cuda()
        s["pos"] = torch.cat([torch.arange(m - r, m) for m, r in zip(lens, rows)]).cuda()
        blocks = [m // BLOCK - (m - r) // BLOCK + (1 if m % BLOCK else 0)
                  for m, r in zip(lens, rows)]
        s["runs"] = sum(blocks)
        s["rope"] = None
        if case["rot"]:
            half = case["rot"] // 2
            freq = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            ang = torch.arange(max(lens), device="cuda", dtype=torch.float64)[:, None] * freq
            s["rope"] = torch.cat([ang.cos(), ang.sin()], 1).float()
        return s

    # attention: sequences with the same number of rows go together in the plain form
    s["groups"] = []
    starts = _sums(rows)
    for r in sorted(set(rows)):
        who = [b for b in range(len(rows)) if rows[b] == r]
        most = max(lens[b] for b in who)
        index = torch.zeros(len(who), most, dtype=torch.int64)
        for i, b in enumerate(who):
            index[i, :lens[b]] = _slots(tables[b], page, 0, lens[b])
        s["groups"].append((r, index.cuda(), torch.tensor([lens[b] for b in who]).cuda(),
                            torch.tensor([starts[b] for b in who]).cuda()))
    if own:
        most = max(len(t) for t in tables)
        s["plan"] = f.Kv8Plan(hq, hkv, dim, page, case["seqs"], most, case["dtype"] == "bf16",
                              pages)
        s["plan"].prepare(starts, _sums([len(t) for t in tables]), _flat(tables),
                          [(n - 1) % page + 1 for n in lens])
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    return {"append": _run_append, "attention": _run_attention, "gather": _run_gather,
            "copy": _run_copy}[s["case"]["op"]](s)


def _run_append(s):
    (kc, ke), (vc, ve) = s["pools"]
    if own:
        _fekv().append_kv8(s["q"], s["k"], s["v"], s["kpool"], s["vpool"], s["slots"], s["pos"],
                           s["rope"], q_out=s["out"])
        return s["out"], kc, ke, vc, ve
    q, k = s["q"].float(), s["k"].float()
    if s["rope"] is not None:
        q, k = _rotate(q, s["pos"], s["rope"]), _rotate(k, s["pos"], s["rope"])
    _store(k, kc, ke, s["slots"], s["runs"])
    _store(s["v"].float(), vc, ve, s["slots"], s["runs"])
    s["out"].copy_(q.to(s["q"].dtype))
    return s["out"], kc, ke, vc, ve


def _rotate(x, pos, rope):
    r = rope.shape[1] // 2
    c, sn = rope[pos, None, :r], rope[pos, None, r:]
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * c - b * sn, b * c + a * sn, x[..., 2 * r:]], -1)


def _store(x, codes, exps, slots, runs):
    block = slots // BLOCK
    first = torch.ones_like(slots, dtype=torch.bool)
    first[1:] = block[1:] != block[:-1]
    run_of = first.long().cumsum(0) - 1
    # slot and block where each run begins
    begin = torch.zeros(runs, dtype=torch.int64, device=x.device)
    begin.scatter_reduce_(0, run_of, slots, "amin", include_self=False)
    blk, kept = begin // BLOCK, begin % BLOCK
    size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    amax = torch.zeros(runs, x.shape[1], device=x.device)
    amax.scatter_reduce_(0, run_of[:, None].expand_as(size), size, "amax")
    old = exps[blk].int()
    new = _needed(amax)
    new = torch.where((kept > 0)[:, None], torch.maximum(new, old), new)
    # codes of the tokens before the run, from the old scale to the new one
    grid = codes.view(torch.uint8).view(-1, BLOCK, *codes.shape[1:])
    was = grid[blk].view(torch.float8_e4m3fn)
    now = _codes(was.float() * (_pow2(old) / _pow2(new))[:, None, :, None])
    keep = torch.arange(BLOCK, device=x.device)[None, :] < kept[:, None]
    grid[blk] = torch.where(keep[..., None, None], now.view(torch.uint8), was.view(torch.uint8))
    codes.view(torch.uint8)[slots] = _codes(x / _pow2(new)[run_of][..., None]).view(torch.uint8)
    exps[blk] = new.to(torch.uint8)


def _values(pool, index):
    codes, exps = pool
    x = codes.view(torch.uint8)[index].view(torch.float8_e4m3fn).float()
    return x * _pow2(exps[index // BLOCK])[..., None]


def _run_attention(s):
    case = s["case"]
    if own:
        s["plan"].attention(s["q"], s["kpool"], s["vpool"], s["out"], case["causal"])
        return s["out"]
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    for r, index, lens, starts in s["groups"]:
        at = starts[:, None] + torch.arange(r, device="cuda")
        q = s["q"][at].float()                                   # [b, r, hq, dim]
        q = q.view(-1, r, hkv, hq // hkv, dim).permute(0, 2, 1, 3, 4)
        q = q.reshape(-1, hkv, r * (hq // hkv), dim)
        k = _values(s["pools"][0], index).permute(0, 2, 3, 1)    # [b, hkv, dim, keys]
        p = torch.matmul(q, k).div_(math.sqrt(dim))
        del k
        t = torch.arange(index.shape[1], device="cuda")
        limit = lens[:, None] - r + 1 + torch.arange(r, device="cuda") if case["causal"] \
            else lens[:, None].expand(-1, r)
        hidden = t >= limit[..., None]                           # [b, r, keys]
        hidden = hidden.repeat_interleave(hq // hkv, 1)[:, None]
        p = p.masked_fill_(hidden, -math.inf)
        p = p.sub_(p.amax(-1, keepdim=True)).exp_()
        p = p.div_(p.sum(-1, keepdim=True))
        v = _values(s["pools"][1], index).permute(0, 2, 1, 3)
        o = torch.matmul(p, v)
        del v, p
        o = o.view(-1, hkv, r, hq // hkv, dim).permute(0, 2, 1, 3, 4).reshape(-1, r, hq, dim)
        s["out"][at] = o.to(s["out"].dtype)
    return s["out"]


def _run_gather(s):
    if own:
        _fekv().gather_kv8(s["kpool"], s["out"], s["kv"], s["pages"], s["last"], s["offset"],
                           s["most"], s["case"]["page"])
        return s["out"]
    s["out"].copy_(_values(s["pools"][0], s["index"]).to(s["out"].dtype))
    return s["out"]


def _run_copy(s):
    case = s["case"]
    if own:
        src, dst, ntok = s["lists"]
        _fekv().copy_blocks_kv8(s["layers"][0], s["layers"][1], src, dst, ntok, case["page"])
    else:
        src, dst, ntok = (x.long() for x in s["lists"])
        page = case["page"]
        keep = torch.arange(page, device="cuda")[None, :] < ntok[:, None]
        part = torch.arange(page // BLOCK, device="cuda")[None, :] * BLOCK < ntok[:, None]
        for codes, exps in s["pools"]:
            c = codes.view(torch.uint8).view(case["layers"], -1, page, case["hkv"], case["dim"])
            c[:, dst] = torch.where(keep[None, :, :, None, None], c[:, src], c[:, dst])
            e = exps.view(case["layers"], -1, page // BLOCK, case["hkv"])
            e[:, dst] = torch.where(part[None, :, :, None], e[:, src], e[:, dst])
    (kc, ke), (vc, ve) = s["pools"]
    return kc, ke, vc, ve


# ---------------------------------------------------------------------------------------------
# the operators' definition in 64 bits
# ---------------------------------------------------------------------------------------------

def _grid64(x):
    """x rounded to e4m3: three fraction bits, exponents down to -6, ties to even, at most 448."""
    e = torch.frexp(x.abs().clamp(min=2.0 ** -40))[1] - 1
    unit = torch.ldexp(torch.ones_like(x), e.clamp(min=-6) - 3)
    return (torch.round(x / unit) * unit).clamp(-448.0, 448.0)


def _pool64(pool, index):
    codes, exps = pool
    x = codes.view(torch.uint8)[index].view(torch.float8_e4m3fn).double()
    return torch.ldexp(x, exps[index // BLOCK].int()[..., None] - 127)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "copy":
        return _exact_copy(case, s)
    if case["op"] == "gather":
        return _pool64(s["pools"][0], s["index"])
    if case["op"] == "attention":
        return _exact_attention(case, s)
    q, k, v = s["q"].double(), s["k"].double(), s["v"].double()
    if s["rope"] is not None:
        rope = s["rope"].double()[s["pos"]][:, None, :]
        r = rope.shape[-1] // 2
        c, sn = rope[..., :r], rope[..., r:]
        turned = []
        for x in (q, k):
            y = x.clone()
            y[..., :r] = x[..., :r] * c - x[..., r:2 * r] * sn
            y[..., r:2 * r] = x[..., r:2 * r] * c + x[..., :r] * sn
            turned.append(y)
        q, k = turned
    slots = s["slots"].tolist()
    runs = []  # rows that share a block
    for i, slot in enumerate(slots):
        if runs and slot // BLOCK == slots[runs[-1][0]] // BLOCK:
            runs[-1][1] += 1
        else:
            runs.append([i, 1])
    first = torch.tensor([a for a, _ in runs], device="cuda")
    count = torch.tensor([n for _, n in runs], device="cuda")
    run_of = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), count)
    begin = s["slots"][first]
    out = [q]
    for x, (codes, exps) in ((k, s["pools"][0]), (v, s["pools"][1])):
        size = torch.segment_reduce(x.abs().amax(-1), "max", lengths=count)
        e = torch.ceil(torch.log2((size / 448.0).clamp(min=2.0 ** -60))).clamp(-32, 64)
        was = exps[begin // BLOCK].double() - 127
        e = torch.where((begin % BLOCK > 0)[:, None], torch.maximum(e, was), e)
        full = codes.double()
        for t in range(BLOCK - 1):  # kept tokens of each run's block
            who = (begin % BLOCK > t).nonzero()[:, 0]
            at = begin[who] // BLOCK * BLOCK + t
            full[at] = _grid64(full[at] * torch.exp2(was[who] - e[who])[..., None])
        full[s["slots"]] = _grid64(x * torch.exp2(-e[run_of])[..., None])
        out += [full, None]
    return out


def _exact_copy(case, s):
    out, page = [], case["page"]
    for codes, _ in s["pools"]:
        full = codes.double().view(case["layers"], -1, page, case["hkv"] * case["dim"])
        for src, dst, n in zip(*_copies(case)):
            full[:, dst, :n] = full[:, src, :n]
        out += [full.view(codes.shape), None]
    return out


def _exact_attention(case, s):
    if work(case)["flops"] > 2e12 or work(case)["bytes"] > 4e9:
        return None
    hq, hkv, dim = case["hq"], case["hkv"], case["dim"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r, index, lens, starts in s["groups"]:
        for i, (n, at) in enumerate(zip(lens.tolist(), starts.tolist())):
            k, v = (_pool64(p, index[i, :n]).transpose(0, 1) for p in s["pools"])  # [hkv, n, dim]
            q = s["q"][at:at + r].double().view(r, hkv, -1, dim).permute(1, 2, 0, 3)
            score = torch.einsum("hgrd,hnd->hgrn", q, k) * dim ** -0.5
            if case["causal"]:
                seen = torch.arange(n, device="cuda") <= \
                    n - r + torch.arange(r, device="cuda")[:, None]
                score = torch.where(seen, score, -math.inf)
            o = torch.einsum("hgrn,hnd->rhgd", torch.softmax(score, -1), v)
            out[at:at + r] = o.reshape(r, hq, dim)
    return out
