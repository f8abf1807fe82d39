"""Selection and compaction restated token by token (test infrastructure)."""
import math

import numpy as np


def slots_of(table, page, n):
    t = np.arange(n)
    return np.asarray(table, np.int64)[t // page] * page + t % page


def select(scores, tables, lens, page, budget, sink, recent):
    """scores float [hkv, cache_slots]; kept int32 [batch, hkv, budget]."""
    out = np.full((len(lens), scores.shape[0], budget), -1, np.int32)
    for b, n in enumerate(lens):
        for h in range(scores.shape[0]):
            if n <= budget:
                out[b, h, :n] = np.arange(n)
                continue
            x = scores[h, slots_of(tables[b], page, n)]
            best = sorted(range(sink, n - recent),
                          key=lambda t: (math.inf if np.isnan(x[t]) else -float(x[t]), t))
            # NaN after -inf too
            best.sort(key=lambda t: np.isnan(x[t]))
            kept = list(range(sink)) + sorted(best[:budget - sink - recent]) + \
                list(range(n - recent, n))
            out[b, h, :len(kept)] = kept
    return out


def compact(pools, scores, kept, tables, lens, page, dst_tables=None):
    """Numpy pools [cache_slots, hkv, dim], changed in place."""
    sources = [p.copy() for p in pools], None if scores is None else scores.copy()
    for b, n in enumerate(lens):
        src = slots_of(tables[b], page, n)
        table = (tables if dst_tables is None else dst_tables)[b]
        dst = slots_of(table, page, len(table) * page)
        for h in range(kept.shape[1]):
            for j, t in enumerate(kept[b, h]):
                if t < 0:
                    break
                for p, s in zip(pools, sources[0]):
                    p[dst[j], h] = s[src[t], h]
                if scores is not None:
                    scores[h, dst[j]] = sources[1][h, src[t]]
