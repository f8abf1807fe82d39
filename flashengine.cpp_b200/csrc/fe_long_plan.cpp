// Host planners of the shared-prefix and the scored plans (see fe_long_plan.h).
#include "fe_long_plan.h"

#include <algorithm>
#include <cstring>

#include "fe_kv.h"
#include "fe_plan_lists.h"

namespace fe {
namespace {

// Costs, as measured on B200, in microseconds of one SM. A 128-key tile of the row
// kernels: the weights of the row lists (fifths of a microsecond). The same keys
// in the key or decode kernel: their bytes at an SM's share of the memory rate. A
// record's bytes, written and read through the L2; one more launch on all SMs.
double tile_us(const PlanConfig& cfg, int64_t P) {
  if (P <= kRowBlock) return 1.75 * cfg.dim / kHeadDim;
  const int rows = row_item_rows(cfg.dim);
  const double per_key = 128.0 / (kTileTokens * cfg.row_tile) / 5.0;
  const int64_t full = P / rows, rest = P % rows;
  const double last = rest == 0 ? 0 : rest > 128 ? cfg.row_weight[1] : cfg.row_weight[0];
  return (full * (rows > 128 ? cfg.row_weight[1] : cfg.row_weight[0]) + last) * per_key;
}
constexpr double kRecordGbs = 27;  // per SM
constexpr double kLaunchUs = 2;
// A 16-key tile and an item of a warp of the key kernel that memory does not hold up
constexpr double kKeyTileUs = 0.65, kKeyItemUs = 2.5;
constexpr double kHbmGbs = 6000;

// Where the records of a sequence's (or row block's) query rows lie; unit
// numbers as in RowInfo.
struct MergeSeq {
  int q_row0 = 0, qrows = 0;
  int own_unit = -1, own_blocks = 0;
  int pre_unit = -1, pre_blocks = 0;
  int pre_row0 = 0;  // its first packed row among the prefix's
  int pre_rows = 0;  // packed rows of the prefix (a KV head)
};

struct Tables {
  std::vector<SeqInfo> seqs;
  std::vector<MergeSeq> merge;  // one per sequence of the step (or row block)
  std::vector<RowInfo> rows;
  std::vector<ScoreChunk> chunks;
  std::vector<int64_t> sink;
};

// The decode list, cut by cost: a piece of a unit costs its tiles and about kKeyItem
// more (its queries, first loads and record). Cut by tiles alone the short
// sequences of a step fall to a few CTAs (three of 24 keys at head_dim 256: six
// items to one CTA, 25 us).
constexpr int kKeyItem = 4;
int decode_view(const PlanConfig& cfg, const std::vector<Unit>& units, int ctas, bool fixed_grid,
                View& v, std::string& err) {
  PlanConfig c = cfg;
  c.row_tile = c.row_weight[0] = 1;
  c.row_item_tiles = kKeyItem;
  c.row_pair_blocks = 0;
  c.row_min_piece = cfg.dec_min_tiles;
  return build_cost_view(c, units, ctas, fixed_grid, v, err);
}

// views: 0 and 1 the row list without and with the mask, 2 the decode list.
// Offsets the decode list's records past the row lists' and packs everything.
int pack(const PlanConfig& cfg, bool keys, View (&views)[3], const Tables& t,
         const int32_t* pages, int total_pages, int batch, int rows, LongResult& out,
         std::string& err) {
  const int64_t row_floats = std::max(views[0].partial_floats, views[1].partial_floats);
  out.partial_floats = row_floats + views[2].partial_floats;
  if (out.partial_floats > cfg.partial_capacity || out.partial_floats > int64_t(INT32_MAX)) {
    err = "attention work exceeds the plan's split-workspace capacity";
    return FE_ERR_CAPACITY;
  }
  for (auto& it : views[2].items)
    if (it.group >= 0) it.part += static_cast<int32_t>(row_floats);
  for (auto& g : views[2].groups) g.part0 += static_cast<int32_t>(row_floats);

  MetaHeader h{};
  std::vector<uint8_t> meta(align16(sizeof(MetaHeader)));
  size_t over = 0;
  auto put = [&](const auto& v) -> int32_t {
    const size_t at = meta.size(), bytes = sizeof(v[0]) * v.size();
    if (at + bytes > size_t(INT32_MAX)) over = at + bytes;
    if (over) return 0;
    meta.resize(align16(at + bytes));
    if (bytes) std::memcpy(meta.data() + at, v.data(), bytes);
    return static_cast<int32_t>(at);
  };
  for (int c = 0; c < 3; ++c) {
    const View& v = views[c];
    h.n_items[c] = static_cast<int32_t>(v.items.size());
    h.n_groups[c] = static_cast<int32_t>(v.groups.size());
    h.grid[c] = out.grid[c] = v.grid;
    h.cta_off_off[c] = put(v.cta_off);
    h.items_off[c] = put(v.items);
    h.groups_off[c] = put(v.groups);
  }
  for (int c = 0; c < 2; ++c) {
    std::vector<UnitRec> unit;
    for (const View* v : {&views[c], &views[2]})
      for (int32_t g : v->unit_group) {
        UnitRec u{0, 0, 0, 0};
        if (g >= 0) {
          const SplitGroup& sg = v->groups[g];
          u = UnitRec{sg.part0, sg.nsplit, sg.rec_floats, sg.rows};
          out.merge[c] = true;
        }
        unit.push_back(u);
      }
    h.unit_off[c] = put(unit);
  }
  if (keys) {
    std::vector<KeyItem> items;
    for (const WorkItem& w : views[2].items) {
      const SeqInfo& s = t.seqs[w.seq];
      items.push_back(KeyItem{s.q_row0, s.qrows, s.length, s.page_off, w.kvh, w.key_mode, w.kt0,
                              w.kt1, w.part, w.group, w.seq, 0});
    }
    h.key_items_off = put(items);
  }
  h.seqs_off = put(t.seqs);
  h.row_info_off = put(t.rows);
  h.chunk_off = put(t.chunks);
  h.sink_off = put(t.sink);
  h.n_chunks = out.n_chunks = static_cast<int32_t>(t.chunks.size());
  h.pages_off = put(std::vector<int32_t>(pages, pages + total_pages));
  if (over) {
    err = "metadata too large";
    return FE_ERR_CAPACITY;
  }
  h.batch = batch;
  h.rows = out.rows = rows;
  h.total_bytes = static_cast<int32_t>(meta.size());
  h.dec_heads = cfg.dec_heads;
  std::memcpy(meta.data(), &h, sizeof(h));
  out.meta.swap(meta);
  return FE_OK;
}

void fill_rows(Tables& t, int rows, int G) {
  t.rows.assign(rows, RowInfo{-1, 0, 0, 0, -1, 0, 0, 0});
  for (const MergeSeq& m : t.merge)
    for (int i = 0; i < m.qrows; ++i)
      t.rows[m.q_row0 + i] = RowInfo{m.own_unit,  m.own_blocks, m.qrows * G, i * G,
                                     m.pre_unit,  m.pre_blocks, m.pre_rows,  m.pre_row0 + i * G};
}

struct Group {
  int first, end;  // sequences
  int pages;       // shared, as far as sharing them pays
  int rows;        // query rows of the members
};

// One layout of the step; `share` off leaves every sequence whole.
int layout(const PlanConfig& cfg, bool keys, const std::vector<SeqInfo>& step,
           const std::vector<Group>& gs,
           const int32_t* pages, int total_pages, int rows, bool share, bool fixed_grid,
           LongResult& out, std::string& err) {
  out = LongResult{};
  const int G = cfg.hq / cfg.hkv, H = cfg.dec_heads, batch = static_cast<int>(step.size());
  const int kRowItem = row_item_rows(cfg.dim);
  Tables t;
  t.seqs = step;
  t.merge.assign(batch, MergeSeq{});
  std::vector<Unit> key, full, causal;
  auto add_rows = [&](int seq, int mode, int P, int qrows, int64_t length, bool record) {
    for (int h = 0; h < cfg.hkv; ++h)
      for (int p0 = 0; p0 < P; p0 += kRowItem) {
        const int n = std::min(kRowItem, P - p0);
        const int64_t limit = mode == 2 ? length : length - qrows + (p0 + n - 1) / G + 1;
        Unit u{seq, h, mode, p0 / kRowBlock, ceil_div(n, kRowBlock), ceil_div(length, kTileTokens),
               n, record};
        full.push_back(u);
        u.tiles = ceil_div(limit, kTileTokens);
        causal.push_back(u);
      }
  };
  auto add_key = [&](int seq, int mode, int P, int64_t length, bool record) {
    for (int h = 0; h < cfg.hkv; h += H)
      key.push_back(Unit{seq, h, mode, 0, 1, ceil_div(length, kTileTokens), H * P, record});
  };
  for (const Group& g : gs) {
    const int shared = share ? g.pages : 0;
    const int64_t plen = int64_t(shared) * cfg.page;
    int pre_unit = -1, pre_blocks = 0;
    const int PP = g.rows * G;
    if (shared > 0) {
      const SeqInfo& s0 = step[g.first];
      const int at = static_cast<int>(t.seqs.size());
      t.seqs.push_back(SeqInfo{s0.q_row0, g.rows, static_cast<int32_t>(plen), s0.page_off});
      ++out.groups_shared;
      if (PP <= kRowBlock) {
        pre_unit = static_cast<int>(key.size());
        add_key(at, 2, PP, plen, true);
      } else {
        pre_unit = static_cast<int>(full.size());
        pre_blocks = ceil_div(PP, kRowItem);
        add_rows(at, 2, PP, g.rows, plen, true);
      }
    }
    for (int b = g.first; b < g.end; ++b) {
      SeqInfo& s = t.seqs[b];
      if (s.qrows == 0) continue;
      s.length -= static_cast<int32_t>(plen);
      s.page_off += shared;
      MergeSeq& m = t.merge[b];
      const int P = s.qrows * G;
      m.q_row0 = s.q_row0;
      m.qrows = s.qrows;
      m.pre_unit = pre_unit;
      m.pre_blocks = pre_blocks;
      m.pre_row0 = (s.q_row0 - step[g.first].q_row0) * G;
      m.pre_rows = PP;
      if (P <= kRowBlock) {
        m.own_unit = static_cast<int>(key.size());
        add_key(b, 1, P, s.length, shared > 0);
      } else {
        m.own_unit = static_cast<int>(full.size());
        m.own_blocks = ceil_div(P, kRowItem);
        add_rows(b, 0, P, s.qrows, s.length, shared > 0);
      }
    }
  }
  const int row_units = static_cast<int>(full.size());
  for (MergeSeq& m : t.merge) {
    if (m.own_unit >= 0 && m.own_blocks == 0) m.own_unit += row_units;
    if (m.pre_unit >= 0 && m.pre_blocks == 0) m.pre_unit += row_units;
  }
  // Both kinds of work: the kernels run side by side, each on SMs of its own, the
  // row list's on as many as let both end together (it is bound by the tensor
  // pipe, the key kernel by memory, which a part of the SMs fills too).
  int row_sms = cfg.grid_cap, key_ctas = cfg.dec_grid_cap;
  if (keys && !full.empty() && !key.empty() && cfg.grid_cap > 1) {
    double row_us = 0, key_us = 0, key_bytes = 0;
    for (const Unit& u : full)
      row_us += (ceil_div(u.tiles, cfg.row_tile) *
                     cfg.row_weight[u.nrb > cfg.row_pair_blocks] + cfg.row_item_tiles) / 5.0;
    for (const Unit& u : key) {
      key_us += u.tiles * kKeyTileUs + kKeyItemUs;
      key_bytes += double(u.tiles) * kTileTokens * cfg.dim * 4;
    }
    const int per_sm = cfg.dec_grid_cap / cfg.grid_cap;
    double best = 1e30;
    for (int n = 1; n < cfg.grid_cap; ++n) {
      const int m = cfg.grid_cap - n;
      const double t = std::max(
          row_us / n, std::max(key_us / (m * per_sm), key_bytes / (kHbmGbs * 1e3)));
      if (t < best) {
        best = t;
        row_sms = n;
        key_ctas = m * per_sm;
      }
    }
  }
  View views[3];
  int rc = build_cost_view(cfg, full, row_sms, fixed_grid, views[0], err);
  if (rc == FE_OK) rc = build_cost_view(cfg, causal, row_sms, fixed_grid, views[1], err);
  if (rc == FE_OK) rc = decode_view(cfg, key, key_ctas, fixed_grid, views[2], err);
  if (rc != FE_OK) return rc;
  fill_rows(t, rows, G);
  return pack(cfg, keys, views, t, pages, total_pages, batch, rows, out, err);
}

}  // namespace

int build_shared_plan(const PlanConfig& cfg, bool keys, const int32_t* qo, const int32_t* kv,
                      const int32_t* pages, const int32_t* last, const int32_t* group_off,
                      const int32_t* shared, int groups, int batch, int rows, bool fixed_grid,
                      LongResult& out, std::string& err) {
  std::vector<SeqInfo> step;
  int rc = read_step(cfg, qo, kv, pages, last, batch, rows, step, err);
  if (rc != FE_OK) return rc;
  if (int64_t(rows) * cfg.hq > INT32_MAX / 2) {
    err = "too many query rows";
    return FE_ERR_CAPACITY;
  }
  if (groups < 0 || (groups > 0 && (!group_off || !shared))) {
    err = "groups need group_off and shared";
    return FE_ERR_INVALID_ARGUMENT;
  }
  std::vector<Group> gs;
  if (groups == 0) {
    for (int b = 0; b < batch; ++b) gs.push_back(Group{b, b + 1, 0, step[b].qrows});
  } else if (group_off[0] != 0 || group_off[groups] != batch) {
    err = "group_off must run from 0 to the batch";
    return FE_ERR_INVALID_ARGUMENT;
  }
  const int G = cfg.hq / cfg.hkv;
  int64_t saved_total = 0;
  for (int g = 0; g < groups; ++g) {
    const int first = group_off[g], end = group_off[g + 1];
    if (end < first || end > batch || shared[g] < 0) {
      err = "group_off must be non-decreasing and shared non-negative (g=" + std::to_string(g) +
            ")";
      return FE_ERR_INVALID_ARGUMENT;
    }
    Group x{first, end, shared[g], 0};
    double apart = 0;  // a tile of the prefix when it is not shared
    int members = 0;
    for (int b = first; b < end; ++b) {
      if (shared[g] > kv[b + 1] - kv[b] ||
          std::memcmp(pages + kv[first], pages + kv[b], sizeof(int32_t) * size_t(shared[g]))) {
        err = "sequence does not begin with its group's shared pages (b=" + std::to_string(b) + ")";
        return FE_ERR_INVALID_ARGUMENT;
      }
      const SeqInfo& s = step[b];
      x.rows += s.qrows;
      if (s.qrows == 0) continue;
      // a causal row sees the whole prefix: the query rows' own keys (one at
      // least) stay out
      x.pages = std::min(x.pages, (s.length - s.qrows) / cfg.page);
      ++members;
      apart += tile_us(cfg, int64_t(s.qrows) * G);
    }
    const int64_t PP = int64_t(x.rows) * G;
    const double tiles = double(x.pages) * cfg.page / 128 * cfg.hkv;
    const double records = 4.0 * PP * cfg.hkv * cfg.dim * sizeof(float) / (kRecordGbs * 1e3);
    const double launch = PP > kRowBlock ? kLaunchUs * cfg.grid_cap : 0;
    if (members < 2 || tile_us(cfg, PP) * tiles + records + launch >= apart * tiles)
      x.pages = 0;
    else
      saved_total += int64_t(members - 1) * x.pages * (cfg.page / kTileTokens) * cfg.hkv;
    gs.push_back(x);
  }
  const int total_pages = batch > 0 ? kv[batch] : 0;
  rc = layout(cfg, keys, step, gs, pages, total_pages, rows, true, fixed_grid, out, err);
  // where the records of the shared parts do not fit, every sequence stays whole
  if (rc == FE_ERR_CAPACITY && saved_total > 0) {
    saved_total = 0;
    rc = layout(cfg, keys, step, gs, pages, total_pages, rows, false, fixed_grid, out, err);
  }
  out.shared_tiles = saved_total;
  return rc;
}

int build_scored_plan(const PlanConfig& cfg, bool keys, const int32_t* qo, const int32_t* kv,
                      const int32_t* pages, const int32_t* last, const int32_t* fresh, int batch,
                      int rows, bool fixed_grid, int64_t sink_capacity, LongResult& out,
                      std::string& err) {
  out = LongResult{};
  std::vector<SeqInfo> step;
  int rc = read_step(cfg, qo, kv, pages, last, batch, rows, step, err);
  if (rc != FE_OK) return rc;
  if (int64_t(rows) * cfg.hq > INT32_MAX / 2) {
    err = "too many query rows";
    return FE_ERR_CAPACITY;
  }
  const int G = cfg.hq / cfg.hkv, H = cfg.dec_heads;
  const int per = kRowBlock / G;  // query rows of a block
  Tables t;
  std::vector<Unit> key;
  std::vector<uint8_t> used(size_t(cfg.num_blocks) + 1, 0);
  for (int b = 0; b < batch; ++b) {
    const SeqInfo& s = step[b];
    if (s.qrows == 0) continue;
    for (int i = kv[b]; i < kv[b + 1]; ++i) {
      if (used[pages[i]]++) {
        err = "page " + std::to_string(pages[i]) +
              " is listed twice: its scores would be added to by two CTAs";
        return FE_ERR_INVALID_ARGUMENT;
      }
    }
    const int f = fresh ? fresh[b] : s.qrows;
    if (f < 0 || f > s.length) {
      err = "fresh[b] must be in [0, length] (b=" + std::to_string(b) + ")";
      return FE_ERR_INVALID_ARGUMENT;
    }
    const int block0 = static_cast<int>(t.seqs.size());
    for (int i = 0; i < s.qrows; i += per) {
      const int n = std::min(per, s.qrows - i), P = n * G;
      // up to the last key that the block's last row sees
      const int length = s.length - s.qrows + i + n;
      const int tiles = ceil_div(length, kTileTokens);
      MergeSeq m;
      m.q_row0 = s.q_row0 + i;
      m.qrows = n;
      m.own_unit = static_cast<int>(key.size());
      t.merge.push_back(m);
      t.seqs.push_back(SeqInfo{s.q_row0 + i, n, length, s.page_off});
      t.sink.push_back(out.sink_floats);
      out.sink_floats += int64_t(cfg.hkv) * tiles * kTileTokens * ((P + 1) & ~1);
      for (int h = 0; h < cfg.hkv; h += H)
        key.push_back(Unit{static_cast<int>(t.seqs.size()) - 1, h, 1, 0, 1, tiles, H * P, true});
    }
    const int blocks = static_cast<int>(t.seqs.size()) - block0;
    for (int t0 = 0; t0 < s.length; t0 += kScoreChunk)
      t.chunks.push_back(ScoreChunk{block0, blocks, s.length, s.page_off, s.length - f, t0});
  }
  if (out.sink_floats > sink_capacity) {
    err = "query rows x keys exceed the plan's max_keys";
    return FE_ERR_CAPACITY;
  }
  View views[3];
  rc = decode_view(cfg, key, cfg.dec_grid_cap, fixed_grid, views[2], err);
  if (rc != FE_OK) return rc;
  fill_rows(t, rows, G);
  return pack(cfg, keys, views, t, pages, batch > 0 ? kv[batch] : 0, batch, rows, out, err);
}

}  // namespace fe
