// The host planner's building blocks (fe_attn_plan.cpp), shared by the planners
// of the different kinds of plans.
#pragma once

#include <string>
#include <vector>

#include "fe_attn_plan.h"

namespace fe {

// One (sequence, KV head or heads, query-row block) against its key tiles.
struct Unit {
  int seq, kvh, key_mode, rb0, nrb, tiles, rows;
  bool record = false;  // lists cut by cost: a record even when it is not cut
};

struct View {
  std::vector<int32_t> cta_off;
  std::vector<WorkItem> items;
  std::vector<SplitGroup> groups;
  std::vector<int> unit_group;  // lists cut by cost: group of each unit, -1 for none
  int grid = 0, chunk = 0, decode_items = 0, prefill_items = 0, split_units = 0;
  int64_t partial_floats = 0;
};

inline int ceil_div(int64_t a, int64_t b) { return static_cast<int>((a + b - 1) / b); }

inline size_t align16(size_t n) { return (n + 15) & ~size_t(15); }

int read_step(const PlanConfig& cfg, const int32_t* qo, const int32_t* kv, const int32_t* pages,
              const int32_t* last, int batch, int rows, std::vector<SeqInfo>& seqs,
              std::string& err);

int build_cost_view(const PlanConfig& cfg, const std::vector<Unit>& units, int grid_cap,
                    bool fixed_grid, View& v, std::string& err);

}  // namespace fe
