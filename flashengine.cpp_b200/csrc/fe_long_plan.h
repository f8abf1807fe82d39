// Host planners of the shared-prefix and the scored plans: work lists for the key
// kernel (at head_dim 256 the decode kernel) and the row kernels whose items write
// partial records, and the tables by which the kernels of fe_long_attn.cu join
// them. "Decode list" below is list 2 of fe_attn_plan.h, whichever kernel serves
// it. Pure C++.
//
// Shared-prefix plans: the sequences of a group begin with the same pages. The
// group's prefix becomes one more sequence of the lists, with the query rows of
// all its members and a mask that hides nothing (key_mode 2); each member keeps
// its own keys, those after the prefix. A query row's result is the joined
// softmax of its records from both.
//
// Scored plans: the query rows of a sequence are cut into blocks of at most 16
// packed rows, each a sequence of the decode list, whose raw scores the kernel
// stores beside the records.
#pragma once

#include <stdint.h>

#include <string>
#include <vector>

#include "fe_attn_plan.h"

namespace fe {

// The records of a unit (one sequence, KV head or heads, and block of rows):
// `n` of them, rec_floats apart. Units are numbered through both lists, row
// units first; n = 0: the unit writes its output itself.
struct UnitRec {  // 16 bytes
  int32_t part0, n, rec_floats, rows;
};

// Where the records of a query row lie: packed rows own_p .. own_p + G - 1 of
// the units from own_unit on, and the same of the prefix (pre_unit -1: none).
struct RowInfo {  // 32 bytes
  int32_t own_unit;
  int32_t own_blocks;  // row blocks (row_item_rows) a KV head; 0: units of the decode list
  int32_t own_rows;    // packed rows a KV head
  int32_t own_p;
  int32_t pre_unit, pre_blocks, pre_rows, pre_p;
};

// Packed rows of a row-kernel item: two tiles of the two-stream kernel, or one of
// the head_dim 256 kernel.
#ifdef __CUDACC__
__host__ __device__
#endif
constexpr int row_item_rows(int dim) { return dim == kHeadDim ? 256 : 128; }

// An item of the key kernel (fe_keys.cu): a WorkItem of the decode list with what
// it needs of its sequence.
struct KeyItem {  // 48 bytes
  int32_t q_row0, qrows, length, page_off;
  int32_t kvh, key_mode, kt0, kt1;
  int32_t part, group, seq, pad;
};

// A stretch of keys whose scores one CTA and KV head update.
struct ScoreChunk {  // 24 bytes
  int32_t block0, blocks;  // the sequence's row blocks (sequences of the lists)
  int32_t length, page_off;
  int32_t fresh;  // first key whose score is set and not added to
  int32_t t0;
};
constexpr int kScoreChunk = 512;  // keys

struct LongResult {
  std::vector<uint8_t> meta;
  int grid[3] = {0, 0, 0};
  bool merge[2] = {false, false};  // by mask: some unit writes records
  int rows = 0, groups_shared = 0, n_chunks = 0;
  int64_t shared_tiles = 0;   // key tiles that the sharing saves
  int64_t partial_floats = 0, sink_floats = 0;
};

// group_off [groups + 1]: runs of consecutive sequences, all of them;
// shared [groups]: pages that the members of each have in common at the start.
// keys: the decode list is the key kernel's (one KV head an item, cut by cost).
int build_shared_plan(const PlanConfig& cfg, bool keys, const int32_t* qo, const int32_t* kv,
                      const int32_t* pages, const int32_t* last, const int32_t* group_off,
                      const int32_t* shared, int groups, int batch, int rows, bool fixed_grid,
                      LongResult& out, std::string& err);

// fresh [batch]: keys at each sequence's end whose score is set (null: the
// query rows). sink_capacity: floats of raw scores.
int build_scored_plan(const PlanConfig& cfg, bool keys, const int32_t* qo, const int32_t* kv,
                      const int32_t* pages, const int32_t* last, const int32_t* fresh, int batch,
                      int rows, bool fixed_grid, int64_t sink_capacity, LongResult& out,
                      std::string& err);

}  // namespace fe
