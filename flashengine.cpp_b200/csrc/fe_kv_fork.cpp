// Copy lists for forked sequences and the prefixes that sequences share
// (fe_kv_fork_copies, fe_kv_shared_prefixes, fe_kv.h). Host code only: no device
// memory is touched, so it runs on a host without a GPU.
//
// The reference's BlockManager shares only whole published pages between
// sequences and never writes a published page (src/scheduler.cpp:6-29, the
// check at :27); the tokens of a prefix it cannot share are recomputed by a
// prefill. A fork that copies instead of recomputing needs, for every page
// of the shared prefix that the child does not share with the parent, one
// copy of the prefix tokens on that page from the parent's page to the
// child's. This file derives those copies from the two block tables, and
// rejects tables that would let one sequence write a page the other reads.
#include <stdint.h>

#include <algorithm>
#include <new>
#include <string>
#include <unordered_set>
#include <vector>

#include "fe_kv.h"

namespace fe {
int fail(int status, const std::string& msg);  // fe_kv_ops.cu: records fe_last_error()
}

extern "C" int fe_kv_fork_copies(int num_forks, const int32_t* parent_tables,
                                 const int32_t* parent_off, const int32_t* child_tables,
                                 const int32_t* child_off, const int64_t* fork_len, int page,
                                 int32_t* src, int32_t* dst, int32_t* ntok, int capacity,
                                 int* num_copies) {
  using fe::fail;
  if (num_copies) *num_copies = 0;
  if (num_forks < 0 || page <= 0 || capacity < 0 || !num_copies)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_fork_copies: bad sizes");
  if (num_forks == 0) return FE_OK;
  if (!parent_tables || !parent_off || !child_tables || !child_off || !fork_len ||
      (capacity > 0 && (!src || !dst || !ntok)))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_fork_copies: null pointer");
  int n = 0;
  for (int f = 0; f < num_forks; ++f) {
    const int32_t* parent = parent_tables + parent_off[f];
    const int32_t* child = child_tables + child_off[f];
    const int64_t np = int64_t(parent_off[f + 1]) - parent_off[f];
    const int64_t nc = int64_t(child_off[f + 1]) - child_off[f];
    const int64_t len = fork_len[f];
    const std::string at = "fe_kv_fork_copies: fork " + std::to_string(f) + ": ";
    if (np < 0 || nc < 0 || len < 0)
      return fail(FE_ERR_INVALID_ARGUMENT, at + "negative table size or fork length");
    const int64_t pages = (len + page - 1) / page;  // pages holding the shared prefix
    if (pages > np || pages > nc)
      return fail(FE_ERR_INVALID_ARGUMENT, at + "fork length beyond a block table");
    std::unordered_set<int32_t> parent_pages(parent, parent + np);
    for (int64_t j = 0; j < pages; ++j) {
      const int64_t tokens = len - j * page < page ? len - j * page : page;
      if (child[j] == parent[j]) {
        // a shared page must be full: both sequences append after `len`, so a
        // partial page would be written by one while the other reads it
        if (tokens < page)
          return fail(FE_ERR_INVALID_ARGUMENT,
                      at + "partial tail page " + std::to_string(parent[j]) +
                          " is shared; give the child a fresh page (copy-on-write)");
        continue;
      }
      if (child[j] < 0 || parent[j] < 0)
        return fail(FE_ERR_INVALID_ARGUMENT, at + "negative page id");
      if (parent_pages.count(child[j]))
        return fail(FE_ERR_INVALID_ARGUMENT,
                    at + "child page " + std::to_string(child[j]) +
                        " belongs to the parent at another position");
      if (n >= capacity)
        return fail(FE_ERR_CAPACITY, "fe_kv_fork_copies: more copies than `capacity`");
      src[n] = parent[j];
      dst[n] = child[j];
      ntok[n] = static_cast<int32_t>(tokens);
      ++n;
    }
    // beyond the prefix the child's pages are its own: none may be the parent's
    for (int64_t j = pages; j < nc; ++j)
      if (parent_pages.count(child[j]))
        return fail(FE_ERR_INVALID_ARGUMENT,
                    at + "child page " + std::to_string(child[j]) +
                        " past the fork belongs to the parent");
  }
  *num_copies = n;
  return FE_OK;
}

namespace fe {
namespace {

// Cuts the batch into groups of neighbours so that sharing saves the most: a group
// [a, e) reads its common pages once and not e - a times. With same[b] the pages in
// common of sequences b - 1 and b, it saves (e - a - 1) * min same[a + 1 .. e - 1];
// best[x] is the most that the sequences before begin[x] can save. Where same[] does
// not change a cut saves no more than at either end of the stretch, so that groups
// begin at those ends only: a batch over few prefixes has few of them. Among equals
// the larger last group is taken. Returns the groups.
int share(const int32_t* kv, const int32_t* pages, int batch, int min_pages, int32_t* group_off,
          int32_t* shared) {
  std::vector<int32_t> same(size_t(batch) + 1, 0);
  for (int b = 1; b < batch; ++b) {
    const int32_t *x = pages + kv[b - 1], *y = pages + kv[b];
    const int32_t most = std::min(kv[b] - kv[b - 1], kv[b + 1] - kv[b]);
    int32_t n = 0;
    while (n < most && x[n] == y[n]) ++n;
    same[b] = n >= min_pages ? n : 0;
  }
  std::vector<int> begin{0};
  for (int b = 1; b < batch; ++b)
    if (same[b] == 0 || b == 1 || b + 1 == batch || same[b] != same[b - 1] ||
        same[b] != same[b + 1])
      begin.push_back(b);
  if (batch > 0) begin.push_back(batch);
  const int ends = static_cast<int>(begin.size());
  std::vector<int64_t> best(ends, 0);
  std::vector<int> from(ends, 0);          // the last group begins at begin[from]
  std::vector<int32_t> common(ends, 0);    // and has so many pages in common
  for (int x = 1; x < ends; ++x) {
    const int end = begin[x];
    int32_t low = INT32_MAX;  // pages in common of the sequences from `a` on
    best[x] = -1;
    for (int y = x - 1; y >= 0; --y) {
      const int a = begin[y];
      if (begin[y + 1] - a > 1) low = std::min(low, same[a + 1]);
      if (y + 1 < x) low = std::min(low, same[begin[y + 1]]);
      if (low == 0) break;
      // no group that begins before can save more
      if (end - a > 1 && best[y] + int64_t(end - 1) * low < best[x]) break;
      const int64_t saved = best[y] + (end - a > 1 ? int64_t(end - a - 1) * low : 0);
      if (saved >= best[x]) {
        best[x] = saved;
        from[x] = y;
        common[x] = end - a > 1 ? low : 0;
      }
    }
  }
  int groups = 0;
  for (int x = ends - 1; x > 0; x = from[x]) ++groups;
  group_off[0] = 0;
  for (int x = ends - 1, g = groups; x > 0; x = from[x]) {
    group_off[g] = begin[x];
    shared[--g] = common[x];
  }
  return groups;
}

}  // namespace
}  // namespace fe

extern "C" int fe_kv_shared_prefixes(const int32_t* kv, const int32_t* pages, int batch,
                                     int min_pages, int32_t* group_off, int32_t* shared,
                                     int* num_groups) {
  using fe::fail;
  if (num_groups) *num_groups = 0;
  if (batch < 0 || min_pages < 1 || !num_groups)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_shared_prefixes: bad sizes");
  if (!group_off || (batch > 0 && (!kv || !pages || !shared)))
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_shared_prefixes: null pointer");
  // before any page is read: every list lies within the first kv[batch] pages
  if (batch > 0 && kv[0] != 0)
    return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_shared_prefixes: kv[0] must be 0");
  for (int b = 0; b < batch; ++b)
    if (kv[b + 1] < kv[b])
      return fail(FE_ERR_INVALID_ARGUMENT, "fe_kv_shared_prefixes: kv decreases (b=" +
                                               std::to_string(b) + ")");
  try {
    *num_groups = fe::share(kv, pages, batch, min_pages, group_off, shared);
  } catch (const std::bad_alloc&) {
    return fail(FE_ERR_CAPACITY, "fe_kv_shared_prefixes: out of host memory");
  }
  return FE_OK;
}
