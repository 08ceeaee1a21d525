// The plan of a shared-prefix decode batch, as the plan kernels write it and the attention kernels read it.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piekv {
namespace sprefix {

constexpr int kTileTokens = 128;           // kv tokens per tile (8 pages of 16)
constexpr int kRowsPerItem = 256;          // query rows (request x head of one kv head) an item covers at most
constexpr int kSpareItems = 2048;          // items beyond one per (group, kv head, row block)

struct Group {
  int first, members;  // requests
  int pages;           // pages the group reads once (0: its requests go on their own)
  int chunks;          // pieces the prefix is cut into
};

// One piece of work: rows [256 row_block, +256) of (group, kv head), chunk `chunk` of the group's prefix.
struct Item {
  int group, kv_head, row_block, chunk;
};

struct PlanView {
  int *header;       // [0] items  [1] prefixes in use  [2] CTAs that work on them  [3] SMs left for the requests' own
                     // pages meanwhile (all of them when the two kernels follow each other)
  Group *groups;     // [num_groups]
  int2 *requests;    // [batch] (pages read with the group, group)
  int *match;        // [batch] scratch: leading full pages equal to the group's first request's
  Item *items;       // [max_items]
  int max_items;
  int64_t bytes;
};

// How many partial results the row `row` (request * heads_per_kv + head of the kv head) of a group has: one per
// chunk, or two where its row block has at most 128 rows, whose other half then works on the rest of the chunk.
__host__ __device__ inline int partials_of(const Group &g, int row, int heads_per_kv, int max_splits) {
  const int left = g.members * heads_per_kv - row / kRowsPerItem * kRowsPerItem;
  return left <= kRowsPerItem / 2 && max_splits >= 2 ? 2 * g.chunks : g.chunks;
}

__host__ __device__ inline PlanView plan_view(void *plan, int batch, int groups, int hq, int hkv) {
  PlanView v;
  const int64_t rows = (int64_t)batch * (hq / hkv);
  v.max_items = (int)((rows / kRowsPerItem + (groups < batch ? groups : batch)) * hkv) + kSpareItems;
  uint8_t *base = reinterpret_cast<uint8_t *>(plan);
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    uint8_t *p = base + off;
    off += (bytes + 255) / 256 * 256;
    return p;
  };
  v.header = reinterpret_cast<int *>(take(256));
  v.groups = reinterpret_cast<Group *>(take((int64_t)groups * sizeof(Group)));
  v.requests = reinterpret_cast<int2 *>(take((int64_t)batch * sizeof(int2)));
  v.match = reinterpret_cast<int *>(take((int64_t)batch * 4));
  v.items = reinterpret_cast<Item *>(take((int64_t)v.max_items * sizeof(Item)));
  v.bytes = off;
  return v;
}

}  // namespace sprefix
}  // namespace piekv
