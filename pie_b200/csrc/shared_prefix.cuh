// The plan of a shared-prefix decode batch, as the plan kernels write it and the attention kernels read it.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piekv {
namespace sprefix {

constexpr int kTileTokens = 128;  // kv tokens per tile (8 pages of 16)
constexpr int kSpareItems = 4096; // items beyond one per segment

// Query rows (request x head of one kv head) of one MMA problem: whole requests, up to 128 rows.  A block is two problems.
__host__ __device__ inline int problem_rows(int heads_per_kv) { return heads_per_kv * (128 / heads_per_kv); }

struct Group {
  int first, members;  // requests
  int pages;           // pages the group reads once (0: its requests go on their own)
  int segment;         // its first segment
};

// A prefix against a block of rows of one kv head, cut into `pieces` items.
struct Segment {
  int rows;  // from the block's first request to the group's end (at most two problems' worth are this segment's)
  int pieces;
};
// One piece of a segment, with what the segment says about it: a CTA starts on its first item after one load.
struct Item {
  int request, list, pages;  // first request of the block, the group's page list's first entry, pages
  int kv_head, rows;
  int t0, t1, piece;  // tiles [t0, t1)
};

struct PlanView {
  int *header;        // [0] CTAs at work on prefixes  [1] prefixes in use  [2] items  [3] SMs left for the requests' own
                      // pages meanwhile (all of them when the two kernels follow each other)
                      // [4] items claimed  [5] CTAs done: zero between runs
  Group *groups;      // [num_groups]
  int2 *requests;     // [batch] (pages read with the group, group)
  int *match;         // [batch] scratch: leading full pages equal to the group's first request's
  Segment *segments;  // [max_segments]
  Item *items;        // [max_segments + kSpareItems]
  int max_segments;
  int64_t bytes;
};

// How many partial results a row of a segment has: one per piece, or two where the block is one problem, whose twin then
// works on the second half of the piece.
__host__ __device__ inline int partials_of(const Segment &s, int problem, int max_splits) {
  return s.rows <= problem && max_splits >= 2 ? 2 * s.pieces : s.pieces;
}

__host__ __device__ inline PlanView plan_view(void *plan, int batch, int groups, int hq, int hkv) {
  PlanView v;
  const int group = hq / hkv;
  const int64_t block = 2 * (group <= 128 ? problem_rows(group) : group);
  v.max_segments = (int)(((int64_t)batch * group / block + (groups < batch ? groups : batch)) * hkv);
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
  v.segments = reinterpret_cast<Segment *>(take((int64_t)v.max_segments * sizeof(Segment)));
  v.items = reinterpret_cast<Item *>(take((int64_t)(v.max_segments + kSpareItems) * sizeof(Item)));
  v.bytes = off;
  return v;
}

}  // namespace sprefix
}  // namespace piekv
