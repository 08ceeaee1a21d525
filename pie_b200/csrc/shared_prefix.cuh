// The plan of a shared-prefix decode batch, as the plan kernels write it and the attention kernels read it.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace piekv {
namespace sprefix {

constexpr int kTileTokens = 128;   // kv tokens per tile (8 pages of 16)
constexpr int kRowsPerBlock = 256; // query rows (request x head of one kv head) that read a tile together at most
constexpr int kMaxCtas = 1024;

struct Group {
  int first, members;  // requests
  int pages;           // pages the group reads once (0: its requests go on their own)
  int segment;         // its first segment
};

// A prefix against a block of rows of one kv head: what a CTA streams without changing its query rows.  Segments are
// cut by the CTAs' shares at any tile; `pieces` of them hold a part, from `first_cta` on.
struct Segment {
  int request, list, pages;   // the group's first request, its page list's first entry, pages
  int kv_head, row0, rows;    // rows row0 .. row0 + min(rows, 256) - 1 of the group
  int first_cta, pieces;
};

struct PlanView {
  int *header;        // [0] CTAs at work on prefixes  [1] prefixes in use  [2] segments  [3] SMs left for the requests'
                      // own pages meanwhile (all of them when the two kernels follow each other)
  int2 *starts;       // [kMaxCtas + 1] (segment, tile) at which each CTA's share starts
  Group *groups;      // [num_groups]
  long long *line;    // [num_groups] where a group starts on the line that the shares divide
  int2 *requests;     // [batch] (pages read with the group, group)
  int *match;         // [batch] scratch: leading full pages equal to the group's first request's
  Segment *segments;  // [max_segments]
  int max_segments;
  int64_t bytes;
};

// How many partial results a row of a segment has: one per piece, or two where the block has at most 128 rows, whose
// second half then works on the second half of the piece.
__host__ __device__ inline int partials_of(const Segment &s, int max_splits) {
  return s.rows <= kRowsPerBlock / 2 && max_splits >= 2 ? 2 * s.pieces : s.pieces;
}

__host__ __device__ inline PlanView plan_view(void *plan, int batch, int groups, int hq, int hkv) {
  PlanView v;
  const int64_t rows = (int64_t)batch * (hq / hkv);
  v.max_segments = (int)((rows / kRowsPerBlock + (groups < batch ? groups : batch)) * hkv);
  uint8_t *base = reinterpret_cast<uint8_t *>(plan);
  int64_t off = 0;
  auto take = [&](int64_t bytes) {
    uint8_t *p = base + off;
    off += (bytes + 255) / 256 * 256;
    return p;
  };
  v.header = reinterpret_cast<int *>(take(256));
  v.starts = reinterpret_cast<int2 *>(take((int64_t)(kMaxCtas + 1) * sizeof(int2)));
  v.groups = reinterpret_cast<Group *>(take((int64_t)groups * sizeof(Group)));
  v.line = reinterpret_cast<long long *>(take((int64_t)groups * sizeof(long long)));
  v.requests = reinterpret_cast<int2 *>(take((int64_t)batch * sizeof(int2)));
  v.match = reinterpret_cast<int *>(take((int64_t)batch * 4));
  v.segments = reinterpret_cast<Segment *>(take((int64_t)v.max_segments * sizeof(Segment)));
  v.bytes = off;
  return v;
}

}  // namespace sprefix
}  // namespace piekv
