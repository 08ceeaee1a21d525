// Decode attention over a part of every request's pages (decode_span.cu).
#pragma once
#include "attn.cuh"
#include "shared_prefix.cuh"

namespace piekv {

// What the prefix kernel left behind for the requests of a shared-prefix batch.
struct SpanPrefix {
  const int2 *requests = nullptr;  // [batch] (pages read with the group, group); nullptr: no prefix
  const sprefix::Group *groups = nullptr;
  const sprefix::Segment *segments = nullptr;
  const int *header = nullptr;     // the plan's
  const float *part_o = nullptr;   // [split][batch][Hq][128]
  const float2 *part_ml = nullptr;
  float *own_o = nullptr;          // [batch][Hq][128]: the requests' own pages, until the prefix's results are there
  float2 *own_ml = nullptr;
  int max_splits = 0;
  int overlap = 0;  // the launch may start before the prefix kernel has ended
};

bool decode_span_supported(const AttnArgs &a, int dtype);
int64_t decode_span_scratch_bytes(int hq, int hkv);
// a.window_left >= 0 with a.first_tokens, or `prefix`
int launch_decode_span(const AttnArgs &a, int dtype, const SpanPrefix &prefix, void *workspace, int64_t workspace_bytes,
                       cudaStream_t st);

}  // namespace piekv
