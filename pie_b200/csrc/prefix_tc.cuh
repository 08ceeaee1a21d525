// Attention of many requests to the pages they share (prefix_tc.cu).
#pragma once
#include "shared_prefix.cuh"

namespace piekv {

struct PrefixTcParams {
  const void *q;  // [batch, Hq, 128], rows 16-byte aligned
  int64_t q_sn, q_sh;
  const int32_t *kv_indices;
  int *header;  // the plan's
  const sprefix::Item *items;
  float *part_o;    // [split][batch][Hq][128], unnormalised
  float2 *part_ml;  // [split][batch][Hq]: reference maximum (log2 units), sum
  int batch, hq, group, num_pages, max_splits;
  int problem;      // rows of one MMA problem: whole requests
  float scale_log2;
  int32_t *err;
};

int launch_prefix_tc(const PrefixTcParams &p, const void *pool, int hkv, int dtype, cudaStream_t st);

}  // namespace piekv
