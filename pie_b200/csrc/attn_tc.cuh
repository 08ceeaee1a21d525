// MMA batches and small arithmetic shared by the two-problem attention kernels (prefill_tc2.cu, prefix_tc.cu).
#pragma once
#include "prefill_common.cuh"
#include "tcgen05.cuh"

namespace piekv {
namespace prefill {

// not volatile: the scheduler may interleave these with the surrounding arithmetic
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
// The MMA batches.  Inlined on purpose: the issuing thread's own instructions sit on the critical path
// between one softmax pass of a head and the next, and a call per batch measured 10 % slower.
// S = Q K^T: eight K = 16 steps over the two 64-element halves of head_dim, then the commit that wakes
// the softmax warps of the head.
__device__ __forceinline__ void issue_scores(uint32_t d_tmem, uint64_t q_desc, uint64_t k_desc, uint32_t idesc,
                                             uint64_t *s_full_bar) {
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
    const uint64_t off = (uint64_t)(((ks >> 2) * kHalfBytes + (ks & 3) * 32) >> 4);
    tc::mma_ss(d_tmem, q_desc + off, k_desc + off, idesc, ks > 0 ? 1u : 0u);
  }
  tc::commit(s_full_bar);
}
// O (+)= P V for 64 kv tokens (four K = 16 steps); P is read from TMEM, two 16-bit values per column
__device__ __forceinline__ void issue_pv_half(uint32_t d_tmem, uint32_t p_tmem, uint64_t v_desc, uint32_t idesc,
                                              uint32_t accumulate_first) {
#pragma unroll
  for (int ks = 0; ks < 4; ++ks)
    tc::mma_ts(d_tmem, p_tmem + ks * 8, v_desc + (uint64_t)((ks * 2048) >> 4), idesc, (accumulate_first || ks > 0) ? 1u : 0u);
}

}  // namespace prefill
}  // namespace piekv
