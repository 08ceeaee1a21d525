// Attention of many requests to the pages they share, on the sm_100a tensor cores (tcgen05 / TMEM).
//
// The query rows of a group and kv head are packed, row = request * (heads per kv head) + head, so a prefix is read
// once for all of them.  A segment is (group, kv head, block of 256 rows); CTAs have equal shares of all segments' tiles
// (the plan, shared_prefix.cu) and work through the pieces of segments in theirs.  Two 128-row problems "A" and "B" run against each other on one SM - while the softmax warps of one work on its scores, the tensor pipe runs
// the other's MMAs:
//   more than 128 rows    A and B are the two halves of the block and share every K and V tile
//   at most 128 rows      A and B are the same rows over the two halves of the piece
// Every problem leaves a partial result (m, l, O) per row, unnormalised and in fp32, for the kernel that folds it with
// the request's own pages (decode_span.cu): M = max m_i, L = sum l_i 2^(m_i - M), O = sum O_i 2^(m_i - M).
//
// What bounds it: with R rows per kv head a prefix token costs 4 * 128 * R flops and 512 bytes, so the tensor and
// special-function pipes from about 200 rows on, HBM below.
//
//   TMEM (512 columns): S_A/P_A [0,128)  S_B/P_B [128,256)  O_A [256,384)  O_B [384,512)
//   smem: Q_A, Q_B (32 KiB each), K ring (3 x 32 KiB), V ring (2 x 32 KiB)
// P stays in TMEM (packed 16-bit pairs over the scores' columns) and the MMA order per step t is
//   O_A(t) S_A(t + 1) O_B(t) S_B(t + 1), as in the prefill kernel (prefill_tc2.cu).
//
// Precision: S, m, l, O in fp32; P is rounded to the storage type because it meets V in one MMA type.
//
// Roles (384 threads): warps 0-3 softmax of A (thread = row = TMEM lane), 4-7 of B, 8 K producer, 9 MMA issuer and
// TMEM owner, 10 V producer, 11 none; the last four give registers to the softmax warps.  The softmax threads bring
// their own query row into shared memory (256 bytes, any strides).  Every wait is bounded; on a timeout the CTA reports,
// all roles leave, bulk copies are drained and TMEM is released.
#include <cuda.h>

#include <type_traits>

#include "attn_tc.cuh"
#include "common.cuh"
#include "prefill_common.cuh"
#include "prefix_tc.cuh"
#include "tcgen05.cuh"
#include "tma.cuh"

namespace piekv {

using namespace prefill;
using namespace sprefix;

namespace {

constexpr int kPxThreads = 384;
constexpr int kPxRegsLaunch = 168, kPxRegsSoftmax = 200, kPxRegsOther = 96;
static_assert(256 * kPxRegsSoftmax + 128 * kPxRegsOther <= kPxThreads * kPxRegsLaunch, "registers the CTA owns");
constexpr int kPxSmemBytes = kTileBytes * (2 + kKStages + kVStages) + 1024;
constexpr int kPxVWarp = kMmaWarp + 1;
static_assert(kTileTokens == kBN && kRowsPerBlock == 2 * kBM, "plan and kernel cut the work alike");
static_assert(sizeof(Segment) == 32, "a segment is read as two vectors");

// A piece of a segment as every role reads it off the plan.
struct Work {
  int request, list, pages;    // the group's first request, its page list, pages of the prefix
  int kv_head, row0;
  int rows[2];                 // rows of A and B
  int n[2], t0[2], split[2];   // tiles, first tile and partial index of A and B
  bool pair;                   // A and B share their tiles
};
__device__ __forceinline__ int4 ld_int4(const void *p) { return __ldg(reinterpret_cast<const int4 *>(p)); }
// tiles [t0, t1) of segment `seg`, by CTA `cta`; t1 < 0: to its end
__device__ __forceinline__ Work work_of(const PrefixTcParams &p, int cta, int seg, int t0, int t1) {
  const int4 a = ld_int4(p.segments + seg), b = ld_int4(reinterpret_cast<const int4 *>(p.segments + seg) + 1);
  Segment s;
  s.request = a.x, s.list = a.y, s.pages = a.z, s.kv_head = a.w;
  s.row0 = b.x, s.rows = b.y, s.first_cta = b.z, s.pieces = b.w;
  Work w;
  w.request = s.request;
  w.list = s.list;
  w.pages = s.pages;
  w.kv_head = s.kv_head;
  w.row0 = s.row0;
  if (t1 < 0) t1 = (s.pages * kPage + kBN - 1) / kBN;
  const int piece = s.pieces > 1 ? cta - s.first_cta : 0;
  w.pair = s.rows > kBM;
  w.t0[0] = t0;
  if (w.pair) {
    w.rows[0] = kBM;
    w.rows[1] = min(kBM, s.rows - kBM);
    w.n[0] = w.n[1] = t1 - t0;
    w.t0[1] = t0;
    w.split[0] = w.split[1] = piece;
  } else {
    const bool two = p.max_splits >= 2;
    w.rows[0] = w.rows[1] = s.rows;
    w.n[0] = two ? (t1 - t0 + 1) / 2 : t1 - t0;
    w.n[1] = t1 - t0 - w.n[0];
    w.t0[1] = t0 + w.n[0];
    w.split[0] = two ? 2 * piece : piece;
    w.split[1] = 2 * piece + 1;
    if (!two) w.rows[1] = 0;
  }
  return w;
}
// the pieces of a CTA's share in order: fn(piece) until it returns false
template <typename F>
__device__ __forceinline__ void for_pieces(const PrefixTcParams &p, int cta, int2 from, int2 to, F fn) {
#pragma unroll 1
  for (int seg = from.x; seg < to.x || (seg == to.x && to.y > 0); ++seg)
    if (!fn(work_of(p, cta, seg, seg == from.x ? from.y : 0, seg == to.x ? to.y : -1))) return;
}

__device__ __forceinline__ void store_v8(float *dst, const uint32_t *r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kPxThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tmap_kv, const __grid_constant__ PrefixTcParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages],
      s_full[2], p_full[2][2], o_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort;

  // The kernel behind this one reads its own pages first and waits for these results only then.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int2 share_from = __ldg(p.starts + blockIdx.x), share_to = __ldg(p.starts + blockIdx.x + 1);
  if (share_from.x == share_to.x && share_from.y == share_to.y) return;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *base_ptr = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t q_smem = base;
  const uint32_t k_smem0 = base + 2 * kTileBytes;
  const uint32_t v_smem0 = base + (2 + kKStages) * kTileBytes;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 4);  // one arrival per softmax warp
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x][0], 4);
      mbar_init(&p_full[x][1], 4);
      mbar_init(&o_done[x], 1);
    }
    sh_abort = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc(&tmem_slot, kTmemCols);
    tc::tmem_relinquish();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = tmem_slot;
  volatile int *abort_flag = &sh_abort;
  constexpr bool kBf16 = !std::is_same<T, __half>::value;
  auto give_up = [&](int where) {
    if (lane == 0 && atomicExch(&sh_abort, 1) == 0)
      report_error(p.err, PIEKV_ERR_WAIT_TIMEOUT, KID_SHARED_PREFIX, blockIdx.x, where);
  };

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPxRegsOther));
    if (warp == kProducerWarp || warp == kPxVWarp) {
      // ================================================================ TMA producers: K tiles / V tiles
      const bool is_v = warp == kPxVWarp;
      const uint32_t ring0 = is_v ? v_smem0 : k_smem0;
      const int stages = is_v ? kVStages : kKStages;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      int armed = 0;
      bool ok = true;
      for_pieces(p, blockIdx.x, share_from, share_to, [&](const Work &w) {
        // tiles in the order they are used: shared ones, or A's and B's in turn.  A tile's page ids are loaded while the
        // ring still waits for room.
        const int total = w.pair ? w.n[0] : w.n[0] + w.n[1];
        const bool turns = !w.pair && w.n[1] > 0;
        auto entry_of = [&](int u) { return (!turns ? w.t0[0] + u : (u & 1 ? w.t0[1] : w.t0[0]) + (u >> 1)) * 8 + lane; };
        auto page_of = [&](int u) -> int {
          if (u >= total || lane >= 8 || entry_of(u) >= w.pages) return p.num_pages;  // outside the tensor map: zeros
          return __ldg(p.kv_indices + w.list + entry_of(u));
        };
        int next = page_of(0);
        for (int u = 0; u < total; ++u) {
          int page = next;
          next = page_of(u + 1);
          const int st = armed % stages;
          if (!wait_or_abort(&empty[st], ((armed / stages) & 1) ^ 1, abort_flag)) {
            give_up(is_v ? 121 : 101);
            ok = false;
            break;
          }
          if (lane < 8 && entry_of(u) < w.pages && (page < 0 || page >= p.num_pages)) {
            report_error(p.err, PIEKV_ERR_PAGE_ID, KID_SHARED_PREFIX, w.list + entry_of(u), page);
            page = p.num_pages;
          }
          if (lane == 0) mbar_arrive_expect_tx(&full[st], kTileBytes);
          __syncwarp();
          if (lane < 8) {
            const uint32_t dst = ring0 + st * kTileBytes + lane * 2048;
            tma_load_5d(dst, &tmap_kv, 0, 0, 0, w.kv_head, page * 2 + (is_v ? 1 : 0), &full[st]);
            tma_load_5d(dst + kHalfBytes, &tmap_kv, 0, 0, 1, w.kv_head, page * 2 + (is_v ? 1 : 0), &full[st]);
          }
          ++armed;
        }
        return ok;
      });
      // drain: the CTA must not retire while a bulk copy may still be landing
      __syncwarp();
      if (lane == 0)
        for (int x = armed > stages ? armed - stages : 0; x < armed; ++x)
          mbar_wait(&full[x % stages], (x / stages) & 1, 200000000ull);
    } else if (warp == kMmaWarp) {
      // ================================================================ MMA issuer
      if (lane == 0) {
        constexpr uint32_t idesc_qk = tc::instr_desc(kBf16, false, false, kBM, kBN);
        constexpr uint32_t idesc_pv = tc::instr_desc(kBf16, false, true, kBM, kDim);
        const uint64_t q_desc[2] = {tc::desc_k_major(q_smem), tc::desc_k_major(q_smem + kTileBytes)};
        const uint64_t k_desc0 = tc::desc_k_major(k_smem0);
        const uint64_t v_desc0 = tc::desc_mn_major(v_smem0, kHalfBytes);
        int kt = 0, vt = 0;        // tiles of the two streams consumed so far
        int done[2] = {0, 0};      // probability tiles of A and B consumed: phases of p_full
        auto wait = [&](uint64_t *bar, int phase) { return wait_or_abort(bar, phase & 1, abort_flag); };
        auto wait_k = [&]() { return wait(&k_full[kt % kKStages], kt / kKStages); };
        auto wait_v = [&]() { return wait(&v_full[vt % kVStages], vt / kVStages); };
        auto scores = [&](int x) {
          tc::fence_after_sync();
          issue_scores(tmem + x * 128, q_desc[x], k_desc0 + (uint64_t)(((kt % kKStages) * kTileBytes) >> 4), idesc_qk, &s_full[x]);
        };
        auto release_k = [&]() {
          tc::commit(&k_empty[kt % kKStages]);
          ++kt;
        };
        auto release_v = [&]() {
          tc::commit(&v_empty[vt % kVStages]);
          ++vt;
        };
        auto pv = [&](int x, bool accumulate) -> bool {
          const uint64_t vd = v_desc0 + (uint64_t)(((vt % kVStages) * kTileBytes) >> 4);
          const uint32_t d = tmem + 256 + x * 128, pa = tmem + x * 128;
          if (!wait(&p_full[x][0], done[x])) return false;
          tc::fence_after_sync();
          issue_pv_half(d, pa, vd, idesc_pv, accumulate ? 1u : 0u);
          if (!wait(&p_full[x][1], done[x])) return false;
          tc::fence_after_sync();
          issue_pv_half(d, pa + 32, vd + (uint64_t)((4 * 2048) >> 4), idesc_pv, 1u);
          ++done[x];
          return true;
        };
        bool ok = true;
        int qi[2] = {0, 0};  // query tiles of A and B taken so far: phases of q_full
        for_pieces(p, blockIdx.x, share_from, share_to, [&](const Work &w) {
          const int na = w.n[0], nb = w.n[1];
          ok = wait(&q_full[0], qi[0]++) && wait_k();
          if (!ok) return false;
          scores(0);
          if (!w.pair) release_k();
          if (nb > 0) {
            ok = wait(&q_full[1], qi[1]++) && wait_k();
            if (!ok) return false;
            scores(1);
            release_k();
          }
#pragma unroll 1
          for (int t = 0; t < na; ++t) {
            ok = wait_v() && pv(0, t > 0);
            if (!ok) return false;
            if (!w.pair) release_v();
            if (t + 1 < na) {
              ok = wait_k();
              if (!ok) return false;
              scores(0);
              if (!w.pair) release_k();
            } else {
              tc::commit(&o_done[0]);
            }
            if (t >= nb) continue;
            ok = wait_v() && pv(1, t > 0);
            if (!ok) return false;
            release_v();
            if (t + 1 < nb) {
              ok = wait_k();
              if (!ok) return false;
              scores(1);
              release_k();
            } else {
              tc::commit(&o_done[1]);
            }
          }
          return true;
        });
        if (!ok) give_up(200);
      }
    }
  } else {
    // ================================================ softmax of problem x (thread = row = TMEM lane)
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPxRegsSoftmax));
    const int x = warp >> 2;
    const int q4 = warp & 3;
    const int row = q4 * 32 + lane;
    const uint32_t lane_base = (uint32_t)(q4 * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + x * 128;
    const uint32_t o_addr = tmem + lane_base + 256 + x * 128;
    const float c = p.scale_log2;
    int sc = 0, oc = 0;  // score tiles and items (with tiles) finished: phases of s_full and o_done
    bool ok = true;

    for_pieces(p, blockIdx.x, share_from, share_to, [&](const Work &w) {
      const int rows = w.rows[x], n = w.n[x];
      const bool row_valid = row < rows;
      const bool warp_valid = q4 * 32 < rows;
      const int r = w.row0 + (w.pair ? x * kBM : 0) + row;  // row of the group
      const int member = r / p.group, g = r - member * p.group;
      const int request = w.request + member, head = w.kv_head * p.group + g;
      if (n == 0) {  // (nothing is announced for it: the barriers' phases count pieces with tiles)
        if (row_valid) p.part_ml[((size_t)w.split[x] * p.batch + request) * p.hq + head] = make_float2(-INFINITY, 0.f);
        return true;
      }
      // ---- the query row into shared memory: K-major, 128-byte swizzle.  Every MMA that read the last item's is done:
      // this warp has seen the scores of all its tiles.
      if (warp_valid) {
        const uint4 *src = reinterpret_cast<const uint4 *>(reinterpret_cast<const T *>(p.q) + (int64_t)request * p.q_sn +
                                                           (int64_t)head * p.q_sh);
        uint4 v[16];
#pragma unroll
        for (int ch = 0; ch < 16; ++ch) v[ch] = row_valid ? __ldg(src + ch) : make_uint4(0, 0, 0, 0);
        uint8_t *dst = base_ptr + x * kTileBytes + row * 128;
#pragma unroll
        for (int ch = 0; ch < 16; ++ch)
          *reinterpret_cast<uint4 *>(dst + (ch >> 3) * kHalfBytes + (((ch & 7) ^ (row & 7)) << 4)) = v[ch];
        fence_proxy_async_smem();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[x]);
      const int limit = w.pages * kPage - 1;
      float m_ref = -INFINITY, l = 0.f;
      for (int t = 0; t < n; ++t) {
        ok = wait_or_abort(&s_full[x], sc & 1, abort_flag);
        if (!ok) break;
        ++sc;
        if (!warp_valid) {  // nobody reads these rows' results
          if (lane == 0) {
            mbar_arrive(&p_full[x][0]);
            mbar_arrive(&p_full[x][1]);
          }
          continue;
        }
        tc::fence_after_sync();
        const int k0 = (w.t0[x] + t) * kBN;
        const bool full_tile = k0 + kBN - 1 <= limit;
        uint4 mw = make_uint4(0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu);
        if (!full_tile) mw = band_bits(k0, 0, 0, limit);
        float mxa[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t sr[64];
          tc::tmem_ld32(s_addr + h * 64, sr);
          tc::tmem_ld32(s_addr + h * 64 + 32, sr + 32);
          tc::tmem_wait_ld();
          if (!full_tile) {
            const uint32_t w0 = h ? mw.z : mw.x, w1 = h ? mw.w : mw.y;
#pragma unroll
            for (int e = 0; e < 64; ++e) sr[e] = ((e < 32 ? w0 : w1) >> (e & 31)) & 1u ? sr[e] : 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e)
            mxa[e & 3] = max3(mxa[e & 3], __uint_as_float(sr[2 * e]), __uint_as_float(sr[2 * e + 1]));
        }
        const float mx = fmaxf(fmaxf(mxa[0], mxa[1]), fmaxf(mxa[2], mxa[3])) * c;  // c > 0
        float alpha = 1.f;
        bool rescale = false;
        if (mx > m_ref + 8.f) {  // the reference moves only when the maximum grows by more than 2^8
          alpha = exp2_approx(m_ref - mx);
          l *= alpha;
          m_ref = mx;
          rescale = t > 0;
        }
        if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
          for (int ch = 0; ch < 4; ++ch) {
            uint32_t oreg[32];
            tc::tmem_ld32(o_addr + ch * 32, oreg);
            tc::tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) oreg[e] = __float_as_uint(__uint_as_float(oreg[e]) * alpha);
            tc::tmem_st32(o_addr + ch * 32, oreg);
          }
        }
        const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
        float suma[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t sr[64];
          uint32_t pk[32];
          tc::tmem_ld32(s_addr + h * 64, sr);
          tc::tmem_ld32(s_addr + h * 64 + 32, sr + 32);
          tc::tmem_wait_ld();
          if (!full_tile) {
            const uint32_t w0 = h ? mw.z : mw.x, w1 = h ? mw.w : mw.y;
#pragma unroll
            for (int e = 0; e < 64; ++e) sr[e] = ((e < 32 ? w0 : w1) >> (e & 31)) & 1u ? sr[e] : 0xff800000u;
          }
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float p0v = exp2_approx(fmaf(__uint_as_float(sr[2 * e]), c, neg_m));
            const float p1v = exp2_approx(fmaf(__uint_as_float(sr[2 * e + 1]), c, neg_m));
            suma[e & 3] += p0v + p1v;
            pk[e] = pack2<T>(p0v, p1v);
          }
          tc::tmem_st16(s_addr + h * 32, pk);
          tc::tmem_st16(s_addr + h * 32 + 16, pk + 16);
          tc::tmem_wait_st();
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[x][h]);
        }
        l += (suma[0] + suma[1]) + (suma[2] + suma[3]);
      }
      // ---- the partial result.  The next item's O_x is not written before this warp has delivered that item's first
      // probabilities.
      if (ok) ok = wait_or_abort(&o_done[x], oc & 1, abort_flag);
      if (!ok) return false;
      ++oc;
      if (!warp_valid) return true;
      tc::fence_after_sync();
      const size_t at = ((size_t)w.split[x] * p.batch + request) * p.hq + head;
#pragma unroll 1
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t oreg[32];
        tc::tmem_ld32(o_addr + ch * 32, oreg);
        tc::tmem_wait_ld();
        if (row_valid) {
          // fragment order (decode_span.cu): element nt * 8 + 2 * q + e at q * 32 + nt * 2 + e, a sector per q
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = oreg[(e >> 1) * 8 + q * 2 + (e & 1)];
            store_v8(p.part_o + at * kDim + q * 32 + ch * 8, v);
          }
        }
      }
      if (row_valid) p.part_ml[at] = make_float2(m_ref, l);
      return true;
    });
    if (!ok) give_up(300 + warp);
  }

  // ---- teardown: every thread arrives here on every path
  tc::fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc::fence_after_sync();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T>
int launch_t(const CUtensorMap &tkv, const PrefixTcParams &p, cudaStream_t st) {
  static unsigned char configured[kMaxDevices] = {0};
  if (int rc = opt_in_dynamic_smem(prefix_tc_kernel<T>, kPxSmemBytes, configured, "shared prefix: cudaFuncSetAttribute"))
    return rc;
  prefix_tc_kernel<T><<<sm_count(), kPxThreads, kPxSmemBytes, st>>>(tkv, p);
  PIEKV_LAUNCH_CHECK("prefix_tc_kernel");
  return 0;
}

}  // namespace

int launch_prefix_tc(const PrefixTcParams &p, const void *pool, int hkv, int dtype, cudaStream_t st) {
  CUtensorMap tkv;
  if (int rc = make_page_tensor_map(&tkv, pool, p.num_pages, hkv, dtype, 1, 1, 1)) return rc;
  return dtype == PIEKV_BF16 ? launch_t<__nv_bfloat16>(tkv, p, st) : launch_t<__half>(tkv, p, st);
}

}  // namespace piekv
