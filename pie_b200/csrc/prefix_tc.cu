// Attention of many requests to the pages they share, on the sm_100a tensor cores (tcgen05 / TMEM).
//
// The query rows of a group and kv head are packed, row = request * (heads per kv head) + head, so a prefix is read
// once for all of them.  A segment is (group, kv head, block of up to 256 rows); it is cut into items, which persistent
// CTAs claim (the plan, shared_prefix.cu).  Two 128-row problems "A" and "B" run against each other on one SM - while the
// softmax warps of one work on its scores, the tensor pipe runs the other's MMAs:
//   more than one problem's rows   A and B are the two halves of the block and share every K and V tile
//   otherwise                      A and B are the same rows over the two halves of the item
// Every problem leaves a partial result (m, l, O) per row, unnormalised and in fp32, for the kernel that folds it with
// the request's own pages (decode_span.cu): M = max m_i, L = sum l_i 2^(m_i - M), O = sum O_i 2^(m_i - M).
//
// What bounds it: with R rows per kv head a prefix token costs 4 * 128 * R flops and 512 bytes, so the tensor and
// special-function pipes from about 200 rows on, HBM below.  A tile against two problems takes 2.1 us; on some boards
// half of the SMs take 2.7 under this load, which is why items are claimed instead of dealt out (with equal shares per
// CTA the fast ones stood idle for a third of the launch there: ends between 67 and 110 us).
// Measured, with the kernel beside it: 16384 shared tokens, 128 requests, 64 / 8 heads, fp16, up to 512 tokens of their
// own (70 GFLOP, 202 MB): 112 us, 0.62 PFLOP/s; of it 3.5 until the first scores, 92 for 43 tiles (96 CTAs), 4 to store
// rows, 12 for the joins.
// 64 requests behind 4096 tokens with 1024 of their own, 32 / 8 heads: 43 us (158 MB); 16 prompts of 4 beams: 33 us.
//
//   TMEM (512 columns): S_A/P_A [0,128)  S_B/P_B [128,256)  O_A [256,384)  O_B [384,512)
//   smem: Q_A, Q_B (32 KiB each), K ring (3 x 32 KiB), V ring (2 x 32 KiB)
// P stays in TMEM (packed 16-bit pairs over the scores' columns).  One thread issues every MMA, per step t
//   O_A(t) S_A(next) O_B(t) S_B(next),  next = tile t + 1 or the following item's first,
// so the streams run across item boundaries: the rings keep filling, a problem's query rows are replaced once its last
// scores are computed, and the next item's first scores run while the softmax warps store the finished one's rows.
//
// Precision: S, m, l, O in fp32; P is rounded to the storage type because it meets V in one MMA type.
//
// Roles (384 threads): warps 0-3 softmax of A (thread = row = TMEM lane), 4-7 of B, 8 K producer, 9 MMA issuer and
// TMEM owner, 10 V producer, 11 scheduler (claims items, describes them in a ring that every role reads, brings query
// rows in); the last four give registers to the softmax warps.  Every wait is bounded; on a timeout the CTA reports, all
// roles leave, bulk copies are drained and TMEM is released.
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
constexpr int kPxVWarp = kMmaWarp + 1, kPxSchedWarp = kMmaWarp + 2;
constexpr int kPxSlots = 4;                         // items the scheduler may describe ahead of the slowest reader
constexpr int kPxReaders = kSoftmaxWarps + 1 + 3;   // softmax warps, MMA thread, K, V and query-row cursors
static_assert(kTileTokens == kBN, "plan and kernel cut the work alike");
static_assert(sizeof(Item) == 32, "read as two vectors");

// An item as the scheduler publishes it.
struct Work {
  int valid;                  // 0: nothing is left
  int list, pages, kv_head;   // the group's page list and its pages
  int request[2], rows[2];    // first request and rows of A and B
  int n[2], t0[2], split[2];  // tiles, first tile and partial index of A and B
  int pair;                   // A and B share their tiles
};

__device__ __forceinline__ void store_v8(float *dst, const uint32_t *r) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kPxThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_kv,
                     const __grid_constant__ PrefixTcParams p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], k_full[kKStages], k_empty[kKStages], v_full[kVStages],
      v_empty[kVStages], s_full[2], p_full[2][2], o_done[2], item_full[kPxSlots], item_empty[kPxSlots];
  __shared__ __align__(16) Work sh_item[kPxSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ int sh_abort;

  // The kernel behind this one reads its own pages first and waits for these results only then.
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // The first item is the CTA's own: it is loaded together with the header (there is room for more items than CTAs).
  const int4 *first = reinterpret_cast<const int4 *>(p.items + blockIdx.x);
  int4 it0 = make_int4(0, 0, 0, 0), it1 = it0;
  if (warp == kPxSchedWarp) {
    it0 = __ldg(first);
    it1 = __ldg(first + 1);
  }
  if (threadIdx.x == 0) {
    tma_prefetch_map(&tmap_q);
    tma_prefetch_map(&tmap_kv);
  }
  const int ctas = __ldg(p.header);
  if ((int)blockIdx.x >= ctas) return;

  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
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
      mbar_init(&q_full[x], 1);
      mbar_init(&q_empty[x], 1);
      mbar_init(&s_full[x], 1);
      mbar_init(&p_full[x][0], 4);  // one arrival per softmax warp
      mbar_init(&p_full[x][1], 4);
      mbar_init(&o_done[x], 1);
    }
    for (int s = 0; s < kPxSlots; ++s) {
      mbar_init(&item_full[s], 1);
      mbar_init(&item_empty[s], kPxReaders);
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
  // item number `n` of this CTA, read by a whole warp; false after a timeout
  auto read_item = [&](int n, Work &w, int where) -> bool {
    const int slot = n % kPxSlots;
    if (!wait_or_abort(&item_full[slot], (n / kPxSlots) & 1, abort_flag)) {
      give_up(where);
      return false;
    }
    w = sh_item[slot];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[slot]);
    return true;
  };

  if (warp >= kSoftmaxWarps) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPxRegsOther));
    if (warp == kPxSchedWarp) {
      // ================================================================ scheduler and query rows
      // Neither is urgent: this warp polls and sleeps instead of occupying issue slots.
      const int items = __ldg(p.header + 2);
      int n = 0, sched_done = 0;             // items described
      int qn = 0, q_x = 2, q_done = 0;       // query-row cursor: item, problem (2: the item is still to be read)
      int q_cnt[2] = {0, 0};                 // query tiles requested
      Work qw{};
      uint64_t idle_since = 0;
      while (!(sched_done && q_done)) {
        bool progressed = false;
        if (!sched_done && __any_sync(0xffffffffu, mbar_test_wait(&item_empty[n % kPxSlots], ((n / kPxSlots) & 1) ^ 1))) {
          int idx = blockIdx.x;  // the first item is the CTA's own, the others are claimed
          if (n > 0) {
            if (lane == 0) idx = ctas + atomicAdd(p.header + 4, 1);
            idx = __shfl_sync(0xffffffffu, idx, 0);
            if (idx < items) {
              it0 = __ldg(reinterpret_cast<const int4 *>(p.items + idx));
              it1 = __ldg(reinterpret_cast<const int4 *>(p.items + idx) + 1);
            }
          }
          Work w{};
          if (idx < items) {  // it0 = request, list, pages, kv head; it1 = rows, t0, t1, piece
            w.valid = 1;
            w.list = it0.y;
            w.pages = it0.z;
            w.kv_head = it0.w;
            w.pair = it1.x > p.problem;
            w.request[0] = w.request[1] = it0.x;
            w.rows[0] = w.rows[1] = min(it1.x, p.problem);
            w.t0[0] = w.t0[1] = it1.y;
            w.n[0] = w.n[1] = it1.z - it1.y;
            w.split[0] = w.split[1] = it1.w;
            if (w.pair) {
              w.request[1] += p.problem / p.group;
              w.rows[1] = min(it1.x - p.problem, p.problem);
            } else if (p.max_splits >= 2) {
              w.n[0] = (it1.z - it1.y + 1) / 2;
              w.n[1] -= w.n[0];
              w.t0[1] += w.n[0];
              w.split[0] = 2 * it1.w;
              w.split[1] = 2 * it1.w + 1;
            } else {
              w.n[1] = w.rows[1] = 0;
            }
          }
          if (lane == 0) {
            sh_item[n % kPxSlots] = w;
            mbar_arrive(&item_full[n % kPxSlots]);  // release: the description is visible to whoever sees the phase
          }
          __syncwarp();
          if (w.valid)
            ++n;
          else
            sched_done = 1;
          progressed = true;
        }
        if (!q_done) {
          if (q_x == 2) {
            if (__any_sync(0xffffffffu, mbar_test_wait(&item_full[qn % kPxSlots], (qn / kPxSlots) & 1))) {
              qw = sh_item[qn % kPxSlots];
              __syncwarp();
              if (lane == 0) mbar_arrive(&item_empty[qn % kPxSlots]);
              ++qn;
              if (qw.valid)
                q_x = 0;
              else
                q_done = 1;
              progressed = true;
            }
          } else if (qw.n[q_x] == 0) {
            ++q_x;
            progressed = true;
          } else if (__any_sync(0xffffffffu, mbar_test_wait(&q_empty[q_x], (q_cnt[q_x] & 1) ^ 1))) {
            if (lane == 0) {
              mbar_arrive_expect_tx(&q_full[q_x], (uint32_t)(p.problem * 256));
              const uint32_t dst = q_smem + q_x * kTileBytes;
              tma_load_4d(dst, &tmap_q, 0, qw.kv_head * p.group, qw.request[q_x], 0, &q_full[q_x]);
              tma_load_4d(dst + kHalfBytes, &tmap_q, 0, qw.kv_head * p.group, qw.request[q_x], 1, &q_full[q_x]);
            }
            ++q_cnt[q_x];
            ++q_x;
            progressed = true;
          }
        }
        if (progressed) {
          idle_since = 0;
        } else {
          __nanosleep(100);
          if (*abort_flag) break;
          const uint64_t now = global_timer_ns();
          if (idle_since == 0) idle_since = now;
          if (now - idle_since > 2000000000ull) {
            give_up(400);
            break;
          }
        }
      }
      // The last scheduler to leave (for want of items, or after a timeout) puts the counters back to zero for the next
      // run: every CTA has made its final claim by then.
      if (lane == 0 && atomicAdd(p.header + 5, 1) == ctas - 1) {
        p.header[4] = 0;
        p.header[5] = 0;
      }
      // drain: the CTA must not retire while a bulk copy may still be landing
      if (lane == 0)
        for (int x = 0; x < 2; ++x)
          if (q_cnt[x] > 0) mbar_wait(&q_full[x], (q_cnt[x] - 1) & 1, 200000000ull);
    } else if (warp == kProducerWarp || warp == kPxVWarp) {
      // ================================================================ TMA producers: K tiles / V tiles
      const bool is_v = warp == kPxVWarp;
      const uint32_t ring0 = is_v ? v_smem0 : k_smem0;
      const int stages = is_v ? kVStages : kKStages;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      int armed = 0;
      bool ok = true;
      Work w;
      for (int n = 0; ok; ++n) {
        ok = read_item(n, w, is_v ? 120 : 100);
        if (!ok || !w.valid) break;
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
      }
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
        int qi[2] = {0, 0};        // query tiles of A and B taken so far: phases of q_full
        auto wait = [&](uint64_t *bar, int phase) { return wait_or_abort(bar, phase & 1, abort_flag); };
        auto wait_k = [&]() { return wait(&k_full[kt % kKStages], kt / kKStages); };
        auto wait_v = [&]() { return wait(&v_full[vt % kVStages], vt / kVStages); };
        // the next scores of problem x; `last` of the item's: its query rows are then no longer needed
        auto scores = [&](int x, bool last) {
          tc::fence_after_sync();
          issue_scores(tmem + x * 128, q_desc[x], k_desc0 + (uint64_t)(((kt % kKStages) * kTileBytes) >> 4), idesc_qk, &s_full[x]);
          if (last) tc::commit(&q_empty[x]);
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
        int n = 0;
        // the tiles of A and B of the following item; 0 when there is none, false after a timeout
        auto next_item = [&](int &na, int &nb, bool &pair) -> bool {
          const int slot = n % kPxSlots;
          if (!wait(&item_full[slot], n / kPxSlots)) return false;
          const bool valid = sh_item[slot].valid != 0;
          na = valid ? sh_item[slot].n[0] : 0;
          nb = valid ? sh_item[slot].n[1] : 0;
          pair = sh_item[slot].pair != 0;
          mbar_arrive(&item_empty[slot]);
          ++n;
          return true;
        };
        // an item's first scores: A has tiles always; B's tile is A's (pair) or the next one of the stream
        auto first_a = [&](int na, bool pair) -> bool {
          if (!wait(&q_full[0], qi[0]++) || !wait_k()) return false;
          scores(0, na == 1);
          if (!pair) release_k();
          return true;
        };
        auto first_b = [&](int nb) -> bool {
          if (nb == 0) return true;
          if (!wait(&q_full[1], qi[1]++) || !wait_k()) return false;
          scores(1, nb == 1);
          release_k();
          return true;
        };
        int na = 0, nb = 0;
        bool pair = false;
        bool ok = next_item(na, nb, pair);
        if (ok && na > 0) ok = first_a(na, pair) && first_b(nb);
        while (ok && na > 0) {
          int na2 = 0, nb2 = 0;
          bool pair2 = false;
#pragma unroll 1
          for (int t = 0; ok && t < na; ++t) {
            const bool last = t + 1 == na;
            if (last) ok = next_item(na2, nb2, pair2);
            ok = ok && wait_v() && pv(0, t > 0);
            if (!ok) break;
            if (!pair) release_v();
            if (!last) {
              ok = wait_k();
              if (!ok) break;
              scores(0, t + 2 == na);
              if (!pair) release_k();
            } else {
              tc::commit(&o_done[0]);  // all of A's MMAs of this item
              if (na2 > 0) ok = first_a(na2, pair2);
              if (!ok) break;
            }
            if (t < nb) {
              ok = wait_v() && pv(1, t > 0);
              if (!ok) break;
              release_v();
              if (t + 1 < nb) {
                ok = wait_k();
                if (!ok) break;
                scores(1, t + 2 == nb);
                release_k();
              } else {
                tc::commit(&o_done[1]);
              }
            }
            // (behind A's, as the tiles come: B may have ended a tile earlier)
            if (last && na2 > 0) ok = first_b(nb2);
          }
          na = na2;
          nb = nb2;
          pair = pair2;
        }
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
    const int member = row / p.group, g = row - member * p.group;
    int sc = 0, oc = 0;  // score tiles and items (with tiles) finished: phases of s_full and o_done
    bool ok = true;

    for (int item = 0; ok; ++item) {
      const int slot = item % kPxSlots;
      if (!wait_or_abort(&item_full[slot], (item / kPxSlots) & 1, abort_flag)) {
        ok = false;
        break;
      }
      const int valid = sh_item[slot].valid, rows = sh_item[slot].rows[x], n = sh_item[slot].n[x];
      const int first_tile = sh_item[slot].t0[x], limit = sh_item[slot].pages * kPage - 1;
      const int request = sh_item[slot].request[x] + member, head = sh_item[slot].kv_head * p.group + g;
      const size_t at = ((size_t)sh_item[slot].split[x] * p.batch + request) * p.hq + head;
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[slot]);
      if (!valid) break;
      const bool row_valid = row < rows;
      const bool warp_valid = q4 * 32 < rows;
      if (n == 0) {
        if (row_valid) p.part_ml[at] = make_float2(-INFINITY, 0.f);
        continue;
      }
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
        const int k0 = (first_tile + t) * kBN;
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
      if (!ok) break;
      ++oc;
      if (!warp_valid) continue;
      tc::fence_after_sync();
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
    }
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
int launch_t(const CUtensorMap &tq, const CUtensorMap &tkv, const PrefixTcParams &p, cudaStream_t st) {
  static unsigned char configured[kMaxDevices] = {0};
  if (int rc = opt_in_dynamic_smem(prefix_tc_kernel<T>, kPxSmemBytes, configured, "shared prefix: cudaFuncSetAttribute"))
    return rc;
  prefix_tc_kernel<T><<<sm_count(), kPxThreads, kPxSmemBytes, st>>>(tq, tkv, p);
  PIEKV_LAUNCH_CHECK("prefix_tc_kernel");
  return 0;
}

}  // namespace

int launch_prefix_tc(const PrefixTcParams &p, const void *pool, int hkv, int dtype, cudaStream_t st) {
  CUtensorMap tq, tkv;
  if (int rc = make_q_rows_tensor_map(&tq, p.q, p.batch, p.hq, p.q_sn, p.q_sh, dtype, p.group, p.problem / p.group)) return rc;
  if (int rc = make_page_tensor_map(&tkv, pool, p.num_pages, hkv, dtype, 1, 1, 1)) return rc;
  return dtype == PIEKV_BF16 ? launch_t<__nv_bfloat16>(tq, tkv, p, st) : launch_t<__half>(tq, tkv, p, st);
}

}  // namespace piekv
