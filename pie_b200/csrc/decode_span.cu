// Paged decode attention over a PART of every request's pages, 16-bit K/V, head_dim 128, page size 16 (sm_100a):
//
//   window with first tokens   the pages of tokens [0, first) and of the window behind the query; the pages between
//                              them are neither listed nor read
//   behind a shared prefix     the pages after the ones the request's group reads once (shared_prefix.cu); the
//                              prefix's partial results are folded in when a request's own pages are done
//
// Mathematics: one pass with a running maximum m, sum l and accumulator O per (request, query head); partial
// results (m, l, O) of page ranges join as M = max m_i, L = sum l_i 2^(m_i - M), O = sum O_i 2^(m_i - M), all in fp32.
//
// What bounds it: HBM.  2 * 2 * 128 bytes per token and kv head are read once, everything else is small.
//
// Work partition (in the kernel, no plan, so a captured graph follows its tables): every CTA reads the page counts
// of the whole batch, scans them, and takes an equal share [X_c, X_{c+1}) of the line on which each request occupies
// its visible pages plus kOpenCost (opening and closing a request costs about as much as streaming that many pages).
// A request cut by a share's end leaves partials in the two slots a share owns; the shares of a request are
// consecutive, so who holds a partial, and how many there are, follows from the line - there is no slot allocator, and
// results are reproducible bit for bit.  The last share to arrive (a counter per request and kv head, left zero) folds.
//
// Data path: a CTA takes HB kv heads of a page (HB = 2, or 1 where the head count is odd): HB * 8 KiB by TMA into a ring
// of stages, 192 KiB in flight per SM.  The producer warp and the consumer warps walk the same sequence independently;
// only the ring's barriers pass between them.  Consumer warp w owns head w: K and V [16 tokens x 128], 128-byte swizzled,
// as the m16n8k16 tensor-core fragments want them.  No step waits for the whole CTA: a warp opens, closes and folds the
// rows of its own head, and arrives only when its stream has ended.  (With block-wide closes through shared memory and
// arrivals on the way, a third of a CTA's time on short requests went into them.)
//
// Partial rows are kept in the order the MMA fragments hold them: element nt * 8 + 2 * q + e of a row at
// q * 32 + nt * 2 + e, so that a lane's 32 values of a row are one run of 128 bytes.
//
// Measured: 64 contexts of 512 .. 4096 tokens, 32 / 8 heads, window 1023, 4 first tokens (260 MB) 54 us, 4.8 TB/s; 128
// contexts of 2049 .. 8191, 64 / 8 heads, window 4095, 16 first tokens (1.97 GB) 316 us, 6.2 TB/s = 0.95 of the copy rate.
// In the 54 us the first bytes are asked for after 3.3 and the last CTAs' joins take 3.  One context: 10.3 us, of which
// streaming is 2.  More stages of one page, one head per CTA, or two shares per CTA changed the long cases by under 3 %.
//
// Precision: a GQA group of up to 8 heads fills rows 0-7 of the 16-row MMA.  Rows 8-15 then carry the part of each
// probability that its 16-bit rounding drops, so P V is formed with 16 bits of P (bf16) at no extra MMA.  Groups of 9 to
// 16 heads (WIDE) need all rows: P is rounded to the storage type there, as in the prefix and prefill kernels.
#include <cuda.h>

#include <type_traits>

#include "attn.cuh"
#include "common.cuh"
#include "decode_span.cuh"
#include "shared_prefix.cuh"
#include "tma.cuh"

namespace piekv {
namespace {

constexpr int kDim = 128;
constexpr int kPage = 16;
constexpr int kTileBytes = 8192;  // one (page, head): K 4 KiB + V 4 KiB
constexpr int kCounterBytes = 65536;
constexpr int kMaxSlice = 512;   // requests per launch: the line is kept in shared memory
static_assert(kMaxSlice * 128 <= 65536 && PIEKV_SHARED_PREFIX_MAX_SPLITS < 128, "sh_closed packs a request and a count");
constexpr int kOpenCost = 4;     // pages
// A share is not made smaller than kMinUnits, nor than sqrt(kUnitsOfLine * a request's part of the line): a page more
// costs a share 0.5 us, a partial more costs the warp that joins a request a quarter of a microsecond.  (One context of 8000
// tokens in a window of 4095, 32 / 8 heads: 20.4 us with shares of 4 pages, 17.1 with 12; of 516 tokens 10.1 and 13.5.)
constexpr int kMinUnits = 4;
constexpr float kUnitsOfLine = 0.45f;

// Launch shape for HB heads per CTA: 12 warps per SM (168 registers each) and 24 tiles in flight.
template <int HB>
struct Shape {
  static constexpr int kThreads = (HB + 1) * 32;
  static constexpr int kCtasPerSm = HB == 1 ? 6 : 4;
  static constexpr int kStages = HB == 1 ? 4 : 3;
  static constexpr int kStageBytes = HB * kTileBytes;
  static constexpr int kSmemBytes = kStages * kStageBytes + 1024;
};

struct SpanParams {
  AttnArgs a;           // pointers of the whole batch
  SpanPrefix prefix;    // requests == nullptr: window with first tokens
  int b0, nb;           // the slice of the batch
  int n_hb, ctas;       // head blocks, CTAs per head block
  int sms;
  int *counters;        // [Hkv][nb], zero between launches
  float *part_o;        // [share][2][Hq][128]
  float2 *part_ml;      // [share][2][Hq]
};

// Four rows per warp, eight lanes a row: maximum, sum and 16 columns of the accumulator, column groups k * 8 + (lane & 7)
// of four.
struct Rows {
  float m, l;
  float4 o[4];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // (without a branch: a batch of folds follows a batch of loads)
  __device__ __forceinline__ void fold(float2 ml, const float4 *v, bool live) {
    live = live && ml.y != 0.f;  // a partial that saw nothing has no meaning in v; one that saw NaN keeps it
    const float mn = live ? fmaxf(m, ml.x) : m;
    const float a = m == mn ? 1.f : fast_exp2(m - mn);  // m = -inf at first: 0
    const float w = live ? fast_exp2(ml.x - mn) : 0.f;
    m = mn;
    l = fmaf(l, a, live ? ml.y * w : 0.f);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      o[k].x = fmaf(o[k].x, a, live ? v[k].x * w : 0.f);
      o[k].y = fmaf(o[k].y, a, live ? v[k].y * w : 0.f);
      o[k].z = fmaf(o[k].z, a, live ? v[k].z * w : 0.f);
      o[k].w = fmaf(o[k].w, a, live ? v[k].w * w : 0.f);
    }
  }
};

// What of request b is streamed: pages [0, front) and [second, np) of its list.
struct Visible {
  int len, front, second, pages;
};
__device__ __forceinline__ Visible visible_part(const SpanParams &p, int b) {
  const AttnArgs &a = p.a;
  const int np = max(0, __ldg(a.kv_indptr + b + 1) - __ldg(a.kv_indptr + b));
  const int last = np > 0 ? min(max(__ldg(a.kv_last_page_len + b), 1), kPage) : 0;
  Visible v;
  v.len = np > 0 ? (np - 1) * kPage + last : 0;
  if (p.prefix.requests != nullptr) {
    v.front = 0;
    v.second = min(__ldg(&p.prefix.requests[b].x), np);
  } else {
    const int low = max(0, v.len - 1 - a.window_left);
    v.front = (min(a.first_tokens, v.len) + kPage - 1) / kPage;
    v.second = max(v.front, low / kPage);
  }
  v.pages = v.front + np - v.second;
  return v;
}

template <typename T, int HB, bool WIDE>
__global__ void __launch_bounds__(Shape<HB>::kThreads, Shape<HB>::kCtasPerSm)
    decode_span_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ SpanParams p) {
  constexpr int kThreads = Shape<HB>::kThreads, kStages = Shape<HB>::kStages, kStageBytes = Shape<HB>::kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ int sh_cost[kMaxSlice + 1];  // prefix sums of pages + kOpenCost
  __shared__ int sh_warp[kThreads / 32];
  // requests whose own pages a warp has finished, for the prefix's join: request * 128 + partial results to fold
  __shared__ unsigned short sh_closed[HB][kMaxSlice];
  __shared__ int sh_abort;

  const AttnArgs &a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hb = blockIdx.x % p.n_hb, c = blockIdx.x / p.n_hb;
  const int nb = p.nb;
  const uint32_t stage0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *stage0_ptr = smem_raw + (stage0 - smem_u32(smem_raw));

  if (tid == 0) {
    tma_prefetch_map(&tmap);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], HB);
    }
    sh_abort = 0;
    mbar_fence_init();
  }
  // ---- the line: visible pages of every request, scanned
  {
    const int per = (nb + kThreads - 1) / kThreads;  // consecutive requests per thread
    int sum = 0;
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < nb) {
        sum += visible_part(p, p.b0 + b).pages + kOpenCost;
        sh_cost[b + 1] = sum;  // relative to this thread's first
      }
    }
    int x = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) sh_warp[warp] = x;
    __syncthreads();
    int before = x - sum;
    for (int w = 0; w < warp; ++w) before += sh_warp[w];
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < nb) sh_cost[b + 1] += before;
    }
    if (tid == 0) sh_cost[0] = 0;
  }
  __syncthreads();
  const long long line = sh_cost[nb];
  // Beside the prefix kernel only the first CTAs find an SM: the line is divided among those.
  const int ctas = p.prefix.requests != nullptr && p.prefix.overlap
                       ? max(1, (int)((long long)p.ctas * __ldg(p.prefix.header + 3) / p.sms))
                       : p.ctas;
  const float part = __fdividef(kUnitsOfLine * (float)line, (float)nb);
  const unsigned units = max(kMinUnits, (int)(part * rsqrtf(part)));  // (approximate, and the same in every CTA)
  const long long shares = max(1, min(ctas, (int)((unsigned)line / units)));
  // share c is [line * c / shares, line * (c + 1) / shares); unit x lies in share ((x + 1) * shares - 1) / line
  const int x0 = c < shares ? (int)(line * c / shares) : (int)line;
  const int x1 = c < shares ? (int)(line * (c + 1) / shares) : (int)line;
  auto share_of = [&](int x) { return (int)((((long long)x + 1) * shares - 1) / line); };
  int b_first = 0;
  {
    int lo = 0, hi = nb;  // first b with sh_cost[b + 1] > x0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sh_cost[mid + 1] > x0)
        hi = mid;
      else
        lo = mid + 1;
    }
    b_first = lo;
  }
  // The pieces of this share: fn(request, first page, end page, pages of the request), pages counted along the
  // visible ones.  A request without visible pages is a piece of the share its opening cost starts in.
  auto for_pieces = [&](auto fn) {
    for (int b = b_first; b < nb && sh_cost[b] < x1; ++b) {
      const int at = sh_cost[b] + kOpenCost;
      const int pages = sh_cost[b + 1] - at;
      const int lo = min(max(x0 - at, 0), pages), hi = min(max(x1 - at, 0), pages);
      if (lo < hi || (pages == 0 && sh_cost[b] >= x0)) fn(b, lo, hi, pages);
    }
  };

  if (warp == HB) {
    // ------------------------------------------------------------------ producer
    int armed = 0;
    bool ok = true;
    for_pieces([&](int b, int lo, int hi, int) {
      const Visible r = visible_part(p, p.b0 + b);
      const int32_t *list = a.kv_indices + __ldg(a.kv_indptr + p.b0 + b);
      int base = lo - 32, id = 0;
      for (int v = lo; v < hi && ok; ++v) {
        if (v >= base + 32) {  // the next 32 page ids in one load
          base = v;
          const int vi = v + lane;
          id = vi < hi ? __ldg(list + (vi < r.front ? vi : vi - r.front + r.second)) : 0;
        }
        int page = __shfl_sync(0xffffffffu, id, v - base);
        if (page < 0 || page >= a.num_pages) {
          if (hb == 0 && lane == 0) report_error(a.err, PIEKV_ERR_PAGE_ID, KID_DECODE, p.b0 + b, page);
          page = a.num_pages;  // outside the tensor map: zeros
        }
        const int s = armed % kStages;
        if (*(volatile int *)&sh_abort || !mbar_wait(&empty_bar[s], ((armed / kStages) & 1) ^ 1)) {
          if (lane == 0 && atomicExch(&sh_abort, 1) == 0)
            report_error(a.err, PIEKV_ERR_WAIT_TIMEOUT, KID_DECODE, blockIdx.x, 500 + s);
          ok = false;
          break;
        }
        if (lane == 0) {
          mbar_arrive_expect_tx(&full_bar[s], (uint32_t)kStageBytes);
          tma_load_5d(stage0 + s * kStageBytes, &tmap, 0, 0, 0, hb * HB, page * 2, &full_bar[s]);
        }
        ++armed;
      }
    });
    // drain: the CTA must not retire while a bulk copy may still be landing
    __syncwarp();
    if (lane == 0)
      for (int x = armed > kStages ? armed - kStages : 0; x < armed; ++x)
        mbar_wait(&full_bar[x % kStages], (x / kStages) & 1, 200000000ull);
    if (p.prefix.requests != nullptr) asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }

  // -------------------------------------------------------------------- consumers: warp = kv head
  const int quad = lane >> 2, qlane = lane & 3;
  const int group = a.hq / a.hkv;
  const int hk = hb * HB + warp;
  const int head0 = hk * group;  // query heads head0 .. head0 + group - 1 are the MMA's rows
  const float scale_log2 = a.sm_scale * 1.4426950408889634f;
  T *out = reinterpret_cast<T *>(a.out);
  const bool prefixed = p.prefix.requests != nullptr;
  int it = 0;      // stages consumed
  int closed = 0;  // entries of sh_closed
  int pend_b[2] = {-1, -1};  // requests with a partial in this share's slots

  // A share's first request may have begun in an earlier share (slot 0); otherwise the piece that has to be joined is
  // the share's last one (slot 1).
  auto slot_base = [&](int share, bool first_piece) -> size_t {
    return ((size_t)share * 2 + (first_piece ? 1 : 0)) * a.hq + head0;
  };
  auto first_share = [&](int b) { return share_of(sh_cost[b] + kOpenCost); };
  auto last_share = [&](int b) { return share_of(sh_cost[b + 1] - 1); };
  auto has_prefix = [&](int b) { return prefixed && __ldg(&p.prefix.requests[p.b0 + b].x) > 0; };
  auto store_lse = [&](int b, int head, float m, float l) {
    if (a.lse != nullptr)
      a.lse[(size_t)(p.b0 + b) * a.hq + head] = l > 0.f ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  };
  for_pieces([&](int b, int lo, int hi, int pages) {
    const Visible seen_part = visible_part(p, p.b0 + b);
    const int len = seen_part.len, front = seen_part.front, second = seen_part.second;
    const int low = prefixed ? 0 : max(0, len - 1 - a.window_left);
    const int first = prefixed ? 0 : a.first_tokens;
    if (hk == 0 && lane == 0 && len > 0) {
      const int last = __ldg(a.kv_last_page_len + p.b0 + b);
      if (last < 1 || last > kPage) report_error(a.err, PIEKV_ERR_LAST_PAGE_LEN, KID_DECODE, p.b0 + b, last);
    }
    // query fragments of this warp's kv head (rows beyond the group are zero)
    uint32_t qa[8][4];
    {
      const T *qb = reinterpret_cast<const T *>(a.q) + (int64_t)(p.b0 + b) * a.q_sn + (int64_t)head0 * a.q_sh;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        const int col = ks * 16 + qlane * 2;
        const uint32_t *r0 = reinterpret_cast<const uint32_t *>(qb + (int64_t)quad * a.q_sh + col);
        const uint32_t *r1 = reinterpret_cast<const uint32_t *>(qb + (int64_t)(quad + 8) * a.q_sh + col);
        qa[ks][0] = quad < group ? __ldg(r0) : 0u;
        qa[ks][2] = quad < group ? __ldg(r0 + 4) : 0u;
        qa[ks][1] = WIDE && quad + 8 < group ? __ldg(r1) : 0u;
        qa[ks][3] = WIDE && quad + 8 < group ? __ldg(r1 + 4) : 0u;
      }
    }
    float o[16][4];
#pragma unroll
    for (int nt = 0; nt < 16; ++nt) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    for (int vi = lo; vi < hi; ++vi) {
      const int s = it % kStages;
      bool ok = *(volatile int *)&sh_abort == 0;
      if (ok && !mbar_wait(&full_bar[s], (it / kStages) & 1)) {
        if (lane == 0 && atomicExch(&sh_abort, 1) == 0)
          report_error(a.err, PIEKV_ERR_WAIT_TIMEOUT, KID_DECODE, blockIdx.x, 600 + s);
        ok = false;
      }
      ++it;
      if (ok) {
        const int t0 = (vi < front ? vi : vi - front + second) * kPage;
        const uint32_t ktile = stage0 + s * kStageBytes + warp * 4096, vtile = ktile + HB * 4096;
        // tokens of the page that are seen: below `first` or from `low` on, and inside the context
        uint32_t seen = 0xffffu >> (kPage - min(kPage, len - t0));
        seen &= ((1u << min(max(first - t0, 0), kPage)) - 1u) | (0xffffu << min(max(low - t0, 0), kPage));
        if (seen != 0xffffu) {
          // unseen rows may hold anything: zero their V so that 0 * garbage stays 0 (their scores are masked below)
          uint8_t *vptr = stage0_ptr + (vtile - stage0);
          for (int x = lane; x < kPage * 16; x += 32) {
            const int row = x >> 4;
            if (!((seen >> row) & 1u))
              *reinterpret_cast<uint4 *>(vptr + ((x >> 3) & 1) * 2048 + row * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();  // the stage is next written by a bulk copy
          __syncwarp();
        }
        // ---- S = Q K^T
        float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
        {
          const int mi = lane >> 3, r = lane & 7;
          const int t = (mi >> 1) * 8 + r;
#pragma unroll
          for (int ks = 0; ks < 8; ++ks) {
            const int ch = (ks & 3) * 2 + (mi & 1);
            uint32_t kb[4];
            ldmatrix_x4(kb, ktile + (ks >> 2) * 2048 + t * 128 + ((ch ^ r) << 4));
            mma_16816<T>(sc[0], qa[ks], kb[0], kb[1]);
            mma_16816<T>(sc[1], qa[ks], kb[2], kb[3]);
          }
        }
        // ---- online softmax (base 2); row `quad` (and quad + 8), tokens nt * 8 + qlane * 2 + {0, 1}
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool in = (seen >> (nt * 8 + qlane * 2 + e)) & 1u;
            sc[nt][e] = in ? sc[nt][e] * scale_log2 : -INFINITY;
            mx0 = fmaxf(mx0, sc[nt][e]);
            if (WIDE) {
              sc[nt][2 + e] = in ? sc[nt][2 + e] * scale_log2 : -INFINITY;
              mx1 = fmaxf(mx1, sc[nt][2 + e]);
            }
          }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        if (WIDE) {
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        }
        const float mn0 = fmaxf(m0, mx0), mn1 = WIDE ? fmaxf(m1, mx1) : 0.f;
        const float mu0 = mn0 == -INFINITY ? 0.f : mn0, mu1 = mn1 == -INFINITY ? 0.f : mn1;
        const float al0 = fast_exp2(m0 - mu0), al1 = WIDE ? fast_exp2(m1 - mu1) : al0;
        m0 = mn0;
        m1 = mn1;
        uint32_t pa[4];
        float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float p0 = fast_exp2(sc[nt][0] - mu0), p1 = fast_exp2(sc[nt][1] - mu0);
          ps0 += p0 + p1;
          pa[nt * 2] = pack2<T>(p0, p1);
          if (WIDE) {
            const float p2 = fast_exp2(sc[nt][2] - mu1), p3 = fast_exp2(sc[nt][3] - mu1);
            ps1 += p2 + p3;
            pa[nt * 2 + 1] = pack2<T>(p2, p3);
          } else {  // what the rounding dropped, in the row eight below
            const float2 kept = unpack2<T>(pa[nt * 2]);
            pa[nt * 2 + 1] = pack2<T>(p0 - kept.x, p1 - kept.y);
          }
        }
        l0 = l0 * al0 + ps0;
        l1 = l1 * al1 + ps1;
        if (__any_sync(0xffffffffu, al0 != 1.f || al1 != 1.f)) {
#pragma unroll
          for (int nt = 0; nt < 16; ++nt) {
            o[nt][0] *= al0;
            o[nt][1] *= al0;
            o[nt][2] *= al1;
            o[nt][3] *= al1;
          }
        }
        // ---- O += P V
        {
          const int mi = lane >> 3, r = lane & 7;
          const int t = (mi & 1) * 8 + r;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int ch = (i & 3) * 2 + (mi >> 1);
            uint32_t vb[4];
            ldmatrix_x4_trans(vb, vtile + (i >> 2) * 2048 + t * 128 + ((ch ^ r) << 4));
            mma_16816<T>(o[2 * i], pa, vb[0], vb[1]);
            mma_16816<T>(o[2 * i + 1], pa, vb[2], vb[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty_bar[s]);
    }

    // ================= the piece is done: its rows straight from the fragments
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
    l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (!WIDE) {
#pragma unroll
      for (int nt = 0; nt < 16; ++nt) {
        o[nt][0] += o[nt][2];
        o[nt][1] += o[nt][3];
      }
    }
    const bool whole = lo == 0 && hi == pages;
    const bool later = has_prefix(b);
    const int s_first = whole ? c : first_share(b);
    float *po;  // where partial rows go
    float2 *pml;
    if (whole) {
      const size_t at = (size_t)(p.b0 + b) * a.hq + head0;
      po = p.prefix.own_o + at * kDim;
      pml = p.prefix.own_ml + at;
    } else {
      const size_t at = slot_base(c, c == s_first);
      po = p.part_o + at * kDim;
      pml = p.part_ml + at;
    }
#pragma unroll
    for (int half = 0; half < (WIDE ? 2 : 1); ++half) {
      const int row = quad + half * 8;
      if (row < group) {
        const float m = half ? m1 : m0;
        float l = half ? l1 : l0;
        if (whole && !later) {
          l = add_sink(l, m, a.sinks, head0 + row);
          const float inv = l > 0.f ? 1.f / l : 0.f;
          uint32_t *orow = reinterpret_cast<uint32_t *>(out + ((size_t)(p.b0 + b) * a.hq + head0 + row) * kDim);
#pragma unroll
          for (int nt = 0; nt < 16; ++nt)
            orow[nt * 4 + qlane] = pack2<T>(o[nt][half * 2] * inv, o[nt][half * 2 + 1] * inv);
          if (qlane == 0) store_lse(b, head0 + row, m, l);
        } else {
          float4 *prow = reinterpret_cast<float4 *>(po + (size_t)row * kDim) + qlane * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            prow[i] = make_float4(o[2 * i][half * 2], o[2 * i][half * 2 + 1], o[2 * i + 1][half * 2], o[2 * i + 1][half * 2 + 1]);
          if (qlane == 0) pml[row] = make_float2(m, l);
        }
      }
    }
    if (!whole) {
      pend_b[c == s_first ? 1 : 0] = b;
    } else if (later) {
      if (lane == 0) sh_closed[warp][closed] = (unsigned short)(b * 128);
      ++closed;
    }
  });

  // ================= joins.  Steps 0 and 1: the requests with a partial in this share's slots, folded by the share that
  // arrives last.  Then, for what is behind a prefix, the prefix's results with the requests' own: waiting for them only
  // now keeps the pages streaming while the prefix kernel works.  One loop, so that this code exists once: on a short
  // call fetching instructions is most of its time.
#pragma unroll 1
  for (int x = 0;; ++x) {
    int b;
    bool later = false;
    if (x < 2) {
      b = x == 0 ? pend_b[0] : pend_b[1];
      if (b < 0) continue;
      int is_last = 0;
      __syncwarp();
      if (lane == 0) {
        __threadfence();
        int *counter = p.counters + hk * nb + b;
        is_last = atomicAdd(counter, 1) == last_share(b) - first_share(b);
        if (is_last) {
          *counter = 0;  // nobody else touches it in this launch
          __threadfence();
        }
      }
      if (!__shfl_sync(0xffffffffu, is_last, 0)) continue;
      later = has_prefix(b);
    } else {
      if (!prefixed) break;
      if (x == 2) {
        // how many partial results each request has, looked up while the prefix kernel may still be at work
        __syncwarp();
        const int problem = sprefix::problem_rows(group);
        for (int i = lane; i < closed; i += 32) {
          const int e = sh_closed[warp][i], request = p.b0 + (e >> 7);
          const sprefix::Group g = p.prefix.groups[__ldg(&p.prefix.requests[request].y)];
          const int block = (request - g.first) * group / (2 * problem);  // a request's rows lie in one block
          const sprefix::Segment &seg = p.prefix.segments[g.segment + block * a.hkv + hk];
          sh_closed[warp][i] = (unsigned short)(e + sprefix::partials_of(seg, problem, p.prefix.max_splits));
        }
        // (also without work: the launch must not end before the one it was allowed to overtake)
        asm volatile("griddepcontrol.wait;" ::: "memory");
        __syncwarp();
      }
      if (x - 2 >= closed) break;
      b = sh_closed[warp][x - 2] >> 7;
    }
    const size_t request = (size_t)(p.b0 + b) * a.hq + head0;
    // Row r's results: partial i of the share slots at `at` + max(2 i - 1, 0) * step + r; behind a prefix the own one
    // first (written above by this warp), then partial i - 1 of the prefix.
    const int n = x < 2 ? last_share(b) - first_share(b) + 1 : 1 + (sh_closed[warp][x - 2] & 127);
    const size_t at = x < 2 ? slot_base(first_share(b), true) : request;
    const size_t step = x < 2 ? (size_t)a.hq : (size_t)a.batch * a.hq;
    const float *po = x < 2 ? p.part_o : p.prefix.part_o, *po0 = x < 2 ? p.part_o : p.prefix.own_o;
    const float2 *pml = x < 2 ? p.part_ml : p.prefix.part_ml, *pml0 = x < 2 ? p.part_ml : p.prefix.own_ml;
#pragma unroll 1
    for (int r0 = 0; r0 < group; r0 += 4) {
      const int r = min(r0 + (lane >> 3), group - 1), sub = lane & 7;
      Rows acc;
      acc.clear();
#pragma unroll 1
      for (int i0 = 0; i0 < n; i0 += 4) {
        float2 ml[4];
        float4 v[4][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = min(i0 + j, n - 1);
          const size_t row = at + (size_t)max(x < 2 ? 2 * i - 1 : i - 1, 0) * step + r;
          ml[j] = ld_batch_cg((i == 0 ? pml0 : pml) + row);
          const float4 *src = reinterpret_cast<const float4 *>((i == 0 ? po0 : po) + row * kDim) + sub;
#pragma unroll
          for (int k = 0; k < 4; ++k) v[j][k] = ld_batch_cg(src + k * 8);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) acc.fold(ml[j], v[j], i0 + j < n);
      }
      if (r0 + (lane >> 3) < group) {
        if (later) {
#pragma unroll
          for (int k = 0; k < 4; ++k) *(reinterpret_cast<float4 *>(p.prefix.own_o + (request + r) * kDim) + k * 8 + sub) = acc.o[k];
          if (sub == 0) p.prefix.own_ml[request + r] = make_float2(acc.m, acc.l);
        } else {
          const float l = add_sink(acc.l, acc.m, a.sinks, head0 + r);
          const float inv = l > 0.f ? 1.f / l : 0.f;
          // fragment order: o[k] holds columns 16 sub + 2 k + {0, 1} and 16 sub + 8 + 2 k + {0, 1}
          uint32_t *row = reinterpret_cast<uint32_t *>(out + (request + r) * kDim) + sub * 8;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            row[k] = pack2<T>(acc.o[k].x * inv, acc.o[k].y * inv);
            row[4 + k] = pack2<T>(acc.o[k].z * inv, acc.o[k].w * inv);
          }
          if (sub == 0) store_lse(b, head0 + r, acc.m, l);
        }
      }
    }
    if (later) {
      if (lane == 0) sh_closed[warp][closed] = (unsigned short)(b * 128);
      ++closed;
    }
  }
}

template <typename T, int HB, bool WIDE>
int launch_t(const CUtensorMap &tm, const SpanParams &p, cudaStream_t st) {
  static unsigned char configured[kMaxDevices] = {0};
  if (int rc = opt_in_dynamic_smem(decode_span_kernel<T, HB, WIDE>, Shape<HB>::kSmemBytes, configured,
                                   "decode span: cudaFuncSetAttribute"))
    return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_hb * p.ctas));
  cfg.blockDim = dim3(Shape<HB>::kThreads);
  cfg.dynamicSmemBytes = Shape<HB>::kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // only behind the prefix kernel, which says when it may be overtaken and whose results are waited for
  cfg.numAttrs = p.prefix.requests != nullptr && p.prefix.overlap ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, decode_span_kernel<T, HB, WIDE>, tm, p);
  if (e != cudaSuccess) return cuda_status(e, "decode_span_kernel");
  return 0;
}

template <typename T>
int launch_h(int heads, bool wide, const CUtensorMap &tm, const SpanParams &p, cudaStream_t st) {
  if (heads == 2) return wide ? launch_t<T, 2, true>(tm, p, st) : launch_t<T, 2, false>(tm, p, st);
  return wide ? launch_t<T, 1, true>(tm, p, st) : launch_t<T, 1, false>(tm, p, st);
}

int heads_per_cta(int hkv) { return hkv % 2 == 0 ? 2 : 1; }
// shares of the line: CTAs of one head block
int shares_of(int hkv) {
  const int heads = heads_per_cta(hkv);
  const int n = (heads == 2 ? Shape<2>::kCtasPerSm : Shape<1>::kCtasPerSm) * sm_count() / (hkv / heads);
  return n > 1 ? n : 1;
}

}  // namespace

bool decode_span_supported(const AttnArgs &a, int dtype) {
  if (dtype != PIEKV_BF16 && dtype != PIEKV_F16) return false;
  if (a.dim != kDim || a.page_size != kPage) return false;
  if (a.hq % a.hkv != 0 || a.hq / a.hkv > 16) return false;
  if (a.hkv > kCounterBytes / 4) return false;
  if ((reinterpret_cast<uintptr_t>(a.pool) & 15) || (reinterpret_cast<uintptr_t>(a.q) & 3) ||
      (reinterpret_cast<uintptr_t>(a.out) & 3))
    return false;
  return !((a.q_sn & 1) || (a.q_sh & 1));
}

// Partials of a launch: two slots per share of the line, one row per query head.
int64_t decode_span_scratch_bytes(int hq, int hkv) {
  const int64_t rows = 2ll * shares_of(hkv) * hq;
  return (rows * 8 + 255) / 256 * 256 + rows * kDim * 4;
}

int launch_decode_span(const AttnArgs &a, int dtype, const SpanPrefix &prefix, void *workspace, int64_t workspace_bytes,
                       cudaStream_t st) {
  const int64_t need = kCounterBytes + decode_span_scratch_bytes(a.hq, a.hkv);
  PIEKV_REQUIRE(workspace != nullptr && workspace_bytes >= need, "decode: workspace too small (%lld < %lld bytes)",
                (long long)workspace_bytes, (long long)need);
  PIEKV_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 255) == 0, "decode: workspace must be 256-byte aligned");
  const int heads = heads_per_cta(a.hkv);
  SpanParams p;
  p.a = a;
  p.prefix = prefix;
  p.n_hb = a.hkv / heads;
  p.ctas = shares_of(a.hkv);
  p.sms = sm_count();
  uint8_t *ws = reinterpret_cast<uint8_t *>(workspace);
  p.counters = reinterpret_cast<int *>(ws);
  const int64_t rows = 2ll * p.ctas * a.hq;
  p.part_ml = reinterpret_cast<float2 *>(ws + kCounterBytes);
  p.part_o = reinterpret_cast<float *>(ws + kCounterBytes + (rows * 8 + 255) / 256 * 256);
  CUtensorMap tm;
  if (int rc = make_page_tensor_map(&tm, a.pool, a.num_pages, a.hkv, dtype, /*box_halves=*/2, /*box_heads=*/heads,
                                    /*box_kv=*/2))
    return rc;
  const int most = kCounterBytes / 4 / a.hkv;
  const int slice = most < kMaxSlice ? most : kMaxSlice;
  for (int b0 = 0; b0 < a.batch; b0 += slice) {
    p.b0 = b0;
    p.nb = a.batch - b0 < slice ? a.batch - b0 : slice;
    p.prefix.overlap = prefix.overlap && b0 == 0;
    const bool wide = a.hq / a.hkv > 8;
    const int rc = dtype == PIEKV_BF16 ? launch_h<__nv_bfloat16>(heads, wide, tm, p, st) : launch_h<__half>(heads, wide, tm, p, st);
    if (rc) return rc;
  }
  return 0;
}

}  // namespace piekv
