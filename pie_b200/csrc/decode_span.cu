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
// A request cut by a share's end leaves partials in the two slots a CTA owns; CTAs of a request are consecutive, so
// who holds a partial, and how many there are, follows from the line - there is no slot allocator, and results are
// reproducible bit for bit.  The last CTA to arrive (one counter per request and head block, left zero) folds them.
//
// Data path: a CTA takes HB kv heads of a page (HB = 4, 2 or 1, whichever divides), 4/HB pages per stage: 32 KiB by
// TMA into three stages, two CTAs per SM (192 KiB in flight per SM).  The producer warp and the consumers walk the
// same sequence independently; only barriers pass between them.  Consumer warp w owns tile (page w / HB, head
// w % HB): K and V [16 tokens x 128], 128-byte swizzled, as the m16n8k16 tensor-core fragments want them.
//
// Precision: a GQA group of up to 8 heads fills rows 0-7 of the 16-row MMA.  Rows 8-15 then carry the part of each
// probability that its 16-bit rounding drops, so P V is formed with 16 bits of P (bf16) at no extra MMA.
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
constexpr int kWarps = 4;  // consumer warps
constexpr int kConsumers = kWarps * 32;
constexpr int kThreads = kConsumers + 32;
constexpr int kStages = 3;
constexpr int kTileBytes = 8192;  // one (page, head): K 4 KiB + V 4 KiB
constexpr int kStageBytes = kWarps * kTileBytes;
constexpr int kSmemBytes = kStages * kStageBytes + 1024;
constexpr int kCtasPerSm = 2;
constexpr int kCounterBytes = 65536;
constexpr int kMaxSlice = 512;  // requests per launch: their page counts are kept in shared memory
constexpr int kOpenCost = 2;    // pages
constexpr int kMinUnits = 4;    // a share is not made smaller than this

struct SpanParams {
  AttnArgs a;           // pointers of the whole batch
  SpanPrefix prefix;    // requests == nullptr: window with first tokens
  int b0, nb;           // the slice of the batch
  int n_hb, ctas;       // head blocks, CTAs per head block
  int sms;
  int *counters;        // [n_hb][nb], zero between launches
  float *part_o;        // [n_hb * ctas][2][HB * group][128]
  float2 *part_ml;      // [n_hb * ctas][2][HB * group]
};

__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers) : "memory"); }

// (maximum, sum, 4 columns of the accumulator) of one row, and the fold of another partial into it
struct Row {
  float m, l;
  float4 o;
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // (without a branch: a batch of folds follows a batch of loads)
  __device__ __forceinline__ void fold(float2 ml, float4 v, bool live = true) {
    live = live && ml.y > 0.f;  // a partial that saw nothing has no meaning in v
    const float mn = live ? fmaxf(m, ml.x) : m;
    const float a = m == mn ? 1.f : fast_exp2(m - mn);  // m = -inf at first: 0
    const float w = live ? fast_exp2(ml.x - mn) : 0.f;
    m = mn;
    l = fmaf(l, a, live ? ml.y * w : 0.f);
    o.x = fmaf(o.x, a, live ? v.x * w : 0.f);
    o.y = fmaf(o.y, a, live ? v.y * w : 0.f);
    o.z = fmaf(o.z, a, live ? v.z * w : 0.f);
    o.w = fmaf(o.w, a, live ? v.w * w : 0.f);
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
__global__ void __launch_bounds__(kThreads, kCtasPerSm)
    decode_span_kernel(const __grid_constant__ CUtensorMap tmap, const __grid_constant__ SpanParams p) {
  constexpr int PG = kWarps / HB;  // pages per stage
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full_bar[kStages], empty_bar[kStages];
  __shared__ int sh_cost[kMaxSlice + 1];       // prefix sums of pages + kOpenCost
  __shared__ __align__(16) int4 sh_req[kMaxSlice];  // first list entry, length, front, second
  __shared__ int sh_warp[kThreads / 32];
  __shared__ float2 sh_ml[kWarps][16];
  __shared__ int sh_abort, sh_last;
  __shared__ short sh_closed[kMaxSlice];  // requests whose own pages this CTA has finished, for the prefix's join

  const AttnArgs &a = p.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hb = blockIdx.x % p.n_hb, c = blockIdx.x / p.n_hb;
  const int nb = p.nb;
  const uint32_t stage0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *stage0_ptr = smem_raw + (stage0 - smem_u32(smem_raw));

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], kWarps);
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
        const Visible v = visible_part(p, p.b0 + b);
        sh_req[b] = make_int4(__ldg(a.kv_indptr + p.b0 + b), v.len, v.front, v.second);
        sum += v.pages + kOpenCost;
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
  const long long shares = max(1ll, min((long long)ctas, line / kMinUnits));
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

  if (warp == kWarps) {
    // ------------------------------------------------------------------ producer
    int armed = 0;
    bool ok = true;
    for_pieces([&](int b, int lo, int hi, int) {
      const int4 r = sh_req[b];
      int base = lo - 32, id = 0;
      for (int v = lo; v < hi && ok; v += PG) {
        const int npg = min(PG, hi - v);
        if (v + npg > base + 32) {  // the next 32 page ids in one load
          base = v;
          const int vi = v + lane;
          id = vi < hi ? __ldg(a.kv_indices + r.x + (vi < r.z ? vi : vi - r.z + r.w)) : 0;
        }
        int page = __shfl_sync(0xffffffffu, id, (v - base + lane) & 31);
        if (lane < npg && (page < 0 || page >= a.num_pages)) {
          if (hb == 0) report_error(a.err, PIEKV_ERR_PAGE_ID, KID_DECODE, p.b0 + b, page);
          page = a.num_pages;  // outside the tensor map: zeros
        }
        const int s = armed % kStages;
        if (*(volatile int *)&sh_abort || !mbar_wait(&empty_bar[s], ((armed / kStages) & 1) ^ 1)) {
          if (lane == 0 && atomicExch(&sh_abort, 1) == 0)
            report_error(a.err, PIEKV_ERR_WAIT_TIMEOUT, KID_DECODE, blockIdx.x, 500 + s);
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(&full_bar[s], (uint32_t)(npg * HB * kTileBytes));
        __syncwarp();
        if (lane < npg)
          tma_load_5d(stage0 + s * kStageBytes + lane * (HB * kTileBytes), &tmap, 0, 0, 0, hb * HB, page * 2, &full_bar[s]);
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

  // -------------------------------------------------------------------- consumers
  const int pslot = warp / HB, h = warp % HB;
  const int quad = lane >> 2, qlane = lane & 3;
  const int group = a.hq / a.hkv;
  const int rows = HB * group;                // query heads of this head block: head0 .. head0 + rows
  const int head0 = hb * HB * group;
  const float scale_log2 = a.sm_scale * 1.4426950408889634f;
  T *out = reinterpret_cast<T *>(a.out);
  int it = 0;             // stages consumed
  int closed = 0;         // entries of sh_closed

  // A share's first request may have begun in an earlier share (slot 0); otherwise the piece that has to be joined is
  // the share's last one (slot 1).
  auto slot_base = [&](int share, bool first_piece) -> size_t {
    return ((size_t)(share * p.n_hb + hb) * 2 + (first_piece ? 1 : 0)) * rows;
  };
  auto store_row = [&](int b, int r, Row x) {
    const int head = head0 + r;
    const float l = add_sink(x.l, x.m, a.sinks, head);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    uint2 pk;
    pk.x = pack2<T>(x.o.x * inv, x.o.y * inv);
    pk.y = pack2<T>(x.o.z * inv, x.o.w * inv);
    const size_t at = (size_t)(p.b0 + b) * a.hq + head;
    *reinterpret_cast<uint2 *>(out + at * kDim + lane * 4) = pk;
    if (a.lse != nullptr && lane == 0) a.lse[at] = l > 0.f ? (x.m + log2f(l)) * 0.6931471805599453f : -INFINITY;
  };
  // Fold stored partials of rows r, r + 4, ... (HW of them, count[u] of each) into acc: partial i of row x is at
  // part(i, x).
  auto fold_rows = [&](auto hw, Row *acc, int r, const int *count, const float *po, const float2 *pml, auto part) {
    constexpr int HW = decltype(hw)::value;
    constexpr int PB = 16 / HW;  // loads of 16 partials are in flight before one is used
    int most = 0;
#pragma unroll
    for (int u = 0; u < HW; ++u) most = max(most, count[u]);
    for (int i0 = 0; i0 < most; i0 += PB) {
      float2 ml[PB][HW];
      float4 v[PB][HW];
#pragma unroll
      for (int j = 0; j < PB; ++j)
#pragma unroll
        for (int u = 0; u < HW; ++u) {
          const size_t at = part(max(min(i0 + j, count[u] - 1), 0), min(r + u * kWarps, rows - 1));
          ml[j][u] = ld_batch_cg(pml + at);
          v[j][u] = ld_batch_cg(reinterpret_cast<const float4 *>(po + at * kDim) + lane);
        }
#pragma unroll
      for (int j = 0; j < PB; ++j)
#pragma unroll
        for (int u = 0; u < HW; ++u)
          acc[u].fold(ml[j][u], v[j][u], i0 + j < count[u]);
    }
  };
  auto for_rows = [&](auto fn) {  // warp w: rows w, w + 4, ..., four at a time
    for (int r = warp; r < rows; r += 4 * kWarps) {
      const int left = (rows - r + kWarps - 1) / kWarps;
      if (left >= 3)
        fn(std::integral_constant<int, 4>{}, r);
      else if (left == 2)
        fn(std::integral_constant<int, 2>{}, r);
      else
        fn(std::integral_constant<int, 1>{}, r);
    }
  };
  // rows r, r + 4, ... of request b are complete, but for a prefix: out, or put by until the prefix's results are there
  auto finish_rows = [&](auto hw, const Row *acc, int r, int b, bool later) {
    constexpr int HW = decltype(hw)::value;
#pragma unroll
    for (int u = 0; u < HW; ++u) {
      const int row = r + u * kWarps;
      if (row >= rows) continue;
      if (!later) {
        store_row(b, row, acc[u]);
      } else {
        const size_t at = (size_t)(p.b0 + b) * a.hq + head0 + row;
        *(reinterpret_cast<float4 *>(p.prefix.own_o + at * kDim) + lane) = acc[u].o;
        if (lane == 0) p.prefix.own_ml[at] = make_float2(acc[u].m, acc[u].l);
      }
    }
  };
  auto has_prefix = [&](int b) { return p.prefix.requests != nullptr && __ldg(&p.prefix.requests[p.b0 + b].x) > 0; };
  // the prefix partials of request b into acc
  auto fold_prefix = [&](auto hw, Row *acc, int r, int b) {
    const int2 rq = __ldg(&p.prefix.requests[p.b0 + b]);
    const sprefix::Group g = p.prefix.groups[rq.y];
    const int member = p.b0 + b - g.first;
    constexpr int HW = decltype(hw)::value;
    int count[HW];
#pragma unroll
    for (int u = 0; u < HW; ++u)
      count[u] = sprefix::partials_of(g, member * group + min(r + u * kWarps, rows - 1) % group, group, p.prefix.max_splits);
    fold_rows(hw, acc, r, count, p.prefix.part_o, p.prefix.part_ml,
              [&](int i, int row) { return ((size_t)i * a.batch + p.b0 + b) * a.hq + head0 + row; });
  };

  for_pieces([&](int b, int lo, int hi, int pages) {
    const int4 rq = sh_req[b];
    const int len = rq.y, front = rq.z, second = rq.w;
    const bool prefix = p.prefix.requests != nullptr;
    const int low = prefix ? 0 : max(0, len - 1 - a.window_left);
    const int first = prefix ? 0 : a.first_tokens;
    if (warp == 0 && lane == 0 && len > 0) {
      const int last = __ldg(a.kv_last_page_len + p.b0 + b);
      if (last < 1 || last > kPage) report_error(a.err, PIEKV_ERR_LAST_PAGE_LEN, KID_DECODE, p.b0 + b, last);
    }
    // query fragments of this warp's kv head (rows beyond the group are zero)
    uint32_t qa[8][4];
    {
      const T *qb = reinterpret_cast<const T *>(a.q) + (int64_t)(p.b0 + b) * a.q_sn + (int64_t)(head0 + h * group) * a.q_sh;
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
    int s = 0;
    for (int v0 = lo; v0 < hi; v0 += PG) {
      s = it % kStages;
      bool ok = *(volatile int *)&sh_abort == 0;
      if (ok && !mbar_wait(&full_bar[s], (it / kStages) & 1)) {
        if (lane == 0 && atomicExch(&sh_abort, 1) == 0)
          report_error(a.err, PIEKV_ERR_WAIT_TIMEOUT, KID_DECODE, blockIdx.x, 600 + s);
        ok = false;
      }
      ++it;
      const int vi = v0 + pslot;
      if (ok && vi < hi) {
        const int t0 = (vi < front ? vi : vi - front + second) * kPage;
        const uint32_t page_base = stage0 + s * kStageBytes + pslot * (HB * kTileBytes);
        const uint32_t ktile = page_base + h * 4096, vtile = page_base + HB * 4096 + h * 4096;
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
          fence_proxy_async_smem();
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
      // the piece's last stage is kept a little longer: its tiles carry the warps' results below
      if (lane == 0 && v0 + PG < hi) mbar_arrive(&empty_bar[s]);
    }

    // ================= the piece is done: every warp puts its rows over its own tile of the last stage
    const bool any = lo < hi;
    if (any) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
      l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
      l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
      // float2 index within a 512-byte row, XORed with the row so that the eight rows of a store hit different banks
      uint8_t *kt = stage0_ptr + s * kStageBytes + pslot * (HB * kTileBytes) + h * 4096;
#pragma unroll
      for (int nt = 0; nt < 16; ++nt) {
        const int at = ((nt * 4 + qlane) ^ (quad << 2)) * 8 + quad * 512;
        if (WIDE) {
          *reinterpret_cast<float2 *>(kt + at) = make_float2(o[nt][0], o[nt][1]);
          *reinterpret_cast<float2 *>(kt + HB * 4096 + at) = make_float2(o[nt][2], o[nt][3]);
        } else {
          *reinterpret_cast<float2 *>(kt + at) = make_float2(o[nt][0] + o[nt][2], o[nt][1] + o[nt][3]);
        }
      }
      if (qlane == 0) {
        sh_ml[warp][quad] = make_float2(m0, l0);
        if (WIDE) sh_ml[warp][quad + 8] = make_float2(m1, l1);
      }
    }
    consumer_sync();
    const uint8_t *stage = stage0_ptr + s * kStageBytes;
    auto own_row = [&](int r) {  // this piece's row r: the warps of its head folded
      Row x;
      x.clear();
      if (any) {
        const int hh = r / group, q = r - hh * group;
#pragma unroll
        for (int ps = 0; ps < PG; ++ps)
          x.fold(sh_ml[ps * HB + hh][q],
                 *reinterpret_cast<const float4 *>(stage + ps * (HB * kTileBytes) + hh * 4096 + (q >> 3) * (HB * 4096) +
                                                   (q & 7) * 512 + ((lane * 2) ^ ((q & 7) << 2)) * 8));
      }
      return x;
    };
    const bool whole = lo == 0 && hi == pages;
    const int s_first = whole ? c : share_of(sh_cost[b] + kOpenCost);
    const bool later = has_prefix(b);
    if (whole) {
      for_rows([&](auto hw, int r) {
        constexpr int HW = decltype(hw)::value;
        Row acc[HW];
#pragma unroll
        for (int u = 0; u < HW; ++u) acc[u] = own_row(min(r + u * kWarps, rows - 1));
        finish_rows(hw, acc, r, b, later);
      });
    } else {
      const size_t base = slot_base(c, c == s_first);
      for (int r = warp; r < rows; r += kWarps) {
        const Row x = own_row(r);
        *(reinterpret_cast<float4 *>(p.part_o + (base + r) * kDim) + lane) = x.o;
        if (lane == 0) p.part_ml[base + r] = make_float2(x.m, x.l);
      }
    }
    fence_proxy_async_smem();  // these tiles are next written by bulk copies
    consumer_sync();
    if (any && lane == 0) mbar_arrive(&empty_bar[s]);
    if (!whole) {
      // ================= partials: the last share of the request to arrive folds them all
      const int n = share_of(sh_cost[b + 1] - 1) - s_first + 1;
      if (tid == 0) {
        __threadfence();
        int *counter = p.counters + hb * nb + b;
        const int old = atomicAdd(counter, 1);
        sh_last = old + 1 == n ? 1 : 0;
        if (sh_last) {
          *counter = 0;  // nobody else touches it in this launch
          __threadfence();
        }
      }
      consumer_sync();
      if (sh_last == 0) return;
      for_rows([&](auto hw, int r) {
        constexpr int HW = decltype(hw)::value;
        Row acc[HW];
        int count[HW];
#pragma unroll
        for (int u = 0; u < HW; ++u) {
          acc[u].clear();
          count[u] = n;
        }
        fold_rows(hw, acc, r, count, p.part_o, p.part_ml, [&](int i, int row) { return slot_base(s_first + i, i == 0) + row; });
        finish_rows(hw, acc, r, b, later);
      });
    }
    if (later) {
      if (tid == 0) sh_closed[closed] = (short)b;
      ++closed;
    }
  });
  if (p.prefix.requests == nullptr) return;
  // ================= the prefix's results, folded with the requests' own.  Waiting only now keeps the pages streaming
  // while the prefix kernel works; the launch must not end before that kernel in any case.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  consumer_sync();
  for (int x = 0; x < closed; ++x) {
    const int b = sh_closed[x];
    for_rows([&](auto hw, int r) {
      constexpr int HW = decltype(hw)::value;
      Row acc[HW];
      float2 ml[HW];
#pragma unroll
      for (int u = 0; u < HW; ++u) {  // written above by this very warp
        const size_t at = (size_t)(p.b0 + b) * a.hq + head0 + min(r + u * kWarps, rows - 1);
        ml[u] = ld_batch_cg(p.prefix.own_ml + at);
        acc[u].o = ld_batch_cg(reinterpret_cast<const float4 *>(p.prefix.own_o + at * kDim) + lane);
      }
#pragma unroll
      for (int u = 0; u < HW; ++u) {
        acc[u].m = ml[u].x;
        acc[u].l = ml[u].y;
      }
      fold_prefix(hw, acc, r, b);
      finish_rows(hw, acc, r, b, false);
    });
  }
}

template <typename T, int HB, bool WIDE>
int launch_t(const CUtensorMap &tm, const SpanParams &p, cudaStream_t st) {
  static unsigned char configured[kMaxDevices] = {0};
  if (int rc = opt_in_dynamic_smem(decode_span_kernel<T, HB, WIDE>, kSmemBytes, configured, "decode span: cudaFuncSetAttribute"))
    return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(p.n_hb * p.ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
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
  if (heads == 4) return wide ? launch_t<T, 4, true>(tm, p, st) : launch_t<T, 4, false>(tm, p, st);
  if (heads == 2) return wide ? launch_t<T, 2, true>(tm, p, st) : launch_t<T, 2, false>(tm, p, st);
  return wide ? launch_t<T, 1, true>(tm, p, st) : launch_t<T, 1, false>(tm, p, st);
}

int heads_per_cta(int hkv) { return hkv % 4 == 0 ? 4 : (hkv % 2 == 0 ? 2 : 1); }
int ctas_per_head_block(int hkv) {
  const int n = kCtasPerSm * sm_count() / (hkv / heads_per_cta(hkv));
  return n > 1 ? n : 1;
}

}  // namespace

bool decode_span_supported(const AttnArgs &a, int dtype) {
  if (dtype != PIEKV_BF16 && dtype != PIEKV_F16) return false;
  if (a.dim != kDim || a.page_size != kPage) return false;
  if (a.hq % a.hkv != 0 || a.hq / a.hkv > 16) return false;
  if (a.hkv / heads_per_cta(a.hkv) > kCounterBytes / 4) return false;
  if ((reinterpret_cast<uintptr_t>(a.pool) & 15) || (reinterpret_cast<uintptr_t>(a.q) & 3) ||
      (reinterpret_cast<uintptr_t>(a.out) & 7))
    return false;
  return !((a.q_sn & 1) || (a.q_sh & 1));
}

// Partials of a launch: two slots per CTA, one row per query head of its head block.
int64_t decode_span_scratch_bytes(int hq, int hkv) {
  const int64_t rows = 2ll * ctas_per_head_block(hkv) * hq;
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
  p.ctas = ctas_per_head_block(a.hkv);
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
  const int most = kCounterBytes / 4 / p.n_hb;
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
