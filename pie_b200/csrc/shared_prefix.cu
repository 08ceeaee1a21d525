// Decode attention for groups of requests that share the leading pages of their contexts.
#include "attn.cuh"
#include "common.cuh"
#include "decode_span.cuh"
#include "prefix_tc.cuh"
#include "shared_prefix.cuh"

namespace piekv {

using namespace sprefix;

namespace {

constexpr int64_t kCounterBytes = 65536;
// A prefix shorter than this is left to the requests: reading it once saves less than joining two parts costs.
constexpr int kMinSharedPages = 4;

// Full pages of request b (the partly filled last page of a fork is a copy of its own).
__device__ __forceinline__ int full_pages(const int32_t *kv_indptr, const int32_t *last, int b, int page_size) {
  const int np = kv_indptr[b + 1] - kv_indptr[b];
  return np <= 0 ? 0 : (last[b] >= page_size ? np : np - 1);
}

// How many leading full pages request b has in common with its group's first request.  One block per request.
__global__ void __launch_bounds__(128) sp_match_kernel(const int32_t *__restrict__ kv_indptr,
                                                       const int32_t *__restrict__ kv_indices,
                                                       const int32_t *__restrict__ last,
                                                       const int32_t *__restrict__ group_indptr, int batch, int groups,
                                                       int page_size, int *match) {
  __shared__ int sh_first;
  const int b = blockIdx.x;
  int lo = 0, hi = groups - 1;  // first g with group_indptr[g + 1] > b
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (group_indptr[mid + 1] > b)
      hi = mid;
    else
      lo = mid + 1;
  }
  const int leader = min(max(group_indptr[lo], 0), batch - 1);  // (a bad grouping is refused by the plan kernel)
  const int n = min(full_pages(kv_indptr, last, b, page_size), full_pages(kv_indptr, last, leader, page_size));
  const int32_t *x = kv_indices + kv_indptr[b], *y = kv_indices + kv_indptr[leader];
  if (threadIdx.x == 0) sh_first = n;
  __syncthreads();
  if (b != leader) {
    for (int base = 0; base < n; base += 4 * 128) {
      int bad = n;
#pragma unroll
      for (int u = 3; u >= 0; --u) {
        const int j = base + u * 128 + threadIdx.x;
        if (j < n && x[j] != y[j]) bad = j;
      }
      if (__syncthreads_or(bad < n)) {
        if (bad < n) atomicMin(&sh_first, bad);
        break;
      }
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) match[b] = sh_first;
}

// The line that the CTAs' shares divide, in units of 0.3 us as measured on the prefix kernel: a tile against at most 128
// rows (bound by its stream) or more (by the tensor and special-function pipes), and opening and closing a piece.
constexpr int kTileSingle = 5, kTilePair = 8, kOpen = 22;
// The same units for the choice of how many SMs work on prefixes: starting that kernel, starting the other one beside it
// or behind it, a tile's worth of own pages there, and one row of partial results folded by an SM.  Two kernels that
// stream at the same time slow each other down by up to kContention.
constexpr float kStartPrefix = 16.f, kStartBeside = 24.f, kStartBehind = 90.f, kOwnTile = 6.f, kFoldRow = 0.03f;
constexpr float kContention = 0.3f;

// Checks the grouping, decides what every group reads once, how many SMs work on that while the others stream the
// requests' own pages, and where each CTA's share of the prefixes starts.  One block.
//
// More CTAs on the prefixes leave fewer SMs to the other kernel, which runs at the same time, and cut them into more
// pieces, whose partial results have to be folded.  Thread x costs x + 1 CTAs with the constants above; the cheapest
// is taken.  Shares are equal parts of the line, so no CTA has more than its part whatever the prefixes' lengths.
__global__ void __launch_bounds__(1024) sp_plan_kernel(const int32_t *__restrict__ kv_indptr,
                                                       const int32_t *__restrict__ group_indptr, int batch, int groups,
                                                       int page_size, int heads_per_kv, int hkv, int max_splits,
                                                       int sms, PlanView v, int32_t *err) {
  __shared__ unsigned long long sh_own, sh_best, sh_longest, sh_rows, sh_row_len;
  __shared__ long long sh_scan[32][2], sh_carry[2];
  __shared__ int sh_used;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    sh_own = sh_longest = sh_rows = sh_row_len = 0;
    sh_best = ~0ull;
    sh_used = 0;
    sh_carry[0] = sh_carry[1] = 0;
  }
  int bad = -1;
  for (int g = tid; g < groups; g += 1024) {
    const int a = group_indptr[g], e = group_indptr[g + 1];
    if (a > e || a < 0 || e > batch || (g == 0 && a != 0) || (g == groups - 1 && e != batch)) bad = g;
  }
  if (bad >= 0) report_error(err, PIEKV_ERR_INDPTR, KID_SHARED_PREFIX, bad, group_indptr[bad]);
  const bool refused = __syncthreads_or(bad >= 0) != 0;
  if (refused) {  // every request on its own
    for (int b = tid; b < batch; b += 1024) v.requests[b] = make_int2(0, 0);
    for (int c = tid; c <= sms; c += 1024) v.starts[c] = make_int2(0, 0);
    if (tid == 0) {
      v.header[0] = v.header[1] = v.header[2] = 0;
      v.header[3] = sms;
    }
    return;
  }
  auto tiles_of = [&](int pages) { return (int)(((long long)pages * page_size + kTileTokens - 1) / kTileTokens); };
  // blocks of more than 128 rows, and whether a smaller one is left
  auto pair_blocks = [&](int members) { return (int)(((long long)members * heads_per_kv + kRowsPerBlock / 2 - 1) / kRowsPerBlock); };
  auto single_blocks = [&](int members) {
    const int left = (int)((long long)members * heads_per_kv % kRowsPerBlock);
    return left > 0 && left <= kRowsPerBlock / 2 ? 1 : 0;
  };
  auto length = [&](int tiles, bool pair) { return (long long)tiles * (pair ? kTilePair : kTileSingle) + kOpen; };
  // ---- a warp per group: pages common to all its requests, pages left to each
  for (int g = warp; g < groups; g += 32) {
    const int a = group_indptr[g], m = group_indptr[g + 1] - a;
    int pages = 1 << 30;
    long long own = 0;
    for (int i = lane; i < m; i += 32) {
      pages = min(pages, v.match[a + i]);
      own += max(0, kv_indptr[a + i + 1] - kv_indptr[a + i]);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      pages = min(pages, __shfl_xor_sync(0xffffffffu, pages, d));
      own += __shfl_xor_sync(0xffffffffu, own, d);
    }
    if (m < 2 || pages < kMinSharedPages) pages = 0;
    for (int i = lane; i < m; i += 32) v.requests[a + i] = make_int2(pages, g);
    if (lane == 0) {
      v.groups[g] = Group{a, m, pages, 0};
      atomicAdd(&sh_own, (unsigned long long)(own - (long long)m * pages));
      if (pages > 0) {
        const int tiles = tiles_of(pages), pb = pair_blocks(m), sb = single_blocks(m);
        const long long rows_single = sb ? (long long)m * heads_per_kv - (long long)pb * kRowsPerBlock : 0;
        const long long rows_pair = (long long)m * heads_per_kv - rows_single;
        atomicMax(&sh_longest, (unsigned long long)length(tiles, pb > 0));
        atomicAdd(&sh_rows, (unsigned long long)(rows_pair + 2 * rows_single));
        atomicAdd(&sh_row_len, (unsigned long long)(rows_pair * length(tiles, true) + 2 * rows_single * length(tiles, false)));
        atomicAdd(&sh_used, 1);
      }
    }
  }
  __syncthreads();
  // ---- the line: segments and lengths of the groups, scanned in order
  for (int g0 = 0; g0 < groups; g0 += 1024) {
    const int g = g0 + tid;
    long long x[2] = {0, 0};
    if (g < groups && v.groups[g].pages > 0) {
      const Group gr = v.groups[g];
      const int tiles = tiles_of(gr.pages), pb = pair_blocks(gr.members), sb = single_blocks(gr.members);
      x[0] = (long long)(pb + sb) * hkv;
      x[1] = hkv * (pb * length(tiles, true) + sb * length(tiles, false));
    }
    const long long own[2] = {x[0], x[1]};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x[k], d);
        if (lane >= d) x[k] += y;
      }
      if (lane == 31) sh_scan[warp][k] = x[k];
    }
    __syncthreads();
    for (int k = 0; k < 2; ++k) {
      for (int w = 0; w < warp; ++w) x[k] += sh_scan[w][k];
      x[k] += sh_carry[k];
    }
    if (g < groups) {
      v.groups[g].segment = (int)(x[0] - own[0]);
      v.line[g] = x[1] - own[1];
    }
    __syncthreads();
    if (tid == 1023) {
      sh_carry[0] = x[0];
      sh_carry[1] = x[1];
    }
    __syncthreads();
  }
  const long long line = sh_carry[1];
  const int segments = (int)sh_carry[0];
  if (line == 0) {
    for (int c = tid; c <= sms; c += 1024) v.starts[c] = make_int2(0, 0);
    if (tid == 0) {
      v.header[0] = v.header[1] = v.header[2] = 0;
      v.header[3] = sms;
    }
    return;
  }
  // ---- how many CTAs.  A share holds a tile at least; no segment is cut into more pieces than there is room for.
  const int max_pieces = max(1, max_splits / 2);
  const bool cut = max_pieces >= 3;
  long long most = min((long long)sms, max(1ll, line / (kOpen + kTilePair)));
  if (cut) most = max(1ll, min(most, (max_pieces - 2) * line / (long long)sh_longest));
  if (tid < (int)most) {
    const int n = tid + 1, left = n < sms ? sms - n : sms;
    const float own = (n < sms ? kStartBeside : kStartBehind) +
                      (float)((double)sh_own * page_size / kTileTokens * hkv) * kOwnTile / (float)left;
    // a share that starts inside a segment opens one piece more than the line counts, one that is not an even part of
    // the segments (or a whole number of them) two
    const bool even = n % segments == 0 || segments % n == 0;
    float prefix = fmaxf((float)line / (float)n, cut ? 0.f : (float)sh_longest) + (even ? kOpen : 2 * kOpen);
    if (n < sms) prefix *= 1.f + kContention * fminf(1.f, own / prefix);
    prefix += kStartPrefix;
    const float fold = kFoldRow * (float)hkv / (float)left * ((float)sh_rows + (cut ? (float)sh_row_len * (float)n / (float)line : 0.f));
    const float cost = (n < sms ? fmaxf(prefix, own) : prefix + own) + fold;
    atomicMin(&sh_best, ((unsigned long long)__float_as_uint(cost) << 32) | (unsigned)tid);
  }
  __syncthreads();
  const int ctas = (int)(sh_best & 0xffffffffu) + 1;
  auto share_of = [&](long long x) { return (int)(((x + 1) * ctas - 1) / line); };
  for (int g = warp; g < groups; g += 32) {
    const Group gr = v.groups[g];
    if (gr.pages == 0) continue;
    const int pb = pair_blocks(gr.members), blocks = pb + single_blocks(gr.members), tiles = tiles_of(gr.pages);
    for (int i = lane; i < blocks * hkv; i += 32) {
      const int block = i / hkv;
      const bool pair = block < pb;
      const long long at = v.line[g] + min(i, pb * hkv) * length(tiles, true) + max(0, i - pb * hkv) * length(tiles, false);
      const int first = cut ? share_of(at + kOpen) : 0;
      const int last = cut ? share_of(at + kOpen + (long long)(tiles - 1) * (pair ? kTilePair : kTileSingle)) : 0;
      v.segments[gr.segment + i] = Segment{gr.first, kv_indptr[gr.first], gr.pages, i % hkv, block * kRowsPerBlock,
                                           gr.members * heads_per_kv - block * kRowsPerBlock, first, last - first + 1};
    }
  }
  for (int c = tid; c <= sms; c += 1024) {  // (CTAs behind the last share start where they end)
    const long long x = c < ctas ? line * c / ctas : 0;
    int lo = 0, hi = groups - 1;  // last group whose start is <= x (of equal starts the one with a prefix: the last)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (v.line[mid] <= x)
        lo = mid;
      else
        hi = mid - 1;
    }
    int2 start = make_int2(segments, 0);
    if (c < ctas) {
      const Group gr = v.groups[lo];
      const int tiles = tiles_of(gr.pages);
      const long long in_pairs = (long long)pair_blocks(gr.members) * hkv * length(tiles, true);
      long long y = x - v.line[lo];
      int seg = gr.segment;
      const bool pair = y < in_pairs;
      if (!pair) {
        seg += pair_blocks(gr.members) * hkv;
        y -= in_pairs;
      }
      seg += (int)(y / length(tiles, pair));
      y %= length(tiles, pair);
      const int step = pair ? kTilePair : kTileSingle;
      // tiles whose first unit lies before x belong to the share before
      int tile = y <= kOpen ? 0 : (int)((y - kOpen + step - 1) / step);
      if (!cut) tile = y > 0 ? tiles : 0;
      if (tile >= tiles) {
        ++seg;
        tile = 0;
      }
      start = make_int2(seg, tile);
    }
    v.starts[c] = start;
  }
  if (tid == 0) {
    v.header[0] = ctas;
    v.header[1] = sh_used;
    v.header[2] = segments;
    v.header[3] = ctas < sms ? sms - ctas : sms;
  }
}

int check_args(const piekv_shared_prefix_args *a, const char *who) {
  PIEKV_REQUIRE(a != nullptr, "%s: null arguments", who);
  PIEKV_REQUIRE(a->dtype >= PIEKV_F32 && a->dtype <= PIEKV_BF16, "%s: unknown dtype %d", who, a->dtype);
  PIEKV_REQUIRE(a->batch >= 0 && a->num_groups >= 0, "%s: negative batch / num_groups", who);
  PIEKV_REQUIRE(a->num_qo_heads > 0 && a->num_kv_heads > 0 && a->num_qo_heads % a->num_kv_heads == 0,
                "%s: num_qo_heads %d not a multiple of num_kv_heads %d", who, a->num_qo_heads, a->num_kv_heads);
  PIEKV_REQUIRE(a->head_dim > 0 && a->page_size > 0, "%s: bad head_dim / page_size", who);
  PIEKV_REQUIRE(a->max_splits >= 1 && a->max_splits <= PIEKV_SHARED_PREFIX_MAX_SPLITS, "%s: max_splits %d not in 1..%d", who,
                a->max_splits, PIEKV_SHARED_PREFIX_MAX_SPLITS);
  if (a->batch == 0) return 0;
  PIEKV_REQUIRE(a->num_groups > 0, "%s: no groups for %d requests", who, a->batch);
  PIEKV_REQUIRE(a->kv_indptr && a->kv_indices && a->kv_last_page_len && a->group_indptr, "%s: null pointer", who);
  const int64_t need = piekv_shared_prefix_plan_bytes(a->batch, a->num_groups, a->num_qo_heads, a->num_kv_heads);
  PIEKV_REQUIRE(a->plan != nullptr && a->plan_bytes >= need, "%s: plan too small (%lld < %lld bytes)", who,
                (long long)a->plan_bytes, (long long)need);
  PIEKV_REQUIRE((reinterpret_cast<uintptr_t>(a->plan) & 255) == 0, "%s: plan must be 256-byte aligned", who);
  return 0;
}

}  // namespace
}  // namespace piekv

using namespace piekv;

extern "C" int64_t piekv_shared_prefix_plan_bytes(int32_t batch, int32_t num_groups, int32_t num_qo_heads,
                                                  int32_t num_kv_heads) {
  if (batch < 0 || num_groups < 0 || num_qo_heads <= 0 || num_kv_heads <= 0) return 0;
  return plan_view(nullptr, batch, num_groups, num_qo_heads, num_kv_heads).bytes;
}

// Partials: max_splits of the prefix and one of the request's own pages per (request, query head).
static int64_t prefix_ml_bytes(int batch, int hq, int max_splits) {
  return (((int64_t)max_splits + 1) * batch * hq * 8 + 255) / 256 * 256;
}

extern "C" int64_t piekv_shared_prefix_workspace_bytes(int32_t batch, int32_t num_qo_heads, int32_t num_kv_heads,
                                                       int32_t head_dim, int32_t max_splits) {
  if (batch < 0 || num_qo_heads <= 0 || num_kv_heads <= 0 || max_splits < 1) return 0;
  if (head_dim != 128) return kCounterBytes;
  return kCounterBytes + (decode_span_scratch_bytes(num_qo_heads, num_kv_heads) + 255) / 256 * 256 +
         prefix_ml_bytes(batch, num_qo_heads, max_splits) + ((int64_t)max_splits + 1) * batch * num_qo_heads * 128 * 4;
}

extern "C" int piekv_shared_prefix_plan(const piekv_shared_prefix_args *args, void *stream) {
  if (int rc = check_args(args, "shared_prefix_plan")) return rc;
  const piekv_shared_prefix_args &a = *args;
  if (a.batch == 0) return 0;
  PIEKV_REQUIRE(sm_count() <= kMaxCtas, "shared_prefix_plan: %d SMs, the plan holds %d shares", sm_count(), kMaxCtas);
  const PlanView v = plan_view(a.plan, a.batch, a.num_groups, a.num_qo_heads, a.num_kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
  sp_match_kernel<<<a.batch, 128, 0, st>>>(a.kv_indptr, a.kv_indices, a.kv_last_page_len, a.group_indptr, a.batch,
                                           a.num_groups, a.page_size, v.match);
  PIEKV_LAUNCH_CHECK("sp_match_kernel");
  sp_plan_kernel<<<1, 1024, 0, st>>>(a.kv_indptr, a.group_indptr, a.batch, a.num_groups, a.page_size,
                                     a.num_qo_heads / a.num_kv_heads, a.num_kv_heads, a.max_splits, sm_count(), v, a.err);
  PIEKV_LAUNCH_CHECK("sp_plan_kernel");
  return 0;
}

extern "C" int piekv_shared_prefix_run(const piekv_shared_prefix_args *args, void *stream) {
  if (int rc = check_args(args, "shared_prefix_run")) return rc;
  if (args->batch == 0) return 0;
  PIEKV_REQUIRE(args->num_pages > 0, "shared_prefix_run: bad num_pages");
  PIEKV_REQUIRE(args->q && args->pool && args->out, "shared_prefix_run: null pointer");
  AttnArgs a{};
  a.q = args->q;
  a.q_sn = args->q_stride_n;
  a.q_sh = args->q_stride_h;
  a.pool = args->pool;
  a.out = args->out;
  a.lse = args->lse;
  a.kv_indptr = args->kv_indptr;
  a.kv_indices = args->kv_indices;
  a.kv_last_page_len = args->kv_last_page_len;
  a.batch = a.nnz = args->batch;
  a.hq = args->num_qo_heads;
  a.hkv = args->num_kv_heads;
  a.dim = args->head_dim;
  a.page_size = args->page_size;
  a.num_pages = args->num_pages;
  a.sm_scale = args->sm_scale;
  a.err = args->err;
  a.sinks = args->sinks;
  cudaStream_t st = (cudaStream_t)stream;
  // a thread of the prefix kernel brings a query row in by 16-byte loads
  const bool rows16 = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.q_sn & 7) == 0 && (a.q_sh & 7) == 0;
  if (!decode_span_supported(a, args->dtype) || !rows16) return launch_attn_generic(a, args->dtype, st);
  const int64_t need = piekv_shared_prefix_workspace_bytes(a.batch, a.hq, a.hkv, a.dim, args->max_splits);
  PIEKV_REQUIRE(args->workspace != nullptr && args->workspace_bytes >= need,
                "shared_prefix_run: workspace too small (%lld < %lld bytes)", (long long)args->workspace_bytes,
                (long long)need);
  PIEKV_REQUIRE((reinterpret_cast<uintptr_t>(args->workspace) & 255) == 0,
                "shared_prefix_run: workspace must be 256-byte aligned");
  const PlanView v = plan_view(args->plan, a.batch, args->num_groups, a.hq, a.hkv);
  uint8_t *ws = reinterpret_cast<uint8_t *>(args->workspace) + kCounterBytes +
                (decode_span_scratch_bytes(a.hq, a.hkv) + 255) / 256 * 256;
  PrefixTcParams px{};
  px.q = a.q;
  px.q_sn = a.q_sn;
  px.q_sh = a.q_sh;
  px.kv_indices = a.kv_indices;
  px.starts = v.starts;
  px.segments = v.segments;
  px.part_ml = reinterpret_cast<float2 *>(ws);
  px.part_o = reinterpret_cast<float *>(ws + prefix_ml_bytes(a.batch, a.hq, args->max_splits));
  px.batch = a.batch;
  px.hq = a.hq;
  px.group = a.hq / a.hkv;
  px.num_pages = a.num_pages;
  px.max_splits = args->max_splits;
  px.scale_log2 = a.sm_scale * 1.4426950408889634f;
  px.err = a.err;
  if (int rc = launch_prefix_tc(px, a.pool, a.hkv, args->dtype, st)) return rc;
  SpanPrefix sp;
  sp.requests = v.requests;
  sp.header = v.header;
  sp.groups = v.groups;
  sp.segments = v.segments;
  sp.part_o = px.part_o;
  sp.part_ml = px.part_ml;
  sp.own_o = px.part_o + (int64_t)args->max_splits * a.batch * a.hq * 128;
  sp.own_ml = px.part_ml + (int64_t)args->max_splits * a.batch * a.hq;
  sp.max_splits = args->max_splits;
  sp.overlap = 1;
  return launch_decode_span(a, args->dtype, sp, args->workspace, args->workspace_bytes, st);
}
