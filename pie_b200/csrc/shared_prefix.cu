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
// A prefix shorter than this is left to the requests.  Measured (32 / 8 heads, bf16, up to 64 tokens of their own, in a
// graph), 3 pages left and 4 read once: one group of 4 requests 11.0 and 9.6 us, of 64 13.3 and 13.9, 16 groups of 4 12.8
// and 13.3.  Many small groups pay for the joins until the prefix is longer: 64 groups of 2, 3 pages left 19.0, 8 read once
// 33.6 (the plain decode call 25.6), 32 pages 41.7 (42.7), 128 pages 105 (128).
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

// Costs in units of 0.3 us, as measured on the two attention kernels.  Prefix kernel: starting it, a tile against one
// problem's rows (bound by its stream) or two (by the tensor and special-function pipes), an item's own costs.  The
// other kernel: starting it beside the prefix kernel or behind it, a tile's worth of own pages; a warp's step of the join
// (four rows, four partial results), of which an SM has kFoldWarps under way.  Two kernels that stream at the same time
// slow each other down by up to kContention.  Every thread walks all groups: 8 us for one group, 20 for 16, 57 for 64, 203 for
// 256 (match and plan, in a graph).
constexpr float kStartPrefix = 16.f, kTileSingle = 5.f, kTilePair = 7.5f, kOpenItem = 6.f;
constexpr float kStartBeside = 24.f, kStartBehind = 90.f, kOwnTile = 6.f, kFoldStep = 4.5f, kFoldWarps = 8.f, kContention = 0.3f;
constexpr int kMaxSearchGroups = 256;

// Checks the grouping, decides what every group reads once, how many CTAs work on that while the other SMs stream the
// requests' own pages, and into how many items each prefix is cut; CTAs claim items.  One block.
//
// More CTAs on the prefixes leave fewer SMs to the other kernel, which runs at the same time; more items balance the
// CTAs (not all SMs are equally fast under this load: by a third on some parts) but leave more partial results to fold.
// Each thread costs one (CTAs, tiles per item) pair with the constants above; the cheapest is taken.
__global__ void __launch_bounds__(1024) sp_plan_kernel(const int32_t *__restrict__ kv_indptr,
                                                       const int32_t *__restrict__ group_indptr, int batch, int groups,
                                                       int page_size, int heads_per_kv, int hkv, int max_splits,
                                                       int sms, PlanView v, int32_t *err) {
  __shared__ unsigned long long sh_own, sh_best;
  __shared__ int sh_scan[32], sh_carry, sh_most, sh_used, sh_items;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    sh_own = 0;
    sh_best = ~0ull;
    sh_carry = sh_most = sh_used = sh_items = 0;
    for (int i = 0; i < 6; ++i) v.header[i] = 0;
    v.header[3] = sms;
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
    return;
  }
  const int problem = problem_rows(heads_per_kv), block_members = 2 * problem / heads_per_kv;
  auto tiles_of = [&](int pages) { return (int)(((long long)pages * page_size + kTileTokens - 1) / kTileTokens); };
  auto blocks_of = [&](int members) { return (members + block_members - 1) / block_members; };
  // whether the last block is one problem
  auto last_single = [&](int members) {
    const int left = members % block_members;
    return left > 0 && left * heads_per_kv <= problem ? 1 : 0;
  };
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
        atomicMax(&sh_most, tiles_of(pages));
        atomicAdd(&sh_used, 1);
      }
    }
  }
  __syncthreads();
  // ---- segments, numbered in the groups' order
  for (int g0 = 0; g0 < groups; g0 += 1024) {
    const int g = g0 + tid;
    const int own = g < groups && v.groups[g].pages > 0 ? blocks_of(v.groups[g].members) * hkv : 0;
    int x = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) sh_scan[warp] = x;
    __syncthreads();
    for (int w = 0; w < warp; ++w) x += sh_scan[w];
    x += sh_carry;
    if (g < groups) v.groups[g].segment = x - own;
    __syncthreads();
    if (tid == 1023) sh_carry = x;
    __syncthreads();
  }
  const int segments = sh_carry;
  if (segments == 0) return;
  // ---- thread = (CTAs: 32 steps up to all SMs, tiles per item: the longest prefix in 1 .. 32 pieces)
  const int most = sh_most, max_pieces = max(1, max_splits / 2);
  auto pieces_of = [&](int tiles, int per) { return min((tiles + per - 1) / per, max_pieces); };
  int ctas = max(1, sms * (warp + 1) / 32), per = (most + lane) / (lane + 1);
  if (groups <= kMaxSearchGroups) {
    const float row_steps = (float)((heads_per_kv + 3) / 4);
    float work = 0.f, folds = 0.f, longest = 0.f, longest_fold = 0.f;
    long long items = 0;
    for (int g = 0; g < groups; ++g) {
      const Group gr = v.groups[g];
      if (gr.pages == 0) continue;
      const int tiles = tiles_of(gr.pages), pieces = pieces_of(tiles, per), blocks = blocks_of(gr.members);
      const int single = last_single(gr.members);
      // join steps of a request: its own result and the prefix's
      const int members_single = single ? gr.members % block_members : 0;
      const float fold = row_steps * (float)((pieces + 4) / 4);
      const float fold_single = row_steps * (float)(((max_splits >= 2 ? 2 : 1) * pieces + 4) / 4);
      items += (long long)blocks * pieces;
      work += (float)tiles * ((float)(blocks - single) * kTilePair + (float)single * kTileSingle);
      folds += (float)(gr.members - members_single) * fold + (float)members_single * fold_single;
      longest_fold = fmaxf(longest_fold, single ? fold_single : fold);
      longest = fmaxf(longest, (float)tiles / (float)pieces * (blocks > single ? kTilePair : kTileSingle));
    }
    if (items * hkv <= segments + kSpareItems) {
      const int n = (int)min((long long)ctas, items * hkv), left = n < sms ? sms - n : sms;
      const float own = (n < sms ? kStartBeside : kStartBehind) +
                        (float)((double)sh_own * page_size / kTileTokens * hkv) * kOwnTile / (float)left;
      float prefix = (work + (float)items * kOpenItem) * (float)hkv / (float)n;
      // claimed items end within one item of each other; fewer items than CTAs: one each
      prefix = items * hkv <= n ? longest + kOpenItem : prefix + 0.5f * (longest + kOpenItem);
      if (n < sms) prefix *= 1.f + kContention * fminf(1.f, own / prefix);
      prefix += kStartPrefix;
      const float cost = (n < sms ? fmaxf(prefix, own) : prefix + own) +
                         kFoldStep * fmaxf(longest_fold, folds * (float)hkv / ((float)left * kFoldWarps));
      atomicMin(&sh_best, ((unsigned long long)__float_as_uint(cost) << 32) | (unsigned)tid);
    }
  }
  __syncthreads();
  // No search for more groups: all SMs, whole prefixes.  For groups alike that costs a little (groups of 2 behind 512 tokens: 256
  // 116 us, 257 129); one long prefix among them is then one item per kv head (16384 tokens, the others 128: 87 and 203 us, the
  // plain decode call 83 and 89).
  const int best = sh_best == ~0ull ? 31 * 32 : (int)(sh_best & 1023);
  ctas = max(1, sms * (best / 32 + 1) / 32);
  per = (most + best % 32) / (best % 32 + 1);
  for (int g = warp; g < groups; g += 32) {
    const Group gr = v.groups[g];
    if (gr.pages == 0) continue;
    const int blocks = blocks_of(gr.members), tiles = tiles_of(gr.pages), n = blocks * hkv;
    int pieces = pieces_of(tiles, per), at = 0;
    if (lane == 0) at = atomicAdd(&sh_items, n * pieces);
    at = __shfl_sync(0xffffffffu, at, 0);
    if (at + n * pieces > v.max_segments + kSpareItems) {  // (cannot happen: nothing is written out of range)
      if (lane == 0) report_error(err, PIEKV_ERR_PAGE_CAPACITY, KID_SHARED_PREFIX, g, pieces);
      pieces = 0;
    }
    const int list = kv_indptr[gr.first];
    for (int i = lane; i < max(n, n * pieces); i += 32) {
      const int piece = i / n, segment = i % n, block = segment / hkv;
      const int request = gr.first + block * block_members, rows = (gr.members - block * block_members) * heads_per_kv;
      if (piece == 0) v.segments[gr.segment + segment] = Segment{rows, pieces};
      if (piece < pieces)
        v.items[at + i] = Item{request, list, gr.pages, segment % hkv, rows, (int)((long long)tiles * piece / pieces),
                               (int)((long long)tiles * (piece + 1) / pieces), piece};
    }
  }
  __syncthreads();
  if (tid == 0) {
    const int items = min(sh_items, v.max_segments + kSpareItems);
    v.header[0] = min(ctas, items);
    v.header[1] = sh_used;
    v.header[2] = items;
    v.header[3] = v.header[0] < sms ? sms - v.header[0] : sms;
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
  const PlanView v = plan_view(a.plan, a.batch, a.num_groups, a.num_qo_heads, a.num_kv_heads);
  cudaStream_t st = (cudaStream_t)stream;
  sp_match_kernel<<<a.batch, 128, 0, st>>>(a.kv_indptr, a.kv_indices, a.kv_last_page_len, a.group_indptr, a.batch,
                                           a.num_groups, a.page_size, v.match);
  PIEKV_LAUNCH_CHECK("sp_match_kernel");
  const int group = a.num_qo_heads / a.num_kv_heads;  // (more than 16 heads run the general kernel, which needs no items)
  sp_plan_kernel<<<1, 1024, 0, st>>>(a.kv_indptr, a.group_indptr, a.batch, a.num_groups, a.page_size,
                                     group < 16 ? group : 16, a.num_kv_heads, a.max_splits, sm_count(), v, a.err);
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
  // the prefix kernel brings query rows in by TMA, and takes the maximum of a row before it scales it
  const bool rows16 = (reinterpret_cast<uintptr_t>(a.q) & 15) == 0 && (a.q_sn & 7) == 0 && (a.q_sh & 7) == 0 &&
                      a.q_sn > 0 && a.q_sh > 0;
  if (!decode_span_supported(a, args->dtype) || !rows16 || !(a.sm_scale > 0.f))
    return launch_attn_generic(a, args->dtype, st);
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
  px.header = v.header;
  px.items = v.items;
  px.part_ml = reinterpret_cast<float2 *>(ws);
  px.part_o = reinterpret_cast<float *>(ws + prefix_ml_bytes(a.batch, a.hq, args->max_splits));
  px.batch = a.batch;
  px.hq = a.hq;
  px.group = a.hq / a.hkv;
  px.problem = problem_rows(px.group);
  px.num_pages = a.num_pages;
  px.max_splits = args->max_splits;
  px.scale_log2 = a.sm_scale * 1.4426950408889634f;
  px.err = a.err;
  const WorkspaceTurn turn(args->workspace);
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
