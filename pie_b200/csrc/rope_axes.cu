// Rotary positions on several axes (time, height, width of an image or a video), with the append into the
// paged cache.
//
// Pair i of a head row turns by the angle pos[axis(i)] * f_i.  Both factors are kept as fractions of a turn in
// 64-bit fixed point: F_i = f_i / (2 pi) * 2^64, and pos * F_i modulo 2^64 IS the angle modulo a turn, exactly,
// for every 32-bit position (an fp32 product of position and frequency is off by 0.01 rad at position 2^18).
// The nearest quarter turn is taken off as an integer, the rest (|r| <= 1/8 turn) goes through sincospif.
// x' = x c - y s, y' = x s + y c with separately rounded products and sums, one rounding to the storage type,
// as the one-axis kernels do (rope.cuh).
//
// What bounds it: HBM.  Per token (2 Hq + 4 Hkv) D elements move, and nothing is read twice.
#include <math.h>

#include "common.cuh"
#include "rope.cuh"

namespace piekv {
namespace {

struct AxesParams {
  const void *q, *k, *v;
  void *q_out, *k_out, *pool;
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, qo_sn, qo_sh, ko_sn, ko_sh;
  const int32_t *pos;
  int64_t pos_stride;
  const int32_t *batch_indices, *positions, *kv_indices, *kv_indptr;
  int32_t *err;
  int nnz, batch, hq, hkv, dim, page_size, num_pages;
  piekv_rope_axes_table t;
};

// cos / sin of pair `pr` of token `tok`; false when the position is outside the table
__device__ __forceinline__ bool pair_cos_sin(const AxesParams &p, int tok, int pr, float &c, float &s) {
  const int pos = __ldg(p.pos + (int64_t)p.t.axis[pr] * p.pos_stride + tok);
  if (p.t.cos_sin_table != nullptr) {
    if (pos < 0 || pos >= p.t.table_len) {
      report_error(p.err, PIEKV_ERR_TABLE_RANGE, KID_ROPE_AXES, tok, pos);
      c = 1.f;
      s = 0.f;
      return false;
    }
    const float *row = p.t.cos_sin_table + (size_t)pos * (2 * p.t.half);
    c = __ldg(row + pr);
    s = __ldg(row + p.t.half + pr);
    return true;
  }
  const uint64_t t = (uint64_t)(int64_t)pos * p.t.turn[pr];
  const uint32_t quarter = (uint32_t)((t + (1ull << 61)) >> 62);
  const int32_t rest = (int32_t)(uint32_t)((t - ((uint64_t)quarter << 62)) >> 32);  // in [-2^29, 2^29): turns * 2^32
  float s0, c0;
  sincospif((float)rest * 4.656612873077393e-10f, &s0, &c0);  // * 2^-31: half turns
  const bool swap = quarter & 1;
  c = swap ? s0 : c0;
  s = swap ? c0 : s0;
  if (quarter == 1 || quarter == 2) c = -c;
  if (quarter & 2) s = -s;
  return true;
}

// The K row of a token in the pool (V half_page elements behind it); nullptr with the error recorded when the
// token's request, slot or page does not exist.
template <typename T>
__device__ __forceinline__ T *pool_row(const AxesParams &p, int tok) {
  const int b = __ldg(p.batch_indices + tok), pos = __ldg(p.positions + tok);
  if (b < 0 || b >= p.batch) {
    report_error(p.err, PIEKV_ERR_BATCH_INDEX, KID_ROPE_AXES, tok, b);
    return nullptr;
  }
  const int p0 = __ldg(p.kv_indptr + b), p1 = __ldg(p.kv_indptr + b + 1);
  const int slot = pos >= 0 ? pos / p.page_size : -1;
  if (slot < 0 || slot >= p1 - p0) {
    report_error(p.err, PIEKV_ERR_PAGE_SLOT, KID_ROPE_AXES, tok, pos);
    return nullptr;
  }
  const int page = __ldg(p.kv_indices + p0 + slot);
  if (page < 0 || page >= p.num_pages) {
    report_error(p.err, PIEKV_ERR_PAGE_ID, KID_ROPE_AXES, tok, page);
    return nullptr;
  }
  const size_t half_page = (size_t)p.page_size * p.hkv * p.dim;
  return reinterpret_cast<T *>(p.pool) + (size_t)page * 2 * half_page + (size_t)(pos % p.page_size) * p.hkv * p.dim;
}

// Any shape: a block per token, a thread per pair or element.
template <typename T>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ AxesParams p) {
  __shared__ float2 sh_cs[kMaxHalfDim];
  __shared__ T *sh_row;
  const int tok = blockIdx.x;
  const int D = p.dim, half = p.t.half;
  if (threadIdx.x == 0) sh_row = p.pool != nullptr ? pool_row<T>(p, tok) : nullptr;
  for (int pr = threadIdx.x; pr < half; pr += blockDim.x) pair_cos_sin(p, tok, pr, sh_cs[pr].x, sh_cs[pr].y);
  __syncthreads();
  T *krow = sh_row;
  const int q_heads = p.q != nullptr ? p.hq : 0;
  const int units = D - half;  // per head: `half` pairs, then the elements behind the rotary width
  for (int x = threadIdx.x; x < (q_heads + p.hkv) * units; x += blockDim.x) {
    const int h = x / units, u = x - h * units;
    const T *src;
    T *d0 = nullptr, *d1 = nullptr;
    if (h < q_heads) {
      src = reinterpret_cast<const T *>(p.q) + (int64_t)tok * p.q_sn + (int64_t)h * p.q_sh;
      d0 = reinterpret_cast<T *>(p.q_out) + (int64_t)tok * p.qo_sn + (int64_t)h * p.qo_sh;
    } else {
      const int hk = h - q_heads;
      src = reinterpret_cast<const T *>(p.k) + (int64_t)tok * p.k_sn + (int64_t)hk * p.k_sh;
      if (krow != nullptr) d0 = krow + (size_t)hk * D;
      if (p.k_out != nullptr) d1 = reinterpret_cast<T *>(p.k_out) + (int64_t)tok * p.ko_sn + (int64_t)hk * p.ko_sh;
    }
    if (u >= half) {
      const int e = half + u;
      const T val = src[e];
      if (d0) d0[e] = val;
      if (d1) d1[e] = val;
      continue;
    }
    const int e0 = p.t.interleave ? 2 * u : u, e1 = p.t.interleave ? 2 * u + 1 : u + half;
    float a, b;
    rope_rotate(Elem<T>::to_f32(src[e0]), Elem<T>::to_f32(src[e1]), sh_cs[u].x, sh_cs[u].y, a, b);
    const T ta = Elem<T>::from_f32(a), tb = Elem<T>::from_f32(b);
    if (d0) {
      d0[e0] = ta;
      d0[e1] = tb;
    }
    if (d1) {
      d1[e0] = ta;
      d1[e1] = tb;
    }
  }
  if (krow == nullptr) return;
  T *vrow = krow + (size_t)p.page_size * p.hkv * D;
  for (int x = threadIdx.x; x < p.hkv * D; x += blockDim.x) {
    const int h = x / D, e = x - h * D;
    vrow[x] = reinterpret_cast<const T *>(p.v)[(int64_t)tok * p.v_sn + (int64_t)h * p.v_sh + e];
  }
}

template <typename T>
int launch_axes(const AxesParams &p, cudaStream_t st) {
  rope_axes_kernel<T><<<p.nnz, 256, 0, st>>>(p);
  PIEKV_LAUNCH_CHECK("rope_axes_kernel");
  return 0;
}

}  // namespace
}  // namespace piekv

using namespace piekv;

extern "C" int piekv_rope_axes_prepare(const piekv_rope_params *rope, const int32_t *sections, int32_t num_axes,
                                       int32_t cyclic, piekv_rope_axes_table *table) {
  const char *who = "rope_axes_prepare";
  PIEKV_REQUIRE(rope != nullptr && sections != nullptr && table != nullptr, "%s: null arguments", who);
  PIEKV_REQUIRE(num_axes >= 1 && num_axes <= PIEKV_MAX_ROPE_AXES, "%s: num_axes %d not in 1..%d", who, num_axes,
                PIEKV_MAX_ROPE_AXES);
  int half = 0;
  for (int i = 0; i < num_axes; ++i) {
    PIEKV_REQUIRE(sections[i] >= 0 && sections[i] <= kMaxHalfDim, "%s: section %d holds %d pairs", who, i, sections[i]);
    half += sections[i];
  }
  PIEKV_REQUIRE(half > 0 && half <= kMaxHalfDim, "%s: sections of %d pairs (1..%d)", who, half, kMaxHalfDim);
  if (cyclic)
    for (int i = 1; i < num_axes; ++i)
      PIEKV_REQUIRE(sections[i] == 0 || i + num_axes * (sections[i] - 1) < half,
                    "%s: %d pairs of axis %d dealt out in turn do not fit %d pairs", who, sections[i], i, half);
  PIEKV_REQUIRE(rope->mode == PIEKV_ROPE_PLAIN || rope->mode == PIEKV_ROPE_LLAMA31 || rope->mode == PIEKV_ROPE_TABLE,
                "%s: rope mode %d (plain, llama31 or table)", who, rope->mode);
  if (int rc = check_rope(rope, 2 * half, who)) return rc;
  memset(table, 0, sizeof(*table));
  table->half = half;
  table->num_axes = num_axes;
  table->interleave = rope->interleave ? 1 : 0;
  int first = 0;  // first pair of the block
  for (int ax = 0; ax < num_axes; ++ax) {
    if (cyclic) {
      if (ax == 0) continue;  // axis 0 has what the others leave
      for (int n = 0; n < sections[ax]; ++n) table->axis[ax + n * num_axes] = (uint8_t)ax;
    } else {
      for (int n = 0; n < sections[ax]; ++n) table->axis[first + n] = (uint8_t)ax;
      first += sections[ax];
    }
  }
  if (rope->mode == PIEKV_ROPE_TABLE) {
    table->cos_sin_table = rope->cos_sin_table;
    table->table_len = rope->table_len;
    return 0;
  }
  const double two_pi = 6.283185307179586476925286766559;
  for (int i = 0; i < half; ++i) {
    double turns = pair_frequency(rope, 2 * half, i) / two_pi;
    turns -= floor(turns);
    // both factors below 2^53 are exact in double; the product's integer part is the fixed-point fraction
    const double high = floor(turns * 4294967296.0);
    const double low = floor((turns * 4294967296.0 - high) * 4294967296.0);
    table->turn[i] = ((uint64_t)high << 32) + (uint64_t)low;
  }
  return 0;
}

extern "C" int piekv_rope_axes(const piekv_rope_axes_args *args, const piekv_rope_axes_table *table, void *stream) {
  const char *who = "rope_axes";
  PIEKV_REQUIRE(args != nullptr && table != nullptr, "%s: null arguments", who);
  const piekv_rope_axes_args &a = *args;
  PIEKV_REQUIRE(a.dtype >= PIEKV_F32 && a.dtype <= PIEKV_BF16, "%s: unknown dtype %d", who, a.dtype);
  PIEKV_REQUIRE(a.nnz >= 0 && a.num_kv_heads > 0 && (a.q == nullptr || a.num_qo_heads > 0), "%s: bad sizes", who);
  PIEKV_REQUIRE(a.head_dim > 0 && a.head_dim <= 2 * kMaxHalfDim, "%s: head_dim %d not in 1..%d", who, a.head_dim,
                2 * kMaxHalfDim);
  PIEKV_REQUIRE(table->half > 0 && 2 * table->half <= a.head_dim, "%s: sections of %d pairs do not fit head_dim %d", who,
                table->half, a.head_dim);
  PIEKV_REQUIRE(table->num_axes >= 1 && table->num_axes <= PIEKV_MAX_ROPE_AXES, "%s: the table is not prepared", who);
  if (a.nnz == 0) return 0;
  PIEKV_REQUIRE(a.k && a.pos, "%s: null pointer", who);
  PIEKV_REQUIRE(a.q == nullptr || a.q_out != nullptr, "%s: q without q_out", who);
  PIEKV_REQUIRE(a.pool != nullptr || a.k_out != nullptr, "%s: rotated k has nowhere to go (no pool, no k_out)", who);
  if (a.pool != nullptr) {
    PIEKV_REQUIRE(a.v && a.batch_indices && a.positions && a.kv_indices && a.kv_indptr, "%s: null pointer", who);
    PIEKV_REQUIRE(a.batch >= 0 && a.page_size > 0 && a.num_pages > 0, "%s: bad batch / page_size / num_pages", who);
  }
  AxesParams p{};
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  p.q_out = a.q_out;
  p.k_out = a.k_out;
  p.pool = a.pool;
  p.q_sn = a.q_stride_n;
  p.q_sh = a.q_stride_h;
  p.k_sn = a.k_stride_n;
  p.k_sh = a.k_stride_h;
  p.v_sn = a.v_stride_n;
  p.v_sh = a.v_stride_h;
  p.qo_sn = a.q_out_stride_n;
  p.qo_sh = a.q_out_stride_h;
  p.ko_sn = a.k_out_stride_n;
  p.ko_sh = a.k_out_stride_h;
  p.pos = a.pos;
  p.pos_stride = a.pos_stride;
  p.batch_indices = a.batch_indices;
  p.positions = a.positions;
  p.kv_indices = a.kv_indices;
  p.kv_indptr = a.kv_indptr;
  p.err = a.err;
  p.nnz = a.nnz;
  p.batch = a.batch;
  p.hq = a.num_qo_heads;
  p.hkv = a.num_kv_heads;
  p.dim = a.head_dim;
  p.page_size = a.page_size > 0 ? a.page_size : 1;
  p.num_pages = a.num_pages;
  p.t = *table;
  cudaStream_t st = (cudaStream_t)stream;
  if (a.dtype == PIEKV_F32) return launch_axes<float>(p, st);
  if (a.dtype == PIEKV_F16) return launch_axes<__half>(p, st);
  return launch_axes<__nv_bfloat16>(p, st);
}
