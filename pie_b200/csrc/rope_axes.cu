// Rotary positions on several axes (time, height, width of an image or a video), with the append into the
// paged cache.
//
// Pair i of a head row turns by the angle pos[axis(i)] * f_i, kept as a fraction of a turn in 64-bit fixed point:
// F_i = f_i / (2 pi) * 2^64, and pos * F_i modulo 2^64 is the angle modulo a turn, without a rounding of its own (an fp32
// product of position and frequency is off by 0.01 rad at position 2^18).  F_i itself comes from a double, within 2^-51
// of itself: the angle is off by up to |pos| * 2^-53 turn, less than the 2^-32 turn that are kept of it up to position
// 2^21, 2^-22 turn (1.5e-6 rad) at position 2^31.
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

// cos / sin of pair `pr` (frequency `turn`) of token `tok` at position `pos`
__device__ __forceinline__ void pair_cos_sin(const AxesParams &p, int tok, int pos, int pr, uint64_t turn, float &c, float &s) {
  if (p.t.cos_sin_table != nullptr) {
    if (pos < 0 || pos >= p.t.table_len) {
      report_error(p.err, PIEKV_ERR_TABLE_RANGE, KID_ROPE_AXES, tok, pos);
      c = 1.f;
      s = 0.f;
      return;
    }
    const float *row = p.t.cos_sin_table + (size_t)pos * (2 * p.t.half);
    c = __ldg(row + pr);
    s = __ldg(row + p.t.half + pr);
    return;
  }
  const uint64_t t = (uint64_t)(int64_t)pos * turn;
  const uint32_t quarter = (uint32_t)((t + (1ull << 61)) >> 62);
  const int32_t rest = (int32_t)(uint32_t)((t - ((uint64_t)quarter << 62)) >> 32);  // in [-2^29, 2^29): turns * 2^32
  float s0, c0;
  sincospif((float)rest * 4.656612873077393e-10f, &s0, &c0);  // * 2^-31: half turns
  const bool swap = quarter & 1;
  c = swap ? s0 : c0;
  s = swap ? c0 : s0;
  if (quarter == 1 || quarter == 2) c = -c;
  if (quarter & 2) s = -s;
}
__device__ __forceinline__ void pair_cos_sin(const AxesParams &p, int tok, int pr, float &c, float &s) {
  pair_cos_sin(p, tok, __ldg(p.pos + (int64_t)p.t.axis[pr] * p.pos_stride + tok), pr, p.t.turn[pr], c, s);
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

// Whole head rows in 16-byte pieces.  A thread owns VEC pairs of one token (two pieces of a row: its halves, or
// neighbours when pairs are interleaved), forms their cos and sin once and keeps them in registers while it walks the
// heads blockIdx.y gives it, q before k before v: no (cos, sin) is formed twice, nothing goes through shared memory.
// kUnits rows are loaded before the first is stored.
constexpr int kUnits = 2;
constexpr int kThreads = 256;
constexpr int kThreadsPerSm = 1024;

template <typename T, bool kNeighbours>
__global__ void __launch_bounds__(kThreads, 3) rope_axes_rows_kernel(const __grid_constant__ AxesParams p, int heads_per_slice) {
  constexpr int VEC = 16 / sizeof(T);
  const int tok = blockIdx.x * blockDim.y + threadIdx.y;
  if (tok >= p.nnz) return;
  const int half = p.t.half;
  const int ch = threadIdx.x;
  const int e0 = kNeighbours ? 2 * ch * VEC : ch * VEC, e1 = kNeighbours ? e0 + VEC : e0 + half;
  const int q_heads = p.q != nullptr ? p.hq : 0, k_end = q_heads + p.hkv, heads = k_end + (p.pool != nullptr ? p.hkv : 0);
  const int h0 = blockIdx.y * heads_per_slice, h1 = min(heads, h0 + heads_per_slice);
  const T *q = reinterpret_cast<const T *>(p.q) + (int64_t)tok * p.q_sn;
  const T *k = reinterpret_cast<const T *>(p.k) + (int64_t)tok * p.k_sn;
  const T *v = reinterpret_cast<const T *>(p.v) + (int64_t)tok * p.v_sn;
  float c[VEC], s[VEC];
  T *krow = nullptr;
  bool ready = false;
  for (int h = h0; h < h1; h += kUnits) {
    uint4 lo[kUnits], hi[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int hh = h + u;
      if (hh < h1) {
        const T *src = hh < q_heads ? q + (int64_t)hh * p.q_sh
                                    : (hh < k_end ? k + (int64_t)(hh - q_heads) * p.k_sh : v + (int64_t)(hh - k_end) * p.v_sh);
        lo[u] = ld_batch(src + e0);
        hi[u] = ld_batch(src + e1);
      }
    }
    if (!ready) {  // while the first rows are on their way
      if (h0 < k_end) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) pair_cos_sin(p, tok, ch * VEC + j, c[j], s[j]);
      }
      if (p.pool != nullptr && h1 > q_heads) krow = pool_row<T>(p, tok);
      ready = true;
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
      const int hh = h + u;
      if (hh >= h1) break;
      if (hh < k_end) {
        T *a = reinterpret_cast<T *>(&lo[u]), *b = reinterpret_cast<T *>(&hi[u]);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          // pair j: (a[j], b[j]) of the row's halves, or neighbours 2j, 2j + 1 of the two pieces in order
          T &x = kNeighbours ? (2 * j < VEC ? a[2 * j] : b[2 * j - VEC]) : a[j];
          T &y = kNeighbours ? (2 * j < VEC ? a[2 * j + 1] : b[2 * j + 1 - VEC]) : b[j];
          float xo, yo;
          rope_rotate(Elem<T>::to_f32(x), Elem<T>::to_f32(y), c[j], s[j], xo, yo);
          x = Elem<T>::from_f32(xo);
          y = Elem<T>::from_f32(yo);
        }
      }
      T *d0 = nullptr, *d1 = nullptr;
      if (hh < q_heads) {
        d0 = reinterpret_cast<T *>(p.q_out) + (int64_t)tok * p.qo_sn + (int64_t)hh * p.qo_sh;
      } else if (hh < k_end) {
        const int hk = hh - q_heads;
        if (krow != nullptr) d0 = krow + (size_t)hk * p.dim;
        if (p.k_out != nullptr) d1 = reinterpret_cast<T *>(p.k_out) + (int64_t)tok * p.ko_sn + (int64_t)hk * p.ko_sh;
      } else if (krow != nullptr) {
        d0 = krow + ((size_t)p.page_size * p.hkv + (size_t)(hh - k_end)) * p.dim;
      }
      if (d0 != nullptr) {
        *reinterpret_cast<uint4 *>(d0 + e0) = lo[u];
        *reinterpret_cast<uint4 *>(d0 + e1) = hi[u];
      }
      if (d1 != nullptr) {
        *reinterpret_cast<uint4 *>(d1 + e0) = lo[u];
        *reinterpret_cast<uint4 *>(d1 + e1) = hi[u];
      }
    }
  }
}

// The same for rows whose heads lie next to each other (a token's q, k and v rows are one run of bytes each), laid out
// for bandwidth: rows move by bulk copies, global to shared memory and back, a ring of stages per block, and only the
// rotation itself passes through registers - in place in the stage; v never does.  A block's positions and page rows
// are looked up 128 tokens at a time, (cos, sin) of the next token are formed while the copies of this one fly.
// Measured (20480 tokens, 32 q / 8 kv heads, bf16, 504 MB moved): 92.6 us, 5.4 TB/s, 0.83 of the copy rate.  Blocks per
// SM: 3 of 50 KB 119.6 us, 5 92.8, 6 98.4; 256 threads 95.4, 64 threads and 8 blocks 108.5.  The same rows with the heads
// eight elements apart, through the registers of the kernel above: 123 us; one element apart, through the element-wise
// kernel: 294; 64 of 128 elements rotated, the same: 342.  A token of more than half of kBulkSmem (two stages have to
// fit) goes through registers too: 8192 tokens of 64 / 8 heads of 256, bf16 (671 MB) 129 us, 5.2 TB/s; of 128, fp32, 115 us,
// 5.8 TB/s; two stages, 64 / 8 heads of 128, bf16: 61 us, 5.5 TB/s.
constexpr int kBulkThreads = 128;
constexpr int kBulkChunk = 128;
constexpr int kMaxStages = 4;
constexpr int kBulkBlocks = 4;       // per SM
constexpr int kBulkSmem = 50 * 1024;  // per block: four blocks per SM

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_store(void *dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, bool kNeighbours>
__global__ void __launch_bounds__(kBulkThreads) rope_axes_bulk_kernel(const __grid_constant__ AxesParams p, int stages,
                                                                      int stage_bytes) {
  constexpr int VEC = 16 / sizeof(T);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxStages];
  __shared__ __align__(16) float sh_c[2][kMaxHalfDim], sh_s[2][kMaxHalfDim];
  __shared__ int sh_pos[PIEKV_MAX_ROPE_AXES][kBulkChunk];
  __shared__ T *sh_row[kBulkChunk];
  const int tid = threadIdx.y * blockDim.x + threadIdx.x, threads = blockDim.x * blockDim.y;
  const int half = p.t.half;
  const uint32_t q_bytes = p.q != nullptr ? (uint32_t)(p.hq * p.dim * sizeof(T)) : 0u;
  const uint32_t k_bytes = (uint32_t)(p.hkv * p.dim * sizeof(T));
  const uint32_t v_bytes = p.pool != nullptr ? k_bytes : 0u;
  const int heads = (p.q != nullptr ? p.hq : 0) + p.hkv;  // rows to rotate, q then k
  const int count = (p.nnz - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;  // tokens of this block
  auto token = [&](int i) { return (int)blockIdx.x + i * (int)gridDim.x; };
  auto load = [&](int i) {  // thread 0
    const int s = i % stages;
    const int64_t tok = token(i);
    const uint32_t dst = smem_u32(smem) + (uint32_t)(s * stage_bytes);
    mbar_arrive_expect_tx(&full[s], q_bytes + k_bytes + v_bytes);
    if (q_bytes) bulk_load(dst, reinterpret_cast<const T *>(p.q) + tok * p.q_sn, q_bytes, &full[s]);
    bulk_load(dst + q_bytes, reinterpret_cast<const T *>(p.k) + tok * p.k_sn, k_bytes, &full[s]);
    if (v_bytes) bulk_load(dst + q_bytes + k_bytes, reinterpret_cast<const T *>(p.v) + tok * p.v_sn, v_bytes, &full[s]);
  };
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    mbar_fence_init();
    for (int i = 0; i < stages && i < count; ++i) load(i);
  }
  // this thread's pair when (cos, sin) are formed
  const uint64_t turn = tid < half ? p.t.turn[tid] : 0;
  const int axis = tid < half ? p.t.axis[tid] : 0;
  auto form = [&](int i) {
    if (tid < half)
      pair_cos_sin(p, token(i), sh_pos[axis][i % kBulkChunk], tid, turn, sh_c[i & 1][tid], sh_s[i & 1][tid]);
  };
  const int ch = threadIdx.x;
  const int e0 = kNeighbours ? 2 * ch * VEC : ch * VEC, e1 = kNeighbours ? e0 + VEC : e0 + half;
  bool ok = true;
  int i = 0;
  for (; i < count; ++i) {
    if (i % kBulkChunk == 0) {
      __syncthreads();  // nobody still reads the last chunk's (and, the first time, the barriers are ready)
      for (int j = tid; j < kBulkChunk && i + j < count; j += threads) {
        const int tok = token(i + j);
        for (int a = 0; a < p.t.num_axes; ++a) sh_pos[a][j] = __ldg(p.pos + (int64_t)a * p.pos_stride + tok);
        sh_row[j] = p.pool != nullptr ? pool_row<T>(p, tok) : nullptr;
      }
      __syncthreads();
      form(i);
      __syncthreads();
    }
    const int s = i % stages;
    uint8_t *stage = smem + s * stage_bytes;
    ok = mbar_wait(&full[s], (i / stages) & 1);
    float c[VEC], sn[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j += 4) {
      *reinterpret_cast<float4 *>(c + j) = *reinterpret_cast<const float4 *>(&sh_c[i & 1][ch * VEC + j]);
      *reinterpret_cast<float4 *>(sn + j) = *reinterpret_cast<const float4 *>(&sh_s[i & 1][ch * VEC + j]);
    }
    for (int h = threadIdx.y; h < heads; h += blockDim.y) {
      T *row = reinterpret_cast<T *>(stage) + h * p.dim;
      uint4 lo = *reinterpret_cast<const uint4 *>(row + e0), hi = *reinterpret_cast<const uint4 *>(row + e1);
      T *a = reinterpret_cast<T *>(&lo), *b = reinterpret_cast<T *>(&hi);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        T &x = kNeighbours ? (2 * j < VEC ? a[2 * j] : b[2 * j - VEC]) : a[j];
        T &y = kNeighbours ? (2 * j < VEC ? a[2 * j + 1] : b[2 * j + 1 - VEC]) : b[j];
        float xo, yo;
        rope_rotate(Elem<T>::to_f32(x), Elem<T>::to_f32(y), c[j], sn[j], xo, yo);
        x = Elem<T>::from_f32(xo);
        y = Elem<T>::from_f32(yo);
      }
      *reinterpret_cast<uint4 *>(row + e0) = lo;
      *reinterpret_cast<uint4 *>(row + e1) = hi;
    }
    if (i + 1 < count && (i + 1) % kBulkChunk != 0) form(i + 1);
    fence_proxy_async_smem();  // the rotated rows before the bulk stores that read them
    ok = __syncthreads_and(ok);
    if (!ok) break;
    if (tid == 0) {
      const int64_t tok = token(i);
      const uint32_t src = smem_u32(stage);
      if (q_bytes) bulk_store(reinterpret_cast<T *>(p.q_out) + tok * p.qo_sn, src, q_bytes);
      if (p.k_out != nullptr) bulk_store(reinterpret_cast<T *>(p.k_out) + tok * p.ko_sn, src + q_bytes, k_bytes);
      T *krow = sh_row[i % kBulkChunk];
      if (krow != nullptr) {
        bulk_store(krow, src + q_bytes, k_bytes);
        bulk_store(krow + (size_t)p.page_size * p.hkv * p.dim, src + q_bytes + k_bytes, v_bytes);
      }
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
      // the stage of the token before is free once its stores have read it
      if (i >= 1 && i - 1 + stages < count) {
        asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
        load(i - 1 + stages);
      }
    }
  }
  if (tid == 0) {  // shared memory outlives the copies
    if (!ok) {
      report_error(p.err, PIEKV_ERR_WAIT_TIMEOUT, KID_ROPE_AXES, blockIdx.x, i);
      // loaded so far: up to token i + stages - 2, at the start stages - 1
      for (int x = i; x < count && x <= max(i - 1, 0) + stages - 1; ++x) mbar_wait(&full[x % stages], (x / stages) & 1, 200000000ull);
    }
    asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
  }
}

template <typename T>
int launch_axes(const AxesParams &p, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  auto rows16 = [](const void *ptr, int64_t sn, int64_t sh) {
    return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && sn % VEC == 0 && sh % VEC == 0;  // (null counts as aligned)
  };
  const int pieces = p.t.half / VEC;
  if (2 * p.t.half == p.dim && p.t.half % VEC == 0 && rows16(p.q, p.q_sn, p.q_sh) && rows16(p.q_out, p.qo_sn, p.qo_sh) &&
      rows16(p.k, p.k_sn, p.k_sh) && rows16(p.k_out, p.ko_sn, p.ko_sh) && rows16(p.v, p.v_sn, p.v_sh) && rows16(p.pool, 0, 0)) {
    const int heads = (p.q != nullptr ? p.hq : 0) + p.hkv + (p.pool != nullptr ? p.hkv : 0);
    // rows that are one run of bytes, and enough tokens that a block works on several: bulk copies
    const bool runs = (p.q == nullptr || (p.q_sh == p.dim && p.qo_sh == p.dim)) && p.k_sh == p.dim &&
                      (p.k_out == nullptr || p.ko_sh == p.dim) && (p.pool == nullptr || p.v_sh == p.dim);
    const int stage_bytes = (heads * p.dim * (int)sizeof(T) + 127) / 128 * 128;
    const int stages = kBulkSmem / stage_bytes < kMaxStages ? kBulkSmem / stage_bytes : kMaxStages;
    const int blocks = kBulkBlocks * sm_count();
    const dim3 bulk_block(pieces, kBulkThreads / pieces);
    if (runs && stages >= 2 && p.nnz >= 2 * blocks && (int)(bulk_block.x * bulk_block.y) >= p.t.half) {
      static unsigned char configured[2][kMaxDevices] = {{0}};
      auto kernel = p.t.interleave ? rope_axes_bulk_kernel<T, true> : rope_axes_bulk_kernel<T, false>;
      if (int rc = opt_in_dynamic_smem(kernel, kBulkSmem, configured[p.t.interleave ? 1 : 0], "rope_axes: cudaFuncSetAttribute"))
        return rc;
      kernel<<<blocks, bulk_block, stages * stage_bytes, st>>>(p, stages, stage_bytes);
      PIEKV_LAUNCH_CHECK("rope_axes_bulk_kernel");
      return 0;
    }
    // a token's heads are divided among threads until every SM has kThreadsPerSm of them
    const long long want = (long long)kThreadsPerSm * sm_count(), have = (long long)p.nnz * pieces;
    const long long slices = have >= want ? 1 : (want + have - 1) / have;
    const int per = slices >= heads ? 1 : (int)((heads + slices - 1) / slices);
    const dim3 block(pieces, kThreads / pieces);
    const dim3 grid((p.nnz + block.y - 1) / block.y, (heads + per - 1) / per);
    if (p.t.interleave)
      rope_axes_rows_kernel<T, true><<<grid, block, 0, st>>>(p, per);
    else
      rope_axes_rows_kernel<T, false><<<grid, block, 0, st>>>(p, per);
    PIEKV_LAUNCH_CHECK("rope_axes_rows_kernel");
    return 0;
  }
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
      for (int i = ax; i < half && i < num_axes * sections[ax]; i += num_axes) table->axis[i] = (uint8_t)ax;
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
