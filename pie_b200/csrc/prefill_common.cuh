// Definitions shared by the prefill attention kernels: tile constants, the device-built plan and the
// kernel parameter block.
#pragma once
#include <cuda.h>

#include "attn.cuh"
#include "common.cuh"

namespace piekv {
namespace prefill {

constexpr int kDim = 128;
constexpr int kPage = 16;
constexpr int kBM = 128;  // query rows per CTA
constexpr int kBN = 128;  // kv tokens per tile (8 pages)
constexpr int kKStages = 3;  // K tiles in flight (needed early, by S = Q K^T)
constexpr int kVStages = 2;  // V tiles in flight (needed a softmax later, by O += P V)
constexpr int kSoftmaxWarps = 8;  // two threads per query row: each owns 64 of the 128 kv columns
constexpr int kProducerWarp = kSoftmaxWarps, kMmaWarp = kSoftmaxWarps + 1;
constexpr int kThreads = (kSoftmaxWarps + 2) * 32;
constexpr int kTileBytes = 32768;  // one 128 x 128 16-bit operand tile
constexpr int kHalfBytes = 16384;  // one 128 x 64 half of it
constexpr int kSmemBytes = kTileBytes * (1 + kKStages + kVStages + 1) + 1024;
constexpr int kTmemCols = 512;
constexpr int kColS = 0, kColO = 256;
constexpr int kCounterBytes = 65536;
constexpr int kSortBins = 1024;

// Plan of one batch, built on the device into the workspace (after the counter area):
//   header (word 0: tiles, words 2-3: items claimed / CTAs finished) | tile_base[B+1] | poff[B+1] | moff[B+1] | tiles[max_tiles] | summary[max_tiles][sw] | packed mask
struct PlanView {
  int *ntiles;             // header word 0
  int32_t *tile_base;      // first q-tile index of every request (prefix of ceil(qo_len / 128))
  long long *poff;         // packed-mask offset of every request, in 16-byte units
  long long *moff;         // byte offset of every request in the flat boolean mask
  int2 *tiles;             // (request, first row within the request), heaviest first
  uint32_t *summary;       // bit j of row t: kv tile j of q tile t has at least one allowed pair
  uint4 *packed;           // per query row ceil(kv_len/128) x 128 mask bits
  int sw;                  // words per summary row
  int max_tiles;
  int64_t bytes;           // total workspace bytes including the counter area
};

struct PrefillParams {
  AttnArgs a;
  const int2 *tiles;
  const int *ntiles;
  int *claim;              // [0] items handed out, [1] CTAs that ran out of items; zero between launches
  const int32_t *tile_base;
  const long long *poff;
  const uint32_t *summary;
  const uint4 *packed;
  int sw;
  int has_mask;
  int tokens;              // two-problem kernel with a band: query tokens per 128-row tile (all heads of a kv head)
};

// bounded wait that also gives up when another role has already aborted
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort_flag) {
  if (mbar_try_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > 2000000000ull) return false;
  }
}

// ---- window with first tokens (kBand kernels): the query at position p sees keys [0, first) and
// [p - window_left, limit], limit = p (causal) or the last key.  Nothing is packed: a row's 128 mask bits of a tile
// follow from three numbers.
__device__ __forceinline__ uint32_t ones_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }
// mask bits of keys t .. t + 31 for a row that sees [0, first), [low, limit]
__device__ __forceinline__ uint32_t band_word(int t, int first, int low, int limit) {
  return (ones_below(first - t) | ~ones_below(low - t)) & ones_below(limit + 1 - t);
}
__device__ __forceinline__ uint4 band_bits(int t, int first, int low, int limit) {
  return make_uint4(band_word(t, first, low, limit), band_word(t + 32, first, low, limit),
                    band_word(t + 64, first, low, limit), band_word(t + 96, first, low, limit));
}
// The kv tiles of a query tile: [0, front) and [low_tile, n_tiles); `low` is the lowest window start of its rows.
struct Band {
  int first, low, front, low_tile;
};
__device__ __forceinline__ Band band_of(const AttnArgs &a, int kv_len, int qo_len, int r0, int n_tiles) {
  Band w;
  w.first = min(a.first_tokens, kv_len);
  w.low = max(0, kv_len - qo_len + r0 - a.window_left);
  w.front = min((w.first + kBN - 1) / kBN, n_tiles);
  w.low_tile = min(max(w.low / kBN, w.front), n_tiles);
  return w;
}
// page `pi` of the request's list holds a key that some row of the query tile may see
__device__ __forceinline__ bool band_page(const Band &w, int pi) { return pi * kPage < w.first || pi * kPage + kPage > w.low; }

// Zero the rows of a staged V tile that belong to the request's last page but lie beyond its last
// token (rows [first, end) of the 128-token tile; a row is 128 bytes in each 64-column half,
// whatever the swizzle does inside it).  Their probabilities are zero, but 0 x NaN is NaN, and a
// recycled page may hold anything there.  Executed by one full warp after the tile has landed.
__device__ __forceinline__ void zero_v_rows(uint32_t v_tile_smem, int first, int end, int lane) {
  for (int x = lane; x < (end - first) * 16; x += 32) {
    const int row = first + (x >> 4), half = (x >> 3) & 1, ch = x & 7;
    asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v_tile_smem + half * kHalfBytes + row * 128 + ch * 16),
                 "r"(0)
                 : "memory");
  }
}

// The same for a band: keys of loaded pages between the first tokens and the window, and behind the context.
// Tells whether tile j has any; with `zero` it clears them.
__device__ __forceinline__ bool band_unseen_v_rows(const Band &w, int kv_len, int j, uint32_t v_tile_smem, int lane, bool zero) {
  const int t0 = j * kBN;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int a, e;
    if (i == 0) {  // rest of the page of the last first token
      a = w.first;
      e = min((w.first + kPage - 1) / kPage * kPage, w.low);
    } else if (i == 1) {  // start of the window's first page
      a = max(w.low / kPage * kPage, w.first);
      e = w.low;
    } else {
      a = kv_len;
      e = (kv_len + kPage - 1) / kPage * kPage;
    }
    a = max(a - t0, 0);
    e = min(e - t0, kBN);
    if (a < e) {
      any = true;
      if (zero) zero_v_rows(v_tile_smem, a, e, lane);
    }
  }
  return any;
}

// The keys an item of the two-problem kernel streams, as a list of pages without the ones nobody sees: pages
// [0, front) and [low_page, ...) of the request, `pages` in all.  Slot s of the list is key s, behind the first
// tokens' pages key s + shift.
struct VisibleKeys {
  int first, low;       // keys [0, first) and [low, ...) are seen by some row
  int front, low_page, pages, shift;
};
__device__ __forceinline__ VisibleKeys visible_keys(const AttnArgs &a, int kv_len, int pos_first, int hi) {
  VisibleKeys w;
  w.first = max(0, min(a.first_tokens, hi));
  w.low = max(0, pos_first - a.window_left);
  w.front = (w.first + kPage - 1) / kPage;
  w.low_page = max(w.front, w.low / kPage);
  w.pages = hi > 0 ? w.front + max(0, (hi + kPage - 1) / kPage - w.low_page) : 0;
  w.shift = (w.low_page - w.front) * kPage;
  return w;
}
// Slots of loaded pages that no row sees, as up to three ranges: behind the first tokens, before the window, behind the
// context.  Tells whether tile j has any; with `zero` it clears their V rows.
__device__ __forceinline__ bool unseen_v_rows(const VisibleKeys &w, int kv_len, int j, uint32_t v_tile_smem, int lane, bool zero) {
  const int t0 = j * kBN, low = w.low - w.shift, len = kv_len - w.shift;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    int a, e;
    if (i == 0) {
      a = w.first;
      e = min(w.front * kPage, low);
    } else if (i == 1) {
      a = max(low / kPage * kPage, w.first);
      e = low;
    } else {
      a = len;
      e = (len + kPage - 1) / kPage * kPage;
    }
    a = max(a - t0, 0);
    e = min(e - t0, kBN);
    if (a < e) {
      any = true;
      if (zero) zero_v_rows(v_tile_smem, a, e, lane);
    }
  }
  return any;
}

}  // namespace prefill
}  // namespace piekv
