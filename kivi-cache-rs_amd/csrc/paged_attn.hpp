// paged_attn.hpp — what the attention kernels of the paged cache share: which tokens a tile of rows
// walks, how a walk is split, where a token's row lies, and the launches of the two kernels.
#pragma once

#include <hip/hip_runtime.h>

#include "paged.hpp"

namespace kivi {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLargest = 3.402823466e+38f;  // |x| <= kLargest: x is finite

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// What the lanes of a wave wrote to its LDS is there for its other lanes.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ int clamped(int64_t x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : (int)x; }

// x of the lanes 16 (32) away, as the vector ALU swaps rows: both results together hold every lane's own
// and its partner's.
template <int BY>
__device__ __forceinline__ void swapped(float x, float* a, float* b) {
  const uint32_t u = __float_as_uint(x);
  if constexpr (BY == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    *a = __uint_as_float(r[0]), *b = __uint_as_float(r[1]);
  } else {
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    *a = __uint_as_float(r[0]), *b = __uint_as_float(r[1]);
  }
}
template <int BY>
__device__ __forceinline__ float sum_with(float x) {
  float a, b;
  swapped<BY>(x, &a, &b);
  return a + b;
}
template <int BY>
__device__ __forceinline__ float max_with(float x) {
  float a, b;
  swapped<BY>(x, &a, &b);
  return fmaxf(a, b);
}
// The largest of three, NaN if one is (of a row's logits: its weights are then NaN too); fmaxf would first
// have to quiet each.
__device__ __forceinline__ float max_of(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// Sum over the lanes of a row of 16 that lie N apart (N 4 or 8), in every lane.
template <int N>
__device__ __forceinline__ float sum_row(float x) {
  x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x128, 0xF, 0xF, true));  // rotated by 8
  if constexpr (N == 4) x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x124, 0xF, 0xF, true));
  return x;
}

// Eight elements of a row.
template <class T>
struct Row;
template <>
struct Row<_Float16> {
  typedef f16x8 Frag;
};
template <>
struct Row<__bf16> {
  typedef bf16x8 Frag;
};
template <>
struct Row<float> {
  typedef f32x8 Frag;
};

// What a call does to one (sequence, KV head): lengths, and which tokens a tile of rows walks.
struct Walk {
  int64_t total;     // tokens: cached, then the new rows where they come as rows
  int64_t hi;        // tokens from here on are seen by no row of the tile
  int64_t lo;        // under a window, tokens in [sinks, lo) neither
  int64_t sinks;
  uint32_t head_tiles, first_tile, tiles;  // token tiles 0 .. head_tiles - 1, then from first_tile on; their number
};

__device__ __forceinline__ Walk walk_of(const PagedAttention& a, const PagedSequence& s, uint32_t row0, uint32_t row1,
                                        uint32_t gq, uint32_t tile) {
  Walk w;
  w.total = s.n + (a.keys.p != nullptr ? s.m : 0);
  const int64_t p0 = w.total - s.m + row0 / gq, p1 = w.total - s.m + (row1 - 1) / gq;
  w.hi = p1 + 1 > 0 ? p1 + 1 : 0;
  w.lo = w.sinks = 0;
  if (a.window != 0) {
    w.lo = p0 + 1 > 0 && (uint64_t)(p0 + 1) > a.window ? p0 + 1 - (int64_t)a.window : 0;
    w.sinks = (uint64_t)w.lo < a.sinks ? w.lo : (int64_t)a.sinks;
  }
  w.head_tiles = (uint32_t)((w.sinks + tile - 1) / tile);
  const uint32_t from = (uint32_t)(w.lo / tile), to = (uint32_t)((w.hi + tile - 1) / tile);
  w.first_tile = from > w.head_tiles ? from : w.head_tiles;
  w.tiles = w.head_tiles + (to > w.first_tile ? to - w.first_tile : 0);
  return w;
}

// Tiles [from, to) of split `split` of at most `splits`, and how many splits the walk takes (at least 1).
struct Part {
  uint32_t from, to, count;
};
__device__ __forceinline__ Part part_of(uint32_t tiles, uint32_t splits, uint32_t split) {
  const uint32_t per = (tiles + splits - 1) / splits;
  Part p;
  p.count = tiles == 0 ? 1 : (tiles + per - 1) / per;
  p.from = split * per < tiles ? split * per : tiles;
  p.to = p.from + per < tiles ? p.from + per : tiles;
  return p;
}

template <class T>
__device__ __forceinline__ float decoded(uint32_t code, float2 pair) {
  return fmaf((float)code, pair.x, pair.y);
}

// Row of token t (t >= what is packed) of one head: in the window, or among the new rows.
template <class T>
__device__ __forceinline__ const T* row_of(const PagedGeometry& g, const void* window, const PagedSequence& s,
                                           uint32_t head, int64_t t, const PagedRows& rows) {
  if (t < s.n)
    return static_cast<const T*>(window) + (((uint64_t)s.slot * g.heads + head) * 2 * g.R + ring_row(g, t)) * g.DW;
  return static_cast<const T*>(rows.p) + (uint64_t)(s.row0 + (t - s.n)) * rows.stride + (uint64_t)head * rows.pitch;
}

// Eight elements as 16-byte pieces and back, by value: through a pointer they would pass through memory.
template <class T>
__device__ __forceinline__ typename Row<T>::Frag frag_of(const u32x4* x) {
  if constexpr (sizeof(T) == 2) {
    return __builtin_bit_cast(typename Row<T>::Frag, x[0]);
  } else {
    return __builtin_bit_cast(f32x8, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
  }
}
template <class T>
__device__ __forceinline__ void pieces_of(typename Row<T>::Frag f, u32x4* x) {
  if constexpr (sizeof(T) == 2) {
    x[0] = __builtin_bit_cast(u32x4, f);
  } else {
    x[0] = __builtin_bit_cast(u32x4, __builtin_shufflevector(f, f, 0, 1, 2, 3));
    x[1] = __builtin_bit_cast(u32x4, __builtin_shufflevector(f, f, 4, 5, 6, 7));
  }
}
// Elements d .. d + 7 of a row (d a multiple of 8 under DW).
template <class T>
__device__ __forceinline__ typename Row<T>::Frag load_frag(const T* p, uint32_t d) {
  u32x4 x[sizeof(T) / 2];
  x[0] = reinterpret_cast<const u32x4*>(p + d)[0];
  if constexpr (sizeof(T) == 4) x[1] = reinterpret_cast<const u32x4*>(p + d)[1];
  return frag_of<T>(x);
}
template <class T>
__device__ __forceinline__ typename Row<T>::Frag zero_frag() {
  return typename Row<T>::Frag{};
}
// Whether any of the eight is infinite or NaN.
template <class T>
__device__ __forceinline__ bool wild(const typename Row<T>::Frag& f) {
  bool any = false;
#pragma unroll
  for (int j = 0; j < 8; ++j) any |= !(fabsf((float)f[j]) <= kLargest);
  return any;
}

// Value (t, d) of one head, t among what the row tile walks; `rec` the record of t's page.
template <class T>
__device__ float value_of(const PagedAttention& a, const PagedSequence& s, const uint32_t* rec, uint32_t head, int64_t t,
                          int64_t vq, uint32_t d) {
  const PagedGeometry& g = a.c.geo;
  if (t >= vq) return (float)row_of<T>(g, a.c.vwin, s, head, t, a.values)[d];
  if (rec == nullptr) return 0.f;
  const uint32_t in_page = token_in_page(g, t), tau = in_page % 32, j = tau % 4 + tau / 16 * 4;
  const uint32_t* words = rec + g.vcodes_at + (uint64_t)(in_page / 32) * g.block_words() + (tau % 16 / 4 * 16 + d % 16) * g.lane_words();
  const float2 pair = reinterpret_cast<const float2*>(rec + g.vparams_at)[(uint64_t)in_page * g.ncg + quotient(d, g.G, g.group_magic)];
  return decoded<T>(words[paged_word(g.bits, d / 16, j)] >> paged_bit(g.bits, d / 16, j) & g.levels(), pair);
}

// Chunks of few rows (kernels_paged_rows_*.hip): sequences whose KV heads have more than `over` and at
// most `most` rows, at most kRowsMost.
constexpr uint32_t kRowsMost = 32;
struct RowsPlan {
  uint32_t over, most;     // rows of a KV head that this launch takes
  uint32_t blocks;         // column groups: 4 (up to 4 rows), 2 (8) or 1 (16 rows a tile)
  uint32_t splits;         // at most this many of a walk's packed blocks,
  uint32_t least;          // each of a multiple of this many 32-token blocks (itself one of 4 * blocks)
  uint32_t tails;          // at most this many of its last blocks
  uint32_t stride;         // rows of a (sequence, head) in the partials
};
// Whether the kernels of few rows take this cache (else the chunk kernel takes everything).
bool paged_rows_take(const PagedGeometry& g);
// Column groups by registers: the codes of a turn's blocks are 16 or 32 words a lane, once for keys and once
// for values.
__host__ __device__ constexpr int rows_most_blocks(uint32_t bits, uint32_t S) {
  return S * bits / 2 <= 8 ? 4 : S * bits / 2 <= 16 ? 2 : 1;
}
// HALVES: G is an odd multiple of 16 (a block's halves may lie in two groups).
template <class T, bool HALVES>
hipError_t launch_paged_rows(const PagedAttention& a, const RowsPlan& p, float* partial, hipStream_t stream);

// Longer chunks (kernels_paged_chunk_*.hip): sequences whose KV heads have more than `over` rows.
struct ChunkPlan {
  uint32_t over, tile_rows, tile, splits;  // rows of a workgroup, tokens of a tile, splits of a walk at most
};
// Rows of a workgroup and tokens of a tile by what the registers (512 a lane of one wave, 256 of two) and
// LDS hold.
constexpr uint32_t paged_chunk_waves(uint32_t type_bytes, uint32_t S) { return type_bytes == 2 && S <= 4 ? 8 : 4; }
constexpr uint32_t paged_chunk_tile(uint32_t S) { return S <= 4 ? 64 : 32; }
inline uint32_t paged_chunk_rows(const PagedGeometry& g) { return 32 * paged_chunk_waves(g.type_bytes(), g.S()); }
inline uint32_t paged_chunk_tokens(const PagedGeometry& g) { return paged_chunk_tile(g.S()); }
template <class T>
hipError_t launch_paged_chunk(const PagedAttention& a, const ChunkPlan& p, float* partial, hipStream_t stream);

}  // namespace kivi
