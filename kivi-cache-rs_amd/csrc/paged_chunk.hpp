// paged_chunk.hpp — attention of a chunk of many rows (a piece of a prompt) over the paged cache: the
// kernel, and its launch for one element type (kernels_paged_chunk_*.hip instantiate it).
#pragma once

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "paged_attn.hpp"

namespace kivi {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

// 32x32 tiles, 16 of the contraction: lane holds row (column) lane % 32, elements 8 (lane / 32) + j;
// accumulator element i is row 8 (i / 4) + 4 (lane / 32) + i % 4 of column lane % 32.
template <class T>
struct Mma;
template <>
struct Mma<_Float16> {
  static __device__ __forceinline__ f32x16 mul(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<__bf16> {
  static __device__ __forceinline__ f32x16 mul(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
// Eight products of two: slice j takes element j of both halves, the same ones of both operands.
template <>
struct Mma<float> {
  static __device__ __forceinline__ f32x16 mul(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
  }
};

// One workgroup: WAVES * 32 rows of one (sequence, KV head), each wave 32 of them, over one split of the
// token tiles. A tile of TT tokens lies in LDS as the products read it, keys by token, values by channel
// (tokens in the order of the code blocks), rows padded by 16 bytes so that the lanes of a read fall on
// different banks. All waves fill it and all read it; there are two, so that a tile is filled while
// the one before is used: its codes or rows are fetched ahead of the products and put after them.
//
// Packed tokens are decoded in float32. One rounding of a key to 16 bits would cost as much precision as
// the output's own (of a bf16 key as much as twice that, as keys have channels of large magnitude), so
// keys are kept in two terms of the type (high and low: twice the first product); values too in f16,
// whose outputs are as exact as the weights, while in bf16 the weights' own rounding is as large.
// Rows are what they are and need one.
//
// Bound by the vector ALU (softmax and decoding, 380 instructions per wave and plain tile) beside the matrix
// cores (48 instructions): 2048 rows over 16384 cached tokens, bf16, 2 bits, 32 query heads of 128: 890 to
// 945 us, 620 to 655 TFLOP/s (one loop for all kinds of tiles: 1370 us, half its instructions addresses and spilled scalars).
// Halves of a tile at different times in a SIMD's two waves: 1030 us, against 980 then.
template <class T>
constexpr int kKeyTerms = sizeof(T) == 2 ? 2 : 1;
template <class T>
constexpr int kValueTerms = std::is_same<T, _Float16>::value ? 2 : 1;

template <class T, int S, int TT>
struct ChunkTile {
  static constexpr int DP = 32 * S, kPad = 16 / sizeof(T);
  static constexpr int kKeyPitch = DP + kPad, kValuePitch = TT + kPad;
  static constexpr int kKeys = TT * kKeyPitch, kValues = DP * kValuePitch;  // elements of one term
  static constexpr int kElements = kKeyTerms<T> * kKeys + kValueTerms<T> * kValues;
  static constexpr size_t kBytes = 2 * kElements * sizeof(T);
};

// x as terms of the type: the rounded value, and in two terms what that leaves out.
template <class T, int TERMS>
__device__ __forceinline__ void put_terms(const float (&x)[8], T* to, int term) {
  typename Row<T>::Frag f, low;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    f[j] = (T)x[j];
    if constexpr (TERMS == 2) low[j] = (T)(x[j] - (float)f[j]);
  }
  *reinterpret_cast<typename Row<T>::Frag*>(to) = f;
  if constexpr (TERMS == 2) *reinterpret_cast<typename Row<T>::Frag*>(to + term) = low;
}

// The eight codes of a fragment as floats, from its word (two at 8 bits; `odd`: the second fragment of a
// 2-bit word). The packed converters take codes as fp4 and fp8 times a scale (exact).
template <int BITS>
__device__ __forceinline__ void codes_to(const uint32_t* w, uint32_t odd, float (&x)[8]) {
  if constexpr (BITS == 2) {
    const uint32_t m = (w[0] >> 2 * odd) & 0x33333333u;
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(m, 2.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(m, 2.0f, 1);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(m, 2.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(m, 2.0f, 3);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
  } else if constexpr (BITS == 4) {
    const uint32_t lo = w[0] & 0x0f0f0f0fu, hi = w[0] >> 4 & 0x0f0f0f0fu;
    const f32x2 a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, true);
    const f32x2 c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, true);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
  } else if constexpr (BITS == 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)(w[j / 4] >> 8 * (j % 4) & 255u);
  }
}

// Last token in front of the window of a row at `pos` (-1: none).
__device__ __forceinline__ int64_t left_of(const PagedAttention& a, int64_t pos) {
  return a.window != 0 ? pos - (int64_t)a.window : -1;
}

// The lane, read anew where it stands: what is derived from it is computed there and not kept in registers
// across the loop (nor the lane itself).
__device__ __forceinline__ uint32_t lane_anew() {
  uint32_t x;
  asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=&v"(x));
  return x;
}

// BITS 0: any layout.
template <class T, int BITS, int S>
__global__ void __launch_bounds__(paged_chunk_waves(sizeof(T), S) * 64)
    k_paged_chunk(PagedAttention a, ChunkPlan plan, float* partial) {
  constexpr int WAVES = paged_chunk_waves(sizeof(T), S), TT = paged_chunk_tile(S);
  typedef typename Row<T>::Frag Frag;
  typedef ChunkTile<T, S, TT> Tile;
  constexpr int DP = Tile::DP, LW = S * (BITS == 0 ? 2 : BITS) / 2, kKeyPitch = Tile::kKeyPitch, kValuePitch = Tile::kValuePitch;
  constexpr int KT = kKeyTerms<T>, VT = kValueTerms<T>;
  constexpr uint32_t kThreads = WAVES * 64, kSub = TT / 32;
  extern __shared__ __align__(16) unsigned char lds[];
  __shared__ uint32_t bad[3][2];  // tokens of a tile with a value that is not finite, where not every row sees all
  __shared__ float bad_row[WAVES][DP];
  const PagedGeometry& g = a.c.geo;
  const uint32_t head = blockIdx.x % g.heads, tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t col = lane % 32, half = lane / 32;
  const PagedSequence s = paged_sequence(a.b, g, blockIdx.z);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq;
  const uint32_t splits = plan.splits;
  const uint32_t tile_row = blockIdx.x / g.heads / splits * (WAVES * 32), split = blockIdx.x / g.heads % splits;
  if (rows <= plan.over || tile_row >= rows) return;
  const uint32_t tile_end = tile_row + WAVES * 32 < rows ? tile_row + WAVES * 32 : rows;
  const Walk w = walk_of(a, s, tile_row, tile_end, gq, TT);
  const Part part = part_of(w.tiles, splits, split);
  if (split >= part.count) return;
  // positions of the wave's first and last row and of the workgroup's first
  const int64_t at0 = w.total - s.m, first_pos = at0 + tile_row / gq;

  const uint32_t D = g.D, DW = g.DW, ncg = g.ncg;
  const int64_t kq = paged_kq(g, s.n), vq = paged_vq(g, s.n);
  // the lane's row of the KV head (the last one in lanes past it): worked out where it is wanted
  const auto row_now = [&] {
    const uint32_t row = tile_row + wave * 32 + lane_anew() % 32;
    return row < rows ? row : rows - 1;
  };
  const uint32_t wr0 = tile_row + wave * 32 < rows ? tile_row + wave * 32 : rows - 1, wr1 = wr0 + 31 < rows ? wr0 + 31 : rows - 1;
  const int64_t all_pos = at0 + wr0 / gq, any_pos = at0 + wr1 / gq;
  // tokens up to here are outside the window: of the wave's last row, of the workgroup's
  const int64_t all_left = a.window != 0 ? any_pos - (int64_t)a.window : -1;
  const int64_t last_left = a.window != 0 ? w.hi - 1 - (int64_t)a.window : -1;
  // Three kinds of tiles, each with a loop of its own, one after the other: [plain_at, plain_at + plains) of the
  // walk are packed and seen by every row (where their pages are there); from dense_at on all tokens are rows;
  // and the others.
  uint32_t dense_at = (uint32_t)((kq + TT - 1) / TT);
  if (dense_at >= w.head_tiles) dense_at = w.head_tiles + (dense_at > w.first_tile ? dense_at - w.first_tile : 0);
  if (dense_at > w.tiles) dense_at = w.tiles;
  const uint32_t denses = w.tiles - dense_at;
  uint32_t plain_at = 0, plains = 0;
  if constexpr (BITS != 0) {
    const int64_t seen = first_pos + 1 < vq ? first_pos + 1 : vq;
    const uint32_t from = last_left < 0 ? 0 : (uint32_t)((last_left + TT) / TT), to = seen < 0 ? 0 : (uint32_t)(seen / TT);
    const uint32_t first = from > w.first_tile ? from : w.first_tile;
    if (to > first) plain_at = w.head_tiles + (first - w.first_tile), plains = to - first;
  }

  // exp2(scale q k) with a scale above zero (hidden logits are -inf): a sign, or a zero, goes to the queries
  const float sign = a.scale < 0.f ? -1.f : a.scale == 0.f ? 0.f : 1.f, scale = a.scale == 0.f ? 1.f : fabsf(a.scale) * kLog2e;
  Frag q[DP / 16];
  {
    const uint32_t row = row_now(), token = row / gq, qhead = head * gq + row % gq;
    const T* p = static_cast<const T*>(a.query.p) + (uint64_t)(s.row0 + token) * a.query.stride + (uint64_t)qhead * a.query.pitch;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const uint32_t d = 16 * i + 8 * half;
      q[i] = d < DW ? load_frag(p, d) : zero_frag<T>();
#pragma unroll
      for (int j = 0; j < 8; ++j) q[i][j] = (T)((float)q[i][j] * sign);
    }
  }
  float top = -INFINITY, sum = 0.f;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{0.f};

  T* const tiles = reinterpret_cast<T*>(lds);
  if (DW < DP)  // channels that no row fills
    for (uint32_t i = tid; i < Tile::kBytes / 16; i += kThreads) reinterpret_cast<u32x4*>(lds)[i] = u32x4{0, 0, 0, 0};
  if (tid < 6) bad[tid / 2][tid % 2] = 0;
  __syncthreads();

  // ---- How a tile is filled. Packed: a thread has two fragments of keys (tokens l % 16 and 16 on of a block,
  // channels 8 S q + 8 i) and two of values (channels 32 i + l % 16 and 16 on, the eight tokens of q), so one set
  // of pairs each. Rows: 8-channel pieces of keys, and of two tokens' values. What is fetched for a piece
  // waits in registers until it is put.
  constexpr int kUnits = kSub * 64 * S, kEach = (kUnits + (int)kThreads - 1) / (int)kThreads;
  constexpr int kKeyPieces = TT * DP / 8, kKeyRows = (kKeyPieces + (int)kThreads - 1) / (int)kThreads;
  constexpr int kValuePieces = TT / 2 * DP / 8, kValueRows = (kValuePieces + (int)kThreads - 1) / (int)kThreads;
  constexpr int kWide = sizeof(T) / 2;  // u32x4s of a fragment
  constexpr int kMost = [](int x, int y, int z) { return x > y ? (x > z ? x : z) : (y > z ? y : z); }(4 * kEach, kKeyRows * kWide, 2 * kValueRows * kWide);
  constexpr int kWords = BITS == 8 ? 4 : 2;  // BITS == 0: any layout, see fill_any
  u32x4 stage[kMost];
  uint32_t words[kEach][kWords];
  struct Next {
    int64_t t0;
    const uint32_t* rec[2];  // of the tile's two blocks (no page: the pool's first, and not held)
    bool held[2];
    uint32_t inner[2];
    int keys, values;  // tokens of the tile whose keys, values are packed; the others are rows
    bool edge;  // some row of the workgroup does not see some token
  };
  const auto locate = [&](uint32_t it) {
    Next n;
    const uint32_t at = it - plains - denses < plain_at ? it - plains - denses : it - denses;  // of the walk
    n.t0 = (int64_t)(at < w.head_tiles ? at : w.first_tile + (at - w.head_tiles)) * TT;
    bool all = true;
    n.keys = clamped(kq - n.t0, 0, TT), n.values = clamped(vq - n.t0, 0, TT);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      n.rec[i] = a.c.pages, n.inner[i] = 0, n.held[i] = true;
      if (i >= (int)kSub || 32 * i >= n.keys) continue;
      const uint32_t block = (uint32_t)(n.t0 / 32) + i, page = quotient(block, g.page_blocks, g.page_magic);
      n.inner[i] = block - page * g.page_blocks;
      const uint32_t* rec = paged_record_of(a.c, a.b, s, head, page);
      n.held[i] = rec != nullptr;
      all &= n.held[i];
      if (n.held[i]) n.rec[i] = rec;
    }
    n.edge = n.t0 + TT - 1 > first_pos || n.t0 <= last_left || !all;
    return n;
  };
  // A thread's unit e of a packed tile: block, step i, lane; its record and place in the page.
  struct Unit {
    uint32_t b, i, l, q, inner;
    const uint32_t* rec;
  };
  const auto unit_of = [&](const Next& n, int e) {
    const uint32_t u = (wave + e * WAVES) * 64 + lane_anew();
    Unit x;
    x.b = u / (64 * S), x.i = u / 64 % S, x.l = u % 64, x.q = x.l / 16;
    x.rec = x.b == 0 ? n.rec[0] : n.rec[1];
    x.inner = x.b == 0 ? n.inner[0] : n.inner[1];
    return x;
  };
  // Place of token tau in a row of values. Values that are not finite are left out of a tile that some row
  // does not see whole (a weight of zero would not keep them from it) and marked.
  const auto slot = [](uint32_t tau) { return tau / 32 * 32 + tau % 16 / 4 * 8 + tau % 32 / 16 * 4 + tau % 4; };
  // Rows of a tile from token `from` of it on: 8-channel pieces.
  const auto fetch_key_rows = [&](u32x4(&stage)[kMost], int64_t t0, int from) {
    const uint32_t me = wave * 64 + lane_anew();
#pragma unroll
    for (int k = 0; k < kKeyRows; ++k) {
      const uint32_t u = me + k * kThreads, tau = u / (DP / 8), d = u % (DP / 8) * 8;
      Frag f = zero_frag<T>();
      if ((int)tau >= from && t0 + tau < w.hi && d < DW && u < kKeyPieces) f = load_frag(row_of<T>(g, a.c.kwin, s, head, t0 + tau, a.keys), d);
      pieces_of<T>(f, &stage[k * kWide]);
    }
  };
  const auto fetch_value_rows = [&](u32x4(&stage)[kMost], int64_t t0, int from) {
    const uint32_t me = wave * 64 + lane_anew();
#pragma unroll
    for (int k = 0; k < kValueRows; ++k) {
      const uint32_t u = me + k * kThreads, tau = u % (TT / 2) * 2, d = u / (TT / 2) * 8;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Frag f = zero_frag<T>();
        if ((int)tau + i >= from && d < DW && t0 + tau + i < w.hi) f = load_frag(row_of<T>(g, a.c.vwin, s, head, t0 + tau + i, a.values), d);
        pieces_of<T>(f, &stage[(2 * k + i) * kWide]);
      }
    }
  };
  const auto put_key_rows = [&](const u32x4(&stage)[kMost], int from, T* kt) {
    const uint32_t me = wave * 64 + lane_anew();
#pragma unroll
    for (int k = 0; k < kKeyRows; ++k) {
      const uint32_t u = me + k * kThreads, tau = u / (DP / 8), d = u % (DP / 8) * 8;
      if ((int)tau < from || (kKeyPieces % kThreads != 0 && u >= kKeyPieces)) continue;
#pragma unroll
      for (int i = 0; i < kWide; ++i) {
        reinterpret_cast<u32x4*>(kt + tau * kKeyPitch + d)[i] = stage[k * kWide + i];
        if (KT == 2 && from > 0) reinterpret_cast<u32x4*>(kt + Tile::kKeys + tau * kKeyPitch + d)[i] = u32x4{0, 0, 0, 0};
      }
    }
  };
  const auto put_value_rows = [&](const u32x4(&stage)[kMost], int from, bool edge, T* vt, uint32_t* marks) {
    const uint32_t me = wave * 64 + lane_anew();
#pragma unroll
    for (int k = 0; k < kValueRows; ++k) {
      const uint32_t u = me + k * kThreads, tau = u % (TT / 2) * 2, d = u / (TT / 2) * 8;
      if (kValuePieces % kThreads != 0 && u >= kValuePieces) continue;
      Frag f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[i] = frag_of<T>(&stage[(2 * k + i) * kWide]);
        if (edge && wild<T>(f[i])) {
          atomicOr(&marks[tau / 32], 1u << (tau + i) % 32);
#pragma unroll
          for (int j = 0; j < 8; ++j) f[i][j] = fabsf((float)f[i][j]) <= kLargest ? f[i][j] : (T)0.f;
        }
      }
      T* to = vt + d * kValuePitch + slot(tau);
      if (from == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          struct alignas(2 * sizeof(T)) Two {
            T x, y;
          };
          *reinterpret_cast<Two*>(to + j * kValuePitch) = Two{f[0][j], f[1][j]};
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if ((int)tau + i < from) continue;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            to[j * kValuePitch + i] = f[i][j];
            if constexpr (VT == 2) to[Tile::kValues + j * kValuePitch + i] = (T)0.f;
          }
        }
      }
    }
  };
  // `packed`: the packed part of tile n, else its rows; only a tile that has both is filled in two passes
  const auto fetch_keys = [&](const Next& n, bool packed) {
    if (packed) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (kUnits % kThreads != 0 && tid + e * kThreads >= kUnits) continue;
        const Unit x = unit_of(n, e);
        const uint32_t* w = x.rec + x.inner * (DP * BITS) + x.l * LW;
        if constexpr (BITS == 2) {
          words[e][0] = w[x.i >> 1], words[e][1] = w[(S + x.i) >> 1];
        } else if constexpr (BITS == 4) {
          words[e][0] = w[x.i], words[e][1] = w[S + x.i];
        } else if constexpr (BITS == 8) {
          words[e][0] = w[2 * x.i], words[e][1] = w[2 * x.i + 1];
          words[e][2] = w[2 * (S + x.i)], words[e][3] = w[2 * (S + x.i) + 1];
        }
        const u32x4* p = reinterpret_cast<const u32x4*>(
            x.rec + g.kparams_at + (quotient(x.inner * 32, g.G, g.group_magic) * DP + 8 * S * x.q + 8 * x.i) * 2);
#pragma unroll
        for (int k = 0; k < 4; ++k) stage[4 * e + k] = p[k];
      }
    } else {
      fetch_key_rows(stage, n.t0, n.keys);
    }
  };
  const auto fetch_values = [&](const Next& n, bool packed) {
    if (packed) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (kUnits % kThreads != 0 && tid + e * kThreads >= kUnits) continue;
        const Unit x = unit_of(n, e);
        const uint32_t* w = x.rec + g.vcodes_at + x.inner * (DP * BITS) + x.l * LW;
#pragma unroll
        for (int k = 0; k < BITS / 2; ++k) words[e][k] = w[BITS / 2 * x.i + k];
        const uint2* p = reinterpret_cast<const uint2*>(x.rec + g.vparams_at) + (x.inner * 32 + 4 * x.q) * ncg +
                         quotient(32 * x.i, g.G, g.group_magic);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint2 y = p[(k / 2 * 16 + k % 2 * 2) * ncg], z = p[(k / 2 * 16 + k % 2 * 2 + 1) * ncg];
          stage[4 * e + k] = u32x4{y.x, y.y, z.x, z.y};
        }
      }
    } else {
      fetch_value_rows(stage, n.t0, n.values);
    }
  };
  // x[j] = code * scale + zero with the pairs of unit e
  const auto decode = [&](int e, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      x[j] = fmaf(x[j], __uint_as_float(stage[4 * e + j / 2][j % 2 * 2]), __uint_as_float(stage[4 * e + j / 2][j % 2 * 2 + 1]));
  };
  const auto put_keys = [&](const Next& n, bool packed, T* kt) {
    if (packed) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (kUnits % kThreads != 0 && tid + e * kThreads >= kUnits) continue;
        const Unit u = unit_of(n, e);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t tau = 32 * u.b + 16 * h + u.l % 16;
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          codes_to<BITS>(words[e] + (BITS == 8 ? 2 * h : h), BITS == 2 ? (h * S + u.i) & 1 : 0, x);
          decode(e, x);
          if ((int)tau < n.keys) put_terms<T, KT>(x, kt + tau * kKeyPitch + 8 * S * u.q + 8 * u.i, Tile::kKeys);
        }
      }
    } else {
      put_key_rows(stage, n.keys, kt);
    }
  };
  const auto put_values = [&](const Next& n, bool packed, T* vt, uint32_t* marks) {
    if (packed) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (kUnits % kThreads != 0 && tid + e * kThreads >= kUnits) continue;
        const Unit u = unit_of(n, e);
        const int rest = n.values - (int)(32 * u.b);  // packed tokens from the block's first on
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          codes_to<BITS>(words[e] + (BITS == 8 ? 2 * h : BITS == 4 ? h : 0), BITS == 2 ? h : 0, x);
          decode(e, x);
          T* to = vt + (32 * u.i + 16 * h + u.l % 16) * kValuePitch + 32 * u.b + 8 * u.q;
          if (n.edge) {
            uint32_t found = 0;
            const bool held = u.b == 0 ? n.held[0] : n.held[1];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int tau = j / 4 * 16 + 4 * (int)u.q + j % 4;
              const bool fine = fabsf(x[j]) <= kLargest, here = held && tau < rest;
              found |= here && !fine ? 1u << tau : 0u;
              x[j] = here && fine ? x[j] : 0.f;
            }
            if (found != 0) atomicOr(&marks[u.b], found);
          }
          if (n.values == TT) {
            put_terms<T, VT>(x, to, Tile::kValues);
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              if (j / 4 * 16 + 4 * (int)u.q + j % 4 >= rest) continue;
              to[j] = (T)x[j];
              if constexpr (VT == 2) to[Tile::kValues + j] = (T)(x[j] - (float)(T)x[j]);
            }
          }
        }
      }
    } else {
      put_value_rows(stage, n.values, n.edge, vt, marks);
    }
  };
  // A layout that the units do not know (groups of no multiple of 32, other head widths): element by element.
  const auto fill_any = [&](const Next& n, T* kt, uint32_t* marks) {
    T* vt = kt + KT * Tile::kKeys;
    const uint32_t bits = g.bits, gs = g.S();
#pragma unroll 1
    for (uint32_t i = tid; i < kKeyPieces; i += kThreads) {
      const uint32_t tau = i / (DP / 8), d = i % (DP / 8) * 8;
      const int64_t t = n.t0 + tau;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if ((int)tau < n.keys) {
        const uint32_t* r = tau < 32 ? n.rec[0] : n.rec[1];
        const uint32_t inner = tau < 32 ? n.inner[0] : n.inner[1];
        if (d < g.DP) {
          const uint32_t o = d / 8, frag = tau % 32 / 16 * gs + o % gs;
          const uint32_t* words = r + inner * g.block_words() + (o / gs * 16 + tau % 16) * g.lane_words();
          const float2* pairs = reinterpret_cast<const float2*>(r + g.kparams_at) + quotient(inner * 32 + tau % 32, g.G, g.group_magic) * g.DP + d;
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            x[j] = decoded<T>(words[paged_word(bits, frag, j)] >> paged_bit(bits, frag, j) & g.levels(), pairs[j]);
        }
      } else if (t < w.hi && d < DW) {
        const Frag f = load_frag(row_of<T>(g, a.c.kwin, s, head, t, a.keys), d);
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = (float)f[j];
      }
      put_terms<T, KT>(x, kt + tau * kKeyPitch + d, Tile::kKeys);
    }
#pragma unroll 1
    for (uint32_t i = tid; i < TT * DP; i += kThreads) {
      const uint32_t d = i % DP, tau = i / DP;
      const int64_t t = n.t0 + tau;
      const bool held = (int)tau >= n.values || (tau < 32 ? n.held[0] : n.held[1]);
      float x = held && d < D && t < w.hi ? value_of<T>(a, s, tau < 32 ? n.rec[0] : n.rec[1], head, t, vq, d) : 0.f;
      if (n.edge && !(fabsf(x) <= kLargest)) {
        atomicOr(&marks[tau / 32], 1u << tau % 32);
        x = 0.f;
      }
      T* to = vt + d * kValuePitch + slot(tau);
      to[0] = (T)x;
      if constexpr (VT == 2) to[Tile::kValues] = (T)(x - (float)to[0]);
    }
  };

  // Both passes of a tile's keys and of its values, one after the other.
  const auto fill_both = [&](const Next& n, bool keys, bool values, T* kt, uint32_t* marks) {
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
      if (keys && (pass == 0 ? n.keys > 0 : n.keys < TT)) {
        fetch_keys(n, pass == 0);
        put_keys(n, pass == 0, kt);
      }
      if (values && (pass == 0 ? n.values > 0 : n.values < TT)) {
        fetch_values(n, pass == 0);
        put_values(n, pass == 0, kt + KT * Tile::kKeys, marks);
      }
    }
  };
  const auto whole = [](int packed) { return packed == 0 || packed == TT; };

  // logit += keys . queries; four fragments are read while the four before are multiplied
  const auto add_logits = [&](f32x16(&logit)[kSub], const T* keys) {
    Frag f[2][4];
    constexpr int kAll = DP / 16 * (int)kSub, kGroups = (kAll + 3) / 4;
    const auto read = [&](int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (4 * n + j) / (int)kSub, sub = (4 * n + j) % (int)kSub;
        if (4 * n + j < kAll) f[n % 2][j] = *reinterpret_cast<const Frag*>(keys + (32 * sub + col) * kKeyPitch + 16 * i + 8 * half);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    read(0);
#pragma unroll
    for (int n = 0; n < kGroups; ++n) {
      if (n + 1 < kGroups) read(n + 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = (4 * n + j) / (int)kSub, sub = (4 * n + j) % (int)kSub;
        if (4 * n + j < kAll) logit[sub] = Mma<T>::mul(f[n % 2][j], q[i], logit[sub]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // acc += values^T . weights; two products of two steps of 32 channels at a time (the last of an odd number: of one)
  const auto add_values = [&](const Frag(&p)[kSub][2], const T* values) {
    Frag f[2][4];
    constexpr int kAll = DP / 32 * (int)kSub * 2, kGroups = (kAll + 3) / 4;
    const auto step = [](int x, int* i, int* sub, int* u) {
      constexpr int kEven = DP / 64 * 2, kOf = 2 * (int)kSub;  // products of a step
      const bool two = x < kEven * kOf;
      *i = two ? x / (2 * kOf) * 2 + x % 2 : kEven;
      const int y = two ? x % (2 * kOf) / 2 : x - kEven * kOf;
      *sub = y / 2, *u = y % 2;
    };
    const auto read = [&](int n) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int i, sub, u;
        step(4 * n + j, &i, &sub, &u);
        if (4 * n + j < kAll) f[n % 2][j] = *reinterpret_cast<const Frag*>(values + (32 * i + col) * kValuePitch + 32 * sub + 16 * u + 8 * half);
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    read(0);
#pragma unroll
    for (int n = 0; n < kGroups; ++n) {
      if (n + 1 < kGroups) read(n + 1);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int i, sub, u;
        step(4 * n + j, &i, &sub, &u);
        if (4 * n + j < kAll) acc[i] = Mma<T>::mul(f[n % 2][j], p[sub][u], acc[i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Softmax: the running maximum and sum, what is summed so far rescaled, logits to weights.
  const auto weigh = [&](const f32x16(&logit)[kSub], Frag(&p)[kSub][2]) {
    float higher = top;
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub)
#pragma unroll
      for (uint32_t i = 0; i < 16; i += 2) higher = max_of(higher, logit[sub][i], logit[sub][i + 1]);
    higher = max_with<32>(higher);
    const float base = higher == -INFINITY ? 0.f : higher * scale;  // a row that has seen nothing yet
    // always: a branch round it has the sums in two sets of registers where it joins
    const float keep = top == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(fmaf(top, scale, -base));
    sum *= keep;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] *= keep;
    top = higher;
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(fmaf(logit[sub][i], scale, -base));
        sum += x;
        // accumulator rows 8 b + 4 half + j: product u takes b = u and b = u + 2
        p[sub][i / 4 % 2][i % 4 + (i >= 8 ? 4 : 0)] = (T)x;
      }
    }
  };

  // Logits of what a row does not see (held: whether the blocks' pages are there) become -inf.
  const auto hide = [&](f32x16(&logit)[kSub], int64_t t0, bool held0, bool held1) {
    const int mine = (int)(lane_anew() / 32 * 4);
    const int64_t pos = at0 + row_now() / gq;
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
      // counted from the sub-tile's first token
      const int64_t from = t0 + 32 * sub;
      const int see_to = clamped(pos - from, -1, 31), see_from = clamped(left_of(a, pos) - from, -1, 31);
      const int sinks = clamped((int64_t)a.sinks - from, 0, 32), held = (sub == 0 ? held0 : held1) ? 0 : clamped(kq - from, 0, 32);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int tau = 8 * (i / 4) + mine + i % 4;
        const bool seen = tau <= see_to && (tau > see_from || tau < sinks) && tau >= held;
        logit[sub][i] = seen ? logit[sub][i] : -INFINITY;
      }
    }
  };
  // Values that were left out of a tile, for the rows that see them.
  const auto add_bad = [&](const Frag(&p)[kSub][2], const uint32_t* marks, int64_t t0, const uint32_t* rec0, const uint32_t* rec1) {
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
      for (uint32_t rest = marks[sub]; rest != 0; rest &= rest - 1) {
        const uint32_t tau = __ffs(rest) - 1;
        const int64_t t = t0 + 32 * sub + tau;
        wave_fence();
#pragma unroll 1
        for (uint32_t d = lane_anew(); d < DP; d += 64) {
          const float x = d < D ? value_of<T>(a, s, sub == 0 ? rec0 : rec1, head, t, vq, d) : 0.f;
          bad_row[wave][d] = fabsf(x) <= kLargest ? 0.f : x;
        }
        wave_fence();
        float weight = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i)
          if (i == tau / 8 * 4 + tau % 4) weight = (float)p[sub][i / 4 % 2][i % 4 + (i >= 8 ? 4 : 0)];
        weight = __shfl(weight, (int)(tau % 8 / 4 * 32 + col));
        const int64_t pos = at0 + row_now() / gq;
        const bool seen = t <= pos && (t > left_of(a, pos) || t < (int64_t)a.sinks);
        const uint32_t mine = lane_anew() / 32 * 4;
#pragma unroll
        for (int i = 0; i < DP / 32; ++i)
#pragma unroll
          for (uint32_t e = 0; e < 16; ++e)
            if (seen) acc[i][e] += weight * bad_row[wave][32 * i + 8 * (e / 4) + mine + e % 4];
      }
    }
  };

  // ---- plain tiles. A wave's units lie in one block each, so all but the lane's place in it is uniform. What
  // the next tile is made of is fetched a tile ahead, its pages a tile before that.
  if constexpr (BITS != 0) {
    const uint32_t to = part.to < plains ? part.to : plains;
    struct {
      u32x4 pairs[kEach][4];
      uint32_t words[kEach][kWords];
    } keys, values;
    const auto tile_of = [&](uint32_t it) {  // in the sequence
      const uint32_t at = plain_at + it;
      return at < w.head_tiles ? at : w.first_tile + (at - w.head_tiles);
    };
    const auto look_up = [&](uint32_t it) {  // lane i: page of block i
      const uint32_t page = quotient(tile_of(it < to ? it : to - 1) * kSub + lane % kSub, g.page_blocks, g.page_magic);
      return page < a.b.per_sequence ? s.table[page] : -1;
    };
    const auto missing = [&](int32_t pages) {  // bit i: block i has no page
      uint32_t bits = 0;
#pragma unroll
      for (uint32_t i = 0; i < kSub; ++i) bits |= (uint32_t)__builtin_amdgcn_readlane(pages, i) < g.pages ? 0u : 1u << i;
      return bits;
    };
    // record and place in the page of the wave's unit e (no page: the pool's first)
    const auto place_of = [&](uint32_t it, int32_t pages, int e, const uint32_t** rec, uint32_t* inner, uint32_t* i) {
      const uint32_t unit = wave + e * WAVES, b = unit / S, block = tile_of(it) * kSub + b;
      *i = unit % S;
      *inner = block - quotient(block, g.page_blocks, g.page_magic) * g.page_blocks;
      const uint32_t page = __builtin_amdgcn_readlane(pages, b);
      *rec = a.c.pages + ((uint64_t)(page < g.pages ? page : 0) * g.heads + head) * g.record_words;
    };
    const auto mine = [&](int e) { return kSub * S % WAVES == 0 || wave + e * WAVES < kSub * S; };
    const auto at = [](const uint32_t* p, uint32_t words) { return reinterpret_cast<const char*>(p) + words * 4; };
    const auto fetch_plain_keys = [&](uint32_t it, int32_t pages) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (!mine(e)) continue;
        const uint32_t* rec;
        uint32_t inner, i;
        place_of(it, pages, e, &rec, &inner, &i);
        const char* from = at(rec + inner * (DP * BITS), lane * LW);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if constexpr (BITS == 8) {
            keys.words[e][2 * h] = reinterpret_cast<const uint32_t*>(from)[2 * (h * S + i)];
            keys.words[e][2 * h + 1] = reinterpret_cast<const uint32_t*>(from)[2 * (h * S + i) + 1];
          } else {
            keys.words[e][h] = reinterpret_cast<const uint32_t*>(from)[BITS == 2 ? (h * S + i) >> 1 : h * S + i];
          }
        }
        const char* p = at(rec + g.kparams_at + (quotient(inner * 32, g.G, g.group_magic) * DP + 8 * i) * 2, lane / 16 * (16 * S));
#pragma unroll
        for (int k = 0; k < 4; ++k) keys.pairs[e][k] = reinterpret_cast<const u32x4*>(p)[k];
      }
    };
    const auto fetch_plain_values = [&](uint32_t it, int32_t pages) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (!mine(e)) continue;
        const uint32_t* rec;
        uint32_t inner, i;
        place_of(it, pages, e, &rec, &inner, &i);
        const char* from = at(rec + g.vcodes_at + inner * (DP * BITS) + BITS / 2 * i, lane * LW);
#pragma unroll
        for (int k = 0; k < BITS / 2; ++k) values.words[e][k] = reinterpret_cast<const uint32_t*>(from)[k];
        const uint32_t* pairs = rec + g.vparams_at + (inner * 32 * ncg + quotient(32 * i, g.G, g.group_magic)) * 2;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t t = k / 2 * 16 + k % 2 * 2;
          const uint2 y = *reinterpret_cast<const uint2*>(at(pairs + t * ncg * 2, lane / 16 * ncg * 8));
          const uint2 z = *reinterpret_cast<const uint2*>(at(pairs + (t + 1) * ncg * 2, lane / 16 * ncg * 8));
          values.pairs[e][k] = u32x4{y.x, y.y, z.x, z.y};
        }
      }
    };
    const auto decode_by = [](const u32x4(&pairs)[4], float(&x)[8]) {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = fmaf(x[j], __uint_as_float(pairs[j / 2][j % 2 * 2]), __uint_as_float(pairs[j / 2][j % 2 * 2 + 1]));
    };
    const auto put_plain_keys = [&](T* kt) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (!mine(e)) continue;
        const uint32_t unit = wave + e * WAVES, b = unit / S, i = unit % S;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
          codes_to<BITS>(keys.words[e] + (BITS == 8 ? 2 * h : h), BITS == 2 ? (h * S + i) & 1 : 0, x);
          decode_by(keys.pairs[e], x);
          put_terms<T, KT>(x, kt + (32 * b + 16 * h + lane % 16) * kKeyPitch + 8 * S * (lane / 16) + 8 * i, Tile::kKeys);
        }
      }
    };
    const auto put_plain_values = [&](T* vt, uint32_t gone) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        if (!mine(e)) continue;
        const uint32_t unit = wave + e * WAVES, b = unit / S, i = unit % S;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
          codes_to<BITS>(values.words[e] + (BITS == 8 ? 2 * h : BITS == 4 ? h : 0), BITS == 2 ? h : 0, x);
          decode_by(values.pairs[e], x);
          if (gone >> b & 1) {  // no weight of zero keeps an infinity out
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
          }
          put_terms<T, VT>(x, vt + (32 * i + 16 * h + lane % 16) * kValuePitch + 32 * b + 8 * (lane / 16), Tile::kValues);
        }
      }
    };
    if (part.from < to) {
      int32_t pages = look_up(part.from), pages_next = look_up(part.from + 1);
      uint32_t gone = missing(pages), gone_next = missing(pages_next);
      fetch_plain_keys(part.from, pages);
      fetch_plain_values(part.from, pages);
      put_plain_keys(tiles);
      put_plain_values(tiles + KT * Tile::kKeys, gone);
      fetch_plain_keys(part.from + 1 < to ? part.from + 1 : part.from, pages_next);
      fetch_plain_values(part.from + 1 < to ? part.from + 1 : part.from, pages_next);
      pages = look_up(part.from + 2);
      T* kt = tiles;
      T* other = tiles + Tile::kElements;
#pragma unroll 1
      for (uint32_t it = part.from; it < to; ++it) {
        __syncthreads();  // this tile is filled, the other one read
        pages_next = look_up(it + 3);
        const uint32_t then = it + 2 < to ? it + 2 : to - 1;  // fetched again behind the end, and dropped
        __builtin_amdgcn_sched_barrier(0);
        f32x16 logit[kSub];
#pragma unroll
        for (uint32_t sub = 0; sub < kSub; ++sub) logit[sub] = f32x16{0.f};
        add_logits(logit, kt);
        if constexpr (KT == 2) add_logits(logit, kt + Tile::kKeys);
        if (gone != 0) {
#pragma unroll
          for (uint32_t sub = 0; sub < kSub; ++sub)
            if (gone >> sub & 1) {
#pragma unroll
              for (uint32_t i = 0; i < 16; ++i) logit[sub][i] = -INFINITY;
            }
        }
        Frag p[kSub][2];
        weigh(logit, p);
        __builtin_amdgcn_sched_barrier(0);
        put_plain_keys(other);
        __builtin_amdgcn_sched_barrier(0);
        gone = gone_next, gone_next = missing(pages);
        fetch_plain_keys(then, pages);
        __builtin_amdgcn_sched_barrier(0);
        add_values(p, kt + KT * Tile::kKeys);
        if constexpr (VT == 2) add_values(p, kt + KT * Tile::kKeys + Tile::kValues);
        put_plain_values(other + KT * Tile::kKeys, gone);  // of the next tile by now
        __builtin_amdgcn_sched_barrier(0);
        fetch_plain_values(then, pages);
        pages = pages_next;
        T* const swap = kt;
        kt = other, other = swap;
      }
      __syncthreads();
    }
  }

  // ---- tiles of rows, fetched a tile ahead
  {
    const uint32_t first = part.from > plains ? part.from : plains, to = part.to < plains + denses ? part.to : plains + denses;
    const auto start_of = [&](uint32_t it) {
      const uint32_t at = dense_at + (it < to ? it : to - 1) - plains;
      return (int64_t)(at < w.head_tiles ? at : w.first_tile + (at - w.head_tiles)) * TT;
    };
    const auto edge_of = [&](int64_t t0) { return t0 + TT - 1 > first_pos || t0 <= last_left; };
    u32x4 key_rows[kMost], value_rows[kMost];
    if (first < to) {
      int64_t t0 = start_of(first), next = start_of(first + 1);
      fetch_key_rows(key_rows, t0, 0);
      fetch_value_rows(value_rows, t0, 0);
      put_key_rows(key_rows, 0, tiles);
      put_value_rows(value_rows, 0, edge_of(t0), tiles + KT * Tile::kKeys, bad[first % 3]);
      fetch_key_rows(key_rows, next, 0);
      fetch_value_rows(value_rows, next, 0);
      T* kt = tiles;
      T* other = tiles + Tile::kElements;
#pragma unroll 1
      for (uint32_t it = first; it < to; ++it) {
        __syncthreads();  // this tile is filled, the other one read
        if (tid < 2) bad[(it + 2) % 3][tid] = 0;
        const int64_t then = start_of(it + 2);  // the last one again behind the end, dropped
        const bool edge = edge_of(t0);
        __builtin_amdgcn_sched_barrier(0);
        f32x16 logit[kSub];
#pragma unroll
        for (uint32_t sub = 0; sub < kSub; ++sub) logit[sub] = f32x16{0.f};
        add_logits(logit, kt);
        if (edge && !(t0 + TT - 1 <= all_pos && t0 > all_left)) hide(logit, t0, true, true);
        Frag p[kSub][2];
        weigh(logit, p);
        __builtin_amdgcn_sched_barrier(0);
        put_key_rows(key_rows, 0, other);
        __builtin_amdgcn_sched_barrier(0);
        fetch_key_rows(key_rows, then, 0);
        __builtin_amdgcn_sched_barrier(0);
        add_values(p, kt + KT * Tile::kKeys);
        if (edge && (bad[it % 3][0] | bad[it % 3][1]) != 0) add_bad(p, bad[it % 3], t0, nullptr, nullptr);
        if (it + 1 < to) put_value_rows(value_rows, 0, edge_of(next), other + KT * Tile::kKeys, bad[(it + 1) % 3]);
        __builtin_amdgcn_sched_barrier(0);
        fetch_value_rows(value_rows, then, 0);
        t0 = next, next = then;
        T* const swap = kt;
        kt = other, other = swap;
      }
      __syncthreads();
      if (tid < 6) bad[tid / 2][tid % 2] = 0;
      __syncthreads();
    }
  }

  // ---- the other tiles
  const uint32_t from = part.from > plains + denses ? part.from : plains + denses;
  Next now = locate(from);
  if (from < part.to) {
    if constexpr (BITS == 0)
      fill_any(now, tiles, bad[from % 3]);
    else
      fill_both(now, true, true, tiles, bad[from % 3]);
  }
#pragma unroll 1
  for (uint32_t it = from; it < part.to; ++it) {
    __syncthreads();  // this tile is filled, the other one read
    if (tid < 2) bad[(it + 2) % 3][tid] = 0;
    const bool more = it + 1 < part.to;
    const Next next = locate(more ? it + 1 : it);
    if (BITS != 0 && more && whole(next.keys)) fetch_keys(next, next.keys > 0);
    const T* kt = tiles + (it - from) % 2 * Tile::kElements;
    const T* vt = kt + KT * Tile::kKeys;
    T* next_kt = tiles + (it + 1 - from) % 2 * Tile::kElements;
    const int64_t t0 = now.t0;
    const bool two_keys = BITS == 0 || now.keys > 0, two_values = BITS == 0 || now.values > 0;  // both terms
    // phases one after the other: interleaved, they want more registers than there are
    __builtin_amdgcn_sched_barrier(0);
    f32x16 logit[kSub];
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) logit[sub] = f32x16{0.f};
    add_logits(logit, kt);
    if (KT == 2 && two_keys) add_logits(logit, kt + Tile::kKeys);
    if (now.edge && !(t0 + TT - 1 <= all_pos && t0 > all_left && t0 >= kq)) hide(logit, t0, now.held[0], now.held[1]);
    Frag p[kSub][2];
    weigh(logit, p);
    __builtin_amdgcn_sched_barrier(0);
    if (BITS != 0 && more) {
      if (whole(next.keys)) put_keys(next, next.keys > 0, next_kt);
      if (whole(next.values)) fetch_values(next, next.values > 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    add_values(p, vt);
    if (VT == 2 && two_values) add_values(p, vt + Tile::kValues);
    if (now.edge && (bad[it % 3][0] | bad[it % 3][1]) != 0) add_bad(p, bad[it % 3], t0, now.rec[0], now.rec[1]);
    if (more) {
      if constexpr (BITS == 0) {
        fill_any(next, next_kt, bad[(it + 1) % 3]);
      } else {
        if (whole(next.values)) put_values(next, next.values > 0, next_kt + KT * Tile::kKeys, bad[(it + 1) % 3]);
        if (!whole(next.keys) || !whole(next.values))
          fill_both(next, !whole(next.keys), !whole(next.values), next_kt, bad[(it + 1) % 3]);
      }
    }
    now = next;
  }

  sum = sum_with<32>(sum);
  if (tile_row + wave * 32 + lane_anew() % 32 >= rows) return;
  top *= scale;
  const uint32_t row = row_now(), token = row / gq, qhead = head * gq + row % gq;
  const uint64_t place = (uint64_t)(s.row0 + token) * a.qh + qhead;
  if (part.count == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.out) + (uint64_t)(s.row0 + token) * a.out_stride + (uint64_t)qhead * D;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (uint32_t b = 0; b < 4; ++b) {
        const uint32_t d = 32 * i + 8 * b + 4 * half;
        if (a.out_vec) {  // D is a multiple of 8: four channels are there or not
          struct alignas(4 * sizeof(T)) Four {
            T x[4];
          } four;
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) four.x[e] = (T)(acc[i][4 * b + e] * inv);
          if (d < D) *reinterpret_cast<Four*>(out + d) = four;
        } else {
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e)
            if (d + e < D) out[d + e] = (T)(acc[i][4 * b + e] * inv);
        }
      }
  } else {
    const uint64_t all = (uint64_t)a.b.rows * a.qh;
    float* to = partial + (split * all + place) * g.DP;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (uint32_t b = 0; b < 4; ++b)
        if (32u * i < g.DP)
          *reinterpret_cast<f32x4*>(to + 32 * i + 8 * b + 4 * half) = f32x4{acc[i][4 * b], acc[i][4 * b + 1], acc[i][4 * b + 2], acc[i][4 * b + 3]};
    if (half == 0)
      *reinterpret_cast<float2*>(partial + splits * all * g.DP + (split * all + place) * 2) =
          make_float2(sum == 0.f ? -INFINITY : top, sum);
  }
}

// Joins the splits of 16 rows of one KV head: a wave takes four at once (one after the other they would wait
// for memory eight times), its lanes over the channels.
constexpr uint32_t kJoinRows = 16;
template <class T>
__global__ void __launch_bounds__(256) k_paged_chunk_join(PagedAttention a, ChunkPlan plan, const float* partial) {
  constexpr int kAtOnce = kJoinRows / 4;
  const PagedGeometry& g = a.c.geo;
  const PagedSequence s = paged_sequence(a.b, g, blockIdx.z);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq, lane = threadIdx.x % 64, head = blockIdx.x % g.heads;
  const uint32_t first = blockIdx.x / g.heads * kJoinRows;
  if (rows <= plan.over || first >= rows) return;
  const uint32_t r0 = first / plan.tile_rows * plan.tile_rows;
  const Walk w = walk_of(a, s, r0, r0 + plan.tile_rows < rows ? r0 + plan.tile_rows : rows, gq, plan.tile);
  const uint32_t count = part_of(w.tiles, plan.splits, 0).count;
  if (count == 1) return;
  const uint64_t all = (uint64_t)a.b.rows * a.qh;
  const float2* state = reinterpret_cast<const float2*>(partial + plan.splits * all * g.DP);
  const uint32_t mine = first + threadIdx.x / 64 * kAtOnce;  // this wave's first row; those past the end are the last one again
  uint64_t place[kAtOnce];
  float2 st[kAtOnce];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    const uint32_t r = mine + i < rows ? mine + i : rows - 1;
    place[i] = (uint64_t)(s.row0 + r / gq) * a.qh + head * gq + r % gq;
    st[i] = lane < count ? state[lane * all + place[i]] : make_float2(-INFINITY, 0.f);  // at most 64 splits
  }
  float factor[kAtOnce], inv[kAtOnce];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    float top = st[i].x;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    factor[i] = __builtin_amdgcn_exp2f(st[i].x - (top == -INFINITY ? 0.f : top));
    float sum = factor[i] * st[i].y;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    inv[i] = sum == 0.f ? 0.f : 1.f / sum;
  }
  for (uint32_t d = lane; d < (g.D + 63) / 64 * 64; d += 64) {
    float x[kAtOnce] = {0.f, 0.f, 0.f, 0.f};
    for (uint32_t k = 0; k < count; ++k) {
      float v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) v[i] = partial[(k * all + place[i]) * g.DP + (d < g.DP ? d : 0)];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) x[i] += __shfl(factor[i], (int)k) * v[i];
    }
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const uint32_t r = mine + i;
      if (r < rows && d < g.D)
        static_cast<T*>(a.out)[(uint64_t)(s.row0 + r / gq) * a.out_stride + (uint64_t)(head * gq + r % gq) * g.D + d] = (T)(x[i] * inv[i]);
    }
  }
}

template <class T, int BITS, int S>
hipError_t chunk_launch(const PagedAttention& a, const ChunkPlan& p, float* partial, hipStream_t stream) {
  constexpr int WAVES = paged_chunk_waves(sizeof(T), S), TT = paged_chunk_tile(S);
  const PagedGeometry& g = a.c.geo;
  const uint64_t rows = (uint64_t)a.b.max_rows * (a.qh / g.heads);
  const uint64_t x = (rows + WAVES * 32 - 1) / (WAVES * 32) * p.splits * g.heads;
  const size_t bytes = ChunkTile<T, S, TT>::kBytes;
  auto kernel = k_paged_chunk<T, BITS, S>;
  hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(kernel), bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)x, 1, a.b.sequences), dim3(WAVES * 64), bytes, stream, a, p, partial);
  if (p.splits > 1) {
    const uint64_t joins = (rows + kJoinRows - 1) / kJoinRows * g.heads;
    hipLaunchKernelGGL(k_paged_chunk_join<T>, dim3((uint32_t)joins, 1, a.b.sequences), dim3(256), 0, stream, a, p, partial);
  }
  return hipGetLastError();
}

template <class T, int BITS>
hipError_t chunk_dims(const PagedAttention& a, const ChunkPlan& p, float* partial, hipStream_t stream) {
  switch (a.c.geo.S()) {
    case 1:
    case 2: return chunk_launch<T, BITS, 2>(a, p, partial, stream);
    case 3: return chunk_launch<T, BITS, 3>(a, p, partial, stream);
    case 4: return chunk_launch<T, BITS, 4>(a, p, partial, stream);
    default: return chunk_launch<T, BITS, 8>(a, p, partial, stream);
  }
}

}  // namespace

template <class T>
hipError_t launch_paged_chunk(const PagedAttention& a, const ChunkPlan& p, float* partial, hipStream_t stream) {
  const uint32_t S = a.c.geo.S();
  if (a.c.geo.G % 32 != 0 || !(S == 2 || S == 3 || S == 4 || S == 8)) return chunk_dims<T, 0>(a, p, partial, stream);
  switch (a.c.geo.bits) {
    case 2: return chunk_dims<T, 2>(a, p, partial, stream);
    case 4: return chunk_dims<T, 4>(a, p, partial, stream);
    default: return chunk_dims<T, 8>(a, p, partial, stream);
  }
}

}  // namespace kivi
