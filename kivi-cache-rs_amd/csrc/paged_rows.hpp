// paged_rows.hpp — attention of few rows (decoded tokens, drafted tokens) over the paged cache: the
// kernel, and its launch for one element type (kernels_paged_rows_*.hip instantiate it).
//
// Bound by the packed bytes it reads (2 bits, D = 128: 4 KB per 32 tokens and KV head), if the vector
// ALU keeps up. So codes go to the matrix cores as they are, and (scale, zero) to the other operand,
// which has few rows:
//
//   q . k_t          = sum_d (q_d s_d) c_td + sum_d q_d z_d         (s, z of the token's group)
//   sum_t p_t v_td   = sum_t (p_t s_t) c_td + sum_t p_t z_t         (s, z of the channel's group)
//
// Codes are exact in bf16 (0 .. 255); q s and p s are split into bf16 terms that add up to 16 bits
// (f16, bf16) or 24 (f32), so nothing depends on the magnitudes and an output of 16 bits loses nothing to
// them. The products accumulate in f32; the z sums are f32.
//
// The 16 columns of the matrix instructions hold BLOCKS groups of 16 / BLOCKS rows, each group with
// the operand of another 32-token block: the scaled operands of BLOCKS blocks (the vector work per
// block, and the softmax) are then made at once, in lanes that would otherwise be idle. Tile (block b)
// times columns of another block is ignored (keys) or zero (values). Every column keeps its own running
// maximum and sum; they are joined at the end.
//
// That is for packed values. The last blocks (the windows, up to R and a few tokens, and new rows that come
// with the call) go block by block, a wave each, in workgroups of their own: keys and values as rows of the
// caller's type, packed keys among them decoded, through the type's own matrix instructions.
#pragma once

#include <algorithm>

#include "common.hpp"
#include "paged_attn.hpp"

namespace kivi {
namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mul16(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mul16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mul16(f32x8 a, f32x8 b, f32x4 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

union Operand {
  uint32_t u[4];
  bf16x8 v;
};

// Fragment f (a constant) of a lane's code words as exact bf16 integers. The packed converters take the
// codes as fp4 (0 1 2 3 are 0, 1/2, 1, 3/2) and fp8 (n is n 2^-9) times a scale.
template <int BITS>
__device__ __forceinline__ bf16x8 codes_of(const uint32_t* w, int f) {
  Operand o;
  if constexpr (BITS == 2) {
    const uint32_t m = (f & 1 ? w[f >> 1] >> 2 : w[f >> 1]) & 0x33333333u;
    o.u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(m, 2.0f, 0));
    o.u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(m, 2.0f, 1));
    o.u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(m, 2.0f, 2));
    o.u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(m, 2.0f, 3));
  } else if constexpr (BITS == 4) {
    const uint32_t lo = w[f] & 0x0f0f0f0fu, hi = w[f] >> 4 & 0x0f0f0f0fu;
    o.u[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false));
    o.u[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true));
    o.u[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false));
    o.u[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true));
  } else {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const uint32_t x = w[2 * f + k];
      const uint32_t a = __float_as_uint((float)(x & 255u)), b = __float_as_uint((float)(x >> 8 & 255u));
      const uint32_t c = __float_as_uint((float)(x >> 16 & 255u)), d = __float_as_uint((float)(x >> 24));
      o.u[2 * k] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      o.u[2 * k + 1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
    }
  }
  return o.v;
}

// x0, x1 as NT bf16 terms each, packed: term k of both in t[k]. All but the last are cut (what is cut
// goes to the next), the last is rounded: NT terms hold 8 NT bits.
template <int NT>
__device__ __forceinline__ void terms_of(float x0, float x1, uint32_t (&t)[NT]) {
#pragma unroll
  for (int k = 0; k < NT - 1; ++k) {
    t[k] = __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
    x0 -= __uint_as_float(__float_as_uint(x0) & 0xffff0000u);
    x1 -= __uint_as_float(__float_as_uint(x1) & 0xffff0000u);
  }
  const bf16x2 last = {(__bf16)x0, (__bf16)x1};
  t[NT - 1] = __builtin_bit_cast(uint32_t, last);
}

// LDS of one wave: staged (scale, zero) pairs of BLOCKS blocks, padded so that the 16 different
// addresses of a read (lanes of one row of 16 differ by column group, rows of 16 by q) fall on
// different banks. Offsets in words.
__host__ __device__ constexpr uint32_t key_pitch(uint32_t S) { return 16 * S + 4; }        // channels of one q
__host__ __device__ inline uint32_t value_pitch(uint32_t ncg) { return 8 * ncg + 4; }       // four tokens
__host__ __device__ inline uint32_t value_block(uint32_t ncg) { return 8 * value_pitch(ncg) + 16; }
__host__ __device__ inline uint32_t rows_wave_words(uint32_t S, uint32_t ncg, uint32_t blocks) {
  const uint32_t k = 4 * key_pitch(S), v = value_block(ncg);
  return blocks * (k + v);
}
// Of the last blocks: values [32 tokens][DP], rows padded so that the four token quads of a transposed
// read fall on different banks (16 bytes: four rows on are 16 words on).
template <class T>
__host__ __device__ constexpr uint32_t tile_pitch(uint32_t S) { return 32 * S + 16 / sizeof(T); }  // elements
template <class T>
__host__ __device__ inline uint32_t wave_words(uint32_t S, uint32_t ncg, uint32_t blocks) {
  const uint32_t pairs = rows_wave_words(S, ncg, blocks), tile = 32 * tile_pitch<T>(S) * sizeof(T) / 4;
  return ((pairs > tile ? pairs : tile) + 3) / 4 * 4;
}
// LDS of a workgroup of four waves: queries [rows][DP + 4], then the waves' pairs, whose place the
// waves' outputs [4][rows][DP], states [4][16] and the rows' 1 / sum take at the end.
template <class T>
__host__ __device__ inline uint32_t rows_lds_words(uint32_t S, uint32_t ncg, uint32_t blocks) {
  const uint32_t rows = 16 / blocks, pairs = 4 * wave_words<T>(S, ncg, blocks), ends = 4 * rows * 32 * S + 128 + 16;
  return rows * (32 * S + 4) + (pairs > ends ? pairs : ends);
}

// A lane's N code words.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&words)[N], const uint32_t* from) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const u32x4 x = reinterpret_cast<const u32x4*>(from)[i];
      words[4 * i] = x[0], words[4 * i + 1] = x[1], words[4 * i + 2] = x[2], words[4 * i + 3] = x[3];
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = reinterpret_cast<const uint2*>(from)[i];
      words[2 * i] = x.x, words[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) words[i] = from[i];
  }
}

// How one row tile's walk is cut: the places [0, main_to) of its list of blocks have packed values and go to
// `mains` splits of `per`; the places from tail_at on have values that are rows and go to `tails` splits of
// `tail_per`. A block that has both is in both: the splits see its packed tokens, and its rows.
struct RowsPart {
  uint32_t main_to, tail_at, per, mains, tail_per, tails, count;
};
__device__ __forceinline__ uint32_t place_of(const Walk& w, uint32_t block) {
  const uint32_t p = block < w.head_tiles ? block : w.head_tiles + (block > w.first_tile ? block - w.first_tile : 0);
  return p < w.tiles ? p : w.tiles;
}
__device__ __forceinline__ RowsPart rows_part(const Walk& w, int64_t vq, const RowsPlan& plan) {
  RowsPart p;
  p.main_to = place_of(w, (uint32_t)((vq + kPagedBlock - 1) / kPagedBlock));
  p.tail_at = place_of(w, (uint32_t)(vq / kPagedBlock));
  p.per = (p.main_to + plan.splits - 1) / plan.splits;
  p.per = (p.per + plan.least - 1) / plan.least * plan.least;
  p.mains = p.main_to == 0 ? 0 : (p.main_to + p.per - 1) / p.per;
  const uint32_t last = w.tiles - p.tail_at;
  p.tail_per = ((last + plan.tails - 1) / plan.tails + 3) / 4 * 4;  // a block a wave, or as few as the plan has room for
  p.tails = last == 0 ? 0 : (last + p.tail_per - 1) / p.tail_per;
  if (p.mains + p.tails == 0) p.tails = 1, p.tail_per = 4;  // nothing seen: zeros
  p.count = p.mains + p.tails;
  return p;
}
__device__ __forceinline__ uint32_t block_at(const Walk& w, uint32_t place) {
  return place < w.head_tiles ? place : w.first_tile + (place - w.head_tiles);
}

// One workgroup: one tile of 16 / BLOCKS rows of one (sequence, KV head), one split of its 32-token
// blocks. In a split of packed blocks each of the four waves takes BLOCKS at a time. Per turn: the
// keys' pairs and codes are there; the values' are fetched while the logits are computed, the next
// turn's keys from the softmax on.
//
// Measured (MI355X, 8 KV heads of 128): 64 sequences of 500 to 32768 tokens, bf16, 2 bits, 32 query heads: 536 MB in
// 171 us (3.1 TB/s) and a join of 12; under a window of 4096, 32 sequences, 4 bits: 206 MB in 56 us. The vector ALU is
// busy 43% of the time, 1.3 waves a SIMD on average (216 registers: two fit). One sequence of 1000 tokens: 12 us, latency.
template <class T, int BITS, int S, int BLOCKS, bool HALVES>
__global__ void __launch_bounds__(256, 2) k_paged_rows(PagedAttention a, RowsPlan plan, float* partial) {
  constexpr int DP = 32 * S, F = 2 * S, LW = S * BITS / 2, ROWS = 16 / BLOCKS, NT = sizeof(T) == 4 ? 3 : 2;
  constexpr int kKeyLoads = (S + 3) / 4, kValueLoads = HALVES ? (S + 1) / 2 : (S + 3) / 4;  // float4s of pairs per lane
  constexpr uint32_t kQueryPitch = DP + 4, kKeyPitch = key_pitch(S);
  extern __shared__ __align__(16) float lds[];
  const PagedGeometry& g = a.c.geo;
  const uint32_t head = blockIdx.x, sequence = blockIdx.y, tid = threadIdx.x, lane = tid % 64;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid / 64);
  const uint32_t col = lane % 16, q = lane / 16, group = col / ROWS, r = col % ROWS;
  const PagedSequence s = paged_sequence(a.b, g, sequence);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq;
  if (rows <= plan.over || rows > plan.most) return;
  const uint32_t places = plan.splits + plan.tails;
  const uint32_t tiles = gridDim.z / places, row0 = blockIdx.z % tiles * ROWS;
  if (row0 >= rows) return;
  const uint32_t row1 = row0 + ROWS < rows ? row0 + ROWS : rows;
  const Walk w = walk_of(a, s, row0, row1, gq, kPagedBlock);
  const int64_t kq = paged_kq(g, s.n), vq = paged_vq(g, s.n);
  const RowsPart part = rows_part(w, vq, plan);
  // The last blocks first: their chain of loads is the longest. Then the first splits of all sequences: those that
  // only long ones have come last, with the workgroups that find nothing to do between them (windowed decode of 32
  // sequences 59 -> 56 us, splits fastest against this).
  const uint32_t turn = blockIdx.z / tiles;
  const bool tail = turn < plan.tails;
  if (tail ? turn >= part.tails : turn - plan.tails >= part.mains) return;
  const uint32_t split = tail ? part.mains + turn : turn - plan.tails;

  const uint32_t D = g.D, G = g.G, ncg = g.ncg, per = G / 16;
  const uint32_t row = row0 + r < rows ? row0 + r : rows - 1;
  const int64_t pos = w.total - s.m + row / gq;
  const int64_t left = a.window != 0 ? pos - (int64_t)a.window : -1;

  float* qs = lds;                                                                       // [ROWS][kQueryPitch]
  float* own = lds + ROWS * kQueryPitch + wave * wave_words<T>(S, ncg, BLOCKS);  // the wave's
  for (uint32_t i = tid; i < ROWS * DP; i += 256) {
    const uint32_t rr = i / DP, d = i % DP, ri = row0 + rr < rows ? row0 + rr : rows - 1;
    const T* p = static_cast<const T*>(a.query.p) + (uint64_t)(s.row0 + ri / gq) * a.query.stride + (uint64_t)(head * gq + ri % gq) * a.query.pitch;
    qs[rr * kQueryPitch + d] = d < D ? (float)p[d] : 0.f;
  }
  __syncthreads();
  const float* qrow = qs + r * kQueryPitch + 8 * S * q;  // this lane's channels: 8 S q + (0 .. 8 S - 1)

  const float scale = a.scale * kLog2e;
  float top = -INFINITY, sum = 0.f;
  f32x4 acc[F];
  float zacc[F];
#pragma unroll
  for (int f = 0; f < F; ++f) {
    acc[f] = f32x4{0.f, 0.f, 0.f, 0.f};
    zacc[f] = 0.f;
  }
  // Softmax of a column's next 32 logits (eight in each of its four lanes): the running maximum and sum,
  // what is summed so far rescaled, logits to weights.
  const auto weigh = [&](float(&x)[8]) {
    float peak = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) peak = fmaxf(peak, x[j]);
    peak = max_with<32>(max_with<16>(peak));
    const float next = fmaxf(top, peak);
    const float base = next == -INFINITY ? 0.f : next;
    const float shrink = __builtin_amdgcn_exp2f(top - base);
    if (__any(next != top)) {
#pragma unroll
      for (int f = 0; f < F; ++f) {
        acc[f] *= shrink;
        zacc[f] *= shrink;
      }
      sum *= shrink;
    }
    top = next;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = __builtin_amdgcn_exp2f(x[j] - base);
      sum += x[j];
    }
  };

  if (!tail) {
    float* kpairs = own;                              // [BLOCKS][4][kKeyPitch]
    float* vpairs = kpairs + BLOCKS * 4 * kKeyPitch;  // [BLOCKS][8][value_pitch] + 16
    const uint32_t vpitch = value_pitch(ncg), vblock = value_block(ncg);
    const uint32_t to = split * part.per + part.per < part.main_to ? split * part.per + part.per : part.main_to;
    // every row sees the blocks [all_from, all_to)
    const int64_t first_pos = w.total - s.m + row0 / gq, last_left = a.window != 0 ? w.hi - 1 - (int64_t)a.window : -1;
    const int64_t all_end = first_pos + 1 < vq ? first_pos + 1 : vq;
    const uint32_t all_to = all_end < 0 ? 0 : (uint32_t)(all_end / kPagedBlock);
    const uint32_t all_from = last_left < 0 ? 0 : (uint32_t)((last_left + kPagedBlock) / kPagedBlock);
    // this lane's float4s of a block's pairs, and where their words go in LDS; lanes past the end take the last
    uint32_t kget[kKeyLoads], kput[kKeyLoads], vget[kValueLoads], vput[kValueLoads];
#pragma unroll
    for (int i = 0; i < kKeyLoads; ++i) {
      kget[i] = lane + 64 * i < 16 * S ? lane + 64 * i : 16 * S - 1;
      kput[i] = 4 * kget[i] / (16 * S) * kKeyPitch + 4 * kget[i] % (16 * S);
    }
#pragma unroll
    for (int i = 0; i < kValueLoads; ++i) {
      vget[i] = lane + 64 * i < 16 * ncg ? lane + 64 * i : 16 * ncg - 1;
      vput[i] = 4 * vget[i] / (8 * ncg) * vpitch + 4 * vget[i] % (8 * ncg);
    }
    // Blocks of a turn: number, place in the page, record. One past the end or of no page is read from the
    // pool's first page (some codes and pairs) and seen by no row. Lane b looks up block b a turn ahead.
    uint32_t block[BLOCKS], inner[BLOCKS];
    const uint32_t* rec[BLOCKS];
    bool held[BLOCKS];
    uint32_t look_block, look_inner;
    int32_t look_page;
    const auto look_up = [&](uint32_t at) {
      const uint32_t place = at + lane % BLOCKS;
      look_block = block_at(w, place < to ? place : to - 1);
      const uint32_t page = quotient(look_block, g.page_blocks, g.page_magic);
      look_inner = look_block - page * g.page_blocks;
      look_page = page < a.b.per_sequence && place < to ? s.table[page] : -1;
    };
    const auto locate = [&] {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        block[b] = __builtin_amdgcn_readlane(look_block, b);
        inner[b] = __builtin_amdgcn_readlane(look_inner, b);
        const uint32_t page = __builtin_amdgcn_readlane(look_page, b);
        held[b] = page < g.pages;
        rec[b] = a.c.pages + ((uint64_t)(held[b] ? page : 0) * g.heads + head) * g.record_words;
      }
    };
    uint32_t kc[BLOCKS][LW], vc[BLOCKS][LW];
    f32x4 kp[BLOCKS][kKeyLoads], vp[BLOCKS][kValueLoads];
    const auto load_key_pairs = [&](f32x4(&pairs)[kKeyLoads], const uint32_t* record, uint32_t in_page) {
      const f32x4* from = reinterpret_cast<const f32x4*>(record + g.kparams_at + quotient(in_page, G, g.group_magic) * (DP * 2));
#pragma unroll
      for (int i = 0; i < kKeyLoads; ++i) pairs[i] = from[kget[i]];
    };
    const auto load_keys = [&] {
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        load_key_pairs(kp[b], rec[b], inner[b] * kPagedBlock);
        load_words<LW>(kc[b], rec[b] + inner[b] * (DP * BITS) + lane * LW);
      }
    };
    const auto put_key_pairs = [&](int b, const f32x4(&from)[kKeyLoads]) {
#pragma unroll
      for (int i = 0; i < kKeyLoads; ++i) *reinterpret_cast<f32x4*>(kpairs + b * 4 * kKeyPitch + kput[i]) = from[i];
    };

    uint32_t at = split * part.per + wave * BLOCKS;
    if (at < to) {
      look_up(at);
      locate();
      load_keys();
      look_up(at + 4 * BLOCKS);
    }
    while (at < to) {
      bool inside = true;  // every row sees every token of the turn
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) inside &= held[b] && block[b] >= all_from && block[b] < all_to;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const f32x4* from = reinterpret_cast<const f32x4*>(rec[b] + g.vparams_at + inner[b] * (kPagedBlock * 2) * ncg);
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) vp[b][i] = from[vget[i]];
        load_words<LW>(vc[b], rec[b] + g.vcodes_at + inner[b] * (DP * BITS) + lane * LW);
      }
      // ---- logits of eight tokens per lane: 16 half + 4 q + i
      wave_fence();
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) put_key_pairs(b, kp[b]);
      wave_fence();
      __builtin_amdgcn_sched_barrier(0);  // phases one after the other: interleaved, they want more registers than there are
      float x[8];
      uint32_t unseen = 0;  // bit j: this lane's row does not see its token j
      {
        uint32_t qk[S][NT][4];  // (q s) of this lane's group: 8 channels each
        float qz = 0.f;
        const auto fold = [&] {
          const float* pairs = kpairs + (group * 4 + q) * kKeyPitch;
          qz = 0.f;
#pragma unroll
          for (int i = 0; i < S; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const f32x4 sz = *reinterpret_cast<const f32x4*>(pairs + 16 * i + 4 * j);
              const f32x2 qq = *reinterpret_cast<const f32x2*>(qrow + 8 * i + 2 * j);
              uint32_t t[NT];
              terms_of<NT>(qq.x * sz.x, qq.y * sz.z, t);
#pragma unroll
              for (int k = 0; k < NT; ++k) qk[i][k][j] = t[k];
              qz = fmaf(qq.x, sz.y, fmaf(qq.y, sz.w, qz));
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          qz = sum_with<32>(sum_with<16>(qz));
        };
        fold();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (HALVES && half == 1) {
            // the second 16 tokens of a block may lie in the next group
            wave_fence();
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) {
              f32x4 more[kKeyLoads];
              load_key_pairs(more, rec[b], inner[b] * kPagedBlock + 16);
              put_key_pairs(b, more);
            }
            wave_fence();
            fold();
          }
          f32x4 mine = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            f32x4 c = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < S; ++i) {
              const bf16x8 codes = codes_of<BITS>(kc[b], half * S + i);
#pragma unroll
              for (int k = 0; k < NT; ++k) {
                Operand o;
#pragma unroll
                for (int j = 0; j < 4; ++j) o.u[j] = qk[i][k][j];
                c = mul16(codes, o.v, c);
              }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[i] = group == b ? c[i] : mine[i];
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) x[4 * half + i] = (mine[i] + qz) * scale;
        }
      }
      if (!inside) {
        // this lane's block, from its first token
        int64_t t0 = 0;
        bool there = false;
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          t0 = group == b ? (int64_t)block[b] * kPagedBlock : t0;
          there = group == b ? held[b] : there;
        }
        const int64_t last = pos < vq - 1 ? pos : vq - 1;  // packed tokens alone
        const int see_to = there ? clamped(last - t0, -1, 31) : -1, see_from = clamped(left - t0, -1, 31);
        const int sinks = clamped((int64_t)a.sinks - t0, 0, 32);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int tau = j / 4 * 16 + 4 * (int)q + j % 4;
          const bool seen = tau <= see_to && (tau > see_from || tau < sinks);
          x[j] = seen ? x[j] : -INFINITY;
          unseen |= seen ? 0u : 1u << j;
        }
      }
      // the next turn's keys are fetched as soon as this one's are done with
      __builtin_amdgcn_sched_barrier(0);
      at += 4 * BLOCKS;
      if (at < to) {
        locate();
        load_keys();
        look_up(at + 4 * BLOCKS);
      }
      __builtin_amdgcn_sched_barrier(0);
      weigh(x);

      // ---- output: the values' pairs go to LDS
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < kValueLoads; ++i) *reinterpret_cast<f32x4*>(vpairs + b * vblock + vput[i]) = vp[b][i];
      wave_fence();
      __builtin_amdgcn_sched_barrier(0);
      constexpr int kStep = HALVES ? 1 : 2;  // fragments that lie in one group of channels whatever G is
      const float* pairs = vpairs + group * vblock + q * vpitch;
#pragma unroll
      for (int f0 = 0; f0 < F; f0 += kStep) {
        const uint32_t cg = quotient(f0, per, g.fragment_magic);
        float y[8], z = 0.f;
        f32x2 sz[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sz[j] = *reinterpret_cast<const f32x2*>(pairs + j / 4 * 4 * vpitch + (j % 4 * ncg + cg) * 2);
        if (!inside) {
          // what is not seen has no weight, whatever its pair
#pragma unroll
          for (int j = 0; j < 8; ++j) sz[j] = unseen >> j & 1 ? f32x2{0.f, 0.f} : sz[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          y[j] = x[j] * sz[j].x;
          z = fmaf(x[j], sz[j].y, z);
        }
        zacc[f0] += cg * per == (uint32_t)f0 ? z : 0.f;
        uint32_t pk[BLOCKS][NT][4];  // (p s) of block b in the columns of group b, else zero
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t t[NT];
          terms_of<NT>(y[2 * j], y[2 * j + 1], t);
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
            for (int k = 0; k < NT; ++k) pk[b][k][j] = BLOCKS == 1 || group == b ? t[k] : 0u;
        }
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
          for (int k = 0; k < NT; ++k) {
            Operand o;
#pragma unroll
            for (int j = 0; j < 4; ++j) o.u[j] = pk[b][k][j];
#pragma unroll
            for (int f = f0; f < f0 + kStep; ++f) acc[f] = mul16(codes_of<BITS>(vc[b], f), o.v, acc[f]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  } else {
    // ---- the last blocks, one at a time, in the columns of group 0
    typedef typename Row<T>::Frag Frag;
    constexpr uint32_t kTilePitch = tile_pitch<T>(S);
    T* tile = reinterpret_cast<T*>(own);  // values [32][kTilePitch]
    const uint32_t DW = g.DW;
    // rows at one position see the same tokens, and what none sees is not read: nothing to keep apart
    const bool apart = s.m > 1;
    const int64_t first_left = a.window != 0 ? w.total - s.m + row0 / gq - (int64_t)a.window : -1;
    const uint32_t to = part.tail_at + (turn + 1) * part.tail_per < w.tiles ? part.tail_at + (turn + 1) * part.tail_per : w.tiles;
#pragma unroll 1
    for (uint32_t i = part.tail_at + turn * part.tail_per + wave; i < to; i += 4) {
      const uint32_t block = block_at(w, i);
      const int64_t t0 = (int64_t)block * kPagedBlock;
      const uint32_t page = quotient(block, g.page_blocks, g.page_magic), inner = block - page * g.page_blocks;
      const uint32_t* rec = t0 < kq ? paged_record_of(a.c, a.b, s, head, page) : nullptr;
      const int kend = clamped(kq - t0, 0, 32), vend = clamped(vq - t0, 0, 32), end = clamped(w.hi - t0, 0, 32);
      const int see_to = group == 0 ? clamped(pos - t0, -1, 31) : -1, see_from = clamped(left - t0, -1, 31);
      const int sinks = clamped((int64_t)a.sinks - t0, 0, 32);
      // the splits of packed blocks have the tokens in front of vend; keys of no page are seen by none
      const int held = rec != nullptr || kend < vend ? vend : kend;
      const int any_from = clamped(first_left - t0, -1, 31);  // no row sees (sinks, any_from]
      const auto seen = [&](int tau) { return tau <= see_to && (tau > see_from || tau < sinks) && tau >= held; };
      const auto read = [&](int tau) { return tau >= vend && tau < end && (tau > any_from || tau < sinks); };
      // rows: keys as the product reads them (token 16 half + col, channels 8 S q + 8 k), values eight lanes a token
      Frag k8[2][S];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int tau = 16 * half + (int)col;
        const bool there = tau >= kend && read(tau);
        const T* p = there ? row_of<T>(g, a.c.kwin, s, head, t0 + tau, a.keys) : nullptr;
#pragma unroll
        for (int k = 0; k < S; ++k) {
          const uint32_t d = 8 * S * q + 8 * k;
          k8[half][k] = zero_frag<T>();
          if (there && d < DW) k8[half][k] = load_frag(p, d);
        }
      }
      constexpr int kOctets = 4 * S;                     // of a row
      constexpr int kPieces = 32 * kOctets / 64;         // of a lane
      constexpr int kAhead = sizeof(T) * S <= 16 ? kPieces : kPieces / 4;  // fetched before the logits, where registers allow
      Frag v8[kAhead];
      uint32_t bad = 0;  // tokens with a value that is not finite: it goes to the rows that see them alone
      const auto piece = [&](int k, int* tau, uint32_t* d) {
        const uint32_t u = lane + 64 * k;
        *tau = (int)(u / kOctets);
        *d = u % kOctets * 8;
        return read(*tau) && *d < DW;
      };
      const auto load_values = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          int tau;
          uint32_t d;
          const bool there = piece(k0 + k, &tau, &d);
          v8[k] = zero_frag<T>();
          if (there) v8[k] = load_frag(row_of<T>(g, a.c.vwin, s, head, t0 + tau, a.values), d);
        }
      };
      const auto put_values = [&](int k0) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
          int tau;
          uint32_t d;
          (void)piece(k0 + k, &tau, &d);
          if (apart && wild<T>(v8[k])) {
            bad |= 1u << tau;
#pragma unroll
            for (int j = 0; j < 8; ++j) v8[k][j] = fabsf((float)v8[k][j]) <= kLargest ? v8[k][j] : (T)0.f;
          }
          u32x4* to = reinterpret_cast<u32x4*>(tile + tau * kTilePitch + d);
          const u32x4* from = reinterpret_cast<const u32x4*>(&v8[k]);
          to[0] = from[0];
          if constexpr (sizeof(T) == 4) to[1] = from[1];
        }
      };
      load_values(0);
      // packed keys among them
      if (kend > 0) {
        const uint32_t* from = rec != nullptr ? rec : a.c.pages;
        uint32_t code[LW];
        load_words<LW>(code, from + inner * (DP * BITS) + lane * LW);
        const f32x4* pairs = reinterpret_cast<const f32x4*>(from + g.kparams_at) + 4 * S * q;
        const uint32_t group0 = quotient(inner * kPagedBlock, G, g.group_magic);
        const uint32_t group1 = HALVES ? quotient(inner * kPagedBlock + 16, G, g.group_magic) : group0;
#pragma unroll
        for (int k = 0; k < S; ++k) {
          f32x4 p[2][4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            p[0][j] = pairs[group0 * (DP / 2) + 4 * k + j];
            p[1][j] = HALVES ? pairs[group1 * (DP / 2) + 4 * k + j] : p[0][j];
          }
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const bf16x8 c = codes_of<BITS>(code, half * S + k);
            Frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = (T)fmaf((float)c[j], p[half][j / 2][j % 2 * 2], p[half][j / 2][j % 2 * 2 + 1]);
            if (16 * half + (int)col < kend) k8[half][k] = f;
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      f32x4 c[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < S; ++k) {
        Frag q8;
#pragma unroll
        for (int j = 0; j < 8; ++j) q8[j] = (T)qrow[8 * k + j];
#pragma unroll
        for (int half = 0; half < 2; ++half) c[half] = mul16(k8[half][k], q8, c[half]);
      }
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = seen(j / 4 * 16 + 4 * (int)q + j % 4) ? c[j / 4][j % 4] * scale : -INFINITY;
      weigh(x);
      Frag p8;
#pragma unroll
      for (int j = 0; j < 8; ++j) p8[j] = (T)x[j];
      wave_fence();
#pragma unroll
      for (int k0 = 0; k0 < kPieces; k0 += kAhead) {
        if (k0 > 0) load_values(k0);
        put_values(k0);
      }
      wave_fence();
#pragma unroll
      for (int f = 0; f < F; ++f) {
        Frag t8;
#pragma unroll
        for (int j = 0; j < 8; ++j) t8[j] = tile[(j / 4 * 16 + 4 * q + j % 4) * kTilePitch + 16 * f + col];
        acc[f] = mul16(t8, p8, acc[f]);
      }
      if (__any(bad != 0)) {
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) bad |= __shfl_xor(bad, o);
        float* line = reinterpret_cast<float*>(tile);  // [DP]
        for (; bad != 0; bad &= bad - 1) {
          const int tau = __ffs(bad) - 1;
          wave_fence();
          for (uint32_t d = lane; d < DP; d += 64) {
            const float v = d < D ? value_of<T>(a, s, rec, head, t0 + tau, vq, d) : 0.f;
            line[d] = fabsf(v) <= kLargest ? 0.f : v;
          }
          wave_fence();
          float weight = 0.f;
#pragma unroll
          for (int j = 0; j < 8; ++j) weight = j == tau / 16 * 4 + tau % 4 ? x[j] : weight;
          weight = __shfl(weight, (int)(tau % 16 / 4 * 16 + col));
          const bool use = seen(tau);
#pragma unroll
          for (int f = 0; f < F; ++f)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (use) acc[f][k] += weight * line[16 * f + 4 * q + k];
        }
      }
    }
  }

  // ---- the columns of a row, over groups and waves
  sum = sum_with<32>(sum_with<16>(sum));
  if (!tail) {
    float z = 0.f;
#pragma unroll
    for (int f = 0; f < F; ++f) {
      z = f % per == 0 ? sum_with<32>(sum_with<16>(zacc[f])) : z;
      acc[f] += z;
    }
  }
  __syncthreads();  // the waves' LDS is done with
  float* outs = lds + ROWS * kQueryPitch;                           // [4][ROWS][DP]
  float2* state = reinterpret_cast<float2*>(outs + 4 * ROWS * DP);  // [4][16]
  float* inverse = reinterpret_cast<float*>(state + 64);            // [ROWS]
  if (q == 0) state[wave * 16 + col] = make_float2(top, sum);
  __syncthreads();
  float all = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4 * BLOCKS; ++i) all = fmaxf(all, state[i / BLOCKS * 16 + i % BLOCKS * ROWS + r].x);
  const float base = all == -INFINITY ? 0.f : all;
  const float factor = __builtin_amdgcn_exp2f(top - base);
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < 4 * BLOCKS; ++i) {
    const float2 st = state[i / BLOCKS * 16 + i % BLOCKS * ROWS + r];
    total += st.y * __builtin_amdgcn_exp2f(st.x - base);
  }
#pragma unroll
  for (int f = 0; f < F; ++f) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      acc[f][i] *= factor;
      if constexpr (ROWS < 16) acc[f][i] = sum_row<ROWS>(acc[f][i]);
    }
    if (group == 0) *reinterpret_cast<f32x4*>(outs + (wave * ROWS + r) * DP + 16 * f + 4 * q) = acc[f];
  }
  const uint64_t home = ((uint64_t)sequence * g.heads + head) * plan.stride;
  float2* states = reinterpret_cast<float2*>(partial + (uint64_t)a.b.sequences * g.heads * plan.stride * places * DP);
  if (part.count > 1 && tid < ROWS && row0 + tid < rows) states[(home + row0 + tid) * places + split] = make_float2(all, total);
  if (tid < ROWS) inverse[tid] = total == 0.f ? 0.f : 1.f / total;  // lane r of wave 0: row r
  __syncthreads();
  for (uint32_t i = tid; i < ROWS * DP; i += 256) {
    const uint32_t rr = i / DP, d = i % DP, ri = row0 + rr;
    if (ri >= rows) break;
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) v += outs[(k * ROWS + rr) * DP + d];
    if (part.count > 1) {
      partial[((home + ri) * places + split) * DP + d] = v;
    } else if (d < D) {
      static_cast<T*>(a.out)[(uint64_t)(s.row0 + ri / gq) * a.out_stride + (uint64_t)(head * gq + ri % gq) * D + d] = (T)(v * inverse[rr]);
    }
  }
}

// Joins the splits of one row: four waves over the splits, lanes over the channels.
template <class T>
__global__ void __launch_bounds__(256) k_paged_rows_join(PagedAttention a, RowsPlan plan, const float* partial) {
  __shared__ float part_out[4][kPagedMaxHeadDim];
  __shared__ float part_state[4];
  const PagedGeometry& g = a.c.geo;
  const uint32_t head = blockIdx.y, row = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const PagedSequence s = paged_sequence(a.b, g, blockIdx.z);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq;
  if (rows <= plan.over || rows > plan.most || row >= rows) return;
  const uint32_t tile = 16 / plan.blocks, row0 = row / tile * tile;
  const Walk w = walk_of(a, s, row0, row0 + tile < rows ? row0 + tile : rows, gq, kPagedBlock);
  const uint32_t count = rows_part(w, paged_vq(g, s.n), plan).count, places = plan.splits + plan.tails;
  if (count == 1) return;
  const uint64_t home = (((uint64_t)blockIdx.z * g.heads + head) * plan.stride + row) * places;
  const float2* states = reinterpret_cast<const float2*>(
      partial + (uint64_t)a.b.sequences * g.heads * plan.stride * places * g.DP);
  // every wave takes a quarter of the splits, 64 at a time: their factors a lane each, then their outputs
  float top = -INFINITY;
  for (uint32_t k = lane; k < count; k += 64) top = fmaxf(top, states[home + k].x);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float base = top == -INFINITY ? 0.f : top;
  const uint32_t quarter = (count + 3) / 4, from = wave * quarter, to = from + quarter < count ? from + quarter : count;
  float sum = 0.f, x[kPagedMaxHeadDim / 64] = {0.f};
  for (uint32_t k0 = from; k0 < to; k0 += 64) {
    const uint32_t n = to - k0 < 64 ? to - k0 : 64;
    float factor = 0.f;
    if (lane < n) {
      const float2 st = states[home + k0 + lane];
      factor = __builtin_amdgcn_exp2f(st.x - base);
      sum += factor * st.y;
    }
#pragma unroll
    for (uint32_t j = 0; j < kPagedMaxHeadDim / 64; ++j) {
      if (j * 64 >= g.DP) continue;
      const float* p = partial + (home + k0) * g.DP + (j * 64 + lane < g.DP ? j * 64 + lane : 0);
      for (uint32_t k = 0; k < n; k += 8) {
        float v[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) v[i] = k + i < n ? p[(uint64_t)(k + i) * g.DP] : 0.f;
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) x[j] += __shfl(factor, (int)((k + i) % 64)) * v[i];  // zero from n on
      }
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
#pragma unroll
  for (uint32_t j = 0; j < kPagedMaxHeadDim / 64; ++j) part_out[wave][j * 64 + lane] = x[j];
  if (lane == 0) part_state[wave] = sum;
  __syncthreads();
  sum = part_state[0] + part_state[1] + part_state[2] + part_state[3];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* out = static_cast<T*>(a.out) + (uint64_t)(s.row0 + row / gq) * a.out_stride + (uint64_t)(head * gq + row % gq) * g.D;
  for (uint32_t d = threadIdx.x; d < g.D; d += 256)
    out[d] = (T)((part_out[0][d] + part_out[1][d] + part_out[2][d] + part_out[3][d]) * inv);
}

template <class T, int BITS, int S, int BLOCKS, bool HALVES>
hipError_t rows_launch(const PagedAttention& a, const RowsPlan& p, float* partial, hipStream_t stream) {
  const PagedGeometry& g = a.c.geo;
  const size_t bytes = rows_lds_words<T>(S, g.ncg, BLOCKS) * 4;
  auto kernel = k_paged_rows<T, BITS, S, BLOCKS, HALVES>;
  hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(kernel), bytes);
  if (e != hipSuccess) return e;
  constexpr uint32_t kTile = 16 / BLOCKS;
  const uint32_t tiles = (p.stride + kTile - 1) / kTile;
  hipLaunchKernelGGL(kernel, dim3(g.heads, a.b.sequences, tiles * (p.splits + p.tails)), dim3(256), bytes, stream, a, p, partial);
  hipLaunchKernelGGL(k_paged_rows_join<T>, dim3(p.stride, g.heads, a.b.sequences), dim3(256), 0, stream, a, p, partial);
  return hipGetLastError();
}

template <class T, int BITS, int S, bool HALVES>
hipError_t rows_blocks(const PagedAttention& a, const RowsPlan& p, float* partial, hipStream_t stream) {
  constexpr int kMost = rows_most_blocks(BITS, S);
  if constexpr (kMost >= 4) {
    if (p.blocks == 4) return rows_launch<T, BITS, S, 4, HALVES>(a, p, partial, stream);
  }
  if constexpr (kMost >= 2) {
    if (p.blocks == 2) return rows_launch<T, BITS, S, 2, HALVES>(a, p, partial, stream);
  }
  return p.blocks == 1 ? rows_launch<T, BITS, S, 1, HALVES>(a, p, partial, stream) : hipErrorInvalidValue;
}

template <class T, int BITS, bool HALVES>
hipError_t rows_dims(const PagedAttention& a, const RowsPlan& p, float* partial, hipStream_t stream) {
  switch (a.c.geo.S()) {
    case 2: return rows_blocks<T, BITS, 2, HALVES>(a, p, partial, stream);
    case 3: return rows_blocks<T, BITS, 3, HALVES>(a, p, partial, stream);
    case 4: return rows_blocks<T, BITS, 4, HALVES>(a, p, partial, stream);
    case 8: return rows_blocks<T, BITS, 8, HALVES>(a, p, partial, stream);
    default: return hipErrorInvalidValue;  // paged_rows_take
  }
}

}  // namespace

template <class T, bool HALVES>
hipError_t launch_paged_rows(const PagedAttention& a, const RowsPlan& p, float* partial, hipStream_t stream) {
  switch (a.c.geo.bits) {
    case 2: return rows_dims<T, 2, HALVES>(a, p, partial, stream);
    case 4: return rows_dims<T, 4, HALVES>(a, p, partial, stream);
    default: return rows_dims<T, 8, HALVES>(a, p, partial, stream);
  }
}

}  // namespace kivi
