// kernels_paged.hip — the paged KIVI cache on CDNA4 (gfx950): new tokens of a ragged batch written
// (what leaves the windows quantized into the pages) and tokens read back as rows.
//
// Quantization is the format's own, bit for bit (src/quant.rs:275-377): scale = span / levels,
// code = round-half-even((x - zero) / scale). Keys take one (scale, zero) per channel over G tokens,
// values one per token over G channels. What is quantized follows from the lengths (paged.hpp), so
// a call needs nothing but them, and a repeated call writes the same bits.
#include "paged.hpp"

#include <algorithm>

#include "common.hpp"

namespace kivi {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kReduce = 2;       // lanes that share the minimum and maximum of a channel's tokens
constexpr uint32_t kReduceAny = 8;    // and of a token's channels, where a group is not whole octets
constexpr uint32_t kWindowRows = 32;  // rows a workgroup copies into the windows
// Elements of a span that one workgroup stages for all channels (32 KB of float32, four workgroups a compute
// unit), else a quarter of them: a span of 512 would not fit.
constexpr uint32_t kMostStaged = 32 * 256;
constexpr uint32_t kMostOctets = 32 * kPagedMaxHeadDim / 8 / kThreads;  // of a 32-token block, per thread

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
__device__ __forceinline__ float to_f(T x) {
  return (float)x;
}

// Eight consecutive elements of a row from p, `count` of which exist (the others read as zero).
template <class T>
__device__ __forceinline__ void load8(const T* p, bool vec, uint32_t count, float (&x)[8]) {
  if (vec && count >= 8) {
    alignas(16) T e[8];
    const uint4* src = reinterpret_cast<const uint4*>(p);
    reinterpret_cast<uint4*>(e)[0] = src[0];
    if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(e)[1] = src[1];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) x[j] = to_f(e[j]);
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j) x[j] = j < count ? to_f(p[j]) : 0.f;
}

template <class T>
__device__ __forceinline__ void store8(T* p, bool vec, uint32_t count, const float (&x)[8]) {
  if (vec && count >= 8) {
    alignas(16) T e[8];
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) e[j] = (T)x[j];
    reinterpret_cast<uint4*>(p)[0] = reinterpret_cast<uint4*>(e)[0];
    if constexpr (sizeof(T) == 4) reinterpret_cast<uint4*>(p)[1] = reinterpret_cast<uint4*>(e)[1];
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (j < count) p[j] = (T)x[j];
}

template <class T>
__device__ __forceinline__ void copy8(const T* from, T* to, bool vec, uint32_t count) {
  if (vec && count >= 8) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = reinterpret_cast<const uint4*>(from)[i];
    return;
  }
#pragma unroll
  for (uint32_t j = 0; j < 8; ++j)
    if (j < count) to[j] = from[j];
}

// What a code stands for: code * scale + zero, rounded once to f32 (src/quant.rs:379-451) before any
// rounding to a narrower type; the empty asm keeps the compiler from folding both into one
// (v_fma_mixlo_f16), which gives other last bits in f16.
__device__ __forceinline__ float decoded(uint32_t code, float2 pair) {
  float x = fmaf((float)code, pair.x, pair.y);
  asm("" : "+v"(x));
  return x;
}

// The row of token t of one head: in the window while t < n, else new row t - n of the tensor.
template <class T>
__device__ __forceinline__ const T* token_row(const PagedGeometry& g, const T* window, const PagedSequence& s,
                                              uint32_t head, int64_t t, const T* rows, uint64_t stride, uint32_t pitch) {
  if (t < s.n)
    return window + (((uint64_t)s.slot * g.heads + head) * 2 * g.R + ring_row(g, t)) * g.DW;
  return rows + (uint64_t)(s.row0 + (t - s.n)) * stride + (uint64_t)head * pitch;
}

// (scale, zero) of the group of `count` elements at p, `stride` apart, by LANES neighbouring lanes,
// each of which gets it. NaN elements are passed over, as by f32::min (src/quant.rs:303, 356).
template <uint32_t LANES>
__device__ __forceinline__ float2 group_pair(const float* p, uint32_t stride, uint32_t count, float levels) {
  float mn = INFINITY, mx = -INFINITY;
  for (uint32_t i = threadIdx.x % LANES; i < count; i += LANES) {
    mn = fminf(mn, p[i * stride]);
    mx = fmaxf(mx, p[i * stride]);
  }
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor(mn, o));
    mx = fmaxf(mx, __shfl_xor(mx, o));
  }
  return make_float2(scale_of(mx - mn, levels), mn);
}

// Codes of one fragment's elements 0 .. 3 and 4 .. 7, a byte each, as they lie in its words (paged_bit): 2
// bits of fragment 0 of the two that share a word, 4 bits, or the first four of 8.
template <int BITS>
__device__ __forceinline__ uint32_t folded(uint32_t lo, uint32_t hi) {
  if constexpr (BITS == 2) {
    const auto nibbles = [](uint32_t x) {
      x = (x | x >> 4) & 0x00ff00ffu;
      return (x | x >> 8) & 0xffffu;
    };
    return nibbles(lo) | nibbles(hi) << 16;
  } else if constexpr (BITS == 4) {
    return lo | hi << 4;
  } else {
    return lo;
  }
}
// Element j of a fragment whose words start with w (2 bits: shifted to the fragment).
template <int BITS>
__device__ __forceinline__ uint32_t code_in(const uint32_t* w, uint32_t j) {
  return w[BITS == 8 ? j / 4 : 0] >> paged_bit(BITS, 0, j) & ((1u << BITS) - 1);
}
// The word or two of fragment f, ready for code_in.
template <int BITS>
__device__ __forceinline__ void fragment_words(const uint32_t* lane_words, uint32_t f, uint32_t (&w)[2]) {
  const uint32_t* p = lane_words + paged_word(BITS, f, 0);
  w[0] = p[0];
  if constexpr (BITS == 2) w[0] >>= 2 * (f & 1);
  if constexpr (BITS == 8) w[1] = p[1];
}

__device__ __forceinline__ void put_word(uint32_t* p, uint32_t bits, uint32_t mask) {
  if (mask == 0) return;
  *p = mask == ~0u ? bits : (*p & ~mask) | (bits & mask);
}

// r[j] holds four bytes of row j: c[i] gets byte i of the four rows.
__device__ __forceinline__ void turn_bytes(const uint32_t (&r)[4], uint32_t (&c)[4]) {
  const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u);
  const uint32_t d = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u), e = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
  c[0] = __builtin_amdgcn_perm(d, a, 0x05040100u);
  c[1] = __builtin_amdgcn_perm(d, a, 0x07060302u);
  c[2] = __builtin_amdgcn_perm(e, b, 0x05040100u);
  c[3] = __builtin_amdgcn_perm(e, b, 0x07060302u);
}

// How an append's grid is cut, and the divisors of its indexes.
struct AppendPlan {
  uint32_t key_spans, parts;  // spans of keys, the channels of each in `parts` (1 or 4: all, or those of one q)
  uint32_t value_items, late;
  uint32_t octets_magic, oct_magic, words_magic, ncg_magic;  // of 4 S / parts, 4 S, a lane's words, D / G
};

// Workgroup items of one (sequence, head): `parts` per key span (no two write one word), one per 32-token
// block of values, and window rows. Every word of the pages belongs to one item, which reads, changes
// and writes it alone.
//
// The reads of a call are window rows of tokens [n - R, n) and new rows; with m <= R its window
// writes (tokens n .. n + m - 1, of 2 R rows) touch none of those. A longer chunk writes its last R rows
// in a second launch (`late`).
//
// Keys pass through LDS as float32 (a channel's group is a column of rows); a thread's values stay in its
// registers and only octet extremes and one byte per code do. Bound by those passes and the code arithmetic in a
// long prompt (nine prompts of 40000 tokens, f32, 2 bits, 8 heads, D = 128: 371 MB in 128 us, 2.9 TB/s, from 245 us
// with the code width and the divisors read at run time) and by latency for single tokens (5.5 us).
template <class T, int BITS>
__global__ void __launch_bounds__(kThreads)
    k_paged_append(PagedView c, PagedBatch b, PagedRows keys, PagedRows values, AppendPlan plan) {
  extern __shared__ __align__(16) float lds[];
  constexpr uint32_t kLevels = (1u << BITS) - 1, kFragments = BITS == 2 ? 2 : 1;  // fragments of a word (of two, 8 bits)
  const PagedGeometry& g = c.geo;
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const PagedSequence s = paged_sequence(b, g, blockIdx.z);
  if (s.slot < 0 || s.m == 0) return;
  const int64_t n = s.n, n2 = s.n + s.m;
  const uint32_t D = g.D, S = g.S(), LW = S * BITS / 2;
  const T* kw = static_cast<const T*>(c.kwin);
  const T* vw = static_cast<const T*>(c.vwin);
  const T* kr = static_cast<const T*>(keys.p);
  const T* vr = static_cast<const T*>(values.p);
  uint32_t item = blockIdx.x;

  if (item < plan.parts * plan.key_spans) {
    const uint32_t part = item % plan.parts, quarters = 4 / plan.parts;
    const uint32_t octets = S * quarters, CH = 8 * octets, ch0 = part * CH, pitch = CH + 4;
    const int64_t kq = paged_kq(g, n), kq2 = paged_kq(g, n2);
    const int64_t base = (kq / g.span + item / plan.parts) * g.span;
    const int64_t lo = base > kq ? base : kq, hi = base + g.span < kq2 ? base + g.span : kq2;
    if (lo >= hi) return;
    uint32_t* rec = paged_record(c, b, s, head, base);
    if (rec == nullptr) return;
    float* tile = lds;                                  // [span][pitch]
    const uint32_t groups = g.span / g.G;
    float *zero = lds + g.span * pitch, *scale = zero + groups * CH, *inv = scale + groups * CH;  // [groups][CH]
    const uint32_t count = (uint32_t)(hi - lo), skip = (uint32_t)(lo - base);
    for (uint32_t i0 = tid; i0 < count * octets; i0 += 2 * kThreads) {
      float x[2][8];
      uint32_t at[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t i = i0 + k * kThreads < count * octets ? i0 + k * kThreads : i0;
        const uint32_t tau = quotient(i, octets, plan.octets_magic), o = i - tau * octets, d = ch0 + 8 * o;
        const int64_t t = lo + tau;
        at[k] = (skip + tau) * pitch + 8 * o;
        load8(token_row(g, kw, s, head, t, kr, keys.stride, keys.pitch) + d, t < n || keys.vec != 0, d < D ? D - d : 0, x[k]);
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<float4*>(tile + at[k] + 4 * j) = make_float4(x[k][4 * j], x[k][4 * j + 1], x[k][4 * j + 2], x[k][4 * j + 3]);
    }
    __syncthreads();
    const uint32_t g0 = quotient(skip, g.G, g.group_magic), ng = quotient(count, g.G, g.group_magic);
    float2* params = reinterpret_cast<float2*>(rec + g.kparams_at) + (uint64_t)quotient(token_in_page(g, base), g.G, g.group_magic) * g.DP;
    for (uint32_t i = tid / kReduce; i < ng * CH; i += kThreads / kReduce) {
      const uint32_t gi = g0 + quotient(i / 8, octets, plan.octets_magic), ch = i - (gi - g0) * CH;
      const float2 p = group_pair<kReduce>(tile + gi * g.G * pitch + ch, pitch, g.G, (float)kLevels);
      if (tid % kReduce == 0) {
        scale[gi * CH + ch] = p.x;
        zero[gi * CH + ch] = p.y;
        inv[gi * CH + ch] = quant_inv(p.x);
        if (ch0 + ch < D) params[(uint64_t)gi * g.DP + ch0 + ch] = p;
      }
    }
    __syncthreads();
    uint32_t* codes = rec + (uint64_t)(token_in_page(g, base) / kPagedBlock) * g.block_words() + part * 16 * LW;
    const uint32_t lanes = 16 * quarters, words = BITS == 8 ? LW / 2 : LW;  // 8 bits: both words of a fragment at once
    for (uint32_t i = tid; i < g.span / kPagedBlock * lanes * words; i += kThreads) {
      const uint32_t lane = quotient(i, words, plan.words_magic), w = i - lane * words;
      const uint32_t blk = lane / lanes, l = lane % lanes;
      uint32_t word[2] = {0, 0}, mask = 0;
#pragma unroll
      for (uint32_t k = 0; k < kFragments; ++k) {
        const uint32_t f = kFragments * w + k, half = f >= S ? 1 : 0, ch = l / 16 * 8 * S + (f - half * S) * 8;
        const uint32_t tau = blk * kPagedBlock + half * 16 + l % 16;  // token - base
        if (tau < skip || tau >= skip + count) continue;
        const uint32_t gi = quotient(tau, g.G, g.group_magic) * CH + ch;
        uint32_t lo4 = 0, hi4 = 0;
#pragma unroll
        for (uint32_t j = 0; j < 8; j += 4) {
          const float4 x = *reinterpret_cast<const float4*>(tile + tau * pitch + ch + j);
          const float4 z = *reinterpret_cast<const float4*>(zero + gi + j), sc = *reinterpret_cast<const float4*>(scale + gi + j);
          const float4 iv = *reinterpret_cast<const float4*>(inv + gi + j);
          const uint32_t four = quant_code_fast(x.x, z.x, sc.x, iv.x, kLevels) | quant_code_fast(x.y, z.y, sc.y, iv.y, kLevels) << 8 |
                                quant_code_fast(x.z, z.z, sc.z, iv.z, kLevels) << 16 | quant_code_fast(x.w, z.w, sc.w, iv.w, kLevels) << 24;
          (j == 0 ? lo4 : hi4) = four;
        }
        word[0] |= folded<BITS>(lo4, hi4) << 2 * k;
        if constexpr (BITS == 8) word[1] = hi4;
        mask |= BITS == 2 ? 0x33333333u << 2 * k : ~0u;
      }
      uint32_t* to = codes + (uint64_t)blk * g.block_words() + l * LW + (BITS == 8 ? 2 * w : w);
      put_word(to, word[0], mask);
      if constexpr (BITS == 8) put_word(to + 1, word[1], mask);
    }
    return;
  }
  item -= plan.parts * plan.key_spans;

  if (item < plan.value_items) {
    const int64_t vq = paged_vq(g, n), vq2 = paged_vq(g, n2);
    const int64_t base = (vq / kPagedBlock + item) * kPagedBlock;
    const int64_t lo = base > vq ? base : vq, hi = base + kPagedBlock < vq2 ? base + kPagedBlock : vq2;
    if (lo >= hi) return;
    uint32_t* rec = paged_record(c, b, s, head, base);
    if (rec == nullptr) return;
    const uint32_t ncg = g.ncg, oct = 4 * S, pitch = g.DP + 4;
    const uint32_t t0 = (uint32_t)(lo - base), count = (uint32_t)(hi - lo);
    float2* params = reinterpret_cast<float2*>(rec + g.vparams_at) + (uint64_t)token_in_page(g, base) * ncg;
    unsigned char* bytes = reinterpret_cast<unsigned char*>(lds);  // codes [32][pitch], a byte each
    float* rest = lds + kPagedBlock * pitch / 4;
    const auto octet_of = [&](uint32_t i, uint32_t* tau, uint32_t* d) {
      const uint32_t t = quotient(i, oct, plan.oct_magic);
      *tau = t0 + t;
      *d = 8 * (i - t * oct);
    };
    const auto load = [&](uint32_t tau, uint32_t d, float(&x)[8]) {
      const int64_t t = base + tau;
      load8(token_row(g, vw, s, head, t, vr, values.stride, values.pitch) + d, t < n || values.vec != 0, d < D ? D - d : 0, x);
    };
    const auto put_bytes = [&](uint32_t tau, uint32_t d, const uint32_t(&code)[8]) {
      uint32_t* to = reinterpret_cast<uint32_t*>(bytes + tau * pitch + d);
      to[0] = code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24;
      to[1] = code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24;
    };
    if (g.G % 8 == 0) {
      // A thread keeps its octets of channels; a group's minimum and maximum come from those of its octets.
      float2* ends = reinterpret_cast<float2*>(rest);  // [32][oct]
      float x[kMostOctets][8];
#pragma unroll
      for (uint32_t k = 0; k < kMostOctets; ++k) {
        const uint32_t i = tid + k * kThreads;
        if (i >= count * oct) break;
        uint32_t tau, d;
        octet_of(i, &tau, &d);
        load(tau, d, x[k]);
      }
#pragma unroll
      for (uint32_t k = 0; k < kMostOctets; ++k) {
        const uint32_t i = tid + k * kThreads;
        if (i >= count * oct) break;
        float mn = INFINITY, mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) mn = fminf(mn, x[k][j]), mx = fmaxf(mx, x[k][j]);
        ends[i] = make_float2(mn, mx);
      }
      __syncthreads();
#pragma unroll
      for (uint32_t k = 0; k < kMostOctets; ++k) {
        const uint32_t i = tid + k * kThreads;
        if (i >= count * oct) break;
        uint32_t tau, d;
        octet_of(i, &tau, &d);
        uint32_t code[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (d < D) {
          const uint32_t cg = quotient(d, g.G, g.group_magic), o = d / 8 - cg * (g.G / 8);  // octet of its group
          float mn = INFINITY, mx = -INFINITY;
          for (uint32_t e = i - o; e < i - o + g.G / 8; ++e) mn = fminf(mn, ends[e].x), mx = fmaxf(mx, ends[e].y);
          const float scale = scale_of(mx - mn, (float)kLevels), inv = quant_inv(scale);
          if (o == 0) params[tau * ncg + cg] = make_float2(scale, mn);
#pragma unroll
          for (int j = 0; j < 8; ++j) code[j] = quant_code_fast(x[k][j], mn, scale, inv, kLevels);
        }
        put_bytes(tau, d, code);
      }
    } else {
      const uint32_t row = g.DP + 1;
      float* tile = rest;                                                                   // [32][row]
      float2* pair = reinterpret_cast<float2*>(rest + ((kPagedBlock * row + 1) & ~1u));  // [32][ncg]
      for (uint32_t i = tid; i < count * oct; i += kThreads) {
        uint32_t tau, d;
        octet_of(i, &tau, &d);
        float x[8];
        load(tau, d, x);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) tile[tau * row + d + j] = x[j];
      }
      __syncthreads();
      for (uint32_t i = tid / kReduceAny; i < count * ncg; i += kThreads / kReduceAny) {
        const uint32_t t = quotient(i, ncg, plan.ncg_magic), tau = t0 + t, cg = i - t * ncg;
        const float2 p = group_pair<kReduceAny>(tile + tau * row + cg * g.G, 1, g.G, (float)kLevels);
        if (tid % kReduceAny == 0) {
          pair[tau * ncg + cg] = p;
          params[tau * ncg + cg] = p;
        }
      }
      __syncthreads();
      for (uint32_t i = tid; i < count * oct; i += kThreads) {
        uint32_t tau, d;
        octet_of(i, &tau, &d);
        uint32_t code[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const float2 p = d + j < D ? pair[tau * ncg + quotient(d + j, g.G, g.group_magic)] : make_float2(0.f, 0.f);
          code[j] = quant_code_fast(tile[tau * row + d + j], p.y, p.x, quant_inv(p.x), kLevels);
        }
        put_bytes(tau, d, code);
      }
    }
    __syncthreads();
    // A thread makes the words of four neighbouring channels: eight tokens of each of their fragments.
    uint32_t* codes = rec + g.vcodes_at + (uint64_t)(token_in_page(g, base) / kPagedBlock) * g.block_words();
    const uint32_t pieces = 2 * S / kFragments;  // words (8 bits: pairs of words) of a lane
    for (uint32_t i = tid; i < 16 * pieces; i += kThreads) {
      const uint32_t l = i % 4 * 4, q = i / 4 % 4, w = i / 16;
      uint32_t lo4[4] = {0, 0, 0, 0}, hi4[4] = {0, 0, 0, 0}, mask[2] = {0, 0};
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t tau = j / 4 * 16 + 4 * q + j % 4;
        mask[j / 4] |= tau >= t0 && tau < t0 + count ? kLevels << 8 * (j % 4) : 0u;
      }
      uint32_t word[4][2];
#pragma unroll
      for (uint32_t k = 0; k < kFragments; ++k) {
        uint32_t r[2][4];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
          r[j / 4][j % 4] = *reinterpret_cast<const uint32_t*>(bytes + (j / 4 * 16 + 4 * q + j % 4) * pitch + 16 * (kFragments * w + k) + l);
        turn_bytes(r[0], lo4);
        turn_bytes(r[1], hi4);
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          const uint32_t x = folded<BITS>(lo4[ch] & mask[0], hi4[ch] & mask[1]) << 2 * k;
          word[ch][0] = k == 0 ? x : word[ch][0] | x;
          word[ch][1] = hi4[ch];
        }
      }
      const uint32_t whole = folded<BITS>(mask[0], mask[1]), both = BITS == 2 ? whole | whole << 2 : whole;
#pragma unroll
      for (int ch = 0; ch < 4; ++ch) {
        uint32_t* to = codes + (q * 16 + l + ch) * LW + (BITS == 8 ? 2 * w : w);
        put_word(to, word[ch][0], both);
        if constexpr (BITS == 8) put_word(to + 1, word[ch][1], mask[1]);
      }
    }
    return;
  }
  item -= plan.value_items;

  if ((s.m > g.R) != (plan.late != 0)) return;
  const int64_t first = n2 - g.R > n ? n2 - g.R : n;
  const int64_t lo = first + (int64_t)item * kWindowRows;
  const int64_t hi = lo + kWindowRows < n2 ? lo + kWindowRows : n2;
  if (lo >= hi) return;
  for (uint32_t i = tid; i < (uint32_t)(hi - lo) * 4 * S; i += kThreads) {
    const uint32_t r = quotient(i, 4 * S, plan.oct_magic), d = 8 * (i - r * 4 * S);
    if (d >= D) continue;
    const int64_t t = lo + r;
    const uint64_t to = (((uint64_t)s.slot * g.heads + head) * 2 * g.R + ring_row(g, t)) * g.DW + d;
    const uint64_t row = (uint64_t)(s.row0 + (t - n));
    copy8(kr + row * keys.stride + (uint64_t)head * keys.pitch + d, static_cast<T*>(c.kwin) + to, keys.vec != 0, D - d);
    copy8(vr + row * values.stride + (uint64_t)head * values.pitch + d, static_cast<T*>(c.vwin) + to, values.vec != 0, D - d);
  }
}

// One wave per (sequence, 32-token block, head): codes become rows. A lane takes an octet of channels of
// eight tokens: of keys a word or two each, of values those of the eight lanes that have its channels, so
// that rows go out in whole pieces and nothing has to turn over. Tokens that the cache does not hold (at
// or behind its length, or in a page or slot outside the pool) read as zeros. Bound by the rows it writes
// (five sequences to 45001 tokens, bf16, 8 bits, 16 heads of 96: 815 MB in 175 us, 4.7 TB/s; turning values
// over in LDS: 573 us); single tokens by latency, of which fetching the code is a good part: VEC (whole octets on
// 16 bytes) has no stores of single elements in it (10 -> 7.5 us).
template <class T, int BITS, bool VEC>
__global__ void __launch_bounds__(kThreads, 4)
    k_paged_read(PagedView c, PagedBatch b, const int32_t* first, PagedRows keys, PagedRows values, uint32_t S_magic, uint32_t oct_magic) {
  const PagedGeometry& g = c.geo;
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t item = blockIdx.x * (kThreads / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t head = item % g.heads;
  const PagedSequence s = paged_sequence(b, g, blockIdx.z);
  if (s.m == 0) return;
  const int32_t from = first != nullptr ? first[blockIdx.z] : 0;
  const int64_t f0 = from > 0 ? from : 0, end = f0 + s.m, n = s.n;
  const int64_t base = (f0 / kPagedBlock + item / g.heads) * kPagedBlock;
  if (base >= end) return;
  const int64_t kq = paged_kq(g, n), vq = paged_vq(g, n);
  const uint32_t D = g.D, G = g.G, S = g.S(), LW = S * BITS / 2, oct = 4 * S, ncg = g.ncg, in_page = token_in_page(g, base);
  const int lo = base > f0 ? 0 : (int)(f0 - base), hi = base + kPagedBlock < end ? (int)kPagedBlock : (int)(end - base);
  // tokens in front of kend (vend) have packed keys (values), those behind and in front of nend lie in the window
  const auto part = [&](int64_t t) { return t <= base ? 0 : t < base + kPagedBlock ? (int)(t - base) : (int)kPagedBlock; };
  const int kend = part(kq), vend = part(vq), nend = part(n);
  const uint32_t* rec = kend > 0 ? paged_record(c, b, s, head, base) : nullptr;
  const bool held = rec != nullptr;
  if (!held) rec = c.pages;  // read, and dropped
  const uint32_t* kcodes = rec + (uint64_t)(in_page / kPagedBlock) * g.block_words();
  const uint32_t* vcodes = kcodes + g.vcodes_at;
  const int64_t row0 = s.row0 + (base - f0);  // of the block's first token

  for (uint32_t u = lane; u < 16 * S; u += 64) {
    const uint32_t p = quotient(u, oct, oct_magic), o = u - p * oct, d = 8 * o;
    if (d >= D) continue;
    const auto put = [&](T* to, uint32_t vec, float(&x)[8]) {
      if (!held) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = 0.f;
      }
      store8(to, VEC || vec != 0, VEC ? 8 : D - d, x);
    };
    // of keys tokens p + 4 i, of values 4 p + i and 16 + 4 p + i
    T* kout = static_cast<T*>(const_cast<void*>(keys.p)) + (row0 + p) * (int64_t)keys.stride + (uint64_t)head * keys.pitch + d;
    T* vout = static_cast<T*>(const_cast<void*>(values.p)) + (uint64_t)head * values.pitch + d;
    uint32_t kwords[8][2], vwords[8][2];
    f32x4 kpairs[4];
    f32x2 vpairs[8];
    const uint32_t q = quotient(o, S, S_magic), k = o - q * S, f = o / 2, group = quotient(in_page, G, g.group_magic);
    const f32x4* pairs = reinterpret_cast<const f32x4*>(rec + g.kparams_at + 2 * d);
    const f32x2* vp = reinterpret_cast<const f32x2*>(rec + g.vparams_at) + (uint64_t)in_page * ncg;
    if (kend > 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) kpairs[i] = pairs[group * (g.DP / 2) + i];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) fragment_words<BITS>(kcodes + (q * 16 + p + 4 * (i % 4)) * LW, i / 4 * S + k, kwords[i]);
    }
    if (vend > 0) {
      const uint32_t cg = quotient(d, G, g.group_magic);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) vpairs[j] = vp[(j / 4 * 16 + 4 * p + j % 4) * ncg + cg];
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) fragment_words<BITS>(vcodes + (p * 16 + 8 * (o % 2) + i) * LW, f, vwords[i]);
    }
    if (kend > 0) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) {
        const int tau = (int)(p + 4 * i);
        if (G % kPagedBlock != 0) {
          const uint32_t mine = quotient(in_page + tau, G, g.group_magic);
#pragma unroll
          for (int j = 0; j < 4; ++j) kpairs[j] = pairs[mine * (g.DP / 2) + j];
        }
        float x[8];
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = decoded(code_in<BITS>(kwords[i], j), make_float2(kpairs[j / 2][j % 2 * 2], kpairs[j / 2][j % 2 * 2 + 1]));
        if (tau >= lo && tau < hi && tau < kend) put(kout + i * 4 * keys.stride, keys.vec, x);
      }
    }
    if (vend > 0) {
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const int tau = (int)(j / 4 * 16 + 4 * p + j % 4);
        float x[8];
#pragma unroll
        for (uint32_t i = 0; i < 8; ++i) {
          f32x2 pair = vpairs[j];
          if (!VEC && G % 8 != 0) pair = vp[tau * ncg + quotient(d + i < D ? d + i : D - 1, G, g.group_magic)];
          x[i] = decoded(code_in<BITS>(vwords[i], j), make_float2(pair.x, pair.y));
        }
        if (tau >= lo && tau < hi && tau < vend) put(vout + (row0 + tau) * (int64_t)values.stride, values.vec, x);
      }
    }
    if (vend < (int)kPagedBlock) {
      // window rows, and zeros behind the cache: all fetched, then all written
      const uint64_t window = ((uint64_t)(s.slot < 0 ? 0 : s.slot) * g.heads + head) * 2 * g.R;
#pragma unroll 1
      for (int w = 0; w < 2; ++w) {
        const T* win = static_cast<const T*>(w == 0 ? c.kwin : c.vwin) + d;
        T* to = w == 0 ? kout : vout + (row0 + p) * (int64_t)values.stride;
        const uint64_t stride = 4 * (w == 0 ? keys.stride : values.stride);
        const uint32_t vec = w == 0 ? keys.vec : values.vec;
        const int packed = w == 0 ? kend : vend;
        constexpr int kAtOnce = 16 / sizeof(T);  // what registers allow
        uint4 raw[kAtOnce][sizeof(T) / 2];
#pragma unroll 1
        for (int tau0 = (int)p; tau0 < (int)kPagedBlock; tau0 += 4 * kAtOnce, to += kAtOnce * stride) {
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int tau = tau0 + 4 * i;
            const T* row = win + (window + ring_row(g, base + tau)) * g.DW;
#pragma unroll
            for (int k = 0; k < (int)sizeof(T) / 2; ++k)
              raw[i][k] = tau >= packed && tau < nend ? reinterpret_cast<const uint4*>(row)[k] : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int i = 0; i < kAtOnce; ++i) {
            const int tau = tau0 + 4 * i;
            if (tau >= lo && tau < hi && tau >= packed)
              copy8(reinterpret_cast<const T*>(raw[i]), to + i * stride, VEC || vec != 0, VEC ? 8 : D - d);
          }
        }
      }
    }
  }
}

template <class T, int BITS>
hipError_t append_typed(const PagedView& c, const PagedBatch& b, const PagedRows& keys, const PagedRows& values,
                        hipStream_t stream) {
  const PagedGeometry& g = c.geo;
  const uint32_t S = g.S();
  AppendPlan p{};
  // key tokens that one chunk can flush, in spans that need not start with it
  const uint64_t flushed = ((uint64_t)b.max_rows + g.R - 1) / g.R * g.R;
  p.key_spans = (uint32_t)(flushed / g.span + (g.R % g.span != 0 ? 2 : 0));
  p.parts = g.span * g.DP <= kMostStaged ? 1 : 4;
  p.value_items = (uint32_t)(((uint64_t)b.max_rows + 2 * (kPagedBlock - 1)) / kPagedBlock);
  p.oct_magic = magic_of(4 * S);
  p.octets_magic = magic_of(4 * S / p.parts);
  p.words_magic = magic_of(BITS == 8 ? 2 * S : S * BITS / 2);
  p.ncg_magic = magic_of(g.ncg);
  const uint32_t window_items = (std::min<uint64_t>(b.max_rows, g.R) + kWindowRows - 1) / kWindowRows;
  const uint32_t ch = g.DP / p.parts;
  const size_t key_lds = (g.span * (ch + 4ull) + 3ull * (g.span / g.G) * ch) * 4;
  const size_t codes = kPagedBlock * (g.DP + 4ull);
  const size_t value_lds = codes + (g.G % 8 == 0 ? kPagedBlock * 4ull * S * 8
                                                 : ((kPagedBlock * (g.DP + 1) + 1) & ~1u) * 4ull + (uint64_t)kPagedBlock * g.ncg * 8);
  const size_t bytes = std::max(key_lds, value_lds);
  hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(&k_paged_append<T, BITS>), bytes);
  if (e != hipSuccess) return e;
  const dim3 grid(p.parts * p.key_spans + p.value_items + window_items, g.heads, b.sequences);
  hipLaunchKernelGGL((k_paged_append<T, BITS>), grid, dim3(kThreads), bytes, stream, c, b, keys, values, p);
  if (b.max_rows > g.R) {
    p.key_spans = p.value_items = 0;
    p.late = 1;
    hipLaunchKernelGGL((k_paged_append<T, BITS>), dim3(window_items, g.heads, b.sequences), dim3(kThreads), 0, stream, c, b, keys,
                       values, p);
  }
  return hipGetLastError();
}
template <class T>
hipError_t append_bits(const PagedView& c, const PagedBatch& b, const PagedRows& keys, const PagedRows& values,
                       hipStream_t stream) {
  switch (c.geo.bits) {
    case 2: return append_typed<T, 2>(c, b, keys, values, stream);
    case 4: return append_typed<T, 4>(c, b, keys, values, stream);
    default: return append_typed<T, 8>(c, b, keys, values, stream);
  }
}

template <class T>
hipError_t read_typed(const PagedView& c, const PagedBatch& b, const int32_t* first, const PagedRows& keys,
                      const PagedRows& values, hipStream_t stream) {
  const PagedGeometry& g = c.geo;
  const uint64_t items = ((uint64_t)b.max_rows + 2 * (kPagedBlock - 1)) / kPagedBlock * g.heads;
  const dim3 grid((uint32_t)((items + kThreads / 64 - 1) / (kThreads / 64)), 1, b.sequences);
  const bool vec = g.G % 8 == 0 && keys.vec != 0 && values.vec != 0;
  const auto kernel = g.bits == 2 ? vec ? k_paged_read<T, 2, true> : k_paged_read<T, 2, false>
                      : g.bits == 4 ? vec ? k_paged_read<T, 4, true> : k_paged_read<T, 4, false>
                                    : vec ? k_paged_read<T, 8, true> : k_paged_read<T, 8, false>;
  hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, stream, c, b, first, keys, values, magic_of(g.S()), magic_of(4 * g.S()));
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const PagedView& c, const PagedBatch& b, PagedRows keys, PagedRows values,
                               hipStream_t stream) {
  switch (c.geo.type) {
    case kPagedF32: return append_bits<float>(c, b, keys, values, stream);
    case kPagedF16: return append_bits<_Float16>(c, b, keys, values, stream);
    default: return append_bits<__bf16>(c, b, keys, values, stream);
  }
}

hipError_t launch_paged_read(const PagedView& c, const PagedBatch& b, const int32_t* first, PagedRows keys,
                             PagedRows values, hipStream_t stream) {
  switch (c.geo.type) {
    case kPagedF32: return read_typed<float>(c, b, first, keys, values, stream);
    case kPagedF16: return read_typed<_Float16>(c, b, first, keys, values, stream);
    default: return read_typed<__bf16>(c, b, first, keys, values, stream);
  }
}

}  // namespace kivi
