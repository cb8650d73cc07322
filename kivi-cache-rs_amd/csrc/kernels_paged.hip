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
constexpr uint32_t kReduce = 8;      // lanes that share one group's minimum and maximum
constexpr uint32_t kWindowRows = 32; // rows a workgroup copies into the windows

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

// (scale, zero) of the group of `count` elements at p, `stride` apart, by kReduce neighbouring lanes,
// each of which gets it. NaN elements are passed over, as by f32::min (src/quant.rs:303, 356).
__device__ __forceinline__ float2 group_pair(const float* p, uint32_t stride, uint32_t count, float levels) {
  float mn = INFINITY, mx = -INFINITY;
  for (uint32_t i = threadIdx.x % kReduce; i < count; i += kReduce) {
    mn = fminf(mn, p[i * stride]);
    mx = fmaxf(mx, p[i * stride]);
  }
#pragma unroll
  for (int o = kReduce / 2; o > 0; o >>= 1) {
    mn = fminf(mn, __shfl_xor(mn, o));
    mx = fmaxf(mx, __shfl_xor(mx, o));
  }
  return make_float2(scale_of(mx - mn, levels), mn);
}

__device__ __forceinline__ uint32_t code_of(float x, float2 pair, uint32_t levels) {
  return quant_code_fast(x, pair.y, pair.x, quant_inv(pair.x), levels);
}

__device__ __forceinline__ void put_word(uint32_t* p, uint32_t bits, uint32_t mask) {
  if (mask == 0) return;
  *p = mask == ~0u ? bits : (*p & ~mask) | bits;
}

// Workgroup items of one (sequence, head): 4 per key span (each a quarter of the channels: the
// channels of one q, so no two write one word), one per 32-token block of values, and window rows.
// Every word of the pages belongs to one item, which reads, changes and writes it alone.
//
// The reads of a call are window rows of tokens [n - R, n) and new rows; with m <= R its window
// writes (tokens n .. n + m - 1, of 2 R rows) touch none of those. A longer chunk writes its last R rows
// in a second launch (`late`).
//
// Bound by memory in a long prompt (rows read, codes and pairs written, nothing twice) and by
// latency for single tokens.
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_paged_append(PagedView c, PagedBatch b, PagedRows keys, PagedRows values, uint32_t key_items,
                   uint32_t value_items, uint32_t late) {
  extern __shared__ float lds[];
  const PagedGeometry& g = c.geo;
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const PagedSequence s = paged_sequence(b, g, blockIdx.z);
  if (s.slot < 0 || s.m == 0) return;
  const int64_t n = s.n, n2 = s.n + s.m;
  const uint32_t D = g.D, S = g.S(), LW = g.lane_words(), levels = g.levels();
  const float flevels = (float)levels;
  const T* kw = static_cast<const T*>(c.kwin);
  const T* vw = static_cast<const T*>(c.vwin);
  const T* kr = static_cast<const T*>(keys.p);
  const T* vr = static_cast<const T*>(values.p);

  if (blockIdx.x < 4 * key_items) {
    const uint32_t q = blockIdx.x % 4, CH = 8 * S, ch0 = q * CH, pitch = CH + 1;
    const int64_t kq = paged_kq(g, n), kq2 = paged_kq(g, n2);
    const int64_t base = (kq / g.span + blockIdx.x / 4) * g.span;
    const int64_t lo = base > kq ? base : kq, hi = base + g.span < kq2 ? base + g.span : kq2;
    if (lo >= hi) return;
    uint32_t* rec = paged_record(c, b, s, head, base);
    if (rec == nullptr) return;
    float* tile = lds;                                                 // [span][pitch]
    float2* pair = reinterpret_cast<float2*>(lds + ((g.span * pitch + 1) & ~1u));  // [span / G][CH]
    const uint32_t count = (uint32_t)(hi - lo);
    for (uint32_t i = tid; i < count * S; i += kThreads) {
      const int64_t t = lo + i / S;
      const uint32_t o = i % S * 8, d = ch0 + o;
      float x[8];
      const T* row = token_row(g, kw, s, head, t, kr, keys.stride, keys.pitch);
      load8(row + d, t < n || keys.vec != 0, d < D ? D - d : 0, x);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) tile[(uint32_t)(t - base) * pitch + o + j] = x[j];
    }
    __syncthreads();
    const uint32_t g0 = (uint32_t)(lo - base) / g.G, ng = count / g.G;
    float2* params = reinterpret_cast<float2*>(rec + g.kparams_at) + (uint64_t)quotient(token_in_page(g, base), g.G, g.group_magic) * g.DP;
    for (uint32_t i = tid / kReduce; i < ng * CH; i += kThreads / kReduce) {
      const uint32_t gi = g0 + i / CH, ch = i % CH;
      const float2 p = group_pair(tile + gi * g.G * pitch + ch, pitch, g.G, flevels);
      if (tid % kReduce == 0) {
        pair[gi * CH + ch] = p;
        if (ch0 + ch < D) params[(uint64_t)gi * g.DP + ch0 + ch] = p;
      }
    }
    __syncthreads();
    uint32_t* codes = rec + (uint64_t)(token_in_page(g, base) / kPagedBlock) * g.block_words();
    for (uint32_t i = tid; i < g.span / kPagedBlock * 16 * LW; i += kThreads) {
      const uint32_t w = i % LW, l = i / LW % 16, blk = i / LW / 16;
      uint32_t word = 0, mask = 0;
      const uint32_t nf = g.bits == 2 ? 2 : 1, j0 = g.bits == 8 ? 4 * (w & 1) : 0, nj = g.bits == 8 ? 4 : 8;
      for (uint32_t k = 0; k < nf; ++k) {
        const uint32_t f = g.bits == 2 ? 2 * w + k : g.bits == 4 ? w : w / 2;
        const uint32_t tau = blk * kPagedBlock + f / S * 16 + l;  // token - base
        if (base + tau < lo || base + tau >= hi) continue;
        for (uint32_t j = j0; j < j0 + nj; ++j) {
          const uint32_t ch = f % S * 8 + j, at = paged_bit(g.bits, f, j);
          mask |= levels << at;
          if (ch0 + ch < D) word |= code_of(tile[tau * pitch + ch], pair[tau / g.G * CH + ch], levels) << at;
        }
      }
      put_word(codes + (uint64_t)blk * g.block_words() + (q * 16 + l) * LW + w, word, mask);
    }
    return;
  }

  if (blockIdx.x < 4 * key_items + value_items) {
    const int64_t vq = paged_vq(g, n), vq2 = paged_vq(g, n2);
    const int64_t base = (vq / kPagedBlock + (blockIdx.x - 4 * key_items)) * kPagedBlock;
    const int64_t lo = base > vq ? base : vq, hi = base + kPagedBlock < vq2 ? base + kPagedBlock : vq2;
    if (lo >= hi) return;
    uint32_t* rec = paged_record(c, b, s, head, base);
    if (rec == nullptr) return;
    const uint32_t pitch = g.DP + 1, ncg = g.ncg, oct = g.DP / 8;
    float* tile = lds;                                                              // [32][pitch]
    float2* pair = reinterpret_cast<float2*>(lds + ((kPagedBlock * pitch + 1) & ~1u));  // [32][ncg]
    const uint32_t t0 = (uint32_t)(lo - base), count = (uint32_t)(hi - lo);
    for (uint32_t i = tid; i < count * oct; i += kThreads) {
      const int64_t t = lo + i / oct;
      const uint32_t d = i % oct * 8;
      float x[8];
      const T* row = token_row(g, vw, s, head, t, vr, values.stride, values.pitch);
      load8(row + d, t < n || values.vec != 0, d < D ? D - d : 0, x);
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) tile[(uint32_t)(t - base) * pitch + d + j] = x[j];
    }
    __syncthreads();
    float2* params = reinterpret_cast<float2*>(rec + g.vparams_at) + (uint64_t)token_in_page(g, base) * ncg;
    for (uint32_t i = tid / kReduce; i < count * ncg; i += kThreads / kReduce) {
      const uint32_t tau = t0 + i / ncg, cg = i % ncg;
      const float2 p = group_pair(tile + tau * pitch + cg * g.G, 1, g.G, flevels);
      if (tid % kReduce == 0) {
        pair[tau * ncg + cg] = p;
        params[tau * ncg + cg] = p;
      }
    }
    __syncthreads();
    uint32_t* codes = rec + g.vcodes_at + (uint64_t)(token_in_page(g, base) / kPagedBlock) * g.block_words();
    for (uint32_t i = tid; i < 64 * LW; i += kThreads) {
      const uint32_t w = i % LW, lane = i / LW, q = lane / 16, l = lane % 16;
      uint32_t word = 0, mask = 0;
      const uint32_t nf = g.bits == 2 ? 2 : 1, j0 = g.bits == 8 ? 4 * (w & 1) : 0, nj = g.bits == 8 ? 4 : 8;
      for (uint32_t j = j0; j < j0 + nj; ++j) {
        const uint32_t tau = (j < 4 ? 4 * q + j : 16 + 4 * q + j - 4);
        if (tau < t0 || tau >= t0 + count) continue;
        for (uint32_t k = 0; k < nf; ++k) {
          const uint32_t f = g.bits == 2 ? 2 * w + k : g.bits == 4 ? w : w / 2;
          const uint32_t d = 16 * f + l, at = paged_bit(g.bits, f, j);
          mask |= levels << at;
          if (d < D) word |= code_of(tile[tau * pitch + d], pair[tau * ncg + d / g.G], levels) << at;
        }
      }
      put_word(codes + lane * LW + w, word, mask);
    }
    return;
  }

  if ((s.m > g.R) != (late != 0)) return;
  const int64_t first = n2 - g.R > n ? n2 - g.R : n;
  const int64_t lo = first + (int64_t)(blockIdx.x - 4 * key_items - value_items) * kWindowRows;
  const int64_t hi = lo + kWindowRows < n2 ? lo + kWindowRows : n2;
  for (int64_t i = tid; lo + i / D < hi; i += kThreads) {
    const int64_t t = lo + i / D;
    const uint32_t d = (uint32_t)(i % D);
    const uint64_t to = (((uint64_t)s.slot * g.heads + head) * 2 * g.R + ring_row(g, t)) * g.DW + d;
    const uint64_t row = (uint64_t)(s.row0 + (t - n));
    static_cast<T*>(c.kwin)[to] = kr[row * keys.stride + (uint64_t)head * keys.pitch + d];
    static_cast<T*>(c.vwin)[to] = vr[row * values.stride + (uint64_t)head * values.pitch + d];
  }
}

// One workgroup per (sequence, 32-token block, head): codes become rows. Values lie channel by
// channel and turn over in LDS. Tokens that the cache does not hold (at or behind its length, or in a page
// or slot outside the pool) read as zeros. Bound by the rows it writes.
template <class T>
__global__ void __launch_bounds__(kThreads)
    k_paged_read(PagedView c, PagedBatch b, const int32_t* first, PagedRows keys, PagedRows values) {
  extern __shared__ float lds[];
  const PagedGeometry& g = c.geo;
  const uint32_t head = blockIdx.y, tid = threadIdx.x;
  const PagedSequence s = paged_sequence(b, g, blockIdx.z);
  if (s.m == 0) return;
  const int32_t from = first != nullptr ? first[blockIdx.z] : 0;
  const int64_t f0 = from > 0 ? from : 0, end = f0 + s.m, n = s.n;
  const uint32_t D = g.D, S = g.S(), LW = g.lane_words(), levels = g.levels(), oct = (D + 7) / 8, ncg = g.ncg;
  const T* kw = static_cast<const T*>(c.kwin);
  const T* vw = static_cast<const T*>(c.vwin);
  T* kout = static_cast<T*>(const_cast<void*>(keys.p));
  T* vout = static_cast<T*>(const_cast<void*>(values.p));
  const int64_t kq = paged_kq(g, n), vq = paged_vq(g, n);
  const uint32_t pitch = g.DP + 8;
  T* turned = reinterpret_cast<T*>(lds);  // [32][pitch]
  for (int64_t blk = f0 / kPagedBlock + blockIdx.x; blk * kPagedBlock < end; blk += gridDim.x) {
    const int64_t base = blk * kPagedBlock;
    const int64_t lo = base > f0 ? base : f0, hi = base + kPagedBlock < end ? base + kPagedBlock : end;
    const uint32_t* rec = base < n ? paged_record(c, b, s, head, base) : nullptr;
    const uint32_t in_page = token_in_page(g, base);
    if (base < vq && rec != nullptr) {
      const uint32_t* codes = rec + g.vcodes_at + (uint64_t)(in_page / kPagedBlock) * g.block_words();
      const float2* pairs = reinterpret_cast<const float2*>(rec + g.vparams_at) + (uint64_t)in_page * ncg;
      for (uint32_t i = tid; i < 64 * 2 * S; i += kThreads) {
        const uint32_t lane = i % 64, f = i / 64, d = 16 * f + lane % 16, q = lane / 16;
        if (d >= D) continue;
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
          const uint32_t tau = j < 4 ? 4 * q + j : 16 + 4 * q + j - 4;
          if (base + tau >= vq) continue;
          const uint32_t code = codes[lane * LW + paged_word(g.bits, f, j)] >> paged_bit(g.bits, f, j) & levels;
          turned[tau * pitch + d] = (T)decoded(code, pairs[tau * ncg + d / g.G]);
        }
      }
    }
    __syncthreads();
    const uint32_t* codes = rec + (uint64_t)(in_page / kPagedBlock) * g.block_words();
    for (uint32_t i = tid; i < (uint32_t)(hi - lo) * oct; i += kThreads) {
      const int64_t t = lo + i / oct;
      const uint32_t d = i % oct * 8, have = D - d, tau = (uint32_t)(t - base);
      const uint64_t row = (uint64_t)(s.row0 + (t - f0));
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (t < kq) {
        if (rec != nullptr) {
          const uint32_t q = d / (8 * S), f = tau / 16 * S + d % (8 * S) / 8;
          const uint32_t* words = codes + (q * 16 + tau % 16) * LW;
          const float2* pairs =
              reinterpret_cast<const float2*>(rec + g.kparams_at) + (uint64_t)((in_page + tau) / g.G) * g.DP + d;
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            x[j] = decoded(words[paged_word(g.bits, f, j)] >> paged_bit(g.bits, f, j) & levels, pairs[j]);
        }
      } else if (t < n) {
        load8(token_row<T>(g, kw, s, head, t, nullptr, 0, 0) + d, true, have, x);
      }
      store8(kout + row * keys.stride + (uint64_t)head * keys.pitch + d, keys.vec != 0, have, x);
      if (t < vq) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = rec != nullptr && j < have ? to_f(turned[tau * pitch + d + j]) : 0.f;
      } else if (t < n) {
        load8(token_row<T>(g, vw, s, head, t, nullptr, 0, 0) + d, true, have, x);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) x[j] = 0.f;
      }
      store8(vout + row * values.stride + (uint64_t)head * values.pitch + d, values.vec != 0, have, x);
    }
    __syncthreads();
  }
}

template <class T>
hipError_t append_typed(const PagedView& c, const PagedBatch& b, const PagedRows& keys, const PagedRows& values,
                        hipStream_t stream) {
  const PagedGeometry& g = c.geo;
  // key tokens that one chunk can flush, in spans that need not start with it
  const uint64_t flushed = ((uint64_t)b.max_rows + g.R - 1) / g.R * g.R;
  const uint32_t key_items = (uint32_t)(flushed / g.span + (g.R % g.span != 0 ? 2 : 0));
  const uint32_t value_items = (uint32_t)(((uint64_t)b.max_rows + 2 * (kPagedBlock - 1)) / kPagedBlock);
  const uint32_t window_items = (std::min<uint64_t>(b.max_rows, g.R) + kWindowRows - 1) / kWindowRows;
  const uint32_t ch = 8 * g.S();
  const size_t key_lds = ((g.span * (ch + 1) + 1) & ~1u) * 4ull + (uint64_t)g.span / g.G * ch * 8;
  const size_t value_lds = ((kPagedBlock * (g.DP + 1) + 1) & ~1u) * 4ull + (uint64_t)kPagedBlock * g.ncg * 8;
  const size_t bytes = std::max(key_lds, value_lds);
  hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(&k_paged_append<T>), bytes);
  if (e != hipSuccess) return e;
  const dim3 grid(4 * key_items + value_items + window_items, g.heads, b.sequences);
  hipLaunchKernelGGL(k_paged_append<T>, grid, dim3(kThreads), bytes, stream, c, b, keys, values, key_items, value_items, 0u);
  if (b.max_rows > g.R) {
    hipLaunchKernelGGL(k_paged_append<T>, dim3(window_items, g.heads, b.sequences), dim3(kThreads), 0, stream, c, b, keys,
                       values, 0u, 0u, 1u);
  }
  return hipGetLastError();
}

template <class T>
hipError_t read_typed(const PagedView& c, const PagedBatch& b, const int32_t* first, const PagedRows& keys,
                      const PagedRows& values, hipStream_t stream) {
  const PagedGeometry& g = c.geo;
  const uint64_t blocks = ((uint64_t)b.max_rows + 2 * (kPagedBlock - 1)) / kPagedBlock;
  const dim3 grid((uint32_t)blocks, g.heads, b.sequences);
  hipLaunchKernelGGL(k_paged_read<T>, grid, dim3(kThreads), kPagedBlock * (g.DP + 8) * sizeof(T), stream, c, b, first, keys,
                     values);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const PagedView& c, const PagedBatch& b, PagedRows keys, PagedRows values,
                               hipStream_t stream) {
  switch (c.geo.type) {
    case kPagedF32: return append_typed<float>(c, b, keys, values, stream);
    case kPagedF16: return append_typed<_Float16>(c, b, keys, values, stream);
    default: return append_typed<__bf16>(c, b, keys, values, stream);
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
