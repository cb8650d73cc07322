// kernels_paged_attn.hip — attention of a chunk of new tokens over the paged KIVI cache on CDNA4
// (gfx950): causal over a ragged batch, one token (decode), a few (drafted tokens) or thousands (a
// piece of a prompt) per sequence, with an optional sliding window and first tokens that stay
// visible.
//
// Row r of a sequence's KV head is query head r % gq of new token r / gq, at position
// p = L - m + r / gq of its L tokens (cached ones, then the new ones where they come as rows). It sees
// token t when t <= p and, under a window W, t > p - W or t < sinks:
//
//   out = sum_t exp(scale q.k_t - max) v_t / sum_t exp(scale q.k_t - max), zeros where it sees none.
//
// The sums run over tiles of tokens with a running maximum and sum in float32 (the base-2 exponent
// takes scale * log2 e). Products are taken as k q^T and v^T p^T: the accumulator of the first then
// holds, in each lane, one row's weights of the very tokens the second wants from that lane.
#include "paged.hpp"

#include <algorithm>

#include "common.hpp"
#include "paged_attn.hpp"

namespace kivi {
namespace {

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

// How the chunk kernel is launched: sequences whose KV heads have more than `over` rows.
struct ChunkPlan {
  uint32_t over, tile_rows, tile, splits, least;
};

// One workgroup: WAVES * 32 rows of one (sequence, KV head), each wave 32 of them, over one split of the
// token tiles. A tile of TT tokens lies in LDS as the products read it, keys by token, values by
// channel (tokens in the order of the code blocks), rows padded by 16 bytes so that the lanes of a
// read fall on different banks. All waves fill it, from codes or from rows, and all read it.
template <class T, int DP, int WAVES, int TT>
__global__ void __launch_bounds__(WAVES * 64)
    k_paged_chunk(PagedAttention a, ChunkPlan plan, float* partial) {
  typedef typename Row<T>::Frag Frag;
  constexpr int kPad = 16 / sizeof(T), kKeyPitch = DP + kPad, kValuePitch = TT + kPad;
  constexpr uint32_t kThreads = WAVES * 64, kSub = TT / 32;
  extern __shared__ __align__(16) unsigned char lds[];
  T* kt = reinterpret_cast<T*>(lds);                    // [TT][kKeyPitch]
  T* vt = kt + TT * kKeyPitch;                          // [DP][kValuePitch]
  __shared__ uint32_t bad[kSub];  // tokens of the tile with a value that is not finite, where not every row sees all
  __shared__ float bad_row[DP];
  const PagedGeometry& g = a.c.geo;
  const uint32_t head = blockIdx.y, tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
  const uint32_t col = lane % 32, half = lane / 32;
  const PagedSequence s = paged_sequence(a.b, g, blockIdx.z);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq;
  const uint32_t splits = plan.splits;
  const uint32_t tile_row = blockIdx.x / splits * (WAVES * 32), split = blockIdx.x % splits;
  if (rows <= plan.over || tile_row >= rows) return;
  const uint32_t tile_end = tile_row + WAVES * 32 < rows ? tile_row + WAVES * 32 : rows;
  const Walk w = walk_of(a, s, tile_row, tile_end, gq, TT);
  const Part part = part_of(w.tiles, splits, plan.least, split);
  if (split >= part.count) return;

  const uint32_t D = g.D, S = g.S(), LW = g.lane_words(), levels = g.levels();
  const int64_t kq = paged_kq(g, s.n), vq = paged_vq(g, s.n);
  const uint32_t row = tile_row + wave * 32 + col;
  const bool live = row < rows;
  const uint32_t token = (live ? row : rows - 1) / gq, qhead = head * gq + (live ? row : rows - 1) % gq;
  const int64_t pos = w.total - s.m + token;
  const int64_t left = a.window != 0 ? pos - (int64_t)a.window : -1;  // tokens up to here are outside the window
  // the wave's rows: every one sees the tokens in (all_left, all_pos]
  const uint32_t wr0 = tile_row + wave * 32 < rows ? tile_row + wave * 32 : rows - 1;
  const uint32_t wr1 = wr0 + 31 < rows ? wr0 + 31 : rows - 1;
  const int64_t all_pos = w.total - s.m + wr0 / gq, any_pos = w.total - s.m + wr1 / gq;
  const int64_t all_left = a.window != 0 ? any_pos - (int64_t)a.window : -1;
  const int64_t first_pos = w.total - s.m + tile_row / gq;  // and those of the workgroup
  const int64_t last_left = a.window != 0 ? w.hi - 1 - (int64_t)a.window : -1;

  Frag q[DP / 16];
  {
    const T* p = static_cast<const T*>(a.query.p) + (uint64_t)(s.row0 + token) * a.query.stride + (uint64_t)qhead * a.query.pitch;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
      const uint32_t d = 16 * i + 8 * half;
      q[i] = d < g.DW ? load_frag(p, d) : zero_frag<T>();
    }
  }
  const float scale = a.scale * kLog2e;
  float top = -INFINITY, sum = 0.f;
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{0.f};

  for (uint32_t it = part.from; it < part.to; ++it) {
    const int64_t t0 = (int64_t)(it < w.head_tiles ? it : w.first_tile + (it - w.head_tiles)) * TT;
    const uint32_t* rec[kSub];
#pragma unroll
    for (uint32_t i = 0; i < kSub; ++i) rec[i] = t0 + 32 * i < kq ? paged_record(a.c, a.b, s, head, t0 + 32 * i) : nullptr;
    // whether some row of the workgroup does not see some token of the tile
    bool edge = t0 + TT - 1 > first_pos || t0 <= last_left;
#pragma unroll
    for (uint32_t i = 0; i < kSub; ++i) edge |= t0 + 32 * i < kq && rec[i] == nullptr;
    __syncthreads();  // the tile before is read
    if (edge) {
      if (tid < kSub) bad[tid] = 0;
      __syncthreads();
    }
    // keys: eight channels of one token a time
    for (uint32_t i = tid; i < TT * (DP / 8); i += kThreads) {
      const uint32_t l = i % 16, o = i / 16 % (DP / 8), tau = i / 16 / (DP / 8) * 16 + l, d = 8 * o;
      const int64_t t = t0 + tau;
      Frag f;
      if (t < kq) {
        const uint32_t* r = rec[tau / 32];
        if (r != nullptr && d < g.DP) {  // DP may be more than the cache's
          const uint32_t in_page = token_in_page(g, t), frag = in_page % 32 / 16 * S + o % S;
          const uint32_t* words = r + (uint64_t)(in_page / 32) * g.block_words() + (o / S * 16 + l) * LW;
          const float2* pairs = reinterpret_cast<const float2*>(r + g.kparams_at) + (uint64_t)(in_page / g.G) * g.DP + d;
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j)
            f[j] = (T)decoded<T>(words[paged_word(g.bits, frag, j)] >> paged_bit(g.bits, frag, j) & levels, pairs[j]);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) f[j] = (T)0.f;
        }
      } else if (t < w.hi && d < g.DW) {
        f = load_frag(row_of<T>(g, a.c.kwin, s, head, t, a.keys), d);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) f[j] = (T)0.f;
      }
      *reinterpret_cast<Frag*>(kt + tau * kKeyPitch + d) = f;
    }
    // values: eight tokens of one channel a time
    for (uint32_t i = tid; i < (TT / 8) * DP; i += kThreads) {
      const uint32_t d = i % DP, sub = i / DP / 4, qq = i / DP % 4;
      Frag f;
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t tau = j < 4 ? 4 * qq + j : 16 + 4 * qq + j - 4;
        const int64_t t = t0 + 32 * sub + tau;
        T x = d < D && t < w.hi ? (T)value_of<T>(a, s, rec[sub], head, t, vq, d) : (T)0.f;
        if (edge && !(fabsf((float)x) <= 3.402823466e+38f)) {
          // a weight of zero would not keep it from the rows that do not see it
          atomicOr(&bad[sub], 1u << tau);
          x = (T)0.f;
        }
        f[j] = x;
      }
      *reinterpret_cast<Frag*>(vt + d * kValuePitch + 32 * sub + 8 * qq) = f;
    }
    __syncthreads();

    f32x16 logit[kSub];
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
      logit[sub] = f32x16{0.f};
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
        logit[sub] = Mma<T>::mul(*reinterpret_cast<const Frag*>(kt + (32 * sub + col) * kKeyPitch + 16 * i + 8 * half), q[i], logit[sub]);
    }
    const bool whole = !edge || (t0 + TT - 1 <= all_pos && t0 > all_left && t0 >= kq);
    float peak = -INFINITY;
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const int64_t t = t0 + 32 * sub + 8 * (i / 4) + 4 * half + i % 4;
        float x = logit[sub][i] * scale;
        if (!whole) {
          const bool seen = t <= pos && (t > left || t < (int64_t)a.sinks) && (t >= kq || rec[sub] != nullptr);
          x = seen ? x : -INFINITY;
        }
        logit[sub][i] = x;
        peak = fmaxf(peak, x);
      }
    }
    peak = fmaxf(peak, __shfl_xor(peak, 32));
    const float next = fmaxf(top, peak);
    const float base = next == -INFINITY ? 0.f : next;  // a row that has seen nothing yet
    const float shrink = __builtin_amdgcn_exp2f(top - base);
    top = next;
    float part_sum = 0.f;
    Frag p[kSub][2];
#pragma unroll
    for (uint32_t sub = 0; sub < kSub; ++sub) {
#pragma unroll
      for (uint32_t i = 0; i < 16; ++i) {
        const float x = __builtin_amdgcn_exp2f(logit[sub][i] - base);
        logit[sub][i] = x;
        part_sum += x;
        // accumulator rows 8 b + 4 half + j: product u takes b = u and b = u + 2
        p[sub][i / 4 % 2][i % 4 + (i >= 8 ? 4 : 0)] = (T)x;
      }
    }
    sum = sum * shrink + part_sum;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      acc[i] *= shrink;
#pragma unroll
      for (uint32_t sub = 0; sub < kSub; ++sub)
#pragma unroll
        for (uint32_t u = 0; u < 2; ++u)
          acc[i] = Mma<T>::mul(*reinterpret_cast<const Frag*>(vt + (32 * i + col) * kValuePitch + 32 * sub + 16 * u + 8 * half),
                               p[sub][u], acc[i]);
    }
    if (edge) {
      for (uint32_t sub = 0; sub < kSub; ++sub) {
        for (uint32_t left_over = bad[sub]; left_over != 0; left_over &= left_over - 1) {
          const uint32_t tau = __ffs(left_over) - 1;
          const int64_t t = t0 + 32 * sub + tau;
          __syncthreads();
          for (uint32_t d = tid; d < DP; d += kThreads) {
            const float x = d < D ? value_of<T>(a, s, rec[sub], head, t, vq, d) : 0.f;
            bad_row[d] = fabsf(x) <= 3.402823466e+38f ? 0.f : x;
          }
          __syncthreads();
          float weight = 0.f;
#pragma unroll
          for (uint32_t k = 0; k < kSub; ++k)
#pragma unroll
            for (uint32_t i = 0; i < 16; ++i)
              if (k == sub && i == tau / 8 * 4 + tau % 4) weight = logit[k][i];
          weight = __shfl(weight, (int)(tau % 8 / 4 * 32 + col));
          const bool seen = t <= pos && (t > left || t < (int64_t)a.sinks);
#pragma unroll
          for (int i = 0; i < DP / 32; ++i)
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e)
              if (seen) acc[i][e] += weight * bad_row[32 * i + 8 * (e / 4) + 4 * half + e % 4];
        }
      }
    }
  }

  sum += __shfl_xor(sum, 32);
  if (!live) return;
  const uint64_t place = (uint64_t)(s.row0 + token) * a.qh + qhead;
  if (part.count == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.out) + (uint64_t)(s.row0 + token) * a.out_stride + (uint64_t)qhead * D;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (uint32_t e = 0; e < 16; ++e) {
        const uint32_t d = 32 * i + 8 * (e / 4) + 4 * half + e % 4;
        if (d < D) out[d] = (T)(acc[i][e] * inv);
      }
  } else {
    const uint64_t all = (uint64_t)a.b.rows * a.qh;
    float* to = partial + (split * all + place) * g.DP;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (uint32_t e = 0; e < 16; ++e)
        if (32u * i < g.DP) to[32 * i + 8 * (e / 4) + 4 * half + e % 4] = acc[i][e];
    if (half == 0)
      *reinterpret_cast<float2*>(partial + splits * all * g.DP + (split * all + place) * 2) = make_float2(top, sum);
  }
}

// Joins the splits of one row and query head per wave, its lanes over the channels.
template <class T>
__global__ void __launch_bounds__(256)
    k_paged_chunk_join(PagedAttention a, ChunkPlan plan, const float* partial) {
  const PagedGeometry& g = a.c.geo;
  const PagedSequence s = paged_sequence(a.b, g, blockIdx.z);
  const uint32_t gq = a.qh / g.heads, rows = s.m * gq, lane = threadIdx.x % 64;
  const uint32_t splits = plan.splits, tile_rows = plan.tile_rows;
  if (rows <= plan.over) return;
  const uint64_t all = (uint64_t)a.b.rows * a.qh;
  for (uint64_t i = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64; i < (uint64_t)s.m * a.qh; i += (uint64_t)gridDim.x * 4) {
    const uint32_t token = (uint32_t)(i / a.qh), qhead = (uint32_t)(i % a.qh), r = token * gq + qhead % gq;
    const uint32_t r0 = r / tile_rows * tile_rows;
    const Walk w = walk_of(a, s, r0, r0 + tile_rows < rows ? r0 + tile_rows : rows, gq, plan.tile);
    const uint32_t count = part_of(w.tiles, splits, plan.least, 0).count;
    if (count == 1) continue;
    const uint64_t place = (uint64_t)s.row0 * a.qh + i;
    const float2* state = reinterpret_cast<const float2*>(partial + splits * all * g.DP);
    float top = -INFINITY;
    for (uint32_t k = 0; k < count; ++k) top = fmaxf(top, state[k * all + place].x);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x[kPagedMaxHeadDim / 64] = {0.f};
    for (uint32_t k = 0; k < count; ++k) {
      const float2 st = state[k * all + place];
      const float f = __builtin_amdgcn_exp2f(st.x - base);
      sum += f * st.y;
#pragma unroll
      for (uint32_t j = 0; j < kPagedMaxHeadDim / 64; ++j)
        if (j * 64 + lane < g.D) x[j] += f * partial[(k * all + place) * g.DP + j * 64 + lane];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    T* out = static_cast<T*>(a.out) + (uint64_t)(s.row0 + token) * a.out_stride + (uint64_t)qhead * g.D;
#pragma unroll
    for (uint32_t j = 0; j < kPagedMaxHeadDim / 64; ++j)
      if (j * 64 + lane < g.D) out[j * 64 + lane] = (T)(x[j] * inv);
  }
}

// Rows as the kernels take them (whole 8-element pieces on 16 bytes), for a caller whose rows are not.
template <class T>
__global__ void __launch_bounds__(256) k_paged_align(PagedRows from, T* to, uint32_t D, uint32_t DW, uint32_t heads, uint64_t rows) {
  const uint64_t all = rows * heads * DW;
  for (uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256) {
    const uint32_t d = (uint32_t)(i % DW), h = (uint32_t)(i / DW % heads);
    to[i] = d < D ? static_cast<const T*>(from.p)[i / DW / heads * from.stride + (uint64_t)h * from.pitch + d] : (T)0.f;
  }
}

// How a call is cut. The lengths are device memory, so the plan goes by the host's bounds: sequences
// shorter than those take fewer of the planned splits, and their other workgroups end at once.
struct Plan {
  RowsPlan rows[2];
  uint32_t row_launches;
  bool chunks;
  ChunkPlan chunk;
  size_t rows_at[2], chunk_at, floats;  // the launches' partials in the workspace
};

// Workgroups that the longest lengths would give: many more than run at once (256 compute units, two or
// so each), so that ragged lengths even out.
constexpr uint64_t kRowsWorkgroups = 8192;
constexpr uint64_t kChunkWorkgroups = 1024;
constexpr uint64_t kMostSplits = 512;

Plan plan_of(const PagedGeometry& g, const PagedBatch& b, uint32_t qh, uint64_t window, uint64_t sinks) {
  Plan p{};
  const uint32_t gq = qh / g.heads;
  const uint64_t rows = (uint64_t)b.max_rows * gq;
  // the workspace is sized without a window, which only ever walks less
  const uint64_t all = b.max_length + b.max_rows;
  const uint64_t tokens =
      window == 0 ? all : std::min(all, window + std::min(sinks, all) + b.max_rows + 2 * kPagedBlock);
  const uint64_t heads = (uint64_t)b.sequences * g.heads;
  if (paged_rows_take(g)) {
    // One launch for what a decoded token brings (gq rows), one for more rows than its tiles hold.
    const uint32_t decode = gq <= 4 ? 4 : gq <= 8 ? 8 : kRowsMost;
    const uint32_t most[2] = {decode, kRowsMost};
    uint32_t over = 0;
    for (uint32_t i = 0; i < 2 && over < rows && over < kRowsMost; ++i) {
      RowsPlan& r = p.rows[p.row_launches];
      r.over = over;
      r.most = most[i];
      r.stride = (uint32_t)std::min<uint64_t>(rows, r.most);
      r.blocks = std::min<uint32_t>(r.stride <= 4 ? 4 : r.stride <= 8 ? 2 : 1, rows_most_blocks(g.bits, g.S()));
      const uint64_t turn = 4 * r.blocks, tiles = (r.stride + 16 / r.blocks - 1) / (16 / r.blocks);
      // blocks of a split and the splits of a walk over n tokens, at most `cap`
      const auto cut = [&](uint64_t n, uint64_t cap) {
        const uint64_t blocks = std::max<uint64_t>(1, (n + kPagedBlock - 1) / kPagedBlock);
        // one to four turns a wave (what surrounds the turns costs about one), more where there are many
        const uint64_t turns = std::clamp<uint64_t>(blocks * heads * tiles / turn / 1024, 1, 4);
        const uint64_t least = std::max({turns * turn, blocks * heads * tiles / kRowsWorkgroups, (blocks + cap - 1) / cap});
        r.least = (uint32_t)((least + turn - 1) / turn * turn);
        r.splits = (uint32_t)((blocks + r.least - 1) / r.least);
      };
      cut(all, kMostSplits);
      const uint64_t most_splits = r.splits;
      if (tokens < all) cut(tokens, most_splits);
      p.rows_at[p.row_launches++] = p.floats;
      p.floats += heads * r.stride * (most_splits + 1) * (g.DP + 2);  // and the last blocks
      over = most[i];
    }
    p.chunk.over = kRowsMost;
  }
  p.chunks = rows > p.chunk.over;
  p.chunk.tile_rows = 128;
  p.chunk.tile = g.type == kPagedF32 && g.DP > 128 ? 32 : 64;
  p.chunk.least = 4;
  const uint64_t groups = std::max<uint64_t>(1, (uint64_t)b.rows * gq / p.chunk.tile_rows) * g.heads;
  const uint64_t want = std::min<uint64_t>((kChunkWorkgroups + groups - 1) / groups, 64);
  const auto chunk_splits = [&](uint64_t n) {
    return (uint32_t)std::max<uint64_t>(1, std::min(want, (n + p.chunk.tile - 1) / p.chunk.tile / p.chunk.least));
  };
  p.chunk.splits = chunk_splits(tokens);
  p.chunk_at = p.floats;
  if (p.chunks && chunk_splits(all) > 1) p.floats += (size_t)chunk_splits(all) * (size_t)b.rows * qh * (g.DP + 2);
  return p;
}

template <class T, int DP>
hipError_t launch_chunk(const PagedAttention& a, const ChunkPlan& p, float* partial, hipStream_t stream) {
  constexpr int WAVES = 4, TT = sizeof(T) == 4 && DP > 128 ? 32 : 64, kPad = 16 / sizeof(T);
  const PagedGeometry& g = a.c.geo;
  const uint64_t rows = (uint64_t)a.b.max_rows * (a.qh / g.heads);
  const uint64_t x = (rows + WAVES * 32 - 1) / (WAVES * 32) * p.splits;
  const size_t bytes = (TT * (DP + kPad) + DP * (TT + kPad)) * sizeof(T);
  auto kernel = k_paged_chunk<T, DP, WAVES, TT>;
  hipError_t e = raise_lds_limit(reinterpret_cast<const void*>(kernel), bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(kernel, dim3((uint32_t)x, g.heads, a.b.sequences), dim3(WAVES * 64), bytes, stream, a, p, partial);
  if (p.splits > 1) {
    const uint64_t joins = std::min<uint64_t>(((uint64_t)a.b.max_rows * a.qh + 3) / 4, 1u << 16);
    hipLaunchKernelGGL(k_paged_chunk_join<T>, dim3((uint32_t)joins, 1, a.b.sequences), dim3(256), 0, stream, a, p, partial);
  }
  return hipGetLastError();
}

// Bytes of the workspace in front of the partials, for rows that have to be aligned first.
size_t aligned_bytes(const PagedGeometry& g, const PagedBatch& b, uint32_t qh) {
  return ((size_t)b.rows * (qh + 2 * g.heads) * g.DW * g.type_bytes() + 255) / 256 * 256;
}

template <class T>
hipError_t align(PagedRows* r, T* to, const PagedAttention& a, uint32_t heads, hipStream_t stream) {
  const PagedGeometry& g = a.c.geo;
  const uint64_t all = (uint64_t)a.b.rows * heads * g.DW;
  hipLaunchKernelGGL(k_paged_align<T>, dim3((uint32_t)std::min<uint64_t>((all + 255) / 256, 1u << 16)), dim3(256), 0, stream, *r, to,
                     g.D, g.DW, heads, (uint64_t)a.b.rows);
  *r = PagedRows{to, (uint64_t)heads * g.DW, g.DW, 1};
  return hipGetLastError();
}

template <class T>
hipError_t attention_typed(PagedAttention a, void* memory, hipStream_t stream) {
  T* rows = static_cast<T*>(memory);
  float* workspace = reinterpret_cast<float*>(static_cast<char*>(memory) + aligned_bytes(a.c.geo, a.b, a.qh));
  hipError_t e = hipSuccess;
  if (!a.query.vec) e = align(&a.query, rows, a, a.qh, stream);
  rows += (uint64_t)a.b.rows * a.qh * a.c.geo.DW;
  if (e == hipSuccess && a.keys.p != nullptr && !a.keys.vec) e = align(&a.keys, rows, a, a.c.geo.heads, stream);
  rows += (uint64_t)a.b.rows * a.c.geo.heads * a.c.geo.DW;
  if (e == hipSuccess && a.keys.p != nullptr && !a.values.vec) e = align(&a.values, rows, a, a.c.geo.heads, stream);
  if (e != hipSuccess) return e;
  const Plan p = plan_of(a.c.geo, a.b, a.qh, a.window, a.sinks);
  for (uint32_t i = 0; i < p.row_launches; ++i) {
    e = a.c.geo.G % 32 != 0 ? launch_paged_rows<T, true>(a, p.rows[i], workspace + p.rows_at[i], stream)
                            : launch_paged_rows<T, false>(a, p.rows[i], workspace + p.rows_at[i], stream);
    if (e != hipSuccess) return e;
  }
  if (!p.chunks) return hipSuccess;
  const uint32_t DP = a.c.geo.DP;
  float* partial = workspace + p.chunk_at;
  if (DP <= 64) return launch_chunk<T, 64>(a, p.chunk, partial, stream);
  if (DP <= 96) return launch_chunk<T, 96>(a, p.chunk, partial, stream);
  if (DP <= 128) return launch_chunk<T, 128>(a, p.chunk, partial, stream);
  return launch_chunk<T, 256>(a, p.chunk, partial, stream);
}

}  // namespace

// The kernel of few rows scales one 16-token tile by one group's pairs, and a wave reads whole words.
bool paged_rows_take(const PagedGeometry& g) {
  const uint32_t S = g.S();
  return g.G % 16 == 0 && (S == 2 || S == 3 || S == 4 || S == 8);
}

size_t paged_attention_workspace(const PagedGeometry& g, const PagedBatch& b, uint32_t qh) {
  return aligned_bytes(g, b, qh) + plan_of(g, b, qh, 0, 0).floats * sizeof(float);
}

hipError_t launch_paged_attention(PagedAttention a, void* workspace, hipStream_t stream) {
  switch (a.c.geo.type) {
    case kPagedF32: return attention_typed<float>(a, workspace, stream);
    case kPagedF16: return attention_typed<_Float16>(a, workspace, stream);
    default: return attention_typed<__bf16>(a, workspace, stream);
  }
}

}  // namespace kivi
