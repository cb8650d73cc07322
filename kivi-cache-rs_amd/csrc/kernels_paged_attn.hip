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
#include <type_traits>

#include "common.hpp"
#include "paged_attn.hpp"

namespace kivi {
namespace {

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
constexpr uint64_t kComputeUnits = 256;
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
    // Where most sequences have to be near the longest chunk, one launch takes all rows of any number (an empty
    // launch and its join cost 7 us).
    const bool alike = (uint64_t)b.rows * 2 > (uint64_t)b.sequences * b.max_rows;
    for (uint32_t i = 0; i < 2 && over < rows && over < kRowsMost; ++i) {
      if (alike && rows > kRowsMost) break;
      if (alike && rows > most[i]) continue;
      RowsPlan& r = p.rows[p.row_launches];
      r.over = over;
      r.most = most[i];
      r.stride = (uint32_t)std::min<uint64_t>(rows, r.most);
      r.blocks = std::min<uint32_t>(r.stride <= 4 ? 4 : r.stride <= 8 ? 2 : 1, rows_most_blocks(g.bits, g.S()));
      const uint64_t turn = 4 * r.blocks, tiles = (r.stride + 16 / r.blocks - 1) / (16 / r.blocks);
      // blocks of a split and the splits of a walk over n tokens, at most `cap`
      const auto cut = [&](uint64_t n, uint64_t cap) {
        const uint64_t blocks = std::max<uint64_t>(1, (n + kPagedBlock - 1) / kPagedBlock);
        // one to eight turns a wave (what surrounds the turns costs about one), more where there are many: 64
        // sequences to 32768 tokens 171 us with at most eight, 178 with four, 182 with sixteen
        const uint64_t turns = std::clamp<uint64_t>(blocks * heads * tiles / turn / 1024, 1, 8);
        const uint64_t least = std::max({turns * turn, blocks * heads * tiles / kRowsWorkgroups, (blocks + cap - 1) / cap});
        r.least = (uint32_t)((least + turn - 1) / turn * turn);
        r.splits = (uint32_t)((blocks + r.least - 1) / r.least);
      };
      // last blocks: the windows' tokens and the new ones, a block a wave
      r.tails = (uint32_t)std::min<uint64_t>((g.R + (r.most + gq - 1) / gq + 2 * kPagedBlock - 2) / (4 * kPagedBlock) + 1, 64);
      cut(all, kMostSplits);
      const uint64_t most_splits = r.splits;
      if (tokens < all) cut(tokens, most_splits);
      p.rows_at[p.row_launches++] = p.floats;
      p.floats += heads * r.stride * (most_splits + r.tails) * (g.DP + 2);
      over = most[i];
    }
    p.chunk.over = alike && rows > kRowsMost ? 0 : kRowsMost;
  }
  p.chunks = rows > p.chunk.over;
  p.chunk.tile_rows = paged_chunk_rows(g);
  p.chunk.tile = paged_chunk_tokens(g);
  const uint64_t groups = std::max<uint64_t>(1, (uint64_t)b.rows * gq / p.chunk.tile_rows) * g.heads;  // about
  // One workgroup fills a compute unit: rounds of workgroups times the tiles of each (and two for its start and
  // end), and what a join costs, in tiles of about 3.5 us: its launch, partial sums written and read. Two sequences of 6000 rows
  // (375 groups) over 18 tiles: 1 split 117 us, 2 splits 124 and a join of 33.
  const auto chunk_splits = [&](uint64_t n) {
    const uint64_t tiles = std::max<uint64_t>(1, (n + p.chunk.tile - 1) / p.chunk.tile);
    uint64_t best = 1, least_cost = ~(uint64_t)0;
    for (uint64_t k = 1; k <= std::max<uint64_t>(1, std::min<uint64_t>(64, tiles / 4)); ++k) {
      const uint64_t rounds = (groups * k + kComputeUnits - 1) / kComputeUnits;
      const uint64_t cost = rounds * ((tiles + k - 1) / k + 2) + (k == 1 ? 0 : 2 + k * groups * g.DP / 6400);
      if (cost < least_cost) least_cost = cost, best = k;
    }
    return (uint32_t)best;
  };
  const uint32_t most_chunk_splits = chunk_splits(all);
  const uint64_t walked = window == 0 ? all : std::min(all, window + std::min(sinks, all) + p.chunk.tile_rows / gq + 3 * p.chunk.tile);
  p.chunk.splits = std::min(chunk_splits(walked), most_chunk_splits);
  p.chunk_at = p.floats;
  if (p.chunks && most_chunk_splits > 1) p.floats += (size_t)most_chunk_splits * (size_t)b.rows * qh * (g.DP + 2);
  return p;
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
  return launch_paged_chunk<T>(a, p.chunk, workspace + p.chunk_at, stream);
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
