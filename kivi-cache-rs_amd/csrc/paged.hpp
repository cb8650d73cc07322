// paged.hpp — device layout of the paged KIVI cache and the launch interface shared by its
// kernels (kernels_paged.hip, kernels_paged_attn.hip) and the host (host.cpp).
//
// A pool of pages holds the quantized tokens of many sequences; a table gives each sequence's
// pages. How much of a sequence is quantized follows from its length n alone, as in a KiviCache
// that got its tokens in any pieces: the first n / R * R keys and the first n - R values. The last
// tokens also lie in windows of the caller's type, 2 R rows per slot and KV head for keys and for
// values (token t in row t % (2 R)). R rows would do for the present; 2 R leave every row that an
// append of up to R tokens quantizes where it was, so that such an append may be repeated or taken
// back by passing the old length (drafted tokens that were refused), and so that it has no reads
// that its own writes could overtake.
//
// Page p, KV head h: one record at pages + (p * heads + h) * record, four arrays in this order:
//
//   key codes    u32 [P/32] blocks   key block: lane-major fragments, see below
//   key params   f32 [P/G][DP][2]    (scale, zero) per (group, channel)
//   value codes  u32 [P/32] blocks
//   value params f32 [P][D/G][2]     (scale, zero) per (token, channel group)
//
// DP is D rounded up to 32 (codes and key params of the channels behind D stay zero). A block of 32
// tokens is stored as the 64 lanes of a wave read it for the matrix cores: lane L holds 2S
// fragments of eight codes (S = DP/32), its words contiguous. With q = L / 16, l = L % 16:
//
//   keys    fragment f = 16-token half * S + s: token half*16 + l, channels 8S q + 8 s + (0..7)
//   values  fragment f: channel 16 f + l, tokens 4q + (0..3) and 16 + 4q + (0..3)
//
// The value tokens follow the accumulator layout of the 16-row matrix instructions (row 4q + i of
// each 16-token tile), so softmax weights go from one product to the next in the lane that has
// them. Inside the words, element j of fragment f lies where the packed fp4 / fp8 converters take
// it without shuffling: 2 bits: word f/2, bit 4j + 2(f%2); 4 bits: word f, bit 8(j%4) + 4(j/4);
// 8 bits: word 2f + j/4, bit 8(j%4).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace kivi {

constexpr uint32_t kPagedBlock = 32;       // tokens per code block
constexpr uint32_t kPagedMaxHeadDim = 256;
constexpr uint32_t kPagedMaxSpan = 512;    // lcm(32, G): tokens a key-quantizing workgroup stages in LDS

enum PagedType : uint32_t { kPagedF32 = 0, kPagedF16 = 1, kPagedBF16 = 2 };

// n / d by a multiplication, any n and d: magic_of(d) falls short of 2^32 / d by less than one (two for d =
// 1), so the estimate falls short of the quotient by at most one.
__host__ inline uint32_t magic_of(uint32_t d) { return d == 1 ? 0xffffffffu : (uint32_t)(((uint64_t)1 << 32) / d); }
__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t d, uint32_t magic) {
  const uint32_t e = __umulhi(n, magic);
  return n - e * d >= d ? e + 1 : e;
}

struct PagedGeometry {
  uint32_t bits, G, R, D, DP;
  uint32_t heads;
  uint32_t P;      // tokens per page
  uint32_t span;   // lcm(32, G)
  uint32_t pages;  // pages of the pool
  uint32_t slots;  // windows
  uint32_t type;   // PagedType
  // what follows from those (finish); offsets in words from a record
  uint32_t ncg, page_blocks;
  uint32_t DW;     // D rounded up to 8: pitch of the windows' rows (zeros behind D)
  uint32_t kparams_at, vcodes_at, vparams_at, record_words;
  uint32_t page_magic, group_magic, fragment_magic, flush_magic, ring_magic;  // of P/32, G, max(1, G/16), R, 2R

  __host__ void finish() {
    ncg = D / G;
    DW = (D + 7) / 8 * 8;
    page_blocks = P / kPagedBlock;
    kparams_at = page_blocks * block_words();
    vcodes_at = kparams_at + P / G * DP * 2;
    vparams_at = vcodes_at + page_blocks * block_words();
    record_words = vparams_at + P * ncg * 2;
    page_magic = magic_of(page_blocks);
    group_magic = magic_of(G);
    fragment_magic = magic_of(G < 16 ? 1 : G / 16);
    flush_magic = magic_of(R);
    ring_magic = magic_of(2 * R);
  }
  __host__ __device__ uint32_t S() const { return DP / 32; }
  __host__ __device__ uint32_t levels() const { return (1u << bits) - 1u; }
  __host__ __device__ uint32_t lane_words() const { return DP / 32 * bits / 2; }
  __host__ __device__ uint32_t block_words() const { return DP * bits; }  // 32 tokens * DP * bits / 32
  __host__ __device__ uint32_t type_bytes() const { return type == kPagedF32 ? 4u : 2u; }
};

struct PagedView {
  PagedGeometry geo;
  uint32_t* pages;
  void* kwin;  // [slots][heads][2R][DW]
  void* vwin;
};

// A ragged batch: device arrays of a kivi_paged_batch and its bounds.
struct PagedBatch {
  const int32_t* slots;
  const int32_t* lengths;
  const int32_t* starts;
  const int32_t* table;
  uint32_t sequences;
  uint32_t per_sequence;  // table entries of a sequence
  int64_t rows;
  uint32_t max_rows;      // longest chunk (the host's bound; longer ones are cut to it)
  uint64_t max_length;    // longest cached length expected (for the grids only)
};

// One sequence of a batch as the kernels see it: whatever the device arrays hold, the ranges stay
// inside the tensors, and a page or slot outside the pool is no page or slot.
struct PagedSequence {
  int64_t n;       // cached tokens
  int64_t row0;    // first row of the new tokens
  uint32_t m;      // new tokens
  int32_t slot;    // -1: none
  const int32_t* table;
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& b, const PagedGeometry& g, uint32_t i) {
  PagedSequence s;
  const int32_t n = b.lengths[i], slot = b.slots[i];
  const int64_t a0 = b.starts[i], a1 = b.starts[i + 1];
  s.slot = slot >= 0 && (uint32_t)slot < g.slots ? slot : -1;
  s.n = n > 0 && s.slot >= 0 ? n : 0;
  s.row0 = a0 < 0 ? 0 : a0 < b.rows ? a0 : b.rows;
  const int64_t end = a1 < s.row0 ? s.row0 : a1 < b.rows ? a1 : b.rows;
  const int64_t m = end - s.row0;
  s.m = m < (int64_t)b.max_rows ? (uint32_t)m : b.max_rows;
  s.table = b.table + (uint64_t)i * b.per_sequence;
  return s;
}

// Record of (the sequence's page p, head), or null where it has no such page.
__device__ __forceinline__ uint32_t* paged_record_of(const PagedView& c, const PagedBatch& b, const PagedSequence& s,
                                                     uint32_t head, uint32_t p) {
  if (p >= b.per_sequence) return nullptr;
  const int32_t page = s.table[p];
  if (page < 0 || (uint32_t)page >= c.geo.pages) return nullptr;
  return c.pages + ((uint64_t)(uint32_t)page * c.geo.heads + head) * c.geo.record_words;
}

// The same of the page of token t.
__device__ __forceinline__ uint32_t* paged_record(const PagedView& c, const PagedBatch& b, const PagedSequence& s,
                                                  uint32_t head, int64_t t) {
  return paged_record_of(c, b, s, head, quotient((uint32_t)(t / kPagedBlock), c.geo.page_blocks, c.geo.page_magic));
}

// Lengths are under 2^31 and a chunk under 2^24 rows: tokens count in 32 bits, positions (which may be
// negative) in 64.
__device__ __forceinline__ int64_t paged_kq(const PagedGeometry& g, int64_t n) {
  return (int64_t)quotient((uint32_t)n, g.R, g.flush_magic) * g.R;
}
__device__ __forceinline__ int64_t paged_vq(const PagedGeometry& g, int64_t n) { return n > g.R ? n - g.R : 0; }
// Window row of token t.
__device__ __forceinline__ uint32_t ring_row(const PagedGeometry& g, int64_t t) {
  return (uint32_t)t - quotient((uint32_t)t, 2 * g.R, g.ring_magic) * 2 * g.R;
}
// Token of its page.
__device__ __forceinline__ uint32_t token_in_page(const PagedGeometry& g, int64_t t) {
  return (uint32_t)t - quotient((uint32_t)(t / kPagedBlock), g.page_blocks, g.page_magic) * g.P;
}

// Word (of a lane's words) and bit of element j of fragment f.
__host__ __device__ inline uint32_t paged_word(uint32_t bits, uint32_t f, uint32_t j) {
  return bits == 2 ? f >> 1 : bits == 4 ? f : 2 * f + (j >> 2);
}
__host__ __device__ inline uint32_t paged_bit(uint32_t bits, uint32_t f, uint32_t j) {
  return bits == 2 ? 4 * j + 2 * (f & 1) : bits == 4 ? 8 * (j & 3) + 4 * (j >> 2) : 8 * (j & 3);
}

// Rows of a ragged tensor: row r, head h at p + r * stride + h * pitch (in elements). `vec`: every row of
// a head is whole 8-element pieces on 16 bytes.
struct PagedRows {
  const void* p;
  uint64_t stride;
  uint32_t pitch;
  uint32_t vec;
};

hipError_t launch_paged_append(const PagedView& c, const PagedBatch& b, PagedRows keys, PagedRows values,
                               hipStream_t stream);
// Rows starts[i] + r of sequence i <- token first[i] + r (first null: 0).
hipError_t launch_paged_read(const PagedView& c, const PagedBatch& b, const int32_t* first, PagedRows keys,
                             PagedRows values, hipStream_t stream);

struct PagedAttention {
  PagedView c;
  PagedBatch b;
  PagedRows query, keys, values;  // keys.p null: the new tokens are cached already. The kernels take `vec` ones.
  void* out;
  uint64_t out_stride;
  uint32_t out_vec;
  uint32_t qh;
  float scale;
  uint64_t window, sinks;  // window 0: none
};
size_t paged_attention_workspace(const PagedGeometry& g, const PagedBatch& b, uint32_t qh);
hipError_t launch_paged_attention(PagedAttention a, void* workspace, hipStream_t stream);

}  // namespace kivi
