// What the kernels of attention over paged caches share (fa_window.hip, fa_tree.hip).
#pragma once
#include "fa_common.hpp"

namespace lsfa {

constexpr float kWinLn2 = 0.6931471805599453f;

// Two e4m3 codes (the low or the high half of w) times a power of two.
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, __bf16) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, _Float16) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

// A sequence's keys, queries and first row of q, and its key tiles of 32: those
// with sinks that its window's tiles do not hold, then the window's from `first` on.
// Keys are those that the block table holds. Draft trees stand at the end of the length itself, which may
// pass the table: there only what is read is held to it, not where the tree begins.
struct KeyTiles {
  int len, seq, n, tok0;
  int sink, first;
  int count;         // all of them; 1 where queries see no key, 0 without queries
};
__device__ __forceinline__ int table_keys(const WindowParams& p) { return min(p.max_seq_len, p.max_blocks << p.block_shift); }
template <bool TREE>
__device__ __forceinline__ KeyTiles key_tiles_of(const WindowParams& p, int len, int n, int tok0) {
  KeyTiles t;
  t.seq = TREE ? min(len, table_keys(p)) : len;
  t.len = len, t.n = n, t.tok0 = tok0;
  t.first = t.sink = 0;
  if (p.window > 0) {
    t.first = max(len - n - p.window + 1, 0);
    if (TREE) t.first = min(t.first, t.seq);
    t.first >>= 5;
    t.sink = min((min(p.sinks, t.seq) + 31) >> 5, t.first);
  }
  t.count = n > 0 ? max(t.sink + ((t.seq + 31) >> 5) - t.first, 1) : 0;
  return t;
}
template <bool TREE>
__device__ __forceinline__ KeyTiles key_tiles(const WindowParams& p, int b) {
  int n = 1, tok0 = b;
  if (p.cu_q != nullptr) {  // (no row outside q, whatever the offsets)
    tok0 = min(max(p.cu_q[b], 0), p.tokens);
    n = max(min(p.cu_q[b + 1], p.tokens) - tok0, 0);
  }
  const int len = max(p.seq_lens[b], 0);
  return key_tiles_of<TREE>(p, TREE ? len : min(len, table_keys(p)), n, tok0);
}

// The kernel's arguments, read again. What only the beginning and the end of a run or item
// need is taken from here: kept in scalar registers through the loop it would push the
// loop's own ones out of them (the wide kernel's reads of LDS then all wait for each other).
__device__ __forceinline__ const __attribute__((address_space(4))) WindowParams* arguments() {
  auto a = (const __attribute__((address_space(4))) WindowParams*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(a));
  return a;
}

// 0 * infinity is NaN, so a row that does not see a key must not add that key's infinities
// and NaN with its weight of zero. The narrow windowed kernel takes such elements of V as zeros
// where a mask cuts a tile for some of a chunk's rows and, if there were any (ordinary caches have
// none), adds them to the rows that see their keys before the sums leave the registers; the
// wide one and the trees' take sums again, with them left out, if they are not finite.
// Ones in the elements of a word of V that are infinite or NaN (e4m3: NaN).
template <typename T, bool Q8>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
  if constexpr (Q8) return ((((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
  constexpr uint32_t e = __is_same(T, _Float16) ? 0x7c007c00u : 0x7f807f80u;  // exponents of ones
  const uint32_t x = w & e;
  return ((x & 0xffffu) == (e & 0xffffu) ? 0xffffu : 0u) | ((x & 0xffff0000u) == (e & 0xffff0000u) ? 0xffff0000u : 0u);
}
template <int N, typename A>
__device__ __forceinline__ bool all_finite(const A (&acc)[N]) {
  float s = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int i = 0; i < (int)(sizeof(A) / 4); ++i) s = fmaf(acc[j][i], 0.f, s);
  return s == 0.f;
}
// Element k of words of V, infinite or NaN, or zero.
template <typename T, bool Q8>
__device__ __forceinline__ float bad_value(const uint32_t* w, int k) {
  if constexpr (Q8) return (w[k / 4] >> (8 * (k & 3)) & 0xff) != 0 ? __builtin_nanf("") : 0.f;
  return (float)__builtin_bit_cast(T, (uint16_t)(w[k / 2] >> (16 * (k & 1))));
}

// Draft trees: bits at .. at + 31 of the mask of query `row`, of n drafts (bits at the number of
// the tile's first key, which may lie before the drafts). Where keys are meant, n is the drafts that the table holds.
template <typename P>
__device__ __forceinline__ uint32_t draft_bits(const P& p, int64_t row, int n, int at) {
  const int i = at >> 5;
  const uint32_t* m = p.tree + row * p.tree_stride;
  const uint32_t w0 = (unsigned)i < (unsigned)p.tree_words ? m[i] : 0u;
  const uint32_t w1 = (unsigned)(i + 1) < (unsigned)p.tree_words ? m[i + 1] : 0u;
  const uint32_t bits = __builtin_amdgcn_alignbit(w1, w0, at & 31);
  const int left = n - at;  // drafts from bit 0 on
  return left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1) : 0u;
}
// An 8-element LDS read of its own alias scope, as lds_read_tr. (The empty asm keeps the scope: without it the
// load is lifted out of the function before its scope is given.)
__device__ __forceinline__ bf16x8 lds_operand(const LDS_AS __bf16* __restrict__ p) {
  asm volatile("");
  return *(const LDS_AS bf16x8*)p;
}
__device__ __forceinline__ f16x8 lds_operand(const LDS_AS _Float16* __restrict__ p) {
  asm volatile("");
  return *(const LDS_AS f16x8*)p;
}
// Position of a query: as many tokens after the last certain one as it sees drafts besides itself.
template <typename P>
__device__ __forceinline__ int draft_position(const P& p, int64_t row, int n, int base) {
  int seen = 0;
  for (int i = 0; i < p.tree_words; ++i) seen += __builtin_popcount(draft_bits(p, row, n, 32 * i));
  return base + max(seen, 1) - 1;
}

}  // namespace lsfa
