// Attention of draft trees over paged KV caches, where a KV head's group has more than
// 16 rows (nodes times query heads), or a few long sequences, for gfx950. The others are fa_window.hip's
// narrow kernel's (its window_plan says which).
//
// A tree's nodes all see the sequence's earlier tokens (under a window its last ones and the
// sinks) and, of one another, those that their masks name: all but the last key tiles are
// whole, and every row tile of a sequence has the same ones. So a workgroup of NW waves takes
// 32 NW (node, query head) rows of a sequence and KV head, wave w rows 32 w .. 32 w + 31: up to 256,
// as the trees and the work of the launch have it (tree_plan), and reads a byte of the cache once for them.
//   key tiles  of BN keys lie in LDS in q's type. 16-bit rows go there by direct loads, two
//              tiles ahead of the one in use; 8-bit ones by way of registers one tile ahead,
//              their scales applied once for all rows.
//   products   S^T = K Q^T and O^T += V^T P^T on v_mfma_f32_32x32x16 (fa_common.hpp has the lane
//              layouts); Q stays in registers.
//   runs       the key tiles of all items (row tiles of a sequence and KV head) are numbered
//              one after another, and every workgroup takes an equal run of them, which may end
//              inside an item or hold several: workgroups end together whatever the lengths. An
//              item in several runs leaves fp32 partial results that a second launch merges.
//
// 32 query heads over 8 KV heads of 128: 16 trees of up to 16 nodes after 512..8192 keys of 16 bits 70 us, bound
// by memory (4.1 TB/s with the merging); 16 of 64 nodes after 1024..8192 of 8 bits 117, where products, softmax, conversions and
// partial results (14 us to merge, 10 to write) share the time (0.67 PFLOP/s); one of 8 nodes after 1500 15, latency.
#include "../../include/lightserve_fa.h"
#include "fa_paged.hpp"

#include <algorithm>
#include <type_traits>

namespace lsfa {

// A sequence's length, keys that the block table holds, nodes and first row of q, and the key tiles that its items have: `sink`
// from key 0 on, then those from tile `first` on (at least one in all, where it has nodes).
template <int BM, int BN>
struct TreeSequence {
  int len, seq, n, tok0;
  int items;  // row tiles times KV heads
  int sink, first, count;
};
template <int BM, int BN, typename P>
__device__ __forceinline__ TreeSequence<BM, BN> tree_sequence(const P& p, int b) {
  TreeSequence<BM, BN> t;
  t.tok0 = min(max(p.cu_q[b], 0), p.tokens);  // (no row outside q, whatever the offsets)
  t.n = min(max(min(p.cu_q[b + 1], p.tokens) - t.tok0, 0), p.max_n);
  // (nodes past max_n are left out at the end of the sequence's rows, not of its keys)
  const int n = max(min(p.cu_q[b + 1], p.tokens) - t.tok0, 0);
  t.len = max(p.seq_lens[b], 0);
  t.seq = min(t.len, min(p.max_seq_len, p.max_blocks << p.block_shift));
  t.items = (int)(((int64_t)t.n * (p.Hq / p.Hkv) + BM - 1) / BM) * p.Hkv;
  t.first = t.sink = 0;
  if (p.window > 0) {
    t.first = min(max(t.len - n - p.window + 1, 0), t.seq) / BN;
    t.sink = min((min(p.sinks, t.seq) + BN - 1) / BN, t.first);
  }
  t.count = t.items > 0 ? max(t.sink + (t.seq + BN - 1) / BN - t.first, 1) : 0;
  t.n = n;
  return t;
}
// All items' key tiles in runs: tiles of a run, and the sequence that holds the first tile of run (ITEMS: item) number `id`
// with the numbers of its own first tile and item; p.B past the last.
constexpr int kRunLeast = 2;  // tiles
struct TreePlace {
  int per, all, b, tile0, item0;
};
template <int BM, int BN, bool ITEMS>
__device__ __forceinline__ TreePlace tree_place(const WindowParams& p, int id, int lane) {
  TreePlace w = {0, 0, p.B, 0, 0};
  TreeSequence<BM, BN> t = {};
  if (lane < p.B) t = tree_sequence<BM, BN>(p, lane);
  int tiles = lanes_sum(t.items * t.count), items = lanes_sum(t.items);  // up to 64 sequences lie in the lanes
  w.all = __builtin_amdgcn_readlane(tiles, 63);
  for (int j = 64; j < p.B; j += 64) {
    TreeSequence<BM, BN> more = {};
    if (j + lane < p.B) more = tree_sequence<BM, BN>(p, j + lane);
    w.all += __builtin_amdgcn_readlane(lanes_sum(more.items * more.count), 63);
  }
  w.per = __builtin_amdgcn_readfirstlane(max((w.all + p.splits - 1) / p.splits, kRunLeast));
  const int64_t at = ITEMS ? (int64_t)id : (int64_t)id * w.per;
  for (int j = 0; j < p.B; j += 64) {
    if (j > 0) {
      t = {};
      if (j + lane < p.B) t = tree_sequence<BM, BN>(p, j + lane);
      tiles = lanes_sum(t.items * t.count), items = lanes_sum(t.items);
    }
    const unsigned long long hit = __ballot(ITEMS ? w.item0 + items > at : w.tile0 + tiles > at);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      w.tile0 += __builtin_amdgcn_readlane(tiles - t.items * t.count, src);
      w.item0 += __builtin_amdgcn_readlane(items - t.items, src);
      w.b = j + src;
      return w;
    }
    w.tile0 += __builtin_amdgcn_readlane(tiles, 63);
    w.item0 += __builtin_amdgcn_readlane(items, 63);
  }
  return w;
}
// Row tile and KV head of item v of sequence b. (The row tiles of a head follow one another; heads are turned from
// sequence to sequence, so that an XCD reads all channels of its L2.)
__device__ __forceinline__ void tree_item(int v, int items, int Hkv, int b, int& rt, int& head) {
  const int rts = items / Hkv, h = v / rts;
  rt = v - h * rts;
  head = (h + b) % Hkv;
}
// Floats of a partial result: (offset, sum for O, sum for the lse, 0) of each row, then O in the
// accumulators' own order, [wave][4-register group][lane].
template <int BM, int DP> constexpr int kTreePart = BM * 4 + BM * DP;

template <typename T> constexpr float kTreeMaxLog2P = 64.0f;
template <> constexpr float kTreeMaxLog2P<_Float16> = 15.0f;

template <typename T, typename C, int DP, int NW, int BN>
__global__ __launch_bounds__((NW * 64), (NW == 8 ? 1 : 2)) void fa_tree_kernel(const WindowParams params) {
  using X8 = typename VecT<T>::x8;
  using X4 = typename VecT<T>::x4;
  constexpr bool Q8 = sizeof(C) == 1;
  constexpr int EB = sizeof(C);
  constexpr int BM = NW * 32;
  constexpr int NS = Q8 ? 2 : 3;           // tiles in LDS
  constexpr int TILE = BN * DP;            // elements of one K or V tile
  constexpr int KSTEPS = DP / 16, DT = DP / 32, KB = BN / 32;
  constexpr int RPW = BN / NW;             // tile rows that a wave loads: 8 or 16, in one cache block
  constexpr int LPR = DP / 8;              // lanes per row, 8 elements each
  constexpr int RPL = 64 / LPR;            // rows per load instruction
  constexpr int NL = RPW / RPL;            // load instructions per wave and tile
  static_assert(NL >= 1 && RPW <= 16 && BN <= 64, "a wave loads whole instructions of one cache block");

  // K, V of tile 0, of tile 1, .., and 16 bytes more. (One variable: between several the compiler sets alias scopes of
  // its own in the place of lds_operand's, and waits for the direct loads of all tiles before each read.)
  __shared__ __attribute__((aligned(1024))) T smem_raw[2 * NS * TILE + 8];
  LDS_AS char* smem = (LDS_AS char*)smem_raw;
  unsigned long long* st_keys = (unsigned long long*)(smem_raw + 2 * NS * TILE);  // keys of a tile whose V is not finite
  int* st_bad = (int*)(st_keys + 1);
  constexpr int BUF = TILE * 2;  // bytes

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const TreePlace place = tree_place<BM, BN, false>(params, blockIdx.x, lane);
  int b = __builtin_amdgcn_readfirstlane(place.b), tile0 = place.tile0;
  if (b >= params.B) return;  // uniform, before any barrier
  int at = blockIdx.x * place.per;
  const int end = min(place.all, at + place.per);

#pragma unroll 1
  do {
    // (the arguments are read again for each item: what the compiler made of them ahead of the loop
    // would not fit the scalar registers through the tiles' one)
    const auto& p = *arguments();
    TreeSequence<BM, BN> sq;
    for (;; ++b) {  // a sequence without nodes has no tiles
      sq = tree_sequence<BM, BN>(p, b);
      if (at < tile0 + sq.items * sq.count) break;
      tile0 += sq.items * sq.count;
    }
    const int seq = __builtin_amdgcn_readfirstlane(sq.seq), n = __builtin_amdgcn_readfirstlane(sq.n);
    const int sink = __builtin_amdgcn_readfirstlane(sq.sink), first = __builtin_amdgcn_readfirstlane(sq.first);
    const int64_t tok0 = __builtin_amdgcn_readfirstlane(sq.tok0);
    const int v = __builtin_amdgcn_readfirstlane((at - tile0) / sq.count);
    const int t_lo = __builtin_amdgcn_readfirstlane(at - tile0 - v * sq.count);
    const int t_hi = __builtin_amdgcn_readfirstlane(min(sq.count, t_lo + end - at));
    const bool whole_item = t_lo == 0 && t_hi == sq.count;
    at += t_hi - t_lo;
    int rt, head;
    tree_item(v, sq.items, p.Hkv, b, rt, head);
    rt = __builtin_amdgcn_readfirstlane(rt), head = __builtin_amdgcn_readfirstlane(head);
    const int len = __builtin_amdgcn_readfirstlane(sq.len);
    const int G = p.Hq / p.Hkv, base = len - n, nrows = min(n, p.max_n) * G;
    const int certain = min(base, seq), drafts = min(n, seq - base);  // keys before the drafts, and drafts, that are there
    const int window = p.window, sinks = window > 0 ? p.sinks : 0;
    const float sl2 = p.scale_abs;

    // The lane's row: it sees keys lo .. certain - 1 (and the sinks) and the drafts of its mask.
    const int r0 = rt * BM + wave * 32, r = r0 + l32, tok = r / G, hq = head * G + (r - tok * G);
    const bool row_ok = r < nrows, live = r0 < nrows;  // live: the wave has rows
    int lo = 0;
    if (window > 0) lo = (row_ok ? draft_position(p, tok0 + tok, n, base) : base) - window + 1;
    const int lo_min = window > 0 ? base - window + 1 : 0, lo_max = window > 0 ? len - window : 0;  // of any row

    u32x4 qraw[KSTEPS];  // the B operand of S^T: row l32, columns 16 kk + 8 hh .. + 7
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const int col = 16 * kk + 8 * hh;
      qraw[kk] = u32x4{0, 0, 0, 0};
      if (row_ok && col < p.D) qraw[kk] = ldg16((const T*)p.q + (tok0 + tok) * p.sqt + (int64_t)hq * p.sqh + col);
    }

    // Loads of the wave's RPW rows of a tile, 8 elements a lane. 8-bit: row (l / LPR) NL + i in
    // instruction i, so that a lane's rows have adjacent scales; 16-bit: what the direct load's linear
    // LDS order makes of the swizzled tile. Rows past the sequence, and pieces (a wave's rows of a tile) that no
    // node sees, read as zeros; what a mask hides within a piece does not matter to S, nor to O where it is finite.
    const __attribute__((address_space(4))) int32_t* table =
        (const __attribute__((address_space(4))) int32_t*)(p.block_tables + (int64_t)b * p.sbt);
    const int block_shift = p.block_shift, D = p.D, num_blocks = p.num_blocks;
    const uint32_t kblock = (uint32_t)(p.skb * EB), kslot = (uint32_t)(p.sks * EB), vblock = (uint32_t)(p.svb * EB), vslot = (uint32_t)(p.svs * EB);
    const char* kbase = (const char*)p.kc + (int64_t)head * p.skh * EB;
    const char* vbase = (const char*)p.vc + (int64_t)head * p.svh * EB;
    const uint8_t* scales = p.scales + ((int64_t)head << (block_shift + 1));
    const uint32_t sblock = (uint32_t)p.Hkv << (block_shift + 1);
    auto key_of = [&](int t) -> int { return (t < sink ? t : t - sink + first) * BN; };
    auto row_at = [&](int i) -> int { return RPW * wave + (Q8 ? lane / LPR * NL + i : i * RPL + lane / LPR); };
    struct Where {
      uint32_t blk, slot;
      int rows;  // that are there; 0: no piece
    };
    auto where = [&](int t) -> Where {
      const int key = key_of(t) + RPW * wave;
      const int blk = t < t_hi && key < seq && (key + RPW > lo_min || key < sinks) ? table[key >> block_shift] : -1;
      const bool ok = (unsigned)blk < (unsigned)num_blocks;
      return {ok ? (uint32_t)blk : 0u, (uint32_t)(key & ((1 << block_shift) - 1)), ok ? min(seq - key, RPW) : 0};
    };
    int ko[NL], vo[NL];  // the lane's offsets in a piece
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int row = row_at(i), col = 8 * (Q8 ? lane % LPR : (lane % LPR) ^ seg_swz<DP>(row));
      ko[i] = col < D ? (row - RPW * wave) * (int)kslot + col * EB : (int)0x80000000;
      vo[i] = col < D ? (row - RPW * wave) * (int)vslot + col * EB : (int)0x80000000;
    }
    auto rows_of = [&](const char* from, uint32_t block, uint32_t slot, const Where& w) -> __amdgpu_buffer_rsrc_t {
      return piece_rsrc(from + ((uint64_t)w.blk * block + (uint64_t)w.slot * slot), w.rows > 0 ? (w.rows - 1) * (int)slot + D * EB : 0);
    };
    constexpr int EW = NL == 4 ? 2 : 1;  // words of a lane's scales (K and V of NL rows)
    struct Codes {
      u32x2 k[NL], v[NL];
      uint32_t e[EW];
    };
    auto load_codes = [&](Codes& c, const Where& w) {
      const __amdgpu_buffer_rsrc_t kr = rows_of(kbase, kblock, kslot, w), vr = rows_of(vbase, vblock, vslot, w);
      const __amdgpu_buffer_rsrc_t er = piece_rsrc(scales + ((uint64_t)w.blk * sblock + w.slot * 2), w.rows > 0 ? 2 * RPW : 0);
#pragma unroll
      for (int i = 0; i < NL; ++i) c.k[i] = load8b(kr, ko[i]);
#pragma unroll
      for (int i = 0; i < NL; ++i) c.v[i] = load8b(vr, vo[i]);
      if constexpr (NL == 1) c.e[0] = load2(er, 2 * (row_at(0) - RPW * wave));
      else load_words<EW>(er, 2 * (row_at(0) - RPW * wave), c.e);
    };
    // (A row past the sequence has codes of zero here, but its scale may be anything: infinity, which
    // 255 stands for, would make NaN of them.)
    auto write_codes = [&](const Codes& c, int buf) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int to = buf * 2 * BUF + swz_off<DP>(row_at(i), 8 * (lane % LPR)) * 2;
        const uint32_t e = c.e[i / 2] >> (16 * (i & 1));
        const float ks = fminf(__uint_as_float((e << 23) & 0x7f800000u), 0x1p127f), vs = fminf(__uint_as_float((e << 15) & 0x7f800000u), 0x1p127f);
        *(LDS_AS u32x4*)(smem + to) = u32x4{codes2<false>(c.k[i][0], ks, T()), codes2<true>(c.k[i][0], ks, T()),
                                            codes2<false>(c.k[i][1], ks, T()), codes2<true>(c.k[i][1], ks, T())};
        *(LDS_AS u32x4*)(smem + to + BUF) = u32x4{codes2<false>(c.v[i][0], vs, T()), codes2<true>(c.v[i][0], vs, T()),
                                                  codes2<false>(c.v[i][1], vs, T()), codes2<true>(c.v[i][1], vs, T())};
      }
    };
    auto load_direct = [&](const Where& w, int buf) {
      const __amdgpu_buffer_rsrc_t kr = rows_of(kbase, kblock, kslot, w), vr = rows_of(vbase, vblock, vslot, w);
      LDS_AS char* to = smem + buf * 2 * BUF + RPW * wave * DP * 2;
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(kr, (LDS_AS void*)(to + i * RPL * DP * 2), ko[i]);
#pragma unroll
      for (int i = 0; i < NL; ++i) dma16(vr, (LDS_AS void*)(to + BUF + i * RPL * DP * 2), vo[i]);
    };

    // LDS offsets of the operands: the segment index of a column step differs from the first one's by
    // an xor of whole bits (swz_off), so that one register each does for all of them; taken through an empty
    // asm in every step, or the compiler hoists all results out of the loop and spills.
    int koff = swz_off<DP>(l32, 8 * hh) * 2;
    const int tr_row = 4 * hh + ((lane & 15) >> 2), tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    int voff0 = swz_off<DP>(tr_row, tr_col) * 2, voff1 = swz_off<DP>(tr_row + 8, tr_col) * 2;
    const float kTileSumMax = __builtin_exp2f(kTreeMaxLog2P<T>);
    // Reads of operands run this many products ahead of the one that takes them (in the written order: the
    // compiler's own has each product wait for its read where registers are short).
    constexpr int kAhead = 4;

    f32x16 acc[DT];
    float m_run, l_run, l_lse;
    // V's infinities and NaN, with the weight of zero of a row that does not see them, make NaN of that row's
    // sums. Sums that are not finite are therefore taken again, with such values left out of the products and
    // added to the rows that see them (ordinary caches have none).
    bool careful = false;
    Codes c;
    Where w2;
    auto load_first = [&]() {
      const Where w1 = where(t_lo + 1);
      w2 = where(t_lo + 2);
      if constexpr (Q8) {
        load_codes(c, where(t_lo));
      } else {
        load_direct(where(t_lo), 0);
        load_direct(w1, 1);
      }
    };
    load_first();
    // (Q is waited for behind the first tiles' loads, and ahead of the tiles' loop)
    X8 q[KSTEPS];
    const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qraw[kk] ^= flip;
      asm volatile("" : "+v"(qraw[kk]));
      q[kk] = __builtin_bit_cast(X8, qraw[kk]);
    }
#pragma unroll 1
    for (int pass = 0; pass < 2; ++pass) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
      m_run = -1e30f, l_run = 0.f, l_lse = 0.f;
      bool begun = false;
      if (tid == 0) *st_bad = 0;
      if constexpr (Q8) {
        write_codes(c, 0);
        load_codes(c, where(t_lo + 1));
      }
      int buf = 0;
#pragma unroll 1
      for (int t = t_lo; t < t_hi; ++t) {
        if constexpr (Q8) {
          // Tile t is in LDS once every wave has written its rows, and none reads tile t - 1 any more.
          __syncthreads();
          write_codes(c, buf ^ 1);
          load_codes(c, w2);
        } else {
          // (2 NL younger loads of the wave are tile t + 1's; LDS operations of its own are done too)
          asm volatile("" ::: "memory");
          __builtin_amdgcn_s_waitcnt(0x0070 | (2 * NL));  // vmcnt(2 NL), lgkmcnt(0)
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          load_direct(w2, buf == 0 ? 2 : buf - 1);
        }
        w2 = where(t + 3);
        LDS_AS char* Ks = smem + buf * 2 * BUF;
        LDS_AS char* Vs = Ks + BUF;
        if constexpr (Q8) buf ^= 1;
        else buf = buf == 2 ? 0 : buf + 1;
        const int key0 = key_of(t);
        unsigned long long bad_keys = 0;
        if (__builtin_expect(careful, 0)) {
          if (tid == 0) *st_keys = 0;
          __syncthreads();
#pragma unroll 1
          for (int i = 0; i < NL; ++i) {
            const int row = RPW * wave + i * RPL + lane / LPR;
            LDS_AS u32x4* at_row = (LDS_AS u32x4*)(Vs + row * DP * 2 + (lane % LPR) * 16);
            u32x4 x = *at_row;
            uint32_t found = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bits = not_finite<T, false>(x[e]);
              found |= bits;
              x[e] &= ~bits;
            }
            *at_row = x;
            if (found != 0) atomicOr(st_keys, 1ull << row);
          }
          __syncthreads();
          bad_keys = *st_keys;
        }
        if (live) {
          f32x16 s[KB];
          __builtin_amdgcn_sched_barrier(0);
          asm volatile("" : "+v"(koff), "+v"(voff0), "+v"(voff1));
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
          auto k_operand = [&](int j) -> X8 {
            return lds_operand((const LDS_AS T*)(Ks + j % KB * 32 * DP * 2 + (koff ^ (j / KB << 5))));
          };
          {
            X8 a[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) a[j] = k_operand(j);
#pragma unroll
            for (int j = 0; j < KSTEPS * KB; ++j) {
              __builtin_amdgcn_sched_barrier(0);
              s[j % KB] = mfma32(a[j % kAhead], q[j / KB], s[j % KB]);
              if (j + kAhead < KSTEPS * KB) a[j % kAhead] = k_operand(j + kAhead);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (!(key0 + BN <= certain && (key0 >= lo_max || key0 + BN <= sinks))) {
            asm volatile("" ::: "memory");  // stays a branch
            const int up = row_ok ? certain - key0 - 4 * hh : 0, dn = lo - key0 - 4 * hh, sk = sinks - key0 - 4 * hh;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              const uint32_t tree = row_ok ? draft_bits(p, tok0 + tok, drafts, key0 + 32 * kb - base) >> (4 * hh) : 0u;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const int k = 32 * kb + 8 * (i >> 2) + (i & 3);
                const bool sees = row_ok && ((k < up && (k >= dn || k < sk)) || (tree >> (k & 31) & 1));
                s[kb][i] = sees ? s[kb][i] : -INFINITY;
              }
            }
          }
          auto row_max = [&]() -> float {
            float mx = s[0][0];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
#pragma unroll
              for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
            mx = half_max(mx);
            return mx == -INFINITY ? -INFINITY : mx * sl2;
          };
          if (!begun) m_run = fmaxf(row_max(), -1e30f), begun = true;
          // Exponentials with the current offset, rounded into the PV operands; x: the lane's part of the sum
          // that normalises O (bf16: of the rounded p, so that the weights sum to one exactly; fp16: of
          // the fp32 p), y: of the fp32 p.
          X8 pb[2 * KB];
          auto softmax = [&]() -> float2 {
            constexpr bool kF16 = __is_same(T, _Float16);
            const float neg_m = -m_run;
            float rs[4] = {-0.f, -0.f, -0.f, -0.f}, re[4] = {-0.f, -0.f, -0.f, -0.f};
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              f32x16 e;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                e[i] = fast_exp2(fmaf(s[kb][i], sl2, neg_m));
                re[i & 3] += e[i];
              }
              pb[2 * kb] = pack8<T>(e, 0);
              pb[2 * kb + 1] = pack8<T>(e, 8);
              if constexpr (!kF16) {
                sum8_into(pb[2 * kb], rs);
                sum8_into(pb[2 * kb + 1], rs);
              }
            }
            float2 x;
            x.y = (re[0] + re[1]) + (re[2] + re[3]);
            x.x = kF16 ? x.y : (rs[0] + rs[1]) + (rs[2] + rs[3]);
            return x;
          };
          // The offset of a row is its first tile's maximum and rises only where p would come near the
          // operands' range: then the tile's exponentials are taken again.
          float2 ts = softmax();
          if (__builtin_amdgcn_ballot_w64(ts.x > kTileSumMax) != 0) {
            const float mx = row_max();
            if (__builtin_amdgcn_ballot_w64(mx > m_run) != 0) {
              const float m_new = fmaxf(m_run, mx);
              const float alpha = fast_exp2(m_run - m_new);
              l_run *= alpha;
              l_lse *= alpha;
              m_run = m_new;
#pragma unroll
              for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
            }
            ts = softmax();
          }
          l_run += ts.x;
          l_lse += ts.y;
          auto v_operand = [&](int j) -> X8 {
            const LDS_AS char* from = Vs + j % (2 * KB) * 16 * DP * 2;
            const int dt = j / (2 * KB);
            return cat4<X8, X4>(lds_read_tr((const LDS_AS T*)(from + (voff0 ^ (dt << 6)))),
                                lds_read_tr((const LDS_AS T*)(from + (voff1 ^ (dt << 6)))));
          };
          {
            X8 a[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) a[j] = v_operand(j);
#pragma unroll
            for (int j = 0; j < DT * 2 * KB; ++j) {
              __builtin_amdgcn_sched_barrier(0);
              acc[j / (2 * KB)] = mfma32(a[j % kAhead], pb[j % (2 * KB)], acc[j / (2 * KB)]);
              if (j + kAhead < DT * 2 * KB) a[j % kAhead] = v_operand(j + kAhead);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          if (__builtin_expect(bad_keys != 0, 0)) {
#pragma unroll 1
            for (unsigned long long left = bad_keys; left != 0; left &= left - 1) {
              int d0 = 4 * hh, most = D;  // (not known ahead of the loop, or what follows from them is kept through it)
              asm volatile("" : "+v"(d0), "+s"(most));
              const int key = key0 + __builtin_ctzll(left);
              const int blk = table[key >> block_shift];
              const bool sees = row_ok && ((key < certain && (key >= lo || key < sinks)) || (draft_bits(p, tok0 + tok, drafts, key - base) & 1));
              if ((unsigned)blk >= (unsigned)num_blocks || !sees) continue;
              const C* from = (const C*)(vbase + (uint64_t)blk * vblock + (uint64_t)(key & ((1 << block_shift) - 1)) * vslot);
#pragma unroll
              for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                  const int d = 32 * dt + 8 * g + d0;
                  if (d >= most) continue;
                  uint32_t w[2] = {*(const uint32_t*)(from + d), 0};
                  if constexpr (!Q8) w[1] = *(const uint32_t*)(from + d + 2);
                  w[0] &= not_finite<T, Q8>(w[0]), w[1] &= not_finite<T, Q8>(w[1]);
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[dt][4 * g + e] += bad_value<T, Q8>(w, e);
                }
            }
          }
        }
      }
      if (!careful && live && __builtin_amdgcn_ballot_w64(!all_finite(acc)) != 0) *st_bad = 1;
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (loads of tiles past the last, of nothing, write zeros to LDS)
      __syncthreads();
      if (*st_bad == 0) break;
      careful = true;
      load_first();
      __syncthreads();  // before the flag is cleared
    }

    const auto& a = *arguments();
    int row0 = r0;  // (as above)
    asm volatile("" : "+s"(row0));
    const float lt = half_sum(l_run), le = half_sum(l_lse);
    if (!whole_item) {
      // (a run has at most two parts of items, the end of one and the beginning of one)
      if (row_ok) {
        float* part = a.part + (2 * (int64_t)blockIdx.x + (t_lo == 0)) * kTreePart<BM, DP>;
        if (hh == 0) *(f32x4*)(part + (wave * 32 + l32) * 4) = f32x4{m_run, lt, le, 0.f};
        f32x4* po = (f32x4*)(part + BM * 4) + wave * DT * 4 * 64 + lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            po[(dt * 4 + g) * 64] = f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
      }
    } else {
      // O leaves through LDS: each wave stages its 32 rows and stores whole ones.
      const float inv = lt == 0.f ? 0.f : 1.f / lt;
      constexpr int BLK = 32 * DP * 2;
      static_assert(NW * BLK <= 2 * NS * TILE * 2, "O staging fits in the K/V buffers");
      LDS_AS char* wb = smem + wave * BLK;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          X4 v4;
#pragma unroll
          for (int e = 0; e < 4; ++e) v4[e] = (T)(acc[dt][4 * g + e] * inv);
          *(LDS_AS X4*)(wb + swz_off<DP>(l32, 32 * dt + 8 * g + 4 * hh) * 2) = v4;
        }
#pragma unroll
      for (int i = 0; i < BLK / 1024; ++i) {
        const int byte = i * 1024 + lane * 16;
        const int row = byte / (DP * 2), seg = (byte % (DP * 2)) / 16;
        const X8 x = *(const LDS_AS X8*)(wb + row * DP * 2 + ((seg ^ seg_swz<DP>(row)) << 4));
        const int rr = row0 + row, tk = rr / G, h = head * G + (rr - tk * G);
        if (rr < nrows && seg * 8 < a.D) *(X8*)((T*)a.o + (tok0 + tk) * a.sot + (int64_t)h * a.soh + seg * 8) = x;
      }
      if (row_ok && hh == 0 && a.lse != nullptr)
        a.lse[(tok0 + tok) * a.slt + (int64_t)hq * a.slh] = le == 0.f ? -INFINITY : (m_run + __log2f(le)) * kWinLn2;
    }
    __syncthreads();  // the next item's tiles take the place of what is staged in LDS
  } while (at < end);
}

// Merges the partial results of items in several runs: workgroup (item, dt) combines 32 channels of the item's
// rows in the accumulators' order. NG groups of waves take every NG-th run and meet in LDS (a sequence of 8000 tokens alone
// lies in some 80 runs, whose results one wave after another would wait for).
template <int NW> constexpr int kGroups = 8 / NW;
template <typename T, int DP, int NW, int BN>
__global__ __launch_bounds__((NW * kGroups<NW> * 64)) void fa_tree_combine_kernel(const WindowParams p) {
  using X4 = typename VecT<T>::x4;
  constexpr int BM = NW * 32, DT = DP / 32, NG = kGroups<NW>, U = 8;  // U: results in flight
  __shared__ f32x4 meet[NG > 1 ? NG - 1 : 1][5][NW * 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6) % NW, dt = blockIdx.y;
  const int group = __builtin_amdgcn_readfirstlane(tid / (NW * 64));
  const int l32 = lane & 31, hh = lane >> 5, G = p.Hq / p.Hkv;
  const TreePlace place = tree_place<BM, BN, true>(p, blockIdx.x, lane);
  const int b = __builtin_amdgcn_readfirstlane(place.b), per = place.per;
  if (b >= p.B) return;
  const TreeSequence<BM, BN> sq = tree_sequence<BM, BN>(p, b);
  const int v = (int)blockIdx.x - place.item0, at = place.tile0 + v * sq.count;
  const int first = __builtin_amdgcn_readfirstlane(at / per), n = __builtin_amdgcn_readfirstlane((at + sq.count - 1) / per) - first + 1;
  if (n <= 1) return;  // already in o
  int rt, head;
  tree_item(v, sq.items, p.Hkv, b, rt, head);
  const int r = rt * BM + wave * 32 + l32, nrows = min(sq.n, p.max_n) * G;
  float M = -1e30f, L = 0.f, E = 0.f;
  f32x4 O[4] = {};
  auto take = [&](const f32x4& st, const f32x4 (&o)[4]) {
    const float m = fmaxf(M, st[0]), a = fast_exp2(M - m), w = fast_exp2(st[0] - m);
    L = a * L + w * st[1];
    E = a * E + w * st[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) O[g] = a * O[g] + w * o[g];
    M = m;
  };
  if (rt * BM + wave * 32 < nrows) {
    for (int i = group; i < n; i += NG * U) {
      f32x4 st[U], o[U][4];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int k = i + NG * u;
        if (k >= n) break;  // (uniform)
        const float* part = p.part + (2 * (int64_t)(first + k) + (k == 0)) * kTreePart<BM, DP>;
        st[u] = *(const f32x4*)(part + (wave * 32 + l32) * 4);
        const f32x4* po = (const f32x4*)(part + BM * 4) + (wave * DT + dt) * 4 * 64 + lane;
#pragma unroll
        for (int g = 0; g < 4; ++g) o[u][g] = po[g * 64];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i + NG * u < n) take(st[u], o[u]);
    }
  }
  if (group > 0) {
    meet[group - 1][0][wave * 64 + lane] = f32x4{M, L, E, 0.f};
#pragma unroll
    for (int g = 0; g < 4; ++g) meet[group - 1][1 + g][wave * 64 + lane] = O[g];
  }
  __syncthreads();
  if (group > 0 || r >= nrows) return;
#pragma unroll 1
  for (int k = 0; k < min(n, NG) - 1; ++k) {
    const f32x4 o[4] = {meet[k][1][wave * 64 + lane], meet[k][2][wave * 64 + lane], meet[k][3][wave * 64 + lane], meet[k][4][wave * 64 + lane]};
    take(meet[k][0][wave * 64 + lane], o);
  }
  const int tok = r / G, hq = head * G + (r - tok * G);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* o = (T*)p.o + ((int64_t)sq.tok0 + tok) * p.sot + (int64_t)hq * p.soh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int d = 32 * dt + 8 * g + 4 * hh;
    X4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (T)(O[g][e] * inv);
    if (d < p.D) *(X4*)(o + d) = x;
  }
  if (dt == 0 && hh == 0 && p.lse != nullptr)
    p.lse[((int64_t)sq.tok0 + tok) * p.slt + (int64_t)hq * p.slh] = E == 0.f ? -INFINITY : (M + __log2f(E)) * kWinLn2;
}

// ---------------------------------------------------------------- launches
constexpr int tree_keys(int waves) { return waves == 8 ? 64 : 32; }

// How a launch goes, from what the host knows (seen: most keys of a sequence).
WindowPlan tree_plan(int B, int tokens, int Hkv, int G, int dp, int max_n, long long seen) {
  WindowPlan w = {};
  const long long rows = (long long)max_n * G;
  // More waves read a key tile for more rows and keep fewer workgroups resident: eight pay from eight tiles a resident
  // workgroup, four from five. Waves 2, 4 and 8 on 32 query heads over 8 of 128 (us): 64 nodes after 1500 keys 27, 30, 33,
  // after 8000 42, 38, 46; four trees of 64 after 1500 keys 43, 33, 38, after 4000 67, 45, 44; 16 after 6000 287, 169, 148.
  for (w.waves = 8;; w.waves /= 2) {
    const long long bm = w.waves * 32, bn = tree_keys(w.waves), slots = w.waves == 8 ? 256 : w.waves == 4 ? 512 : 768;
    w.items = (int)(Hkv * std::min((long long)tokens * G / bm + B, (rows + bm - 1) / bm * B));
    const long long tiles = ((seen + bn - 1) / bn + 1) * w.items;
    if (w.waves > 2 && (rows <= bm / 2 || tiles < slots * (w.waves == 8 ? 8 : 5))) continue;
    // As many runs as workgroups are resident, of at least kRunLeast tiles.
    w.splits = (int)std::max(1LL, std::min(slots, (tiles + kRunLeast - 1) / kRunLeast));
    break;
  }
  const long long bm = w.waves * 32;
  w.part_bytes = LSFA_GEMV_COUNTER_BYTES + (uint64_t)w.splits * 2 * (bm * (4 + dp)) * 4;
  return w;
}

template <typename T, typename C, int DP, int NW>
static hipError_t launch_tree(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  hipLaunchKernelGGL((fa_tree_kernel<T, C, DP, NW, tree_keys(NW)>), dim3(w.splits), dim3(NW * 64), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((fa_tree_combine_kernel<T, DP, NW, tree_keys(NW)>), dim3(w.items, DP / 32), dim3(NW * kGroups<NW> * 64), 0, s, p);
  return hipGetLastError();
}
template <typename T, typename C, int DP>
static hipError_t launch_waves(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  if (w.waves == 8) return launch_tree<T, C, DP, 8>(p, w, s);
  return w.waves == 4 ? launch_tree<T, C, DP, 4>(p, w, s) : launch_tree<T, C, DP, 2>(p, w, s);
}
template <typename T>
static hipError_t dispatch_tree(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  if (p.scales != nullptr) return p.D <= 64 ? launch_waves<T, uint8_t, 64>(p, w, s) : launch_waves<T, uint8_t, 128>(p, w, s);
  return p.D <= 64 ? launch_waves<T, T, 64>(p, w, s) : launch_waves<T, T, 128>(p, w, s);
}
hipError_t tree_attention(const WindowParams& p, const WindowPlan& w, bool is_bf16, hipStream_t s) {
  return is_bf16 ? dispatch_tree<__bf16>(p, w, s) : dispatch_tree<_Float16>(p, w, s);
}

}  // namespace lsfa
