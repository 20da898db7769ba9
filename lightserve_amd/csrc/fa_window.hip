// Attention over paged KV caches of 8 or 16 bits, with a sliding window and
// sinks, for gfx950.
//
// A query at position p sees key j where j <= p (causal) and, under a window of
// w tokens with s sinks, j > p - w or j < s. Sequence b's queries are the last
// n of its seq_lens[b] cached tokens (one for a decode step). An 8-bit cache
// holds e4m3 codes and one power-of-two scale for each row (fa_kvq.hip).
// In a tree of drafted tokens (TREE) the n queries see the tokens before them and, of
// one another, those that their masks name; trees of more rows are fa_tree.hip's (window_plan).
//
// Few rows per KV head (decode, and chunks of a few tokens): the narrow kernel.
// Many: the wide one, further down.
// The narrow path is bound by HBM (64 sequences of 8192 tokens, 8 KV heads of 128, 8
// bits: 203 us, 5.3 TB/s; 64 windows of 4096: 112-114 us, 4.8, of 16 bits 193 us, 5.6) or,
// for one sequence, by latency (1500 tokens 10 us, 32768 27, 131072 64), so it is built
// around bytes in flight, and each byte of the cache is read once for all query heads that
// share it. (Where comments below set two variants side by side, both were timed in replayed
// graphs of a few calls, 2 to 3 us above the kernels' own time.)
//   rows       (token, query head of the KV head's group) pairs, 16 or 32 to a row
//              tile, are the columns of S^T = K Q^T and of O^T += V^T P^T on
//              v_mfma_f32_16x16x32. Q lies in LDS: registers hold loads in flight.
//   key tiles  of 32 keys: two pieces of 16 that each lie in one cache block,
//              so that a piece takes one buffer descriptor built from one
//              block-table entry (scalar work); pieces past the sequence and
//              entries outside the cache read as zeros.
//   K          straight from the cache into the A operand: lane (g, c) = (l / 16,
//              l % 16) holds key c's elements g D/4 .. of a piece (any order of
//              the summed dimension does, as long as Q has the same).
//   V          lane (g, c) holds 8 keys (4g .. 4g + 3 of both pieces, which are
//              the keys whose P the lane computed) times D / 16 adjacent
//              channels; the operand of MFMA j, channel (D/16) c + j of the 8
//              keys, is put together by v_perm. No LDS, no shuffle of P.
//   8 bits     codes become bf16 or fp16 (exact) on load, V's with its rows'
//              scales (the conversion takes one), K's scales multiply S.
// A wave keeps one tile of K and V in flight while it works on the one before.
//
// Work is shared out evenly whatever the lengths: the key tiles of all sequences
// are numbered one after another and every workgroup takes an equal run of
// them, which may end inside a sequence or hold several. A sequence that lies
// in several runs leaves fp32 partial results: a second launch merges those of
// long runs, the last run to arrive those of short ones, whose launches are a few
// microseconds. Either way they are added in the runs' order, whichever ends first.
#include "../../include/lightserve_fa.h"
#include "fa_paged.hpp"

#include <algorithm>
#include <type_traits>

namespace lsfa {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Tiles of a run: the tiles there are over the runs there are, no less than one for each wave.
__device__ __forceinline__ int run_tiles(int all, int runs) {
  return __builtin_amdgcn_readfirstlane(max((all + runs - 1) / runs, 4));
}
// Runs of at least long_run tiles (WindowPlan's, from what a partial result weighs) are long
// ones: a workgroup then takes two or four adjacent KV heads (a wave each, or two) for as
// many times fewer tiles, and runs meet in fa_window_combine_kernel.
__device__ __forceinline__ bool long_runs(const WindowParams& p, int all) {
  return p.long_run > 0 && run_tiles(all, p.runs) >= p.long_run;
}
// KV heads of a workgroup in a launch of long runs.
__device__ __forceinline__ int heads_per_group(const WindowParams& p) { return (p.Hkv & 3) == 0 ? 4 : (p.Hkv & 1) == 0 ? 2 : 1; }
// Partial result of run r of a row tile and KV head: O of part_rows rows, then (offset,
// sum for O, sum for the lse, 0) of each. A run has two: the end of a sequence and,
// first_run, the beginning of one.
template <int DP, typename P>
__device__ __forceinline__ float* part_of(const P& p, int rt, int head, int runs, int r, bool first_run) {
  return p.part + (((int64_t)rt * p.Hkv + head) * 2 * runs + 2 * r + first_run) * (p.part_rows * (DP + 4));
}
// Sums over the keys of one row (offset M in log2 units) taking in those of others.
struct RowSums {
  float M = -1e30f, L = 0.f, E = 0.f;
  f32x4 O = {};
  __device__ __forceinline__ void take(const f32x4& st, const f32x4& o) {
    const float m = fmaxf(M, st[0]), a = fast_exp2(M - m), w = fast_exp2(st[0] - m);
    L = a * L + w * st[1];
    E = a * E + w * st[2];
    O = a * O + w * o;
    M = m;
  }
};

// Channels d .. d + 3 of row r of a sequence and KV head from the sums over its keys
// (offset M in log2 units), and its lse with channel 0.
template <typename T, typename P>
__device__ __forceinline__ void store_row(const P& p, int64_t tok0, int r, int G, int head, int d, float M, float L,
                                          float E, const f32x4& O) {
  const int tok = r / G, h = head * G + (r - tok * G);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  if (d < p.D) {
    typename VecT<T>::x4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = (T)(O[e] * inv);
    *(typename VecT<T>::x4*)((T*)p.o + (tok0 + tok) * p.sot + (int64_t)h * p.soh + d) = out;
  }
  if (d == 0 && p.lse != nullptr)
    p.lse[(tok0 + tok) * p.slt + (int64_t)h * p.slh] = E == 0.f ? -INFINITY : (M + __log2f(E)) * kWinLn2;
}

// Four floats at device scope: written through to, and read from, where all XCDs see them.
__device__ __forceinline__ void store_device(float* to, const f32x4& v) {
  const u32x4 w = __builtin_bit_cast(u32x4, v);
  __hip_atomic_store((uint64_t*)to, w[0] | (uint64_t)w[1] << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __hip_atomic_store((uint64_t*)to + 1, w[2] | (uint64_t)w[3] << 32, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x4 load_device(const float* from) {
  const uint64_t a = __hip_atomic_load((uint64_t*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  const uint64_t b = __hip_atomic_load((uint64_t*)from + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return f32x4{__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32)), __uint_as_float((uint32_t)b),
               __uint_as_float((uint32_t)(b >> 32))};
}

constexpr int kRowTile = 16;  // rows of a column block; a row tile has one or two

// NC column blocks of 16 rows share the tile's K and V operands. ONE: of a decode step, whose
// rows all see the same keys. TREE: of draft trees.
template <typename T, typename C, int DP, int NC, bool ONE, bool TREE>
__global__ __launch_bounds__(256, 2) void fa_window_narrow_kernel(const WindowParams p) {
  using X8 = typename VecT<T>::x8;
  constexpr bool Q8 = sizeof(C) == 1;
  constexpr int EB = sizeof(C);           // bytes of a cached element
  constexpr int NW = 4;
  constexpr int RT = kRowTile * NC;       // rows of a row tile
  constexpr int KK = DP / 32;             // MFMAs of S per 16 keys
  constexpr int KD = DP * EB / 64;        // 16-byte loads of K per lane and piece
  constexpr int VJ = DP / 16;             // channels per lane, MFMAs of O
  constexpr int VW = VJ * EB / 4;         // 32-bit words of V per lane and key
  constexpr int QS = DP + 8;              // elements between rows of Q in LDS (8: the 16 lanes' rows on other banks)
  constexpr float kThreshold = 8.0f;      // log2 units

  __shared__ float st_o[NW][kRowTile][DP];
  __shared__ __attribute__((aligned(16))) T st_q[NW][RT * QS];  // of each head
  __shared__ float st_m[NW][RT], st_l[NW][RT], st_e[NW][RT];
  __shared__ bool st_last;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int G = p.Hq / p.Hkv;

  // The runs' tiles, this run's, the sequence that holds its first one, and the number of
  // that sequence's first tile. (Up to 64 sequences lie in the lanes.)
  KeyTiles mine = {};
  if (lane < p.B) mine = key_tiles<TREE>(p, lane);
  int upto = lanes_sum(mine.count), all = __builtin_amdgcn_readlane(upto, 63);
  for (int j = 64; j < p.B; j += 64) {
    const int more = j + lane < p.B ? key_tiles<TREE>(p, j + lane).count : 0;
    all += __builtin_amdgcn_readlane(lanes_sum(more), 63);
  }
  // Adjacent heads' rows of a token are adjacent in the cache: read by one workgroup
  // they are asked for together, in pieces of 2 or 4 rows (512 bytes at head dim 128 and 8
  // bits) where one head's alone reach HBM as 128-byte ones (64 sequences of 8192 tokens,
  // 8 KV heads: 210 us, 227 with a head each; 64 windows of 4096, 120 and 130). Few tiles
  // stay shared out over the waves of one head, which end sooner.
  const bool deferred = long_runs(p, all);
  const int hw = deferred ? heads_per_group(p) : 1;
  const int groups = p.Hkv / hw, columns = gridDim.x / hw, runs = p.runs * hw, nk = NW / hw;  // nk: waves that share a head's tiles
  const int id = blockIdx.y * gridDim.x + blockIdx.x;
  const int run = __builtin_amdgcn_readfirstlane(id / columns), column = id - run * columns;
  const int rt = __builtin_amdgcn_readfirstlane(column / groups), head_0 = (column - rt * groups) * hw;
  const int wave_k = wave / hw, head = head_0 + wave - wave_k * hw;
  const int per = run_tiles(all, runs);
  if ((int64_t)run * per >= all) return;  // uniform, before any barrier
  const int start = run * per, end = min(all, start + per);
  int b = 0, at = 0, have = mine.count;
  for (int j = 0; j < p.B; j += 64) {
    if (j > 0) {
      have = j + lane < p.B ? key_tiles<TREE>(p, j + lane).count : 0;
      upto = lanes_sum(have);
    }
    const unsigned long long hit = __ballot(at + upto > start);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      b = j + src;
      at += __builtin_amdgcn_readlane(upto - have, src);
      break;
    }
    at += __builtin_amdgcn_readlane(upto, 63);
  }

  const uint32_t kOut = 0x80000000u;  // past every descriptor: reads as zero
  uint32_t ko[KD];
#pragma unroll
  for (int i = 0; i < KD; ++i) {
    const int byte = 64 * i + 16 * g;  // a load takes 64 bytes of each of the 16 rows
    ko[i] = byte < p.D * EB ? (uint32_t)(c * (int)p.sks * EB + byte) : kOut;
  }
  const uint32_t vo = c * VJ < p.D ? (uint32_t)(4 * g * (int)p.svs * EB + c * VJ * EB) : kOut;
  const uint32_t vstep = vo == kOut ? 0 : (uint32_t)((int)p.svs * EB);
  const int kbytes = (15 * (int)p.sks + p.D) * EB, vbytes = (15 * (int)p.svs + p.D) * EB;
  // Byte strides of a block (below 2^32, so that a block's address is one 32 x 32-bit
  // product) and of a slot, and where the head's rows of block 0 are.
  const uint32_t kblock = (uint32_t)(p.skb * EB), vblock = (uint32_t)(p.svb * EB), sblock = (uint32_t)p.Hkv << (p.block_shift + 1);
  const uint32_t kslot = (uint32_t)(p.sks * EB), vslot = (uint32_t)(p.svs * EB);
  const char* kbase = (const char*)p.kc + (int64_t)head * p.skh * EB;
  const char* vbase = (const char*)p.vc + (int64_t)head * p.svh * EB;
  const char* sbase = (const char*)p.scales + ((int64_t)head << (p.block_shift + 1));
  const int slot_mask = (1 << p.block_shift) - 1;
  const int sinks = p.window > 0 ? p.sinks : 0;

  for (; b < p.B && at < end; ++b) {
    KeyTiles kt;
    if (p.B <= 64) {
      kt = key_tiles_of<TREE>(p, __builtin_amdgcn_readlane(mine.len, b), __builtin_amdgcn_readlane(mine.n, b),
                        __builtin_amdgcn_readlane(mine.tok0, b));
    } else {
      kt = key_tiles<TREE>(p, b);
      kt = key_tiles_of<TREE>(p, __builtin_amdgcn_readfirstlane(kt.len), __builtin_amdgcn_readfirstlane(kt.n),
                        __builtin_amdgcn_readfirstlane(kt.tok0));
    }
    const int count = kt.count, seq = kt.seq, n = kt.n, sink = kt.sink, first = kt.first, head0 = at;
    const int base = kt.len - n;  // TREE: the first draft's key
    if (count == 0) continue;
    const int ta = max(start - at, 0), tb = min(count, end - at);
    at += count;
    const int nrows = min(n, p.max_n) * G - rt * RT;  // of this row tile
    if (nrows <= 0) continue;
    const int64_t tok0 = kt.tok0;

    // Q, the B operand of S^T, to LDS: kept in registers it would cost the waves that
    // keep the loads of K and V in flight.
    const auto* args = arguments();
    for (int i = tid; i < hw * RT * (DP / 8); i += 256) {
      const int hs = i / (RT * (DP / 8)), row = i / (DP / 8) % RT, d = i % (DP / 8) * 8, r = rt * RT + row, tok = r / G;
      u32x4 raw = {0, 0, 0, 0};
      if (row < nrows && d < args->D)
        raw = ldg16((const T*)args->q + (tok0 + tok) * args->sqt + (int64_t)((head_0 + hs) * G + (r - tok * G)) * args->sqh + d);
      *(u32x4*)(st_q[hs] + row * QS + d) = raw;
    }
    // The lane's rows see keys lo .. hi.
    int hi[NC], lo[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      const bool row_ok = 16 * x + c < nrows;
      int pos = p.causal ? seq - n + (rt * RT + 16 * x + c) / G : seq - 1;
      if constexpr (TREE) pos = row_ok && p.window > 0 ? draft_position(p, tok0 + (rt * RT + 16 * x + c) / G, n, base) : 0;
      hi[x] = row_ok ? (TREE ? min(base, seq) - 1 : pos) : -1;  // (TREE: beside the drafts of its mask)
      lo[x] = p.window > 0 ? pos - p.window + 1 : 0;
    }
    // TREE: drafts that the lane's row of column block x sees among the 32 keys from key0 on.
    auto drafts = [&](int x, int key0) -> uint32_t {
      return 16 * x + c < nrows ? draft_bits(p, tok0 + (rt * RT + 16 * x + c) / G, min(n, seq - base), key0 - base) : 0u;
    };
    // The same of the tile's first and last rows.
    const int t0 = rt * RT / G, t1 = (rt * RT + min(nrows, RT) - 1) / G;
    const int hi_min = __builtin_amdgcn_readfirstlane(TREE ? min(base, seq) - 1 : p.causal ? seq - n + t0 : seq - 1);
    const int hi_max = __builtin_amdgcn_readfirstlane(!TREE && p.causal ? seq - n + t1 : seq - 1);
    const int lo_min = p.window > 0 ? (TREE ? min(base - p.window + 1, seq) : hi_min - p.window + 1) : 0;
    const int lo_max = p.window > 0 ? (TREE ? kt.len - 1 : hi_max) - p.window + 1 : 0;

    // Of the run's tiles ta .. tb - 1 of this sequence those that the row tile sees,
    // u = 0 .. nt - 1: n1 with sinks (numbered by their keys) from tile ta on, then
    // those of its own window, keys from 32 (f2 + u) on.
    const int own = sink + (max(lo_min, 0) >> 5) - first, a2 = max(ta, own);
    const int n1 = max(min(min(tb, own), (min(sinks, seq) + 31) >> 5) - ta, 0);
    const int nt = n1 + max(min(tb, sink + ((hi_max + 32) >> 5) - first) - a2, 0), f2 = first + a2 - sink - n1;
    const __attribute__((address_space(4))) int32_t* table =
        (const __attribute__((address_space(4))) int32_t*)(p.block_tables + (int64_t)b * p.sbt);
    auto key_of = [&](int u) -> int { return (u < n1 ? ta + u : f2 + u) * 32; };
    auto block_at = [&](int u, int piece) -> int {
      const int key = key_of(u) + 16 * piece;
      return u < nt && key < seq ? table[key >> p.block_shift] : -1;
    };
    // A piece's block and slot; one that is not there has descriptors of no bytes.
    struct Piece {
      uint32_t blk, slot;
      int live;  // all bits or none
    };
    auto piece_of = [&](int u, int blk, int piece) -> Piece {
      const bool live = (unsigned)blk < (unsigned)p.num_blocks;
      return {live ? (uint32_t)blk : 0u, (uint32_t)((key_of(u) + 16 * piece) & slot_mask), live ? -1 : 0};
    };
    // One tile of a wave in flight or in use.
    struct Tile {
      u32x4 k[2][KD];
      uint32_t v[2][4][VW];
      u32x2 sc[2];
    };
    auto load_k = [&](Tile& t, const Piece& c, int piece) {
      const __amdgpu_buffer_rsrc_t rs = piece_rsrc(kbase + ((uint64_t)c.blk * kblock + (uint64_t)c.slot * kslot), kbytes & c.live);
#pragma unroll
      for (int i = 0; i < KD; ++i) {
        const uint32_t o = ko[i];
        t.k[piece][i] = load16(rs, (int)o);
      }
    };
    auto load_s = [&](Tile& t, const Piece& c, int piece) {
      if constexpr (Q8) t.sc[piece] = load8b(piece_rsrc(sbase + ((uint64_t)c.blk * sblock + c.slot * 2), 32 & c.live), 8 * g);
    };
    auto load_v = [&](Tile& t, const Piece& c, int piece) {
      const __amdgpu_buffer_rsrc_t rs = piece_rsrc(vbase + ((uint64_t)c.blk * vblock + (uint64_t)c.slot * vslot), vbytes & c.live);
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VW>(rs, (int)(vo + i * vstep), t.v[piece][i]);
    };

    f32x4 acc[NC][VJ];
    // l_run: sum of the rounded p (normalises O: the weights of the V rows then
    // sum to one exactly); l_lse: of the fp32 p (the logsumexp).
    float m_run[NC], l_run[NC], l_lse[NC];
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      m_run[x] = -1e30f, l_run[x] = 0.f, l_lse[x] = 0.f;
#pragma unroll
      for (int j = 0; j < VJ; ++j) acc[x][j] = f32x4{};
    }

    auto whole = [&](int key0) -> bool { return key0 + 31 <= hi_min && (key0 >= lo_max || key0 + 31 < sinks); };
    bool bad = false;  // V had infinities or NaN in a tile that the mask cuts
    const T* my_q = st_q[head - head_0];
    int b0 = block_at(wave_k, 0), b1 = block_at(wave_k, 1);
    Piece c0 = piece_of(wave_k, b0, 0), c1 = piece_of(wave_k, b1, 1);
    b0 = block_at(wave_k + nk, 0), b1 = block_at(wave_k + nk, 1);
    Tile t;
    load_k(t, c0, 0), load_k(t, c1, 1);
    load_s(t, c0, 0), load_s(t, c1, 1);
    load_v(t, c0, 0), load_v(t, c1, 1);
    __syncthreads();  // Q is in LDS
    // Registers of tile u take the wave's next one as they become free.
    for (int u = wave_k; u < nt; u += nk) {
      const int un = u + nk, key0 = key_of(u);
      c0 = piece_of(un, b0, 0), c1 = piece_of(un, b1, 1);
      f32x4 s[NC][2];
#pragma unroll
      for (int x = 0; x < NC; ++x) s[x][0] = s[x][1] = f32x4{};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        X8 qr[NC];  // elements d .. d + 7 of row c, as ko has K's
        const int d = Q8 ? 64 * (kk / 2) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g;
#pragma unroll
        for (int x = 0; x < NC; ++x) qr[x] = *(const X8*)(my_q + (16 * x + c) * QS + d);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4 a;
          if constexpr (Q8) {
            const uint32_t w0 = t.k[h][kk / 2][2 * (kk & 1)], w1 = t.k[h][kk / 2][2 * (kk & 1) + 1];
            a = u32x4{codes2<false>(w0, 1.f, T()), codes2<true>(w0, 1.f, T()), codes2<false>(w1, 1.f, T()), codes2<true>(w1, 1.f, T())};
          } else {
            a = t.k[h][kk];
          }
#pragma unroll
          for (int x = 0; x < NC; ++x) s[x][h] = mfma16(__builtin_bit_cast(X8, a), qr[x], s[x][h]);
        }
      }
      load_k(t, c0, 0), load_k(t, c1, 1);
      b0 = block_at(un + nk, 0), b1 = block_at(un + nk, 1);
      __builtin_amdgcn_sched_barrier(0);

      // Scores in log2 units, masked to -inf where the row does not see the key.
      float vs[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float ks = p.scale_log2;
          vs[h][i] = 1.f;
          if constexpr (Q8) {
            const uint32_t w = t.sc[h][i >> 1];
            const uint32_t ke = (i & 1) ? w << 7 : w << 23, ve = (i & 1) ? w >> 1 : w << 15;
            ks *= __uint_as_float(ke & 0x7f800000u);
            vs[h][i] = __uint_as_float(ve & 0x7f800000u);
          }
#pragma unroll
          for (int x = 0; x < NC; ++x) s[x][h][i] *= ks;
        }
      load_s(t, c0, 0), load_s(t, c1, 1);
      if (!whole(key0)) {
        uint32_t found = 0, tree[NC];
#pragma unroll
        for (int x = 0; x < NC; ++x) tree[x] = TREE ? drafts(x, key0) >> (4 * g) : 0u;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * h + 4 * g + i;
#pragma unroll
            for (int x = 0; x < NC; ++x)
              if (!(key <= hi[x] && (key >= lo[x] || key < sinks)) && !(TREE && (tree[x] >> (16 * h + i) & 1))) s[x][h][i] = -INFINITY;
            // Rows of V that no query sees are not read as numbers (0 * NaN is NaN).
            const bool used = key <= hi_max && (key >= lo_min || key < sinks);
            if (!used) vs[h][i] = 1.f;
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              t.v[h][i][w] = used ? t.v[h][i][w] : 0u;
              if constexpr (!ONE) {
                const uint32_t x = not_finite<T, Q8>(t.v[h][i][w]);
                t.v[h][i][w] &= ~x;
                found |= x;
              }
            }
          }
        if (!ONE) bad |= __builtin_amdgcn_ballot_w64(found != 0) != 0;
      }
      X8 pb[NC];
#pragma unroll
      for (int x = 0; x < NC; ++x) {
        const f32x4 s0 = s[x][0], s1 = s[x][1];
        float mx = fmaxf(fmaxf(fmaxf(s0[0], s0[1]), fmaxf(s0[2], s0[3])), fmaxf(fmaxf(s1[0], s1[1]), fmaxf(s1[2], s1[3])));
        mx = quarter_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_run[x] + kThreshold) != 0) {
          const float m_new = fmaxf(m_run[x], mx);
          const float alpha = fast_exp2(m_run[x] - m_new);
          l_run[x] *= alpha;
          l_lse[x] *= alpha;
          m_run[x] = m_new;
#pragma unroll
          for (int j = 0; j < VJ; ++j) acc[x][j] *= alpha;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float e = fast_exp2(s[x][h][i] - m_run[x]);
            l_lse[x] += e;
            pb[x][4 * h + i] = (T)e;
          }
        float rs[4] = {0.f, 0.f, 0.f, 0.f};
        sum8_into(pb[x], rs);
        l_run[x] += (rs[0] + rs[1]) + (rs[2] + rs[3]);
      }

      __builtin_amdgcn_sched_barrier(0);
      // Channels (D/16) c + 2 w and + 1 of the 8 keys: converted (8 bits), then two keys to
      // a word.
#pragma unroll
      for (int w = 0; w < VJ / 2; ++w) {
        uint32_t v2[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if constexpr (Q8)
              v2[h][i] = (w & 1) ? codes2<true>(t.v[h][i][w / 2], vs[h][i], T()) : codes2<false>(t.v[h][i][w / 2], vs[h][i], T());
            else
              v2[h][i] = t.v[h][i][w];
          }
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          u32x4 a;
#pragma unroll
          for (int k = 0; k < 4; ++k)
            a[k] = __builtin_amdgcn_perm(v2[k / 2][2 * (k & 1) + 1], v2[k / 2][2 * (k & 1)], odd ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int x = 0; x < NC; ++x) acc[x][2 * w + odd] = mfma16(__builtin_bit_cast(X8, a), pb[x], acc[x][2 * w + odd]);
        }
        if (w & 1) __builtin_amdgcn_sched_barrier(0);
      }
      load_v(t, c0, 0), load_v(t, c1, 1);
    }

    if (!ONE && __builtin_expect(bad, 0)) {
#pragma unroll 1
      for (int u = wave_k; u < nt; u += nk) {
        const int key0 = key_of(u);
        if (whole(key0)) continue;
#pragma unroll 1
        for (int key = key0; key < key0 + 32; ++key) {
          const int piece = (key - key0) >> 4;
          const Piece at_key = piece_of(u, block_at(u, piece), piece);
          const __amdgpu_buffer_rsrc_t rs =
              piece_rsrc(vbase + ((uint64_t)at_key.blk * vblock + (uint64_t)(at_key.slot + (key & 15)) * vslot), (p.D * EB) & at_key.live);
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // channels (4 g + i) VJ ..
            uint32_t v[VW];
            load_words<VW>(rs, (4 * g + i) * VJ < p.D ? (4 * g + i) * VJ * EB : (int)kOut, v);
#pragma unroll
            for (int w = 0; w < VW; ++w) v[w] &= not_finite<T, Q8>(v[w]);
#pragma unroll
            for (int x = 0; x < NC; ++x)
              if ((key <= hi[x] && (key >= lo[x] || key < sinks)) || (TREE && (drafts(x, key) & 1))) {
#pragma unroll
                for (int j = 0; j < VJ; ++j) acc[x][j][i] += bad_value<T, Q8>(v, j);
              }
          }
        }
      }
    }

    // Merge the waves, a column block at a time. A wave without a tile has m = -1e30
    // and sums of zero.
#pragma unroll
    for (int x = 0; x < NC; ++x) {
      const float lt = quarter_sum(l_run[x]), le = quarter_sum(l_lse[x]);
      if (g == 0) {
        st_m[wave][16 * x + c] = m_run[x];
        st_l[wave][16 * x + c] = lt;
        st_e[wave][16 * x + c] = le;
      }
    }
    // A sequence within the run is done. Of one in several runs the partial sums go to
    // the workspace. Long runs leave them for the combine kernel (waiting for the
    // stores and the counter at the end of every run took 20 us of 129 over 64 windows of
    // 4096 tokens, the kernel 5); of short ones, whose launches are a few microseconds, the
    // run that arrives last merges them. That handoff is the skinny GEMM's (fa_gemv.hip):
    // partials are device-scope atomic stores (written through past the XCD's L2),
    // every wave waits for its own before the barrier ahead of the counter's add, and
    // the last run reads them with device-scope loads.
    const bool complete = ta == 0 && tb == count;
    args = arguments();
#pragma unroll
    for (int x = 0; x < NC; ++x) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VJ; ++j) st_o[wave][c][(4 * g + i) * VJ + j] = acc[x][j][i];
      __syncthreads();
      const int items = min(nrows - 16 * x, kRowTile) * (DP / 4);
      for (int idx = tid; idx < items * hw; idx += 256) {
        const int hs = idx / items, row = (idx - hs * items) / (DP / 4), d = (idx - hs * items) % (DP / 4) * 4, rr = 16 * x + row;
        float M = st_m[hs][rr];
        for (int w = hs + hw; w < NW; w += hw) M = fmaxf(M, st_m[w][rr]);
        float L = 0.f, E = 0.f;
        f32x4 O = {};
        for (int w = hs; w < NW; w += hw) {
          const float a = fast_exp2(st_m[w][rr] - M);
          L += a * st_l[w][rr];
          E += a * st_e[w][rr];
          O += a * *(const f32x4*)&st_o[w][row][d];
        }
        if (complete) {
          store_row<T>(*args, tok0, rt * RT + rr, G, head_0 + hs, d, M, L, E, O);
        } else {
          float* part = part_of<DP>(*args, rt, head_0 + hs, runs, run, ta == 0);
          const f32x4 st = {M, L, E, 0.f};
          if (deferred) {
            *(f32x4*)(part + rr * DP + d) = O;
            if (d == 0) *(f32x4*)(part + args->part_rows * DP + 4 * rr) = st;
          } else {
            store_device(part + rr * DP + d, O);
            if (d == 0) store_device(part + args->part_rows * DP + 4 * rr, st);
          }
        }
      }
      __syncthreads();  // the next merge reuses the arrays
    }
    if (complete || deferred) continue;
    const int r0 = head0 / per, r1 = (head0 + count - 1) / per;  // the sequence's runs
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the partials have reached device scope
    __syncthreads();
    if (tid == 0) {
      int* counter = args->counters + column * runs + r0;
      const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == r1 - r0;
      if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      st_last = last;
    }
    __syncthreads();
    if (!st_last) continue;
    // (one head a workgroup here) Groups of threads take every ng-th run, four at a time,
    // and meet in LDS.
    const int items = min(nrows, RT) * (DP / 4), ng = max(256 / items, 1), grp = tid / items;
    f32x4* meet = (f32x4*)&st_o[0][0][0];
    for (int i0 = 0; i0 < items; i0 += 256) {
      const int idx = i0 + (ng > 1 ? tid - grp * items : tid), row = idx / (DP / 4), d = idx % (DP / 4) * 4;
      RowSums sum;
      if (idx < items && (ng == 1 || grp < ng)) {
        constexpr int U = 4;
        for (int r = r0 + (ng > 1 ? grp : 0); r <= r1; r += ng * U) {
          f32x4 st[U], o[U];
#pragma unroll
          for (int k = 0; k < U; ++k) {
            const int rk = min(r + k * ng, r1);
            const float* from = part_of<DP>(*args, rt, head, runs, rk, rk == r0);
            st[k] = load_device(from + args->part_rows * DP + 4 * row);
            o[k] = load_device(from + row * DP + d);
          }
#pragma unroll
          for (int k = 0; k < U; ++k)
            if (r + k * ng <= r1) sum.take(st[k], o[k]);
        }
      }
      if (ng > 1) {
        if (grp < ng) {
          meet[2 * tid] = f32x4{sum.M, sum.L, sum.E, 0.f};
          meet[2 * tid + 1] = sum.O;
        }
        __syncthreads();
        if (tid < items)
          for (int k = 1; k < ng; ++k) sum.take(meet[2 * (tid + k * items)], meet[2 * (tid + k * items) + 1]);
      }
      if (idx < items && (ng == 1 || tid < items)) store_row<T>(*args, tok0, rt * RT + row, G, head, d, sum.M, sum.L, sum.E, sum.O);
    }
    __syncthreads();
  }
}

// Merges the partial results of long runs: a workgroup takes CH channels of a sequence, KV
// head and row tile; groups of threads take every ng-th run and meet in LDS. Bound by latency.
// Many sequences lie in few runs each: two of them in flight a thread do, and 64 channels a
// workgroup, where there are 256 of them or more (64 windows of 4096 tokens of 8 heads, 5 runs
// each: 116 us in all, 32 channels 118, with eight runs in flight 121, which load what others
// have). A long one lies in hundreds: eight in flight and 32 channels, for more groups
// (32768 tokens: 30 us in all, 64 channels with two in flight 47).
template <typename T, int DP, int NC, int CH>
__global__ __launch_bounds__(256) void fa_window_combine_kernel(const WindowParams p) {
  constexpr int RT = kRowTile * NC;
  static_assert(RT * CH / 4 <= 256, "a thread has at most one row's four channels");
  __shared__ f32x4 meet[512];
  const int tid = threadIdx.x, lane = tid & 63;
  const int head = blockIdx.x % p.Hkv, rt = blockIdx.x / p.Hkv, b = blockIdx.y;
  const int G = p.Hq / p.Hkv;
  int all = 0, at = 0, tok0 = 0, count = 0, nrows = 0;  // tiles of all sequences, tiles before b's; b's
  for (int j = 0; j < p.B; j += 64) {
    KeyTiles mine = {};
    if (j + lane < p.B) mine = p.tree != nullptr ? key_tiles<true>(p, j + lane) : key_tiles<false>(p, j + lane);
    const int upto = lanes_sum(mine.count);
    if (j <= b && b < j + 64) {
      at = all + __builtin_amdgcn_readlane(upto - mine.count, b - j);
      count = __builtin_amdgcn_readlane(mine.count, b - j);
      tok0 = __builtin_amdgcn_readlane(mine.tok0, b - j);
      nrows = min(min(__builtin_amdgcn_readlane(mine.n, b - j), p.max_n) * G - rt * RT, RT);
    }
    all += __builtin_amdgcn_readlane(upto, 63);
  }
  if (!long_runs(p, all) || count == 0 || nrows <= 0) return;
  const int runs = p.runs * heads_per_group(p), per = run_tiles(all, runs);
  const int r0 = at / per, r1 = (at + count - 1) / per;
  if (r0 == r1) return;  // already in o
  const int items = nrows * (CH / 4), ng = 256 / items, grp = tid / items, idx = tid - grp * items;
  const int row = idx / (CH / 4), d = blockIdx.z * CH + idx % (CH / 4) * 4;
  RowSums sum;
  auto merge = [&](auto in_flight) {
    constexpr int U = decltype(in_flight)::value;
    for (int r = r0 + grp; r <= r1; r += ng * U) {
      f32x4 st[U], o[U];
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int rk = min(r + k * ng, r1);
        const float* from = part_of<DP>(p, rt, head, runs, rk, rk == r0);
        st[k] = *(const f32x4*)(from + p.part_rows * DP + 4 * row);
        o[k] = *(const f32x4*)(from + row * DP + d);
      }
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (r + k * ng <= r1) sum.take(st[k], o[k]);
    }
  };
  if (grp < ng) {
    if (r1 - r0 >= 4 * ng) merge(std::integral_constant<int, 8>());
    else merge(std::integral_constant<int, 2>());
    meet[2 * tid] = f32x4{sum.M, sum.L, sum.E, 0.f};
    meet[2 * tid + 1] = sum.O;
  }
  __syncthreads();
  if (grp > 0) return;
  for (int k = 1; k < min(ng, r1 - r0 + 1); ++k) sum.take(meet[2 * (tid + k * items)], meet[2 * (tid + k * items) + 1]);
  store_row<T>(p, tok0, rt * RT + row, G, head, d, sum.M, sum.L, sum.E, sum.O);
}

// ---------------------------------------------------------------- wide kernel
// Many rows per KV head (chunks of new tokens): a workgroup of NW waves takes
// 32 NW (token, query head) rows of one sequence and KV head, wave w rows 32 w ..
// 32 w + 31, so that every key tile brought into LDS serves the whole group of
// query heads. Key tiles of 64 lie in LDS in q's type, K and V double-buffered;
// 8-bit rows are loaded into registers one step ahead and written to LDS with
// their scales applied (each value once per workgroup, where every wave would
// convert it again on reading codes), 16-bit rows go there by direct loads.
// Rows that none of the workgroup's queries sees read as zeros. S^T = K Q^T and
// O^T += V^T P^T on v_mfma_f32_32x32x16 (fa_common.hpp has the lane layouts), the
// scores of tile t + 1 beside the softmax of tile t. Bound by the matrix pipe and the
// exponentials that share its issue slots (batched chunks over 8-bit prefixes 327 to 339
// us by the card, 960 to 1000 TFLOP/s, where a large bf16 product of normal operands
// reaches 1230 to 1330; the first 25 ms after a pause take up to a third longer), short
// ones by their steps' latency (2.7 us a tile of 64 keys, and 6 us before the first).
constexpr int kWideTile = 64;  // keys

// The sequence (with its key tiles) and row tile of an item; false past the last. Row
// tiles go longest first (ranked_item) where their lengths differ: up to 64 sequences
// without a window. Else they go in order, the last of a sequence first.
template <int BM>
__device__ __forceinline__ bool wide_item(const WindowParams& p, int item, int lane, int& b, int& rt, KeyTiles& kt) {
  const int G = p.Hq / p.Hkv;
  auto tiles_of = [&](const KeyTiles& t) -> int { return (int)(((int64_t)min(t.n, p.max_n) * G + BM - 1) / BM); };
  KeyTiles mine = {};
  if (lane < p.B) mine = key_tiles<false>(p, lane);
  int tq = tiles_of(mine);
  bool found = false;
  if (p.B > 1 && p.B <= 64 && p.window == 0) {
    const int nk = mine.seq, off = nk - mine.n;
    auto above = [&](int x) -> int {
      if (x < 0) return tq;
      if (tq == 0 || nk <= kWideTile * x) return 0;
      if (!p.causal) return tq;
      const long long y = ((long long)kWideTile * x - off) * G;  // row tile t ends past key 64 x iff t >= y / BM
      return y < 0 ? tq : 1 + (int)max(0LL, tq - 1 - y / BM);
    };
    int d;
    b = ranked_item(p.B, item, lane, tq, nk > 0 ? (nk + kWideTile - 1) / kWideTile : 0, above, d);
    found = b >= 0;
    if (found) rt = __builtin_amdgcn_readlane(tq, b) - 1 - d;
  } else {
    int at = 0;
    for (int j = 0; j < p.B && !found; j += 64) {
      if (j > 0) {
        mine = {};
        if (j + lane < p.B) mine = key_tiles<false>(p, j + lane);
        tq = tiles_of(mine);
      }
      const int upto = lanes_sum(tq);
      const unsigned long long hit = __ballot(at + upto > item);
      if (hit != 0) {
        const int src = __builtin_ctzll(hit);
        b = j + src;
        rt = at + __builtin_amdgcn_readlane(upto, src) - 1 - item;
        found = true;
      }
      at += __builtin_amdgcn_readlane(upto, 63);
    }
  }
  if (!found) return false;
  const int src = b & 63;
  kt = key_tiles_of<false>(p, __builtin_amdgcn_readlane(mine.len, src), __builtin_amdgcn_readlane(mine.n, src),
                    __builtin_amdgcn_readlane(mine.tok0, src));
  return true;
}

// Its KV head: an XCD takes the same head of all row tiles of a sequence, which share
// keys, and another one of the next sequence, so that it reads all channels of its L2.
__device__ __forceinline__ int wide_head(const WindowParams& p, int b) {
  return ranked_head((blockIdx.x + b) % p.Hkv, p.Hkv);
}

// A row tile's key tiles: `sink` of them from key 0 on, then those from tile
// `first` on.
struct WideSpan {
  int sink, first, count;
  int hi_max, lo_min;  // keys past hi_max, or before lo_min and no sinks, are seen by no row
};
template <int BM>
__device__ __forceinline__ WideSpan wide_span(const WindowParams& p, const KeyTiles& kt, int rt) {
  const int G = p.Hq / p.Hkv, rows = kt.n * G;
  const int t0 = rt * BM / G, t1 = (min(rows, (rt + 1) * BM) - 1) / G;
  WideSpan s;
  s.hi_max = p.causal ? kt.seq - kt.n + t1 : kt.seq - 1;
  s.lo_min = p.window > 0 ? kt.seq - kt.n + t0 - p.window + 1 : 0;
  const int end = max(s.hi_max + 1, 0);
  s.first = min(max(s.lo_min, 0), end) / kWideTile;
  s.sink = p.window > 0 ? min((min(p.sinks, end) + kWideTile - 1) / kWideTile, s.first) : 0;
  s.count = s.sink + (end + kWideTile - 1) / kWideTile - s.first;
  return s;
}
// Tiles of one of an item's splits: an even share, at least kSplitLeast (333 tokens under a
// window of 1024: 29.2 us, 33.8 with 8; 64 tokens of 4 sequences of 16 bits: 16.3, 20.3 with
// 8, 16.7 with 1).
constexpr int kSplitLeast = 3;
__device__ __forceinline__ int split_share(int count, int splits) {
  return max((count + splits - 1) / splits, kSplitLeast);
}
// Floats of one split's partial results: (offset, sum for O, sum for the lse, 0) of
// each row, then O in the accumulators' own order, [wave][4-register group][lane].
template <int BM, int DP> constexpr int kWidePart = BM * 4 + BM * DP;

template <typename T> constexpr float kWideMaxLog2P = 64.0f;
template <> constexpr float kWideMaxLog2P<_Float16> = 15.0f;

template <typename T, typename C, int DP, int NW, bool LSE, bool SPLIT>
__global__ __launch_bounds__((NW * 64), (8 / NW)) void fa_window_wide_kernel(const WindowParams p) {
  using X8 = typename VecT<T>::x8;
  using X4 = typename VecT<T>::x4;
  constexpr bool Q8 = sizeof(C) == 1;
  constexpr int EB = sizeof(C);
  constexpr int BM = NW * 32, BN = kWideTile;
  constexpr int TILE = BN * DP;            // elements of one K or V tile in LDS
  constexpr int KSTEPS = DP / 16, DT = DP / 32, KB = BN / 32;
  constexpr int RPW = BN / NW;             // tile rows that a wave loads: 8 or 16, in one cache block
  constexpr int LPR = DP / 8;              // lanes per row, 8 elements each
  constexpr int RPL = 64 / LPR;            // rows per load instruction
  constexpr int NL = RPW / RPL;            // load instructions per wave and tile
  static_assert(NL >= 1, "a wave loads whole instructions");

  __shared__ __attribute__((aligned(1024))) T smem_raw[4 * TILE];  // K0 K1 V0 V1
  LDS_AS char* smem = (LDS_AS char*)smem_raw;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, hh = lane >> 5;
  const int G = p.Hq / p.Hkv;
  int b, rt;
  KeyTiles kt;
  if (!wide_item<BM>(p, blockIdx.x / p.Hkv, lane, b, rt, kt)) return;  // uniform, before any barrier
  const int head = wide_head(p, b);
  const int64_t tok0 = kt.tok0;
  WideSpan sp = wide_span<BM>(p, kt, rt);
  const int sink = __builtin_amdgcn_readfirstlane(sp.sink), first = __builtin_amdgcn_readfirstlane(sp.first);
  const int hi_max = __builtin_amdgcn_readfirstlane(sp.hi_max), lo_min = __builtin_amdgcn_readfirstlane(sp.lo_min);
  int t_lo = 0, t_hi = __builtin_amdgcn_readfirstlane(sp.count);
  bool whole_item = true;
  if constexpr (SPLIT) {
    const int share = __builtin_amdgcn_readfirstlane(split_share(t_hi, p.splits));
    whole_item = t_hi <= share;
    t_lo = blockIdx.y * share;
    if (blockIdx.y > 0 && t_lo >= t_hi) return;  // uniform, before any barrier
    t_hi = min(t_hi, t_lo + share);
  }
  const int seq = kt.seq, nrows = min(kt.n, p.max_n) * G;
  const int sinks = p.window > 0 ? p.sinks : 0;
  const float sl2 = p.scale_abs;

  // The lane's row and what it sees, and the same over the wave's rows.
  const int r0 = rt * BM + wave * 32, r = r0 + l32, tok = r / G, hq = head * G + (r - tok * G);
  const bool row_ok = r < nrows;
  const int pos = p.causal ? seq - kt.n + tok : seq - 1;
  const int hi = row_ok ? pos : -1, lo = p.window > 0 ? pos - p.window + 1 : 0;
  const int w0 = seq - kt.n + r0 / G, w1 = seq - kt.n + (min(r0 + 32, nrows) - 1) / G;
  const int whi_min = __builtin_amdgcn_readfirstlane(p.causal ? w0 : seq - 1);
  const int whi_max = __builtin_amdgcn_readfirstlane(r0 >= nrows ? -1 : p.causal ? w1 : seq - 1);
  const int wlo_min = __builtin_amdgcn_readfirstlane(p.window > 0 ? w0 - p.window + 1 : 0);
  const int wlo_max = __builtin_amdgcn_readfirstlane(p.window > 0 ? w1 - p.window + 1 : 0);

  X8 qreg[KSTEPS];
  auto key_of = [&](int t) -> int { return (t < sink ? t : t - sink + first) * BN; };
  const __attribute__((address_space(4))) int32_t* table =
      (const __attribute__((address_space(4))) int32_t*)(p.block_tables + (int64_t)b * p.sbt);
  // Cache block of the wave's rows of tile t (-1: none).
  auto block_at = [&](int t) -> int {
    const int key = key_of(t) + RPW * wave;
    return t < t_hi && key < seq ? table[key >> p.block_shift] : -1;
  };

  // Loads of the wave's RPW rows of a tile, 8 elements a lane. 8-bit: row (l / LPR)
  // NL + i in instruction i, so that a lane's rows have adjacent scales; 16-bit: what
  // the direct load's linear LDS order makes of the swizzled tile.
  auto row_at = [&](int i) -> int { return Q8 ? lane / LPR * NL + i : i * RPL + lane / LPR; };
  auto offset = [&](int i, uint32_t slot, int key0) -> int {
    const int row = row_at(i), key = key0 + RPW * wave + row;
    const int col = 8 * (Q8 ? lane % LPR : (lane % LPR) ^ seg_swz<DP>(RPW * wave + row));
    const bool used = col < p.D && key <= hi_max && (key >= lo_min || key < sinks);
    return used ? row * (int)slot + col * EB : (int)0x80000000;
  };
  // The head's rows of block 0 and the byte strides (below 2^32) of a block and a slot.
  struct Cache {
    const char* base;
    uint32_t block, slot;
  };
  const Cache K = {(const char*)p.kc + (int64_t)head * p.skh * EB, (uint32_t)(p.skb * EB), (uint32_t)(p.sks * EB)};
  const Cache V = {(const char*)p.vc + (int64_t)head * p.svh * EB, (uint32_t)(p.svb * EB), (uint32_t)(p.svs * EB)};
  auto rows_of = [&](const Cache& c, int t, int blk) -> __amdgpu_buffer_rsrc_t {
    const bool live = (unsigned)blk < (unsigned)p.num_blocks;
    const uint32_t slot = (key_of(t) + RPW * wave) & ((1 << p.block_shift) - 1);
    return tile_rsrc(c.base + (live ? (uint64_t)blk * c.block + (uint64_t)slot * c.slot : 0),
                     live ? (int)((RPW - 1) * c.slot + p.D * EB) : 0);
  };
  constexpr int EW = NL == 4 ? 2 : 1;  // words of a lane's scales (K and V of NL rows)
  struct Codes {
    u32x2 w[NL];
    uint32_t e[EW];
  };
  auto load_codes = [&](Codes& c, const Cache& of, int t, int blk) {
    const __amdgpu_buffer_rsrc_t rs = rows_of(of, t, blk);
    const bool live = (unsigned)blk < (unsigned)p.num_blocks;
    const int slot = (key_of(t) + RPW * wave) & ((1 << p.block_shift) - 1);
    const uint8_t* sb8 = p.scales + (live ? ((((int64_t)blk * p.Hkv + head) << p.block_shift) + slot) * 2 : 0);
    const __amdgpu_buffer_rsrc_t es = tile_rsrc(sb8, live ? 2 * RPW : 0);
#pragma unroll
    for (int i = 0; i < NL; ++i) c.w[i] = load8b(rs, offset(i, of.slot, key_of(t)));
    if constexpr (NL == 1) c.e[0] = load2(es, 2 * row_at(0));
    else load_words<EW>(es, 2 * row_at(0), c.e);
  };
  // (A row that no query sees has codes of zero here, but its scale may be anything:
  // infinity, which 255 stands for, would make NaN of them.)
  int woff = swz_off<DP>(RPW * wave + row_at(0), 8 * (lane % LPR)) * 2;
  auto write_codes = [&](const Codes& c, int buf, int which) {
    asm volatile("" : "+v"(woff));
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const uint32_t e = c.e[i / 2] >> (16 * (i & 1) + 8 * which) << 23;
      const float s = fminf(__uint_as_float(e & 0x7f800000u), 0x1p127f);
      const u32x4 v = {codes2<false>(c.w[i][0], s, T()), codes2<true>(c.w[i][0], s, T()), codes2<false>(c.w[i][1], s, T()),
                       codes2<true>(c.w[i][1], s, T())};
      // row + i: the row and its swizzle (swz_off) differ from the first one's in whole bits
      *(LDS_AS u32x4*)(smem + buf * TILE * 2 + (woff ^ (i * (DP == 128 ? 0x140 : 0x80)))) = v;
    }
  };
  auto load_direct = [&](const Cache& of, int t, int blk, int buf) {
    const __amdgpu_buffer_rsrc_t rs = rows_of(of, t, blk);
#pragma unroll
    for (int i = 0; i < NL; ++i)
      dma16(rs, (LDS_AS void*)(smem + buf * TILE * 2 + (RPW * wave + i * RPL) * DP * 2), offset(i, of.slot, key_of(t)));
  };

  // LDS offsets of the operands: the segment index of a column step differs from
  // the first one's by an xor of whole bits (swz_off), so one register each does
  // for all of them; taken through an empty asm in every step, or the compiler
  // hoists all 14 results out of the loop and spills.
  int koff = swz_off<DP>(l32, 8 * hh) * 2;
  const int tr_row = 4 * hh + ((lane & 15) >> 2);
  const int tr_col = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  int voff0 = swz_off<DP>(tr_row, tr_col) * 2, voff1 = swz_off<DP>(tr_row + 8, tr_col) * 2;

  f32x16 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
  float m_run = -1e30f, l_run = 0.f, l_lse = 0.f;
  const float kTileSumMax = __builtin_exp2f(kWideMaxLog2P<T>);

  // LDS operand reads run this many MFMAs ahead of the one that takes them. (The order is
  // kept apart from the code around, which else undoes it in some instances: chunks of 128
  // tokens 43.4 -> 42.1 us, of 1024 60.8 -> 59.3.)
  constexpr int kReadAhead = 4;
  auto scores = [&](int buf, f32x16* s) {
    const LDS_AS char* Ks = smem + buf * TILE * 2;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(koff));
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const X8 a = *(const LDS_AS X8*)(Ks + kb * 32 * DP * 2 + (koff ^ (kk << 5)));
        s[kb] = mfma32(a, qreg[kk], s[kb]);
      }
    constexpr int NM = KSTEPS * KB;
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
#pragma unroll
    for (int j = 0; j < NM; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (j + kReadAhead < NM) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  auto mask = [&](int t, f32x16* s) {
    const int key0 = key_of(t);
    if (!(key0 + BN - 1 <= whi_min && (key0 >= wlo_max || key0 + BN - 1 < sinks))) {
      asm volatile("" ::: "memory");  // stays a branch
      const int up = hi - key0 - 4 * hh, dn = lo - key0 - 4 * hh, sk = sinks - key0 - 4 * hh;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = 32 * kb + 8 * (i >> 2) + (i & 3);
          s[kb][i] = k <= up && (k >= dn || k < sk) ? s[kb][i] : -INFINITY;
        }
    }
  };
  auto sees = [&](int t) -> bool {
    const int key0 = key_of(t);
    return key0 <= whi_max && (key0 + BN - 1 >= wlo_min || key0 < sinks);
  };
  auto row_max = [&](const f32x16* s) -> float {
    float mx = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[kb][i]);
    mx = half_max(mx);
    return mx == -INFINITY ? -INFINITY : mx * sl2;
  };
  // Exponentials with the current offset, rounded into the PV operands; x: the
  // lane's part of the sum that normalises O (bf16: of the rounded p, so that
  // the weights sum to one exactly; fp16: of the fp32 p), y: of the fp32 p.
  auto softmax = [&](const f32x16* s, X8* pb) -> float2 {
    constexpr bool kF16 = sizeof(T) == 2 && __is_same(T, _Float16);
    const float neg_m = -m_run;
    float rs[4] = {-0.f, -0.f, -0.f, -0.f}, re[4] = {-0.f, -0.f, -0.f, -0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      f32x16 e;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        e[i] = fast_exp2(fmaf(s[kb][i], sl2, neg_m));
        if constexpr (LSE || kF16) re[i & 3] += e[i];
      }
      pb[2 * kb] = pack8<T>(e, 0);
      pb[2 * kb + 1] = pack8<T>(e, 8);
      if constexpr (!kF16) {
        sum8_into(pb[2 * kb], rs);
        sum8_into(pb[2 * kb + 1], rs);
      }
    }
    float2 x;
    x.y = (LSE || kF16) ? (re[0] + re[1]) + (re[2] + re[3]) : 0.f;
    x.x = kF16 ? x.y : (rs[0] + rs[1]) + (rs[2] + rs[3]);
    return x;
  };
  // The offset of a row is its first tile's maximum and rises only where p would
  // come near the operands' range: then the tile's exponentials are taken again.
  auto softmax_checked = [&](const f32x16* s, X8* pb) {
    float2 ts = softmax(s, pb);
    if (__builtin_amdgcn_ballot_w64(ts.x > kTileSumMax) != 0) {
      const float mx = row_max(s);
      if (__builtin_amdgcn_ballot_w64(mx > m_run) != 0) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = fast_exp2(m_run - m_new);
        l_run *= alpha;
        if constexpr (LSE) l_lse *= alpha;
        m_run = m_new;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      ts = softmax(s, pb);
    }
    l_run += ts.x;
    if constexpr (LSE) l_lse += ts.y;
  };
  auto pv = [&](int buf, const X8* pb) {
    const LDS_AS char* Vs = smem + buf * TILE * 2;
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(voff0), "+v"(voff1));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int ks = 0; ks < 2 * KB; ++ks) {
        const LDS_AS char* base = Vs + ks * 16 * DP * 2;
        const X8 a = cat4<X8, X4>(lds_read_tr((const LDS_AS T*)(base + (voff0 ^ (dt << 6)))),
                                  lds_read_tr((const LDS_AS T*)(base + (voff1 ^ (dt << 6)))));
        acc[dt] = mfma32(a, pb[ks], acc[dt]);
      }
    constexpr int NM = DT * 2 * KB;
#pragma unroll
    for (int i = 0; i < kReadAhead; ++i) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
    for (int j = 0; j < NM; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (j + kReadAhead < NM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  // K of tile t lies in buffer t & 1, V in 2 + (t & 1) (counted from t_lo on).
  // Step t needs K(t + 1), V(t) and scores(t); it brings K(t + 2) and V(t + 1) to LDS.
  auto load_q = [&]() {  // the B operand of S^T: row l32, columns 16 kk + 8 hh .. + 7
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const int col = 16 * kk + 8 * hh;
      u32x4 raw = {0, 0, 0, 0};
      if (row_ok && col < p.D) raw = ldg16((const T*)p.q + (tok0 + tok) * p.sqt + (int64_t)hq * p.sqh + col);
      if (p.scale_log2 < 0.f) raw ^= 0x80008000u;
      qreg[kk] = __builtin_bit_cast(X8, raw);
    }
  };
  Codes kc, vc;
  int b1 = block_at(t_lo + 1), b2 = block_at(t_lo + 2), b3 = block_at(t_lo + 3);
  {
    const int bl = block_at(t_lo);
    if constexpr (Q8) {
      Codes k1;
      load_codes(kc, K, t_lo, bl);
      load_codes(k1, K, t_lo + 1, b1);
      load_codes(vc, V, t_lo, bl);
      load_q();
      write_codes(kc, 0, 0);
      load_codes(kc, K, t_lo + 2, b2);
      write_codes(k1, 1, 0);
      write_codes(vc, 2, 1);
      load_codes(vc, V, t_lo + 1, b1);
    } else {
      load_direct(K, t_lo, bl, 0);
      load_direct(K, t_lo + 1, b1, 1);
      load_direct(V, t_lo, bl, 2);
      load_q();
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
  }
  __syncthreads();
  f32x16 s0[KB], s1[KB];
  if (t_lo < t_hi && sees(t_lo)) {
    scores(0, s0);
    mask(t_lo, s0);
    m_run = fmaxf(row_max(s0), -1e30f);
  }
  __syncthreads();  // K buffer 0 is refilled by the first step
  auto step = [&](int t, int par, f32x16* cur, f32x16* nxt) {
    if constexpr (Q8) {
      write_codes(kc, par, 0);
      write_codes(vc, 2 + (par ^ 1), 1);
      load_codes(kc, K, t + 3, b3);
      load_codes(vc, V, t + 2, b2);
    } else {
      load_direct(K, t + 2, b2, par);
      load_direct(V, t + 1, b1, 2 + (par ^ 1));
    }
    if (t + 1 < t_hi && sees(t + 1)) {
      scores(par ^ 1, nxt);
      mask(t + 1, nxt);
    }
    if (sees(t)) {
      X8 pb[2 * KB];
      softmax_checked(cur, pb);
      pv(2 + par, pb);
    }
    if constexpr (!Q8) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    b1 = b2, b2 = b3, b3 = block_at(t + 4);
    __syncthreads();
  };
  int t = t_lo;
  for (; t + 1 < t_hi; t += 2) {
    step(t, 0, s0, s1);
    step(t + 1, 1, s1, s0);
  }
  if (t < t_hi) step(t, 0, s0, s1);

  const float lt = half_sum(l_run), le = half_sum(l_lse);
  auto leave = [&]() {
    const auto* q = arguments();
    if constexpr (SPLIT) {
      if (!whole_item) {
        float* part = q->part + ((int64_t)blockIdx.x * q->splits + blockIdx.y) * kWidePart<BM, DP>;
        if (hh == 0) *(f32x4*)(part + (wave * 32 + l32) * 4) = f32x4{m_run, lt, le, 0.f};
        f32x4* po = (f32x4*)(part + BM * 4) + wave * DT * 4 * 64 + lane;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            po[(dt * 4 + g) * 64] = f32x4{acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
        return;
      }
    }
    // O leaves through LDS (the tiles' buffers are free after the last barrier):
    // each wave stages its 32 rows and stores whole ones.
    const float inv = lt == 0.f ? 0.f : 1.f / lt;
    {
      constexpr int BLK = 32 * DP * 2;
      static_assert(NW * BLK <= 4 * TILE * 2, "O staging fits in the K/V buffers");
      LDS_AS char* wb = smem + wave * BLK;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          X4 v;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = (T)(acc[dt][4 * g + e] * inv);
          *(LDS_AS X4*)(wb + swz_off<DP>(l32, 32 * dt + 8 * g + 4 * hh) * 2) = v;
        }
#pragma unroll
      for (int c = 0; c < BLK / 1024; ++c) {
        const int byte = c * 1024 + lane * 16;
        const int row = byte / (DP * 2), seg = (byte % (DP * 2)) / 16;
        const X8 v = *(const LDS_AS X8*)(wb + row * DP * 2 + ((seg ^ seg_swz<DP>(row)) << 4));
        const int rr = r0 + row, tk = rr / G, h = head * G + (rr - tk * G);
        if (rr < nrows && seg * 8 < q->D) *(X8*)((T*)q->o + (tok0 + tk) * q->sot + (int64_t)h * q->soh + seg * 8) = v;
      }
    }
    if constexpr (LSE) {
      if (row_ok && hh == 0 && q->lse != nullptr)
        q->lse[(tok0 + tok) * q->slt + (int64_t)hq * q->slh] = le == 0.f ? -INFINITY : (m_run + __log2f(le)) * kWinLn2;
    }
  };
  leave();

  // Sums that are not finite while V has infinities or NaN in a tile that the mask cuts are
  // taken again. (Looking for them in every such tile of the loop, before they are
  // multiplied, made 111 us of 98 of windowed prompts of a 16-bit cache.)
  if (__builtin_expect(__builtin_amdgcn_ballot_w64(!all_finite(acc)) != 0, 0)) {
    auto row_of = [&](const Cache& c, int key, int blk) -> const C* {
      return (const C*)(c.base + (uint64_t)blk * c.block + (uint64_t)(key & ((1 << p.block_shift) - 1)) * c.slot);
    };
    bool bad = false;
#pragma unroll 1
    for (int u = t_lo; u < t_hi; ++u) {
      const int key0 = key_of(u), key = key0 + lane;
      if (key0 + BN - 1 <= whi_min && (key0 >= wlo_max || key0 + BN - 1 < sinks)) continue;
      // (whatever the tile holds: other waves may see more than this one)
      const bool used = key <= hi_max && (key >= lo_min || key < sinks);
      const int blk = used ? table[key >> p.block_shift] : -1;
      if ((unsigned)blk >= (unsigned)p.num_blocks) continue;
      const C* row = row_of(V, key, blk);
#pragma unroll 1
      for (int i = 0; i < p.D; i += 8) {
        const u32x2 w = *(const u32x2*)(row + i);
        bad |= (not_finite<T, Q8>(w[0]) | not_finite<T, Q8>(w[1])) != 0;
        if constexpr (!Q8) {
          const u32x2 w4 = *(const u32x2*)(row + i + 4);
          bad |= (not_finite<T, Q8>(w4[0]) | not_finite<T, Q8>(w4[1])) != 0;
        }
      }
    }
    // The wave does so alone, with the offset that its rows ended with, 32 keys at a time
    // through the part of LDS that O left by. V's infinities and NaN stay out of the products
    // where the mask cuts the 32 keys and are added to the rows that see them. (8.5 us for 32
    // keys, of head dim 128: a call over 8192 keys 0.37 -> 2.5 ms, over 32768 1.2 -> 8.8.)
    if (__builtin_amdgcn_ballot_w64(bad) != 0) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16{};
      LDS_AS char* wb = smem + wave * 32 * DP * 2;
      int lrow = lane / LPR, lcol = 8 * (lane % LPR);
      // (LDS is in order within a wave; this keeps the compiler's order)
      auto in_order = [&]() { asm volatile("" ::: "memory"); };
#pragma unroll 1
      for (int i = 0; i < 2 * (t_hi - t_lo); ++i) {
        const int key0 = key_of(t_lo + (i >> 1)) + 32 * (i & 1);
        if (key0 > whi_max || (key0 + 31 < wlo_min && key0 >= sinks)) continue;
        const bool cut = !(key0 + 31 <= whi_min && (key0 >= wlo_max || key0 + 31 < sinks));
        asm volatile("" : "+v"(koff), "+v"(voff0), "+v"(voff1), "+v"(lrow), "+v"(lcol));  // (nothing made of them stays in registers)
        uint32_t found = 0;
        auto to_lds = [&](const Cache& of, int which, bool finite_only) {
          u32x4 w[32 / RPL];
#pragma unroll
          for (int j = 0; j < 32 / RPL; ++j) {
            const int key = key0 + j * RPL + lrow, slot = key & ((1 << p.block_shift) - 1);
            const bool used = lcol < p.D && key <= whi_max && (key >= wlo_min || key < sinks);
            const int blk = used ? table[key >> p.block_shift] : -1;
            w[j] = u32x4{0, 0, 0, 0};
            if ((unsigned)blk >= (unsigned)p.num_blocks) continue;
            const C* row = row_of(of, key, blk) + lcol;
            if constexpr (Q8) {
              const u32x2 codes = *(const u32x2*)row;
              w[j] = u32x4{codes[0], codes[1], p.scales[((((int64_t)blk * p.Hkv + head) << p.block_shift) + slot) * 2 + which], 0};
            } else {
              w[j] = ldg16((const T*)row);
            }
          }
          in_order();
#pragma unroll
          for (int j = 0; j < 32 / RPL; ++j) {
            u32x4 v = w[j];
            if (finite_only) {
#pragma unroll
              for (int c = 0; c < (Q8 ? 2 : 4); ++c) {
                const uint32_t x = not_finite<T, Q8>(v[c]);
                v[c] &= ~x;
                found |= x;
              }
            }
            if constexpr (Q8) {
              const float s = fminf(__uint_as_float(w[j][2] << 23), 0x1p127f);
              v = u32x4{codes2<false>(v[0], s, T()), codes2<true>(v[0], s, T()), codes2<false>(v[1], s, T()), codes2<true>(v[1], s, T())};
            }
            *(LDS_AS u32x4*)(wb + swz_off<DP>(j * RPL + lrow, lcol) * 2) = v;
          }
          in_order();
        };
        to_lds(K, 0, false);
        f32x16 s = {};
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) s = mfma32(*(const LDS_AS X8*)(wb + (koff ^ (kk << 5))), qreg[kk], s);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const int key = key0 + 4 * hh + 8 * (k >> 2) + (k & 3);
          s[k] = key <= hi && (key >= lo || key < sinks) ? fast_exp2(fmaf(s[k], sl2, -m_run)) : 0.f;
        }
        const X8 pb[2] = {pack8<T>(s, 0), pack8<T>(s, 8)};
        in_order();
        to_lds(V, 1, cut);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int ks = 0; ks < 2; ++ks) {
            const LDS_AS char* base = wb + ks * 16 * DP * 2;
            acc[dt] = mfma32(cat4<X8, X4>(lds_read_tr((const LDS_AS T*)(base + (voff0 ^ (dt << 6)))),
                                          lds_read_tr((const LDS_AS T*)(base + (voff1 ^ (dt << 6))))),
                             pb[ks], acc[dt]);
          }
        if (__builtin_amdgcn_ballot_w64(found != 0) == 0) continue;
#pragma unroll 1
        for (int key = key0; key < key0 + 32; ++key) {
          if (key > whi_max || (key < wlo_min && key >= sinks)) continue;
          const int blk = table[key >> p.block_shift];
          if ((unsigned)blk >= (unsigned)p.num_blocks || !(key <= hi && (key >= lo || key < sinks))) continue;
          const C* row = row_of(V, key, blk);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const int d = 32 * dt + 8 * g + 4 * hh;
              if (d >= p.D) continue;
              uint32_t w[2] = {*(const uint32_t*)(row + d), 0};
              if constexpr (!Q8) w[1] = *(const uint32_t*)(row + d + 2);
              w[0] &= not_finite<T, Q8>(w[0]), w[1] &= not_finite<T, Q8>(w[1]);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[dt][4 * g + e] += bad_value<T, Q8>(w, e);
            }
        }
      }
      in_order();
      leave();
    }
  }
}

// Merges the key splits of fa_window_wide_kernel<..., SPLIT>: workgroup (item,
// dt) combines 32 channels of the item's rows in the accumulators' order.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void fa_window_wide_combine_kernel(const WindowParams p) {
  using X4 = typename VecT<T>::x4;
  constexpr int BM = NW * 32, DT = DP / 32;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, dt = blockIdx.y;
  const int l32 = lane & 31, hh = lane >> 5, G = p.Hq / p.Hkv;
  int b, rt;
  KeyTiles kt;
  if (!wide_item<BM>(p, blockIdx.x / p.Hkv, lane, b, rt, kt)) return;
  const int head = wide_head(p, b);
  const int count = wide_span<BM>(p, kt, rt).count, share = split_share(count, p.splits);
  if (count <= share) return;  // already in o
  const int n = (count + share - 1) / share;
  const int r = rt * BM + wave * 32 + l32, nrows = min(kt.n, p.max_n) * G;
  float M = -1e30f, L = 0.f, E = 0.f;
  f32x4 O[4] = {};
  for (int i = 0; i < n; ++i) {
    const float* part = p.part + ((int64_t)blockIdx.x * p.splits + i) * kWidePart<BM, DP>;
    const f32x4 st = *(const f32x4*)(part + (wave * 32 + l32) * 4);
    const f32x4* po = (const f32x4*)(part + BM * 4) + (wave * DT + dt) * 4 * 64 + lane;
    const float m = fmaxf(M, st[0]), a = fast_exp2(M - m), w = fast_exp2(st[0] - m);
    L = a * L + w * st[1];
    E = a * E + w * st[2];
#pragma unroll
    for (int g = 0; g < 4; ++g) O[g] = a * O[g] + w * po[g * 64];
    M = m;
  }
  if (r >= nrows) return;
  const int tok = r / G, hq = head * G + (r - tok * G);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T* o = (T*)p.o + ((int64_t)kt.tok0 + tok) * p.sot + (int64_t)hq * p.soh;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int d = 32 * dt + 8 * g + 4 * hh;
    X4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)(O[g][e] * inv);
    if (d < p.D) *(X4*)(o + d) = v;
  }
  if (dt == 0 && hh == 0 && p.lse != nullptr)
    p.lse[((int64_t)kt.tok0 + tok) * p.slt + (int64_t)hq * p.slh] = E == 0.f ? -INFINITY : (M + __log2f(E)) * kWinLn2;
}

// ------------------------------------------------------------------- launches
// Most rows of a sequence and KV head in the narrow kernel: 16 chunks of 8 tokens, group 4 (32
// rows), take 66 us there and 88 in the wide one, 4 chunks of 64 tokens (256 rows) 73 and 46.
constexpr long long kNarrowRows = 32;
// Trees of more than 16 rows go to the tile kernel (8 nodes of group 4 after 1500 keys 16 us there, 25 here), and
// of fewer where a sequence's runs leave more rows of partial results than this to the one that merges them, of up to 8 rows and
// of more (trees of 2 nodes after 4500 keys 20.8 us here and 21.7 there, after 8000 28.6 and 24.7; of 4 nodes after 1500
// 16.7 and 17.4, after 2200 20.8 and 18.3, four of them after 2000 29.6 and 19.6, 64 after 4000 211 and 225).
constexpr long long kTreeMerge[2] = {400, 200};

WindowPlan tree_plan(int B, int tokens, int Hkv, int G, int dp, int max_n, long long seen);  // fa_tree.hip
hipError_t tree_attention(const WindowParams& p, const WindowPlan& w, bool is_bf16, hipStream_t s);

// How a launch goes, from what the host knows (sizes and bounds, not lengths).
WindowPlan window_plan(int B, int tokens, int Hkv, int G, int D, int eb, int max_n, long long max_keys, int window, int sinks, bool tree) {
  WindowPlan w = {};
  const int dp = D <= 64 ? 64 : 128;
  const long long rows = (long long)max_n * G;
  const long long seen = window > 0 ? std::min(max_keys, (long long)window + max_n + sinks + 96) : max_keys;
  const long long narrow_runs = std::min(std::max(512 / (long long)Hkv, 1LL), std::max(1LL, ((seen + 31) / 32 * B + 3) / 4));
  if (tree && (rows > kRowTile || rows * (narrow_runs / B) > kTreeMerge[rows > 8])) return tree_plan(B, tokens, Hkv, G, dp, max_n, seen);
  if (rows <= kNarrowRows) {
    w.columns = rows > kRowTile ? 2 : 1;
    const int rt = kRowTile * w.columns;
    w.part_rows = (int)std::min<long long>(rows, rt);
    const long long tiles = (rows + rt - 1) / rt * Hkv;
    // Two workgroups a CU, all resident at once: all start together and, their work being
    // equal, end together. Three of them, which the registers would allow, start and merge
    // more runs (64 windows of 4096 tokens 117 -> 123 us, 64 sequences of 8192 206 -> 217).
    const long long most = std::max(1LL, ((seen + 31) / 32 * B + 3) / 4);
    w.runs = (int)std::min(std::max(512 / tiles, 1LL), most);
    // A long run's partial result, written and read, is to be less than an eighth of the
    // keys and values that its waves read, and a workgroup to have 16 tiles. (Short runs
    // only: 64 windows of 4096 tokens 127 us for 120, a batch of 32 of mixed lengths 77 for 75.)
    const int tile_bytes = 64 * dp * eb, part_bytes = w.part_rows * (dp + 4) * 4;
    w.long_run = std::max(16, 4 * 16 * part_bytes / tile_bytes);
    if (w.runs == 1 || (seen + 31) / 32 * B <= (long long)w.runs * (w.long_run - 1)) w.long_run = 0;
    if (w.runs > 1)  // (long runs are up to four times as many)
      w.part_bytes = LSFA_GEMV_COUNTER_BYTES + (uint64_t)tiles * 2 * w.runs * (w.long_run > 0 ? 4 : 1) * part_bytes;
    return w;
  }
  auto items = [&](int bm) {
    return Hkv * std::min((long long)tokens * G / bm + B, (rows + bm - 1) / bm * B);
  };
  // Eight waves bring each key tile in once for 256 rows, four fill the chip with half as
  // many: at 256 items (2048 tokens of 8 KV heads, group 4) 36.2 us and 40.4, and more
  // of them 353 and 415; at 128 (1024 tokens) 69.4 and 62.5.
  w.waves = items(256) >= 256 ? 8 : 4;
  w.items = (int)items(w.waves * 32);
  // Few items share their keys out over two workgroups a CU (4 chunks of 64 tokens after
  // up to 4096: 46 us, 115 without; 256, 384, 640 and 768 workgroups took no less).
  w.splits = 1;
  if (w.waves == 4) {
    const long long tiles = (std::min(seen, window > 0 ? (long long)window + sinks + 32 * 4 / G + 128 : seen) + 63) / 64;
    w.splits = (int)std::max(1LL, std::min(512 / std::max(1, w.items), (int)(tiles / kSplitLeast)) * 1LL);
    if (w.splits > 1) w.part_bytes = LSFA_GEMV_COUNTER_BYTES + (uint64_t)w.items * w.splits * (128 * 4 + 128 * dp) * 4;
  }
  return w;
}

template <typename T, typename C, int DP, int NC, bool TREE>
static hipError_t launch_narrow(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  const int rt = kRowTile * NC, tiles = (p.max_n * (p.Hq / p.Hkv) + rt - 1) / rt;
  if (!TREE && p.max_n == 1)
    hipLaunchKernelGGL((fa_window_narrow_kernel<T, C, DP, NC, !TREE, false>), dim3(p.Hkv * tiles, p.runs), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((fa_window_narrow_kernel<T, C, DP, NC, false, TREE>), dim3(p.Hkv * tiles, p.runs), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || w.long_run == 0) return e;
  const dim3 parts(p.Hkv * tiles, p.B, DP / 32);
  if (NC == 1 && (long long)parts.x * p.B * (DP / 64) >= 256)
    hipLaunchKernelGGL((fa_window_combine_kernel<T, DP, NC, 64 / NC>), dim3(parts.x, p.B, DP / 64), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((fa_window_combine_kernel<T, DP, NC, 32>), parts, dim3(256), 0, s, p);
  return hipGetLastError();
}
template <typename T, typename C, int DP>
static hipError_t launch_wide(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  if (w.splits > 1) {
    hipLaunchKernelGGL((fa_window_wide_kernel<T, C, DP, 4, true, true>), dim3(w.items, w.splits), dim3(256), 0, s, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((fa_window_wide_combine_kernel<T, DP, 4>), dim3(w.items, DP / 32), dim3(256), 0, s, p);
    return hipGetLastError();
  }
  if (w.waves == 8) {
    if (p.lse != nullptr) hipLaunchKernelGGL((fa_window_wide_kernel<T, C, DP, 8, true, false>), dim3(w.items), dim3(512), 0, s, p);
    else hipLaunchKernelGGL((fa_window_wide_kernel<T, C, DP, 8, false, false>), dim3(w.items), dim3(512), 0, s, p);
  } else {
    if (p.lse != nullptr) hipLaunchKernelGGL((fa_window_wide_kernel<T, C, DP, 4, true, false>), dim3(w.items), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((fa_window_wide_kernel<T, C, DP, 4, false, false>), dim3(w.items), dim3(256), 0, s, p);
  }
  return hipGetLastError();
}
template <typename T, typename C, int DP>
static hipError_t launch_window(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  if (p.tree != nullptr) return launch_narrow<T, C, DP, 1, true>(p, w, s);
  if (w.items > 0) return launch_wide<T, C, DP>(p, w, s);
  return w.columns == 1 ? launch_narrow<T, C, DP, 1, false>(p, w, s) : launch_narrow<T, C, DP, 2, false>(p, w, s);
}
template <typename T>
static hipError_t dispatch_window(const WindowParams& p, const WindowPlan& w, hipStream_t s) {
  if (p.scales != nullptr) return p.D <= 64 ? launch_window<T, uint8_t, 64>(p, w, s) : launch_window<T, uint8_t, 128>(p, w, s);
  return p.D <= 64 ? launch_window<T, T, 64>(p, w, s) : launch_window<T, T, 128>(p, w, s);
}

// Host entry used by the C ABI layer (arguments already validated).
hipError_t window_attention(WindowParams p, const WindowPlan& w, bool is_bf16, hipStream_t s) {
  p.runs = w.runs;
  p.part_rows = w.part_rows;
  p.long_run = w.long_run;
  p.splits = w.splits;
  if (p.tree != nullptr && w.items > 0) return tree_attention(p, w, is_bf16, s);
  return is_bf16 ? dispatch_window<__bf16>(p, w, s) : dispatch_window<_Float16>(p, w, s);
}

}  // namespace lsfa
