// Attention over paged KV caches of 8 or 16 bits, with a sliding window and
// sinks, for gfx950.
//
// A query at position p sees key j where j <= p (causal) and, under a window of
// w tokens with s sinks, j > p - w or j < s. Sequence b's queries are the last
// n of its seq_lens[b] cached tokens (one for a decode step). An 8-bit cache
// holds e4m3 codes and one power-of-two scale for each row (fa_kvq.hip).
//
// Few rows per KV head (decode, and chunks of a few tokens): the narrow kernel.
// The path is bound by HBM, so it is built around bytes in flight, and each
// byte of the cache is read once for all query heads that share it:
//   rows       (token, query head of the KV head's group) pairs, 16 to a row
//              tile, are the columns of S^T = K Q^T and of O^T += V^T P^T on
//              v_mfma_f32_16x16x32.
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
// in several runs leaves fp32 partial results that fa_window_combine_kernel
// merges.
#include "fa_common.hpp"

#include <algorithm>

namespace lsfa {

constexpr float kWinLn2 = 0.6931471805599453f;

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// Two e4m3 codes (the low or the high half of w) times a power of two.
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, __bf16) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
}
template <bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w, float scale, _Float16) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
}

// Key tiles of 32 of a sequence: those with sinks that its window's tiles do
// not hold, then the window's from `first` on.
struct KeyTiles {
  int seq, n, tok0;  // cached tokens, queries, the first one's row
  int sink, first;   // tiles of sinks ahead of the window's, the window's first tile
  int count;         // all of them; 1 where queries see no key, 0 without queries
};
__device__ __forceinline__ KeyTiles key_tiles(const WindowParams& p, int b) {
  KeyTiles t;
  t.tok0 = b, t.n = 1;
  if (p.cu_q != nullptr) {  // (no row outside q, whatever the offsets)
    t.tok0 = min(max(p.cu_q[b], 0), p.tokens);
    t.n = max(min(p.cu_q[b + 1], p.tokens) - t.tok0, 0);
  }
  t.seq = min(max(p.seq_lens[b], 0), min(p.max_seq_len, p.max_blocks << p.block_shift));
  t.first = t.sink = 0;
  if (p.window > 0) {
    t.first = max(t.seq - t.n - p.window + 1, 0) >> 5;
    t.sink = min((min(p.sinks, t.seq) + 31) >> 5, t.first);
  }
  t.count = t.n > 0 ? max(t.sink + ((t.seq + 31) >> 5) - t.first, 1) : 0;
  return t;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int lanes_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15, rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31, rows 2 and 3
  return v;
}
// Key tiles of all sequences.
__device__ __forceinline__ int all_tiles(const WindowParams& p, int lane) {
  int sum = 0;
  for (int j = 0; j < p.B; j += 64) {
    const int mine = j + lane < p.B ? key_tiles(p, j + lane).count : 0;
    sum += __builtin_amdgcn_readlane(lanes_sum(mine), 63);
  }
  return sum;
}
// Tiles of a run: the tiles there are over the runs there are, no less than one for each wave.
__device__ __forceinline__ int run_tiles(const WindowParams& p, int all) {
  return max((all + p.runs - 1) / p.runs, 4);
}

constexpr int kRowTile = 16;

template <typename T, typename C, int DP>
__global__ __launch_bounds__(256, 2) void fa_window_narrow_kernel(const WindowParams p) {
  using X8 = typename VecT<T>::x8;
  constexpr bool Q8 = sizeof(C) == 1;
  constexpr int EB = sizeof(C);           // bytes of a cached element
  constexpr int NW = 4;
  constexpr int KK = DP / 32;             // MFMAs of S per 16 keys
  constexpr int KD = DP * EB / 64;        // 16-byte loads of K per lane and piece
  constexpr int VJ = DP / 16;             // channels per lane, MFMAs of O
  constexpr int VW = VJ * EB / 4;         // 32-bit words of V per lane and key
  constexpr float kThreshold = 8.0f;      // log2 units

  __shared__ float st_o[NW][kRowTile][DP];
  __shared__ float st_m[NW][kRowTile], st_l[NW][kRowTile], st_e[NW][kRowTile];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;
  const int head = blockIdx.x % p.Hkv, rt = blockIdx.x / p.Hkv;
  const int run = blockIdx.y;
  const int G = p.Hq / p.Hkv;

  const int all = all_tiles(p, lane), per = run_tiles(p, all);
  if ((int64_t)run * per >= all) return;  // uniform, before any barrier
  const int start = run * per, end = min(all, start + per);
  // The sequence that holds tile `start`, and its first tile's number.
  int b = 0, at = 0;
  for (int j = 0; j < p.B; j += 64) {
    const int mine = j + lane < p.B ? key_tiles(p, j + lane).count : 0;
    const int upto = lanes_sum(mine);
    const unsigned long long hit = __ballot(at + upto > start);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      b = j + src;
      at += __builtin_amdgcn_readlane(upto - mine, src);
      break;
    }
    at += __builtin_amdgcn_readlane(upto, 63);
  }

  const uint32_t kOut = 0x80000000u;  // past every descriptor: reads as zero
  uint32_t ko[KD];
#pragma unroll
  for (int i = 0; i < KD; ++i) {
    const int byte = g * (DP * EB / 4) + 16 * i;
    ko[i] = byte < p.D * EB ? (uint32_t)(c * (int)p.sks * EB + byte) : kOut;
  }
  const uint32_t vo = c * VJ < p.D ? (uint32_t)(4 * g * (int)p.svs * EB + c * VJ * EB) : kOut;
  const uint32_t vstep = vo == kOut ? 0 : (uint32_t)((int)p.svs * EB);
  const int kbytes = (15 * (int)p.sks + p.D) * EB, vbytes = (15 * (int)p.svs + p.D) * EB;

  for (; b < p.B && at < end; ++b) {
    const KeyTiles kt = key_tiles(p, b);
    const int count = __builtin_amdgcn_readfirstlane(kt.count);
    if (count == 0) continue;
    const int seq = __builtin_amdgcn_readfirstlane(kt.seq), n = __builtin_amdgcn_readfirstlane(kt.n);
    const int sink = __builtin_amdgcn_readfirstlane(kt.sink), first = __builtin_amdgcn_readfirstlane(kt.first);
    const int ta = max(start - at, 0), tb = min(count, end - at);
    at += count;
    const int nrows = n * G - rt * kRowTile;  // of this row tile
    if (nrows <= 0) continue;
    const int64_t tok0 = __builtin_amdgcn_readfirstlane(kt.tok0);

    // The lane's row, and the keys that it sees.
    const int r = rt * kRowTile + c, tok = r / G, hq = head * G + (r - tok * G);
    const bool row_ok = c < nrows;
    const int pos = p.causal ? seq - n + tok : seq - 1;
    const int hi = row_ok ? pos : -1, lo = p.window > 0 ? pos - p.window + 1 : 0;
    // The same of the tile's first and last rows.
    const int t0 = rt * kRowTile / G, t1 = (rt * kRowTile + min(nrows, kRowTile) - 1) / G;
    const int hi_min = p.causal ? seq - n + t0 : seq - 1, hi_max = p.causal ? seq - n + t1 : seq - 1;
    const int lo_min = p.window > 0 ? hi_min - p.window + 1 : 0, lo_max = p.window > 0 ? hi_max - p.window + 1 : 0;
    const int sinks = p.window > 0 ? p.sinks : 0;

    // Q as the B operand of S^T: elements g D/4 + 8 kk .. + 7 of row c.
    X8 qr[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = g * (DP / 4) + 8 * kk;
      u32x4 raw = {0, 0, 0, 0};
      if (row_ok && d < p.D) raw = ldg16((const T*)p.q + (tok0 + tok) * p.sqt + (int64_t)hq * p.sqh + d);
      qr[kk] = __builtin_bit_cast(X8, raw);
    }

    const __attribute__((address_space(4))) int32_t* table =
        (const __attribute__((address_space(4))) int32_t*)(p.block_tables + (int64_t)b * p.sbt);
    auto key_of = [&](int t) -> int { return (t < sink ? t : t - sink + first) * 32; };
    auto block_at = [&](int t, int piece) -> int {
      const int key = key_of(t) + 16 * piece;
      return t < tb && key < seq ? table[key >> p.block_shift] : -1;
    };
    u32x4 kr[2][KD];
    uint32_t vr[2][4][VW];
    u32x2 sc[2];
    auto load_k = [&](int t, int blk, int piece) {
      const bool live = (unsigned)blk < (unsigned)p.num_blocks;
      const int slot = (key_of(t) + 16 * piece) & ((1 << p.block_shift) - 1);
      const C* base = (const C*)p.kc + (live ? (int64_t)blk * p.skb + (int64_t)slot * p.sks + (int64_t)head * p.skh : 0);
      const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base, live ? kbytes : 0);
#pragma unroll
      for (int i = 0; i < KD; ++i) {
        const uint32_t o = ko[i];
        kr[piece][i] = load16(rs, (int)o);
      }
    };
    auto load_s = [&](int t, int blk, int piece) {
      if constexpr (Q8) {
        const bool live = (unsigned)blk < (unsigned)p.num_blocks;
        const int slot = (key_of(t) + 16 * piece) & ((1 << p.block_shift) - 1);
        const uint8_t* base = p.scales + (live ? ((((int64_t)blk * p.Hkv + head) << p.block_shift) + slot) * 2 : 0);
        sc[piece] = load8b(tile_rsrc(base, live ? 32 : 0), 8 * g);
      }
    };
    auto load_v = [&](int t, int blk, int piece) {
      const bool live = (unsigned)blk < (unsigned)p.num_blocks;
      const int slot = (key_of(t) + 16 * piece) & ((1 << p.block_shift) - 1);
      const C* base = (const C*)p.vc + (live ? (int64_t)blk * p.svb + (int64_t)slot * p.svs + (int64_t)head * p.svh : 0);
      const __amdgpu_buffer_rsrc_t rs = tile_rsrc(base, live ? vbytes : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) load_words<VW>(rs, (int)(vo + i * vstep), vr[piece][i]);
    };

    f32x4 acc[VJ];
#pragma unroll
    for (int j = 0; j < VJ; ++j) acc[j] = f32x4{};
    // l_run: sum of the rounded p (normalises O: the weights of the V rows then
    // sum to one exactly); l_lse: of the fp32 p (the logsumexp).
    float m_run = -1e30f, l_run = 0.f, l_lse = 0.f;

    int t = ta + wave;
    int b0 = block_at(t, 0), b1 = block_at(t, 1);
    load_k(t, b0, 0), load_k(t, b1, 1);
    load_s(t, b0, 0), load_s(t, b1, 1);
    load_v(t, b0, 0), load_v(t, b1, 1);
    b0 = block_at(t + NW, 0), b1 = block_at(t + NW, 1);
    for (; t < tb; t += NW) {
      const int tn = t + NW, key0 = key_of(t);
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{};
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          u32x4 a;
          if constexpr (Q8) {
            const uint32_t w0 = kr[h][kk / 2][2 * (kk & 1)], w1 = kr[h][kk / 2][2 * (kk & 1) + 1];
            a = u32x4{codes2<false>(w0, 1.f, T()), codes2<true>(w0, 1.f, T()), codes2<false>(w1, 1.f, T()), codes2<true>(w1, 1.f, T())};
          } else {
            a = kr[h][kk];
          }
          s[h] = mfma16(__builtin_bit_cast(X8, a), qr[kk], s[h]);
        }
      }
      load_k(tn, b0, 0), load_k(tn, b1, 1);

      // Scores in log2 units, masked to -inf where the row does not see the key.
      float vs[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (Q8) {
            const uint32_t w = sc[h][i >> 1];
            const uint32_t ke = (i & 1) ? w << 7 : w << 23, ve = (i & 1) ? w >> 1 : w << 15;
            s[h][i] *= __uint_as_float(ke & 0x7f800000u) * p.scale_log2;
            vs[h][i] = __uint_as_float(ve & 0x7f800000u);
          } else {
            s[h][i] *= p.scale_log2;
            vs[h][i] = 1.f;
          }
        }
      load_s(tn, b0, 0), load_s(tn, b1, 1);
      const bool whole = key0 + 31 <= hi_min && (key0 >= lo_max || key0 + 31 < sinks);
      if (!whole) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = key0 + 16 * h + 4 * g + i;
            if (!(key <= hi && (key >= lo || key < sinks))) s[h][i] = -INFINITY;
            // Rows of V that no query sees are not read as numbers (0 * NaN is NaN).
            const bool used = key <= hi_max && (key >= lo_min || key < sinks);
            if (!used) vs[h][i] = 1.f;
#pragma unroll
            for (int w = 0; w < VW; ++w) vr[h][i][w] = used ? vr[h][i][w] : 0u;
          }
      }
      float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
      mx = quarter_max(mx);
      if (__builtin_amdgcn_ballot_w64(mx > m_run + kThreshold) != 0) {
        const float m_new = fmaxf(m_run, mx);
        const float alpha = fast_exp2(m_run - m_new);
        l_run *= alpha;
        l_lse *= alpha;
        m_run = m_new;
#pragma unroll
        for (int j = 0; j < VJ; ++j) acc[j] *= alpha;
      }
      X8 pb;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(s[h][i] - m_run);
          l_lse += e;
          pb[4 * h + i] = (T)e;
        }
      float rs[4] = {0.f, 0.f, 0.f, 0.f};
      sum8_into(pb, rs);
      l_run += (rs[0] + rs[1]) + (rs[2] + rs[3]);

      // Channel (D/16) c + j of the 8 keys, two keys to a word.
      uint32_t x[2][4][VJ / 2];  // words of two adjacent channels of one key
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < VJ / 2; ++w) {
            if constexpr (Q8)
              x[h][i][w] = (w & 1) ? codes2<true>(vr[h][i][w / 2], vs[h][i], T()) : codes2<false>(vr[h][i][w / 2], vs[h][i], T());
            else
              x[h][i][w] = vr[h][i][w];
          }
#pragma unroll
      for (int j = 0; j < VJ; ++j) {
        const uint32_t sel = (j & 1) ? 0x07060302u : 0x05040100u;
        u32x4 a;
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = __builtin_amdgcn_perm(x[k / 2][2 * (k & 1) + 1][j / 2], x[k / 2][2 * (k & 1)][j / 2], sel);
        acc[j] = mfma16(__builtin_bit_cast(X8, a), pb, acc[j]);
      }
      load_v(tn, b0, 0), load_v(tn, b1, 1);
      b0 = block_at(tn + NW, 0), b1 = block_at(tn + NW, 1);
    }

    // Merge the waves. A wave without a tile has m = -1e30 and sums of zero.
    const float lt = quarter_sum(l_run), le = quarter_sum(l_lse);
    if (g == 0) {
      st_m[wave][c] = m_run;
      st_l[wave][c] = lt;
      st_e[wave][c] = le;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < VJ; ++j) st_o[wave][c][(4 * g + i) * VJ + j] = acc[j][i];
    __syncthreads();
    const bool complete = ta == 0 && tb == count;
    const int rows = min(nrows, kRowTile);
    const int64_t slot = (int64_t)blockIdx.x * 2 * p.runs + 2 * run + (ta == 0);
    float* part = p.part + slot * (kRowTile * (DP + 4));
    for (int idx = tid; idx < rows * (DP / 4); idx += 256) {
      const int row = idx / (DP / 4), d = (idx - row * (DP / 4)) * 4;
      float M = st_m[0][row];
#pragma unroll
      for (int w = 1; w < NW; ++w) M = fmaxf(M, st_m[w][row]);
      float L = 0.f, E = 0.f;
      f32x4 O = {};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float a = fast_exp2(st_m[w][row] - M);
        L += a * st_l[w][row];
        E += a * st_e[w][row];
        O += a * *(const f32x4*)&st_o[w][row][d];
      }
      if (complete) {
        const int rr = rt * kRowTile + row, tk = rr / G, h = head * G + (rr - tk * G);
        const float inv = L == 0.f ? 0.f : 1.f / L;
        if (d < p.D) {
          typename VecT<T>::x4 out;
#pragma unroll
          for (int e = 0; e < 4; ++e) out[e] = (T)(O[e] * inv);
          *(typename VecT<T>::x4*)((T*)p.o + (tok0 + tk) * p.sot + (int64_t)h * p.soh + d) = out;
        }
        if (d == 0 && p.lse != nullptr)
          p.lse[(tok0 + tk) * p.slt + (int64_t)h * p.slh] = E == 0.f ? -INFINITY : (M + __log2f(E)) * kWinLn2;
      } else {
        *(f32x4*)(part + row * DP + d) = O;
        if (d == 0) *(f32x4*)(part + kRowTile * DP + 4 * row) = f32x4{M, L, E, 0.f};
      }
    }
    __syncthreads();  // the next sequence's merge reuses the arrays
  }
}

// Merges the partial results of a sequence's row tile that lies in several runs:
// o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
template <typename T, int DP>
__global__ __launch_bounds__(256) void fa_window_combine_kernel(const WindowParams p) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int head = blockIdx.x % p.Hkv, rt = blockIdx.x / p.Hkv, b = blockIdx.y;
  const int G = p.Hq / p.Hkv;
  const KeyTiles kt = key_tiles(p, b);
  const int nrows = kt.n * G - rt * kRowTile;
  if (kt.count == 0 || nrows <= 0) return;
  int all = 0, at = 0;  // tiles of all sequences, tiles before b's
  for (int j = 0; j < p.B; j += 64) {
    const int mine = j + lane < p.B ? key_tiles(p, j + lane).count : 0;
    const int upto = lanes_sum(mine);
    if (j <= b && b < j + 64) at = all + __builtin_amdgcn_readlane(upto - mine, b - j);
    all += __builtin_amdgcn_readlane(upto, 63);
  }
  const int per = run_tiles(p, all);
  const int r0 = at / per, r1 = (at + kt.count - 1) / per;
  if (r0 == r1) return;  // already in o
  const int64_t tok0 = kt.tok0;
  const float* base = p.part + (int64_t)blockIdx.x * 2 * p.runs * (kRowTile * (DP + 4));
  for (int idx = tid; idx < min(nrows, kRowTile) * (DP / 4); idx += 256) {
    const int row = idx / (DP / 4), d = (idx - row * (DP / 4)) * 4;
    float M = -1e30f, L = 0.f, E = 0.f;
    f32x4 O = {};
    for (int r = r0; r <= r1; ++r) {
      const float* part = base + (int64_t)(2 * r + (r == r0)) * (kRowTile * (DP + 4));
      const f32x4 st = *(const f32x4*)(part + kRowTile * DP + 4 * row);
      const f32x4 o = *(const f32x4*)(part + row * DP + d);
      const float m = fmaxf(M, st[0]), a = fast_exp2(M - m), w = fast_exp2(st[0] - m);
      L = a * L + w * st[1];
      E = a * E + w * st[2];
      O = a * O + w * o;
      M = m;
    }
    const int rr = rt * kRowTile + row, tk = rr / G, h = head * G + (rr - tk * G);
    const float inv = L == 0.f ? 0.f : 1.f / L;
    if (d < p.D) {
      typename VecT<T>::x4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = (T)(O[e] * inv);
      *(typename VecT<T>::x4*)((T*)p.o + (tok0 + tk) * p.sot + (int64_t)h * p.soh + d) = out;
    }
    if (d == 0 && p.lse != nullptr)
      p.lse[(tok0 + tk) * p.slt + (int64_t)h * p.slh] = E == 0.f ? -INFINITY : (M + __log2f(E)) * kWinLn2;
  }
}

template <typename T, typename C, int DP>
static hipError_t launch_narrow(const WindowParams& p, hipStream_t s) {
  const int G = p.Hq / p.Hkv, tiles = (p.max_n * G + kRowTile - 1) / kRowTile;
  hipLaunchKernelGGL((fa_window_narrow_kernel<T, C, DP>), dim3(p.Hkv * tiles, p.runs), dim3(256), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.runs == 1) return e;
  hipLaunchKernelGGL((fa_window_combine_kernel<T, DP>), dim3(p.Hkv * tiles, p.B), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <typename T>
static hipError_t dispatch_narrow(const WindowParams& p, hipStream_t s) {
  if (p.scales != nullptr) return p.D <= 64 ? launch_narrow<T, uint8_t, 64>(p, s) : launch_narrow<T, uint8_t, 128>(p, s);
  return p.D <= 64 ? launch_narrow<T, T, 64>(p, s) : launch_narrow<T, T, 128>(p, s);
}

// Runs that the key tiles of a launch are shared out over (per KV head and row
// tile): as many as fill the GPU, no more than there can be for the longest
// sequences.
int window_runs(int B, int Hkv, int G, int max_n, long long max_keys) {
  const long long tiles = (long long)Hkv * (((long long)max_n * G + kRowTile - 1) / kRowTile);
  const long long fill = std::max(1LL, 1024 / std::max(1LL, tiles));
  const long long most = std::max(1LL, ((max_keys + 31) / 32 * B + 3) / 4);
  return (int)std::min(std::max(fill, std::min<long long>(B, 64)), most);
}
uint64_t window_part_bytes(int B, int Hkv, int G, int max_n, int D, int runs) {
  if (runs <= 1) return 0;
  const uint64_t tiles = (uint64_t)Hkv * (((uint64_t)max_n * G + kRowTile - 1) / kRowTile);
  return tiles * 2 * runs * kRowTile * ((D <= 64 ? 64 : 128) + 4) * 4;
}

// Host entry used by the C ABI layer (arguments already validated).
hipError_t window_attention(const WindowParams& p, bool is_bf16, hipStream_t s) {
  return is_bf16 ? dispatch_narrow<__bf16>(p, s) : dispatch_narrow<_Float16>(p, s);
}

}  // namespace lsfa
