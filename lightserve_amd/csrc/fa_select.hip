// Choices among a step's logits where a sequence has several candidates, for gfx950:
//
//   accept   The drafted tokens of a tree that the model itself would have chosen. a_i is the
//            largest logit of node i (torch's order: NaN above all, the first of equals). From
//            node 0 on, the path goes to the first child whose token is a_cur, until there is none;
//            a_cur is then the token that follows. A child of i is a node j > i that sees what i
//            sees and itself, and no more.
//   beams    The `num` best of s_k + x_kv - lse_k over a sequence's beams k and the vocabulary v, with
//            lse_k = log sum_v exp x_kv; the first k V + v of equals.
//
// Both read each logit once (that and, for few rows, latency is what bounds them; 556 rows of 128256 in bf16 29 us, 4.8
// TB/s, 8 of them 10; eight beams of 32 sequences over 50257 in fp32 28 us, some 20 of them the chunks): a workgroup takes a
// chunk of a row into registers and leaves the chunk's largest value, or its sorted `num`
// largest with the chunk's maximum and sum of exponentials; the last workgroup of a sequence to
// arrive does the rest. Values are compared as integers whose order is the floats' (the sign bit
// flipped for positives, all bits for negatives, -0 as +0), with the position below them
// inverted, so that no two are equal and ties go to the lower index by themselves.
//
// Beams of one sequence are ranked by sums whose differences 32 bits would lose, so lse and scores are
// held in 64. Exponentials are exp2's in 32 bits (within 2^-23 of themselves, and so is a sum of them), with all
// that was rounded off their arguments put back.
#include "../../include/lightserve_fa.h"
#include "fa_common.hpp"

#include <cfloat>
#include <algorithm>
#include <type_traits>

namespace lsfa {

constexpr int kThreads = 256, kWaves = 4;

__device__ __forceinline__ void store_agent(uint64_t* to, uint64_t v) {
  __hip_atomic_store(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_agent(const uint64_t* from) {
  return __hip_atomic_load((uint64_t*)from, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Whole numbers in the order of values that are no NaN (-0 as +0), and back.
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
constexpr uint32_t kKeyNan = 0xffffffffu, kKeyLow = 0x007fffffu;  // above all numbers; of -inf, below them

// Largest of two, NaN where one is (one instruction for three of them).
__device__ __forceinline__ float nan_max(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// All lanes' values by one operation, in every lane. The steps within and across rows of 16 lanes leave
// the result in the last one.
template <typename F>
__device__ __forceinline__ float wave_all(float v, F f) {
#define LSFA_STEP(ctrl, rows) \
  v = f(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(v), (int)__float_as_uint(v), ctrl, rows, 0xf, false)))
  LSFA_STEP(0x111, 0xf);  // row_shr 1, 2, 4, 8
  LSFA_STEP(0x112, 0xf);
  LSFA_STEP(0x114, 0xf);
  LSFA_STEP(0x118, 0xf);
  LSFA_STEP(0x142, 0xa);  // row_bcast 15, 31
  LSFA_STEP(0x143, 0xc);
#undef LSFA_STEP
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_all(v, [](float a, float b) { return nan_max(a, b); });
}
// One chunk of a row in a workgroup's registers: U 16-byte loads a thread, of whole 16-byte
// words of memory (a row may begin anywhere: chunks count from the word that it begins in).
template <typename T, int U>
struct Chunk {
  static constexpr int EPV = 16 / sizeof(T), E = EPV * U;  // values of a load, of a thread
  static constexpr int C = kThreads * E;
  static_assert(C <= 65536, "positions have 16 bits");
  u32x4 v[U];
  int lo, hi;  // positions of the row's values in the chunk
  int first;   // index in the row of position 0

  __device__ __forceinline__ void load(const void* logits, int64_t row, int64_t stride, int cols, int chunk) {
    const uintptr_t at = (uintptr_t)logits + (uint64_t)(row * stride) * sizeof(T);
    const int skip = (int)(at & 15) / (int)sizeof(T);
    const int64_t start = (int64_t)chunk * C;
    const int64_t bytes = (((int64_t)(skip + cols) * (int)sizeof(T) + 3) & ~3ll) - start * (int)sizeof(T);
    const __amdgpu_buffer_rsrc_t rs =
        tile_rsrc((const void*)((at & ~(uintptr_t)15) + start * sizeof(T)), (int)std::min<int64_t>(std::max<int64_t>(bytes, 0), C * (int)sizeof(T)));
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = load16(rs, (u * kThreads + (int)threadIdx.x) * 16);
    lo = (int)std::max<int64_t>(skip - start, 0);
    hi = (int)std::min<int64_t>(skip + cols - start, C);
    first = (int)(start - skip);
  }
  __device__ __forceinline__ int pos(int i) const { return (i / EPV * kThreads + (int)threadIdx.x) * EPV + i % EPV; }
  // -inf in the places of the first and last chunk that the row does not have.
  __device__ __forceinline__ void cut() {
    if (lo <= 0 && hi >= C) return;  // uniform
#pragma unroll
    for (int i = 0; i < E; ++i) {
      if (pos(i) >= lo && pos(i) < hi) continue;
      const int e = i % EPV;
      const int j = sizeof(T) == 4 ? e : e / 2;
      uint32_t w = v[i / EPV][j];
      if constexpr (sizeof(T) == 4) w = 0xff800000u;
      else {
        constexpr uint32_t low = __is_same(T, _Float16) ? 0xfc00u : 0xff80u;
        w = e & 1 ? (w & 0xffffu) | low << 16 : (w & 0xffff0000u) | low;
      }
      v[i / EPV][j] = w;
    }
  }
  __device__ __forceinline__ float value(int i) const {
    const int e = i % EPV;
    const uint32_t w = v[i / EPV][sizeof(T) == 4 ? e : e / 2];
    if constexpr (sizeof(T) == 4) return __uint_as_float(w);
    else if constexpr (__is_same(T, _Float16)) return (float)__builtin_bit_cast(_Float16, (uint16_t)(e & 1 ? w >> 16 : w));
    else return __uint_as_float(e & 1 ? w & 0xffff0000u : w << 16);
  }
  __device__ __forceinline__ float largest() const {
    float m[2] = {value(0), value(1)};
#pragma unroll
    for (int i = 2; i < E; i += 2) m[i / 2 & 1] = nan_max(nan_max(m[i / 2 & 1], value(i)), value(i + 1));
    return nan_max(m[0], m[1]);
  }
};
// A key above an index, inverted: of equal keys the lower index is the larger.
__device__ __forceinline__ uint64_t entry_of(uint32_t key, int index) { return (uint64_t)key << 32 | (uint32_t)~index; }
__device__ __forceinline__ int index_of(uint64_t g) { return (int)~(uint32_t)g; }

// Where sequence b's counter lies: arrivals at one cache line wait for one another (32 sequences' next to
// each other cost 1792 workgroups 8 us), so up to 1024 sequences have lines of their own.
__device__ __forceinline__ int counter_of(int b, int B) { return B <= LSFA_GEMV_COUNTER_BYTES / 256 ? b * 64 : b; }

// Whether this workgroup is the last of `all` that arrive at the counter, whose partial
// results are then there to be read with load_agent. (Stores of the others have left for device
// scope before they arrive; the counter is left at zero.)
__device__ __forceinline__ bool last_to_arrive(int* counter, int all, int* flag) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    const bool last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == all - 1;
    if (last) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *flag = last;
  }
  __syncthreads();
  return *flag != 0;
}

// ------------------------------------------------------------------ accept
// A sequence's nodes: n rows of the logits from tok0 on (no row outside them, whatever the offsets).
__device__ __forceinline__ void nodes_of(const AcceptParams& p, int b, int& tok0, int& n) {
  tok0 = min(max(p.cu[b], 0), p.rows);
  n = min(max(min(p.cu[b + 1], p.rows) - tok0, 0), p.max_nodes);
}

// A workgroup takes p.per chunks of a row, the next one in flight while it looks at one, and leaves the
// largest value and its index.
template <typename T, int U>
__global__ __launch_bounds__(kThreads) void fa_accept_kernel(const AcceptParams p) {
  using Ch = Chunk<T, U>;
  __shared__ float st_m[kWaves];
  __shared__ int st_k[kWaves], st_at;
  __shared__ int st_last;
  __shared__ unsigned long long st_best[LSFA_TREE_MAX_NODES];
  __shared__ uint64_t st_mask[LSFA_TREE_MAX_NODES][LSFA_TREE_MAX_NODES / 64];
  __shared__ int64_t st_token[LSFA_TREE_MAX_NODES];
  __shared__ int st_path[LSFA_TREE_MAX_NODES];
  __shared__ int st_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (blockIdx.x == (unsigned)(p.rows * p.parts)) {  // sequences without nodes
    for (int b = 0; b < p.B; ++b) {
      int tok0, n;
      nodes_of(p, b, tok0, n);
      if (n > 0) continue;
      for (int i = tid; i < p.max_nodes; i += kThreads) p.path[(int64_t)b * p.max_nodes + i] = -1;
      if (tid == 0) p.counts[b] = 0, p.next[b] = -1;
    }
    return;
  }
  const int part = (int)(blockIdx.x % (unsigned)p.parts);
  // The nodes of all sequences are numbered one after another; a workgroup takes those p.rows apart
  // (one, unless offsets that are none let sequences share rows).
  for (int64_t id = blockIdx.x / (unsigned)p.parts;; id += p.rows) {
    int b = -1, tok0 = 0, n = 0, node = 0;
    int64_t at = 0;
    for (int j = 0; j < p.B && b < 0; j += 64) {
      int t = 0, c = 0;
      if (j + lane < p.B) nodes_of(p, j + lane, t, c);
      const int upto = lanes_sum(c);
      const unsigned long long hit = __ballot(at + upto > id);
      if (hit != 0) {
        const int src = __builtin_ctzll(hit);
        b = j + src;
        tok0 = __builtin_amdgcn_readlane(t, src);
        n = __builtin_amdgcn_readlane(c, src);
        node = (int)(id - at) - (__builtin_amdgcn_readlane(upto, src) - n);
      }
      at += __builtin_amdgcn_readlane(upto, 63);
    }
    if (b < 0) return;  // uniform

    const int k0 = part * p.per, k1 = min(k0 + p.per, p.chunks);
    const int64_t row = tok0 + node;
    constexpr int AHEAD = 2;  // chunks in registers (three 34.5 us for 33.5, 556 rows of 128256 that no cache holds)
    Ch ring[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (k0 + j < k1) ring[j].load(p.logits, row, p.stride, p.cols, k0 + j);
    float best = -INFINITY;  // the thread's, and the first chunk that has it
    int best_k = k0;
    for (int k = k0; k < k1; k += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        if (k + j >= k1) break;
        Ch& x = ring[j];
        x.cut();
        const float m = x.largest();
        if (m > best || (m != m && best == best)) best = m, best_k = k + j;
        if (k + j + AHEAD < k1) x.load(p.logits, row, p.stride, p.cols, k + j + AHEAD);
      }
    }
    Ch& x = ring[0];  // (a single chunk's still)
    // Of equal ones the lowest chunk, then the lowest position in it.
    auto same = [](float a, float b) -> bool { return a == b || (a != a && b != b); };
    const float wm = wave_max(best);
    int wk = same(best, wm) ? best_k : 0x7fffffff;
    for (int o = 32; o > 0; o >>= 1) wk = min(wk, __shfl_xor(wk, o));
    if (lane == 0) st_m[wave] = wm, st_k[wave] = wk;
    if (tid == 0) st_at = 0x7fffffff;
    __syncthreads();
    float top = st_m[0];
    for (int w = 1; w < kWaves; ++w) top = nan_max(top, st_m[w]);
    int k = 0x7fffffff;
    for (int w = 0; w < kWaves; ++w)
      if (same(st_m[w], top)) k = min(k, st_k[w]);
    if (p.per > 1) {
      x.load(p.logits, row, p.stride, p.cols, k);
      x.cut();
    }
    if (same(wm, top) && wk == k) {  // (a wave without it there has nothing to look for)
      int found = 0x7fffffff;
#pragma unroll
      for (int i = Ch::E - 1; i >= 0; --i) found = same(x.value(i), top) ? x.pos(i) : found;
      if (found != 0x7fffffff) atomicMin(&st_at, found);
    }
    __syncthreads();
    if (tid == 0)
      store_agent(p.part + row * p.parts + part, entry_of(top != top ? kKeyNan : key_of(top), x.first + st_at));
    if (!last_to_arrive(p.counters + counter_of(b, p.B), n * p.parts, &st_last)) continue;

    // (bits past the sequence's nodes say nothing, as in the attention)
    const int words = p.mask_words, nodes = min(p.cu[b + 1], p.rows) - tok0;
    for (int i = tid; i < n; i += kThreads) {
      st_best[i] = 0;
      st_token[i] = p.tokens[tok0 + i];
      for (int w = 0; w < words; ++w) {
        const int bits = nodes - 64 * w;
        const uint64_t m = p.mask[(int64_t)(tok0 + i) * p.mask_stride + w];
        st_mask[i][w] = bits >= 64 ? m : bits > 0 ? m & ((1ull << bits) - 1) : 0;
      }
    }
    __syncthreads();
    for (int t0 = 0; t0 < n * p.parts; t0 += 4 * kThreads) {
      uint64_t g[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = t0 + u * kThreads + tid;
        g[u] = t < n * p.parts ? load_agent(p.part + (int64_t)tok0 * p.parts + t) : 0;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = t0 + u * kThreads + tid;
        if (t < n * p.parts) atomicMax(&st_best[t / p.parts], (unsigned long long)g[u]);
      }
    }
    __syncthreads();
    // (a row of -inf only: its first value)
    auto choice = [&](int i) -> int { return (uint32_t)(st_best[i] >> 32) == kKeyLow ? 0 : index_of(st_best[i]); };
    if (wave == 0) {
      int cur = 0, count = 1;
      if (lane == 0) st_path[0] = 0;
      while (true) {
        const int64_t want = choice(cur);
        int next = -1;
        for (int j0 = 0; j0 < n && next < 0; j0 += 64) {
          const int j = j0 + lane;
          bool child = j > cur && j < n && st_token[j] == want;
          if (child)
            for (int w = 0; w < words; ++w) child &= st_mask[j][w] == (st_mask[cur][w] | (w == j >> 6 ? 1ull << (j & 63) : 0ull));
          const unsigned long long hit = __ballot(child);
          if (hit != 0) next = j0 + __builtin_ctzll(hit);
        }
        if (next < 0) break;
        cur = next;  // (paths only rise: at most n steps)
        if (lane == 0) st_path[count] = cur;
        ++count;
      }
      if (lane == 0) {
        st_count = count;
        p.counts[b] = count;
        p.next[b] = choice(cur);
        if (p.seq_lens != nullptr) p.seq_lens[b] += count;
      }
    }
    __syncthreads();
    for (int i = tid; i < p.max_nodes; i += kThreads) p.path[(int64_t)b * p.max_nodes + i] = i < st_count ? st_path[i] : -1;
    __syncthreads();
  }
}

// ------------------------------------------------------------------- beams
// Adds exp(x - top), x <= top, to a sum that is `sum` + `rest`. The difference is rounded (t, by up to 2^-22 between four and
// eight, and alike for all equal x, of which a vocabulary may be full) and so is its product with log2(e) (y): what both left
// out is small, and exp of it one more than itself. Below exp(-100), which no sum with exp(0) in it shows, t is held there.
// (Without the difference's rounding 32 x 8 beams of 50257 in fp32 take 26.6 us for 28.3.)
__device__ __forceinline__ void add_exp(float x, float top, double& sum, float& rest) {
  constexpr float kLog2e = 1.44269502162933349609375f, kLn2 = 0.693147182464599609375f, kLn2Rest = -1.904654323148236e-9f;
  const float t = x - top, back = t - x;
  const float off = (x - (t - back)) - (top + back);  // x - top - t
  const float c = fmaxf(t, -100.f), y = c * kLog2e;
  const float left = fmaf(-y, kLn2Rest, fmaf(-y, kLn2, c)) + (t > -100.f ? off : 0.f);
  const float e = fast_exp2(y);
  sum += (double)e;
  rest = fmaf(e, left, rest);
}

// The Nth largest of all threads' keys (0 where fewer are above 0): at least N values are at or above it where each is its
// thread's largest, and few more.
__device__ __forceinline__ uint32_t nth_of_threads(uint32_t key, int N, uint32_t* st_key) {
  __syncthreads();
  st_key[threadIdx.x] = key;
  __syncthreads();
  uint32_t k[kWaves], from = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) k[w] = st_key[w * 64 + (threadIdx.x & 63)];
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = from | 1u << bit;
    int c = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) c += __builtin_popcountll(__ballot(k[w] >= t));
    if (c >= N) from = t;
    if (c == N) break;
  }
  return from;
}

// Most entries of a sequence's lists that its merging takes whole (eight beams of 128256, the best 16: 2048 entries 16.8 us,
// in two steps 18.9; 16 x 16 of 32000, the best 32 26.0 and 30.2; 56 lists of 16 27.4 and 29.7).
constexpr int kFew = 8 * kThreads;

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void fa_beams_kernel(const BeamParams p) {
  using Ch = Chunk<T, U>;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float st_m[kWaves];
  __shared__ double st_l[kWaves];
  __shared__ uint32_t st_key[kThreads];
  __shared__ int st_n[kWaves], st_put, st_last, st_found, st_kept, st_chosen[LSFA_BEAMS_NUM_MAX];
  __shared__ double st_lse[LSFA_BEAMS_MAX], st_score[LSFA_BEAMS_MAX], st_floor;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = p.num, S = p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)S), row = (int)(blockIdx.x / (unsigned)S), b = row / p.K;
  const int64_t list = (int64_t)row * S + chunk;

  Ch x;
  x.load(p.logits, row, p.stride, p.cols, chunk);
  x.cut();
  const float mine = x.largest(), top = wave_max(mine);  // NaN where there is one
  double l = 0.;
  if (top > -INFINITY) {
    float rest = 0.f;
#pragma unroll
    for (int i = 0; i < Ch::E; ++i) add_exp(x.value(i), top, l, rest);
    l += (double)rest;
  }
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if (lane == 0) st_m[wave] = top, st_l[wave] = l;
  if (tid == 0) st_put = 0;

  // The chunk's N largest are at or above the Nth largest of its threads' largest, and little else is
  // (finite values: -inf is no candidate, and a row with NaN has none).
  const uint32_t from = nth_of_threads(mine > -INFINITY ? key_of(mine) : 0u, N, st_key);
  const float least = from == 0 ? -FLT_MAX : fmaxf(value_of(from), -FLT_MAX);
  auto entry = [&](int i) -> uint64_t { return entry_of(key_of(x.value(i)), x.first + x.pos(i)); };
  uint64_t* pool = (uint64_t*)lds;  // [kThreads]
  int c = 0;
#pragma unroll
  for (int i = 0; i < Ch::E; ++i) c += x.value(i) >= least;
  const int upto = lanes_sum(c), n = __builtin_amdgcn_readlane(upto, 63);
  int at = 0;
  if (lane == 0) at = atomicAdd(&st_put, n);
  at = __builtin_amdgcn_readfirstlane(at) + upto - c;
#pragma unroll
  for (int i = 0; i < Ch::E; ++i)
    if (x.value(i) >= least) {
      if (at < kThreads) pool[at] = entry(i);
      ++at;
    }
  __syncthreads();
  int all = st_put, have = all;
  if (all > kThreads) {  // (many equal ones): of each wave the entries that exactly N are at or above, or all
    uint64_t exact = 0;
    for (int bit = 63; bit >= 0; --bit) {
      const uint64_t t = exact | 1ull << bit;
      int k = 0;
#pragma unroll
      for (int i = 0; i < Ch::E; ++i) k += __builtin_popcountll(__ballot(x.value(i) >= least && entry(i) >= t));
      if (k >= N) exact = t;
      if (k == N) break;
    }
    pool[tid] = 0;
    c = 0;
#pragma unroll
    for (int i = 0; i < Ch::E; ++i) c += x.value(i) >= least && entry(i) >= exact;
    at = wave * 64 + lanes_sum(c) - c;
#pragma unroll
    for (int i = 0; i < Ch::E; ++i)
      if (x.value(i) >= least && entry(i) >= exact) pool[at++] = entry(i);
    if (lane == 0) st_n[wave] = min(n, N);
    __syncthreads();
    all = kThreads;
    have = 0;
    for (int w = 0; w < kWaves; ++w) have += st_n[w];
  }
  // Each at its rank.
  uint64_t* out = p.lists + list * N;
  const uint64_t cand = tid < all ? pool[tid] : 0;
  int rank = 0;
  if (cand != 0) {
#pragma unroll 4
    for (int j = 0; j < all; ++j) rank += pool[j] > cand;
    if (rank < N) store_agent(out + rank, cand);
  }
  for (int j = have + tid; j < N; j += kThreads) store_agent(out + j, 0);
  if (tid == 0) {
    float M = st_m[0];
    for (int w = 1; w < kWaves; ++w) M = nan_max(M, st_m[w]);
    double L = 0.;
    for (int w = 0; w < kWaves; ++w)
      if (st_m[w] > -INFINITY) L += st_l[w] * exp((double)st_m[w] - (double)M);
    store_agent(p.sums + 2 * list, __float_as_uint(M));
    store_agent(p.sums + 2 * list + 1, (uint64_t)__double_as_longlong(L));
  }
  if (!last_to_arrive(p.counters + counter_of(b, p.B), p.K * S, &st_last)) return;

  // The sequence's lists meet: K S of them, in the order of k V + v. What is read was written elsewhere and
  // takes a microsecond to come: all of it is asked for at once, or of many entries the lists' first ones, then the N lists
  // with the best of them.
  const int lists = p.K * S;
  const int64_t list0 = (int64_t)b * lists;
  double* sum = (double*)lds;                 // [lists]; then the scores of their first entries
  uint64_t* firsts = (uint64_t*)(sum + lists);  // [lists]
  float* lmax = (float*)(firsts + lists);     // [lists]
  const int entries = lists * N;
  const bool few = entries <= kFew;
  uint64_t mine_of[kFew / kThreads];  // few: the thread's entries
  if (few) {
#pragma unroll
    for (int u = 0; u < kFew / kThreads; ++u)
      mine_of[u] = u * kThreads + tid < entries ? load_agent(p.lists + list0 * N + u * kThreads + tid) : 0;
  }
  for (int t = tid; t < lists; t += kThreads) {
    const uint64_t m = load_agent(p.sums + 2 * (list0 + t)), l2 = load_agent(p.sums + 2 * (list0 + t) + 1);
    if (!few) firsts[t] = load_agent(p.lists + (list0 + t) * N);
    lmax[t] = __uint_as_float((uint32_t)m);
    sum[t] = __longlong_as_double((long long)l2);
  }
  const double own = tid < p.K ? (double)p.scores[(int64_t)b * p.K + tid] : 0.;
  if (tid < N) st_chosen[tid] = -1;
  if (tid == 0) st_found = st_kept = 0, st_floor = -(double)INFINITY;
  __syncthreads();
  for (int t = tid; t < lists; t += kThreads) {
    const int k0 = t / S * S;
    float M = lmax[k0];
#pragma unroll 4
    for (int s = 1; s < S; ++s) M = nan_max(M, lmax[k0 + s]);
    if (lmax[t] > -INFINITY) sum[t] *= exp((double)lmax[t] - (double)M);
    if (t == k0) st_lse[t / S] = M;  // (K <= LSFA_BEAMS_MAX)
  }
  __syncthreads();
  if (tid < p.K) {
    double L = 0.;
#pragma unroll 4
    for (int s = 0; s < S; ++s) L += sum[tid * S + s];
    const double lse = st_lse[tid] + log(L);
    st_lse[tid] = lse > -(double)INFINITY && lse < (double)INFINITY ? lse : (double)NAN;  // a row without lse offers nothing
    st_score[tid] = own;
  }
  __syncthreads();
  auto score = [&](int k, uint64_t g) -> double {
    const double sc = st_score[k] + ((double)value_of((uint32_t)(g >> 32)) - st_lse[k]);
    return g != 0 && sc > -(double)INFINITY ? sc : -(double)INFINITY;
  };
  // What is at or above the Nth largest, in 32 bits, of the threads' best candidates is ranked: the N best and few others.
  double* cs = (double*)lds;                       // [entries or N * N] of those
  int* ci = (int*)(cs + (few ? entries : N * N));  // k V + v
  float best = -INFINITY;
  if (few) {
    double sc[kFew / kThreads];
#pragma unroll
    for (int u = 0; u < kFew / kThreads; ++u) {
      sc[u] = mine_of[u] != 0 ? score((u * kThreads + tid) / N / S, mine_of[u]) : -(double)INFINITY;
      best = fmaxf(best, (float)sc[u]);
    }
    const uint32_t low = nth_of_threads(best > -INFINITY ? key_of(best) : 0u, N, st_key);
#pragma unroll
    for (int u = 0; u < kFew / kThreads; ++u) {
      if (!(sc[u] > -(double)INFINITY) || key_of((float)sc[u]) < low) continue;
      const int to = atomicAdd(&st_found, 1);
      cs[to] = sc[u];
      ci[to] = (u * kThreads + tid) / N / S * p.cols + index_of(mine_of[u]);
    }
    __syncthreads();
  } else {
    // The N best lie in the N lists with the best first entries, at or above the Nth of those.
    for (int t = tid; t < lists; t += kThreads) {
      sum[t] = score(t / S, firsts[t]);
      best = fmaxf(best, (float)sum[t]);
    }
    uint32_t low = nth_of_threads(best > -INFINITY ? key_of(best) : 0u, N, st_key);
    double* ks = (double*)firsts;  // [lists]: the scores of those lists that may be, and in lmax their numbers
    int* kt = (int*)lmax;
    for (int t = tid; t < lists; t += kThreads) {
      const double h = sum[t];
      if (!(h > -(double)INFINITY) || key_of((float)h) < low) continue;
      const int at = atomicAdd(&st_kept, 1);
      ks[at] = h;
      kt[at] = t;
    }
    __syncthreads();
    const int kept = st_kept;
    for (int i = tid; i < kept; i += kThreads) {
      const double h = ks[i];
      const int t = kt[i];
      int rank = 0;
#pragma unroll 4
      for (int j = 0; j < kept; ++j) rank += ks[j] > h || (ks[j] == h && kt[j] < t);
      if (rank < N) st_chosen[rank] = t;
      if (rank == N - 1) st_floor = h;
    }
    __syncthreads();
    const double floor = st_floor;
    best = -INFINITY;
    for (int e0 = tid; e0 < N * N; e0 += 4 * kThreads) {
      uint64_t g[4];
      int of[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * kThreads;
        of[u] = e < N * N ? st_chosen[e / N] : -1;
        g[u] = of[u] >= 0 ? load_agent(p.lists + (list0 + of[u]) * N + e % N) : 0;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int e = e0 + u * kThreads;
        const double sc = g[u] != 0 ? score(of[u] / S, g[u]) : -(double)INFINITY;
        if (e >= N * N) break;
        cs[e] = sc >= floor ? sc : -(double)INFINITY;
        ci[e] = of[u] / S * p.cols + index_of(g[u]);
        best = fmaxf(best, (float)cs[e]);
      }
    }
    // Moved to the front: no more than have been read.
    low = nth_of_threads(best > -INFINITY ? key_of(best) : 0u, N, st_key);
    for (int e0 = 0; e0 < N * N; e0 += kThreads) {
      const int e = e0 + tid;
      const double sc = e < N * N ? cs[e] : -(double)INFINITY;
      const int id = e < N * N ? ci[e] : 0;
      __syncthreads();
      if (sc > -(double)INFINITY && key_of((float)sc) >= low) {
        const int to = atomicAdd(&st_found, 1);
        cs[to] = sc;
        ci[to] = id;
      }
      __syncthreads();
    }
  }
  const int found = st_found;
  for (int i = tid; i < found; i += kThreads) {
    const double sc = cs[i];
    const int id = ci[i];
    int rank = 0;
    for (int j = 0; j < found; ++j) rank += cs[j] > sc || (cs[j] == sc && ci[j] < id);
    if (rank < N) {
      const int64_t to = (int64_t)b * N + rank;
      p.out_scores[to] = (float)sc;
      p.out_beams[to] = id / p.cols;
      p.out_tokens[to] = id % p.cols;
    }
  }
  for (int i = found + tid; i < N; i += kThreads) {
    const int64_t to = (int64_t)b * N + i;
    p.out_scores[to] = -INFINITY;
    p.out_beams[to] = 0;
    p.out_tokens[to] = 0;
  }
}

// ---------------------------------------------------------------- launches
// Chunks of a row of `cols` values for U loads a thread (one more where the row begins inside a word).
static int chunks_of(int cols, int size, int U) {
  const int epv = 16 / size, c = kThreads * epv * U;
  return (int)(((long long)cols + epv - 1 + c - 1) / c);
}
SelectPlan select_plan(long long rows, int cols, int dtype, bool beams) {
  const int size = dtype == 0 ? 4 : 2;
  SelectPlan s;
  // Beams: chunks of 8192 values (half of that 30.5 us for 28.3, 256 rows of 50257 in fp32, and 33.3 for 29.8 in bf16).
  // Acceptance reads ahead: 4096 (2048 in fp32; 556 rows of 128256 29.3 us, with twice of that 31).
  s.loads = !beams ? 2 : size == 4 ? 8 : 4;
  // Smaller chunks where there are few of them. (Not for the sake of more CUs: all that arrive at a sequence's counter wait
  // for one another, and their partial results for the last one. 512 chunks of 8 rows of 128256 12.7 us, 128 9.6; 252 of
  // four beams 16.4, 64 14.6.)
  while (s.loads > 1 && rows * chunks_of(cols, size, s.loads) < 64) s.loads /= 2;
  s.chunks = chunks_of(cols, size, s.loads);
  // Acceptance: as many chunks to a workgroup as leave 256 of them or one for each row. (556 rows of 128256 29.3 us; one
  // chunk to a workgroup 76 us for 512 rows, 2048 workgroups 33, 256 27. 32 rows: 512 workgroups 13.7, 256 11.1.) Beams: one chunk,
  // since the selection of a chunk has waits that only another workgroup fills (32 x 8 beams of 50257 in fp32: 28.3 us,
  // several chunks with the best so far as a floor 31 at best).
  s.per = beams ? 1 : (int)std::max(1LL, std::min<long long>(s.chunks, (rows * s.chunks + 255) / 256));
  s.parts = (s.chunks + s.per - 1) / s.per;
  return s;
}

template <typename T, int U>
static void launch_accept(const AcceptParams& p, hipStream_t s) {
  hipLaunchKernelGGL((fa_accept_kernel<T, U>), dim3((unsigned)(p.rows * p.parts + 1)), dim3(kThreads), 0, s, p);
}
template <typename T, int U>
static void launch_beams(const BeamParams& p, hipStream_t s) {
  const size_t lists = (size_t)p.K * p.chunks;
  const size_t lds = std::max({(size_t)kThreads * 8, lists * 20,
                               12 * (lists * p.num <= (size_t)kFew ? lists * p.num : (size_t)p.num * p.num)});
  hipLaunchKernelGGL((fa_beams_kernel<T, U>), dim3((unsigned)(p.B * p.K * p.chunks)), dim3(kThreads), lds, s, p);
}
template <typename T>
static void by_loads(const AcceptParams& p, int loads, hipStream_t s) {
  if (loads == 2) launch_accept<T, 2>(p, s);
  else launch_accept<T, 1>(p, s);
}
template <typename T>
static void by_loads(const BeamParams& p, int loads, hipStream_t s) {
  if constexpr (sizeof(T) == 4)
    if (loads == 8) return launch_beams<T, 8>(p, s);
  if (loads == 4) launch_beams<T, 4>(p, s);
  else if (loads == 2) launch_beams<T, 2>(p, s);
  else launch_beams<T, 1>(p, s);
}
// Host entries used by the C ABI layer (arguments validated there).
hipError_t accept_drafts(const AcceptParams& p, int dtype, int loads, hipStream_t s) {
  if (dtype == 0) by_loads<float>(p, loads, s);
  else if (dtype == 1) by_loads<_Float16>(p, loads, s);
  else by_loads<__bf16>(p, loads, s);
  return hipGetLastError();
}
hipError_t beam_select(const BeamParams& p, int dtype, int loads, hipStream_t s) {
  if (dtype == 0) by_loads<float>(p, loads, s);
  else if (dtype == 1) by_loads<_Float16>(p, loads, s);
  else by_loads<__bf16>(p, loads, s);
  return hipGetLastError();
}

}  // namespace lsfa
