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
// Both read each logit once (that and, for few rows, latency is what bounds them): a workgroup takes a
// chunk of a row into registers and leaves the chunk's largest value, or its sorted `num`
// largest with the chunk's maximum and sum of exponentials; the last workgroup of a sequence to
// arrive does the rest. Values are compared as integers whose order is the floats' (the sign bit
// flipped for positives, all bits for negatives, -0 as +0), with the position below them
// inverted, so that no two are equal and ties go to the lower index by themselves.
//
// Beams of one sequence are ranked by sums whose differences 32 bits would lose, so lse and scores are
// held in 64, and exponentials are taken with the rounding of their argument put back.
#include "../../include/lightserve_fa.h"
#include "fa_common.hpp"

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

// Whole numbers in the order of the values; 0 is below all of them.
template <typename T> struct Order;
template <> struct Order<float> {
  using Raw = uint32_t;
  static __device__ __forceinline__ uint32_t key(uint32_t u) {
    u = u == 0x80000000u ? 0u : u;
    const uint32_t k = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (u & 0x7fffffffu) > 0x7f800000u ? 0xffffffffu : k;
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k); }
};
template <typename T> struct Order16 {
  using Raw = uint16_t;
  static constexpr uint32_t kInf = __is_same(T, _Float16) ? 0x7c00u : 0x7f80u;
  static __device__ __forceinline__ uint32_t key(uint32_t u) {
    u = u == 0x8000u ? 0u : u;
    const uint32_t k = (u & 0x8000u) ? (~u & 0xffffu) : (u | 0x8000u);
    return (u & 0x7fffu) > kInf ? 0xffffu : k;
  }
  static __device__ __forceinline__ float value(uint32_t k) {
    return (float)__builtin_bit_cast(T, (uint16_t)((k & 0x8000u) ? k ^ 0x8000u : ~k));
  }
};
template <> struct Order<_Float16> : Order16<_Float16> {};
template <> struct Order<__bf16> : Order16<__bf16> {};

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
  return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o);
    v = w > v ? w : v;
  }
  return v;
}

// One chunk of a row in a workgroup's registers: U 16-byte loads a thread, of whole 16-byte
// words of memory (a row may begin anywhere: chunks count from the word that it begins in).
template <typename T, int U>
struct Chunk {
  using O = Order<T>;
  static constexpr int EPV = 16 / sizeof(T), E = EPV * U;  // values of a load, of a thread
  static constexpr int C = kThreads * E;
  // A value's key above its position in the chunk, inverted.
  using Comp = std::conditional_t<sizeof(T) == 2, uint32_t, uint64_t>;
  static constexpr int kShift = sizeof(T) == 2 ? 16 : 32;
  static constexpr int kBits = sizeof(T) == 2 ? 32 : 64;
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
  __device__ __forceinline__ uint32_t raw(int i) const {
    const int e = i % EPV;
    if constexpr (sizeof(T) == 4) return v[i / EPV][e];
    else return e & 1 ? v[i / EPV][e / 2] >> 16 : v[i / EPV][e / 2] & 0xffffu;
  }
  __device__ __forceinline__ bool has(int i) const { return pos(i) >= lo && pos(i) < hi; }
  // Value i of the thread; 0 where the row has none.
  __device__ __forceinline__ Comp comp(int i) const {
    return has(i) ? ((Comp)O::key(raw(i)) << kShift) | (Comp)(65535 - pos(i)) : (Comp)0;
  }
  __device__ __forceinline__ float value(int i) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(raw(i));
    else return (float)__builtin_bit_cast(T, (uint16_t)raw(i));
  }
  // The same with the index in the row below the key: comparable over a row's chunks.
  __device__ __forceinline__ uint64_t global(Comp c) const {
    if (c == 0) return 0;
    const uint32_t index = (uint32_t)(first + 65535 - (int)(c & 0xffffu));
    return (uint64_t)(uint32_t)(c >> kShift) << 32 | (uint32_t)~index;
  }
};
__device__ __forceinline__ int index_of(uint64_t g) { return (int)~(uint32_t)g; }
template <typename T> __device__ __forceinline__ float value_of(uint64_t g) { return Order<T>::value((uint32_t)(g >> 32)); }

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

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void fa_accept_kernel(const AcceptParams p) {
  using Ch = Chunk<T, U>;
  __shared__ uint64_t st_best[kWaves];
  __shared__ int st_last;
  __shared__ uint64_t st_mask[LSFA_TREE_MAX_NODES][LSFA_TREE_MAX_NODES / 64];
  __shared__ int64_t st_token[LSFA_TREE_MAX_NODES];
  __shared__ int st_choice[LSFA_TREE_MAX_NODES], st_path[LSFA_TREE_MAX_NODES];
  __shared__ int st_count;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (blockIdx.x == (unsigned)(p.rows * p.chunks)) {  // sequences without nodes
    for (int b = 0; b < p.B; ++b) {
      int tok0, n;
      nodes_of(p, b, tok0, n);
      if (n > 0) continue;
      for (int i = tid; i < p.max_nodes; i += kThreads) p.path[(int64_t)b * p.max_nodes + i] = -1;
      if (tid == 0) p.counts[b] = 0, p.next[b] = -1;
    }
    return;
  }
  const int chunk = (int)(blockIdx.x % (unsigned)p.chunks);
  // The nodes of all sequences are numbered one after another; a workgroup takes those p.rows apart
  // (one, unless offsets that are none let sequences share rows).
  for (int64_t id = blockIdx.x / (unsigned)p.chunks;; id += p.rows) {
    int b = -1, tok0 = 0, n = 0, node = 0;
    int64_t at = 0;
    for (int j = 0; j < p.B && b < 0; j += 64) {
      int t = 0, c = 0;
      if (j + lane < p.B) nodes_of(p, j + lane, t, c);
      int upto = c;
      for (int o = 1; o < 64; o <<= 1) {
        const int w = __shfl_up(upto, o);
        if (lane >= o) upto += w;
      }
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

    Ch x;
    x.load(p.logits, tok0 + node, p.stride, p.cols, chunk);
    typename Ch::Comp m = 0;
#pragma unroll
    for (int i = 0; i < Ch::E; ++i) {
      const typename Ch::Comp c = x.comp(i);
      m = c > m ? c : m;
    }
    m = wave_max(m);
    if (lane == 0) st_best[wave] = x.global(m);
    __syncthreads();
    if (tid == 0) {
      uint64_t best = st_best[0];
      for (int w = 1; w < kWaves; ++w) best = st_best[w] > best ? st_best[w] : best;
      store_agent(p.part + (int64_t)(tok0 + node) * p.chunks + chunk, best);
    }
    if (!last_to_arrive(p.counters + b, n * p.chunks, &st_last)) continue;

    const int words = p.mask_words;
    for (int i = tid; i < n; i += kThreads) {
      uint64_t best = 0;
#pragma unroll 8
      for (int s = 0; s < p.chunks; ++s) {
        const uint64_t g = load_agent(p.part + (int64_t)(tok0 + i) * p.chunks + s);
        best = g > best ? g : best;
      }
      st_choice[i] = index_of(best);
      st_token[i] = p.tokens[tok0 + i];
      for (int w = 0; w < words; ++w) st_mask[i][w] = p.mask[(int64_t)(tok0 + i) * p.mask_stride + w];
    }
    __syncthreads();
    if (wave == 0) {
      int cur = 0, count = 1;
      if (lane == 0) st_path[0] = 0;
      while (true) {
        const int64_t want = st_choice[cur];
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
        p.next[b] = st_choice[cur];
        if (p.seq_lens != nullptr) p.seq_lens[b] += count;
      }
    }
    __syncthreads();
    for (int i = tid; i < p.max_nodes; i += kThreads) p.path[(int64_t)b * p.max_nodes + i] = i < st_count ? st_path[i] : -1;
    __syncthreads();
  }
}

// ------------------------------------------------------------------- beams
// exp(t) of a difference t <= 0 in 32 bits, the argument's rounding put back.
__device__ __forceinline__ float exp_near(float t) {
  constexpr float kLog2e = 1.44269502162933349609375f, kRest = 1.925963033500011079e-8f, kLn2 = 0.6931471805599453f;
  const float y = t * kLog2e, low = fmaf(t, kRest, fmaf(t, kLog2e, -y));
  const float e = fast_exp2(y);
  return e == 0.f ? 0.f : fmaf(e, low * kLn2, e);
}

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void fa_beams_kernel(const BeamParams p) {
  using Ch = Chunk<T, U>;
  using Comp = typename Ch::Comp;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float st_m[kWaves];
  __shared__ double st_l[kWaves];
  __shared__ int st_n[kWaves], st_last, st_found;
  __shared__ double st_lse[LSFA_BEAMS_MAX], st_floor;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int N = p.num, S = p.chunks;
  const int chunk = (int)(blockIdx.x % (unsigned)S), row = (int)(blockIdx.x / (unsigned)S), b = row / p.K;
  const int64_t list = (int64_t)row * S + chunk;

  Ch x;
  x.load(p.logits, row, p.stride, p.cols, chunk);
  Comp m = 0;
#pragma unroll
  for (int i = 0; i < Ch::E; ++i) {
    const Comp c = x.comp(i);
    m = c > m ? c : m;
  }
  const Comp wm = wave_max(m);
  // The wave's sum of exponentials: NaN where it has a NaN or +inf.
  const float top = wm == 0 ? -INFINITY : Order<T>::value((uint32_t)(wm >> Ch::kShift));
  double l = 0.;
  if (top != -INFINITY) {
#pragma unroll
    for (int i = 0; i < Ch::E; ++i)
      if (x.has(i)) l += (double)exp_near(x.value(i) - top);
  }
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o);
  if (lane == 0) st_m[wave] = top, st_l[wave] = l;

  // The wave's N largest: those from the Nth largest of its lanes' largest on hold them all, the
  // few more that there are go by a second search (no two values are equal).
  auto nth_largest = [&](auto count_from) -> Comp {  // the largest c with count_from(c) >= N, or 1
    Comp c = 0;
    for (int bit = Ch::kBits - 1; bit >= 0; --bit) {
      const Comp t = c | (Comp)1 << bit;
      const int n = count_from(t);
      if (n >= N) c = t;
      if (n == N) break;
    }
    return c == 0 ? (Comp)1 : c;
  };
  const Comp from = nth_largest([&](Comp t) -> int { return __builtin_popcountll(__ballot(m >= t)); });
  Comp* mine = (Comp*)lds + wave * (64 * Ch::E);
  int hits = 0;
#pragma unroll
  for (int i = 0; i < Ch::E; ++i) hits += x.comp(i) >= from;
  int upto = hits;
  for (int o = 1; o < 64; o <<= 1) {
    const int w = __shfl_up(upto, o);
    if (lane >= o) upto += w;
  }
  int n = __builtin_amdgcn_readlane(upto, 63), put = upto - hits;
#pragma unroll
  for (int i = 0; i < Ch::E; ++i) {
    const Comp c = x.comp(i);
    if (c >= from) mine[put++] = c;
  }
  asm volatile("" ::: "memory");
  Comp cand = lane < n ? mine[lane] : (Comp)0;
  if (n > 64) {  // uniform over the wave
    const Comp least = nth_largest([&](Comp t) -> int {
      int k = 0;
      for (int j = 0; j < n; j += 64) k += __builtin_popcountll(__ballot(j + lane < n && mine[j + lane] >= t));
      return k;
    });
    int kept = 0;
    cand = 0;
    for (int j = 0; j < n; j += 64) {
      const Comp c = j + lane < n ? mine[j + lane] : (Comp)0;
      const bool in = c >= least;
      const unsigned long long ones = __ballot(in);
      // (at most N <= 64 of them: a slot for each, in places that the loop has read)
      asm volatile("" ::: "memory");
      if (in) mine[kept + __builtin_popcountll(ones & ((1ull << lane) - 1))] = c;
      kept += __builtin_popcountll(ones);
    }
    asm volatile("" ::: "memory");
    n = kept;
    cand = lane < n ? mine[lane] : (Comp)0;
  }
  if (lane == 0) st_n[wave] = n;
  __syncthreads();
  // The workgroup's, one after another, each at its rank.
  int base = 0, all = 0;
  for (int w = 0; w < kWaves; ++w) {
    base += w < wave ? st_n[w] : 0;
    all += st_n[w];
  }
  Comp* pool = (Comp*)lds;
  __syncthreads();  // (the waves' own parts are in registers)
  if (lane < n) pool[base + lane] = cand;
  __syncthreads();
  uint64_t* out = p.lists + list * N;
  if (lane < n) {
    int rank = 0;
    for (int j = 0; j < all; ++j) rank += pool[j] > cand;
    if (rank < N) store_agent(out + rank, x.global(cand));
  }
  for (int j = all + tid; j < N; j += kThreads) store_agent(out + j, 0);
  if (tid == 0) {
    float M = st_m[0];
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, st_m[w]);
    double L = 0.;
    bool nan = false;
    for (int w = 0; w < kWaves; ++w) {
      nan |= !(st_l[w] < (double)INFINITY) || st_m[w] != st_m[w];
      if (st_m[w] > -INFINITY) L += st_l[w] * exp((double)st_m[w] - (double)M);
    }
    store_agent(p.sums + 2 * list, __float_as_uint(M));
    store_agent(p.sums + 2 * list + 1, (uint64_t)__double_as_longlong(nan ? (double)NAN : L));
  }
  if (!last_to_arrive(p.counters + b, p.K * S, &st_last)) return;

  // The sequence's lists meet: K S of them, in the order of k V + v.
  const int lists = p.K * S;
  const int64_t list0 = (int64_t)b * lists;
  double* sum = (double*)lds;               // [lists]; then the scores of their first entries
  float* lmax = (float*)(sum + lists);      // [lists]
  for (int t = tid; t < lists; t += kThreads) {
    lmax[t] = __uint_as_float((uint32_t)load_agent(p.sums + 2 * (list0 + t)));
    sum[t] = __longlong_as_double((long long)load_agent(p.sums + 2 * (list0 + t) + 1));
  }
  if (tid == 0) st_found = 0, st_floor = -(double)INFINITY;
  __syncthreads();
  for (int t = tid; t < lists; t += kThreads) {
    const int k0 = t / S * S;
    float M = lmax[k0];
    for (int s = 1; s < S; ++s) M = fmaxf(M, lmax[k0 + s]);
    if (lmax[t] > -INFINITY) sum[t] *= exp((double)lmax[t] - (double)M);
    if (t == k0) st_lse[t / S] = M;  // (K <= LSFA_BEAMS_MAX)
  }
  __syncthreads();
  for (int k = tid; k < p.K; k += kThreads) {
    double L = 0.;
    for (int s = 0; s < S; ++s) L += sum[k * S + s];
    const double lse = st_lse[k] + log(L);
    st_lse[k] = lse > -(double)INFINITY && lse < (double)INFINITY ? lse : (double)NAN;  // a row without lse offers nothing
  }
  __syncthreads();
  auto score = [&](int k, uint64_t g) -> double {
    const double sc = (double)p.scores[(int64_t)b * p.K + k] + ((double)value_of<T>(g) - st_lse[k]);
    return g != 0 && sc > -(double)INFINITY ? sc : -(double)INFINITY;
  };
  for (int t = tid; t < lists; t += kThreads) sum[t] = score(t / S, load_agent(p.lists + (list0 + t) * N));
  __syncthreads();
  // The N best lie in the N lists with the best first entries, at or above the Nth of those.
  uint32_t chosen = 0;  // of the thread's lists (t = tid + 256 i)
  for (int t = tid, i = 0; t < lists; t += kThreads, ++i) {
    const double h = sum[t];
    int rank = 0;
    for (int j = 0; j < lists; ++j) rank += sum[j] > h || (sum[j] == h && j < t);
    if (rank < N && h > -(double)INFINITY) chosen |= 1u << i;
    if (rank == N - 1) st_floor = h;
  }
  __syncthreads();
  double* cs = (double*)lds;       // [N * N]
  int* ci = (int*)(cs + N * N);    // k V + v
  const double least = st_floor;
  for (int t = tid, i = 0; t < lists; t += kThreads, ++i) {
    if (!(chosen >> i & 1)) continue;
    for (int j = 0; j < N; ++j) {
      const uint64_t g = load_agent(p.lists + (list0 + t) * N + j);
      const double sc = score(t / S, g);
      if (!(sc >= least) || sc == -(double)INFINITY) break;
      const int at = atomicAdd(&st_found, 1);
      cs[at] = sc;
      ci[at] = t / S * p.cols + index_of(g);
    }
  }
  __syncthreads();
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
SelectPlan select_plan(long long rows, int cols, int dtype) {
  const int size = dtype == 0 ? 4 : 2;
  SelectPlan s;
  s.loads = 4;
  while (s.loads > 1 && rows * chunks_of(cols, size, s.loads) < 512) s.loads /= 2;
  s.chunks = chunks_of(cols, size, s.loads);
  return s;
}

template <typename T, int U>
static void launch_accept(const AcceptParams& p, hipStream_t s) {
  hipLaunchKernelGGL((fa_accept_kernel<T, U>), dim3((unsigned)(p.rows * p.chunks + 1)), dim3(kThreads), 0, s, p);
}
template <typename T, int U>
static void launch_beams(const BeamParams& p, hipStream_t s) {
  using Ch = Chunk<T, U>;
  const size_t lists = (size_t)p.K * p.chunks;
  const size_t lds = std::max({sizeof(typename Ch::Comp) * kWaves * 64 * Ch::E, lists * 12, (size_t)p.num * p.num * 12});
  hipLaunchKernelGGL((fa_beams_kernel<T, U>), dim3((unsigned)(p.B * p.K * p.chunks)), dim3(kThreads), lds, s, p);
}
template <typename T>
static void by_loads(const AcceptParams& p, int loads, hipStream_t s) {
  if (loads == 4) launch_accept<T, 4>(p, s);
  else if (loads == 2) launch_accept<T, 2>(p, s);
  else launch_accept<T, 1>(p, s);
}
template <typename T>
static void by_loads(const BeamParams& p, int loads, hipStream_t s) {
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
