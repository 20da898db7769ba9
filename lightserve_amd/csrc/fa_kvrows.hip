// Rows of a paged KV cache moved inside it, for gfx950: what a step with several
// candidates per sequence leaves to be put in order. Rows are moved as bytes, in all
// layers by one launch; nothing is computed.
//
//   keep     row start + keep[i] of a sequence becomes its row start + i (keep[i] > i; others stay).
//            A thread has one column of a sequence's rows (16 or 4 bytes of one layer's K or V) and
//            goes through i upwards, some rows read, then written: what it overwrites lies at or below
//            every i that it has read, and what it still has to read above, so the move needs
//            neither a second buffer nor any wait between threads.
//   reorder  beam k of a sequence continues its beam parents[k]: the table entries of complete blocks
//            are the parent's, the rows of the last, incomplete block are copied into the beam's
//            own one. A thread reads its column of one row of that block for all beams before it
//            writes any, so that parents may be permuted at will.
//
// Both are bound by HBM (half of 2500..4001 rows of 7 sequences in 4 layers of 8 bits 37 us, a copy's rate; the last
// blocks of 8-bit beams, rows of 128 bytes, 117 us, 4.1 TB/s), or for few rows by the chain of their loads (index, table
// entry, row; 3.6 us in 32 layers).
#include "fa_common.hpp"

#include <algorithm>

namespace lsfa {

template <int BYTES> struct Column;
template <> struct Column<16> { using V = u32x4; };
template <> struct Column<4> { using V = uint32_t; };
template <> struct Column<2> { using V = uint16_t; };

// Where a lane's column of the rows of a cache is, and the cache's byte strides (a wave's lanes are all of K's, all of V's or
// all of the scales).
struct Place {
  char* base;
  int64_t block, slot;
};
// Groups of 64 columns (of BYTES bytes; K's and V's rows, then scales of 2 bytes a head) of a layer.
template <int BYTES>
__host__ __device__ __forceinline__ int row_groups(const KvRowsParams& p) { return (p.Hkv * (p.row_bytes / BYTES) + 63) / 64; }
__host__ __device__ __forceinline__ int scale_groups(const KvRowsParams& p) { return p.scales != nullptr ? (p.Hkv + 63) / 64 : 0; }
// The lane's column of a group. Lanes past the last column have that one too: they read and write what
// its own lane does, in the same instructions, and no row needs a branch for them.
template <int BYTES>
__device__ __forceinline__ Place place_of(const KvRowsParams& p, int layer, int group, int lane) {
  const int per = p.row_bytes / BYTES, groups = row_groups<BYTES>(p);
  const bool v = group >= groups;
  const int c = min((v ? group - groups : group) * 64 + lane, p.Hkv * per - 1), head = c / per;
  const int64_t* st = v ? p.sv : p.sk;
  return {(char*)(v ? p.v : p.k) + layer * st[0] + head * st[3] + (int64_t)(c - head * per) * BYTES, st[1], st[2]};
}
__device__ __forceinline__ Place scale_of(const KvRowsParams& p, int layer, int group, int lane) {
  const int head = min(group * 64 + lane, p.Hkv - 1);
  return {(char*)p.scales + layer * p.scale_layer + ((int64_t)head << (p.block_shift + 1)), (int64_t)p.Hkv << (p.block_shift + 1), 2};
}
// Byte offset of a sequence's row at a position; -1 where the cache has none.
__device__ __forceinline__ int slot_of(const KvRowsParams& p, const int32_t* table, int64_t pos, int& blk) {
  blk = -1;
  if (pos < 0 || pos >= (int64_t)p.max_blocks << p.block_shift) return 0;
  const int id = table[pos >> p.block_shift];
  if ((unsigned)id < (unsigned)p.num_blocks) blk = id;
  return (int)(pos & ((1 << p.block_shift) - 1));
}

// The waves of a workgroup that share a column group (W of them, this one is number w) take R rows each
// of W R at a time. Row i is read before any of them writes a row of the same W R, and what is read
// later lies above those.
template <int BYTES, int R, int W>
__device__ __forceinline__ void keep_rows(const KvRowsParams& p, int b, int w, const Place& at) {
  using V = typename Column<BYTES>::V;
  static_assert(R <= 64, "a lane finds one row's place");
  const int lane = threadIdx.x & 63;
  const int32_t* table = p.tables + (int64_t)b * p.sbt;
  const int32_t* keep = p.index + (int64_t)b * p.si;
  const int n = min(max(p.counts[b], 0), p.width);
  const int64_t start = (int64_t)p.seq_lens[b] - n;
  // Lane j: byte offsets of where row i0 + j of the sequence's kept ones comes from and goes to.
  int64_t from = 0, to = 0, next_from = 0, next_to = 0;
  bool moves = false, next_moves = false;
  auto find = [&](int i0, int64_t& f, int64_t& t, bool& m) {
    const int i = i0 + lane;
    m = false;
    if (lane >= R || i >= n) return;
    const int k = keep[i];
    if (k <= i) return;
    int fb, tb;
    const int fs = slot_of(p, table, start + k, fb), ts = slot_of(p, table, start + i, tb);
    m = fb >= 0 && tb >= 0;
    f = fb * at.block + fs * at.slot;
    t = tb * at.block + ts * at.slot;
  };
  find(w * R, from, to, moves);
  for (int i0 = 0; i0 < n; i0 += W * R) {
    const unsigned long long which = __ballot(moves);
    V v[R];
    auto address = [&](int64_t off, int j) -> char* {
      return at.base + ((int64_t)__builtin_amdgcn_readlane((int)(off >> 32), j) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)off, j));
    };
    // (all of them, as in the middle of a long list: without a branch for each row)
    const bool full = which == (R == 64 ? ~0ull : (1ull << (R & 63)) - 1);
    if (full) {
#pragma unroll
      for (int j = 0; j < R; ++j) v[j] = *(const V*)address(from, j);
    } else if (which != 0) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (which >> j & 1) v[j] = *(const V*)address(from, j);
    }
    if (i0 + W * R < n) find(i0 + W * R + w * R, next_from, next_to, next_moves);
    if (W > 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows are there
      __syncthreads();
    }
    if (full) {
#pragma unroll
      for (int j = 0; j < R; ++j) *(V*)address(to, j) = v[j];
    } else if (which != 0) {
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (which >> j & 1) *(V*)address(to, j) = v[j];
    }
    from = next_from, to = next_to, moves = next_moves;
  }
}

// Workgroups (column groups, NW / W each; layers; sequences).
template <int BYTES, int R, int NW, int W>
__global__ __launch_bounds__(NW * 64) void fa_kv_keep_kernel(const KvRowsParams p) {
  const int layer = blockIdx.y, b = blockIdx.z, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int group = blockIdx.x * (NW / W) + wave / W, rows = 2 * row_groups<BYTES>(p);
  if (group >= rows + scale_groups(p)) return;  // (all waves of the group)
  if (group < rows) keep_rows<BYTES, R, W>(p, b, wave % W, place_of<BYTES>(p, layer, group, lane));
  else keep_rows<2, R, W>(p, b, wave % W, scale_of(p, layer, group - rows, lane));
}

template <int BYTES, int KMAX>
__device__ __forceinline__ void reorder_row(const KvRowsParams& p, int b, int full, int row, const Place& at) {
  using V = typename Column<BYTES>::V;
  const int lane = threadIdx.x & 63;
  // Lane k: beam k's own block, and its parent's (itself where that is none of the sequence's beams).
  int own = -1, from = -1;
  if (lane < p.width) {
    const int64_t first = (int64_t)b * p.width;
    int parent = p.index[(int64_t)b * p.si + lane];
    if ((unsigned)parent >= (unsigned)p.width) parent = lane;
    if (parent != lane) {
      own = p.tables[(first + lane) * p.sbt + full];
      from = p.tables[(first + parent) * p.sbt + full];
    }
    if ((unsigned)own >= (unsigned)p.num_blocks || (unsigned)from >= (unsigned)p.num_blocks) own = from = -1;
  }
  const unsigned long long which = __ballot(own >= 0);
  V v[KMAX];
  char* to = at.base + row * at.slot;
#pragma unroll
  for (int k = 0; k < KMAX; ++k)
    if (which >> k & 1) v[k] = *(const V*)(to + (int64_t)__builtin_amdgcn_readlane(from, k) * at.block);
#pragma unroll
  for (int k = 0; k < KMAX; ++k)
    if (which >> k & 1) *(V*)(to + (int64_t)__builtin_amdgcn_readlane(own, k) * at.block) = v[k];
}

// Workgroups (x, y, z) = (columns of K and V, then scales; rows of a block for each layer; sequence), and
// behind the last layer's rows one that reorders the sequence's table.
template <int BYTES, int KMAX>
__global__ __launch_bounds__(256) void fa_kv_reorder_kernel(const KvRowsParams p) {
  const int b = blockIdx.z, rows = 1 << p.block_shift;
  const int64_t first = (int64_t)b * p.width;
  const int len = min(max(p.seq_lens[first], 0), (int)min((int64_t)p.max_blocks << p.block_shift, (int64_t)0x7fffffff));
  const int full = len >> p.block_shift;
  if ((int)blockIdx.y == p.layers * rows) {
    // Entry i of all beams is read before one is written.
    for (int i = blockIdx.x * 256 + threadIdx.x; i < full; i += gridDim.x * 256) {
      int e[KMAX];
#pragma unroll
      for (int k = 0; k < KMAX; ++k)
        if (k < p.width) {
          int parent = p.index[(int64_t)b * p.si + k];
          if ((unsigned)parent >= (unsigned)p.width) parent = k;
          e[k] = p.tables[(first + parent) * p.sbt + i];
        }
#pragma unroll
      for (int k = 0; k < KMAX; ++k)
        if (k < p.width) p.tables_out[(first + k) * p.sbt + i] = e[k];
    }
    return;
  }
  const int layer = blockIdx.y >> p.block_shift, row = blockIdx.y & (rows - 1);
  if (row >= (len & (rows - 1))) return;
  const int lane = threadIdx.x & 63, group = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), of_rows = 2 * row_groups<BYTES>(p);
  if (group >= of_rows + scale_groups(p)) return;
  if (group < of_rows) reorder_row<BYTES, KMAX>(p, b, full, row, place_of<BYTES>(p, layer, group, lane));
  else reorder_row<2, KMAX>(p, b, full, row, scale_of(p, layer, group - of_rows, lane));
}

// Host entries used by the C ABI layer (arguments validated there).
template <int BYTES>
static unsigned groups_of(const KvRowsParams& p) { return (unsigned)(2 * row_groups<BYTES>(p) + scale_groups(p)); }

template <int BYTES, int R, int NW, int W>
static void launch_keep(const KvRowsParams& p, hipStream_t s) {
  constexpr unsigned per = NW / W;
  hipLaunchKernelGGL((fa_kv_keep_kernel<BYTES, R, NW, W>), dim3((groups_of<BYTES>(p) + per - 1) / per, p.layers, p.B), dim3(NW * 64), 0, s, p);
}
// A wave by itself for few rows, or where the columns alone fill the chip; else 16 waves together, with 4-byte columns for long
// lists, so that there are four times as many workgroups. In this order, 8 heads of 128 in bf16 (us): 8 rows in 32 layers of
// 16 sequences 4.6, 15, 51, 256 rows 91, 105, 116, 700 rows 311, 334, 312; 64 rows in 32 layers of one 6.0, 4.3, 6.1; 700 rows
// in 4 layers of one 40, 11, 8.5; 3000 in 4 of seven 215, 78, 62, in 32 of four 367, 335, 328.
hipError_t kv_keep(const KvRowsParams& p, hipStream_t s) {
  if (p.width <= 32 || (long long)groups_of<16>(p) * p.layers * p.B >= 1024) launch_keep<16, 16, 4, 1>(p, s);
  else if (p.width <= 512) launch_keep<16, 16, 16, 16>(p, s);
  else launch_keep<4, 32, 16, 16>(p, s);
  return hipGetLastError();
}
template <int BYTES, int KMAX>
static void launch_reorder(const KvRowsParams& p, hipStream_t s) {
  const unsigned rows = (unsigned)p.layers << p.block_shift;
  hipLaunchKernelGGL((fa_kv_reorder_kernel<BYTES, KMAX>), dim3((groups_of<BYTES>(p) + 3) / 4, rows + 1, p.B), dim3(256), 0, s, p);
}
// More than 16 beams' rows of 16 bytes do not fit the registers; columns of 4 bytes take, for 4 beams in 32 layers, 13.7 us
// for 4.7, for 8 x 16 beams 71 for 49.
hipError_t kv_reorder(const KvRowsParams& p, hipStream_t s) {
  if (p.width <= 16) launch_reorder<16, 16>(p, s);
  else launch_reorder<4, 64>(p, s);
  return hipGetLastError();
}

}  // namespace lsfa
