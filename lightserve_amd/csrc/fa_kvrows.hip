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
// Both are bound by HBM, or for few rows by the chain of their loads (index, table entry, row).
#include "fa_common.hpp"

#include <algorithm>

namespace lsfa {

template <int BYTES> struct Column;
template <> struct Column<16> { using V = u32x4; };
template <> struct Column<4> { using V = uint32_t; };
template <> struct Column<2> { using V = uint16_t; };

// A cache's byte strides and where its rows are.
struct Place {
  char* base;
  int64_t block, slot;
};
// Column `c` (of BYTES bytes) of the rows of a cache: K, V or, where c lies past both, the scales of a
// head (2 bytes). False past the last.
template <int BYTES>
__device__ __forceinline__ bool place_of(const KvRowsParams& p, int layer, int c, Place& at) {
  const int per = p.row_bytes / BYTES, columns = p.Hkv * per;
  const bool v = c >= columns;
  c -= v ? columns : 0;
  if (c >= columns) return false;
  const int head = c / per;
  const int64_t* st = v ? p.sv : p.sk;
  at.base = (char*)(v ? p.v : p.k) + layer * st[0] + head * st[3] + (int64_t)(c - head * per) * BYTES;
  at.block = st[1], at.slot = st[2];
  return true;
}
__device__ __forceinline__ bool scale_of(const KvRowsParams& p, int layer, int head, Place& at) {
  if (head >= p.Hkv) return false;
  at.base = (char*)p.scales + layer * p.scale_layer + ((int64_t)head << (p.block_shift + 1));
  at.block = (int64_t)p.Hkv << (p.block_shift + 1), at.slot = 2;
  return true;
}
// Byte offset of a sequence's row at a position; -1 where the cache has none.
__device__ __forceinline__ int slot_of(const KvRowsParams& p, const int32_t* table, int64_t pos, int& blk) {
  blk = -1;
  if (pos < 0 || pos >= (int64_t)p.max_blocks << p.block_shift) return 0;
  const int id = table[pos >> p.block_shift];
  if ((unsigned)id < (unsigned)p.num_blocks) blk = id;
  return (int)(pos & ((1 << p.block_shift) - 1));
}

template <int BYTES, int R>
__device__ __forceinline__ void keep_rows(const KvRowsParams& p, int b, bool has, const Place& at) {
  using V = typename Column<BYTES>::V;
  const int lane = threadIdx.x & 63;
  const int32_t* table = p.tables + (int64_t)b * p.sbt;
  const int32_t* keep = p.index + (int64_t)b * p.si;
  const int n = min(max(p.counts[b], 0), p.width);
  const int64_t start = (int64_t)p.seq_lens[b] - n;
  for (int i0 = 0; i0 < n; i0 += R) {
    // Lane j: where row i0 + j comes from and goes to (blocks -1: it stays where it is).
    int from_blk = -1, to_blk = -1, from_slot = 0, to_slot = 0;
    if (lane < R && i0 + lane < n) {
      const int k = keep[i0 + lane];
      if (k > i0 + lane) {
        from_slot = slot_of(p, table, start + k, from_blk);
        to_slot = slot_of(p, table, start + i0 + lane, to_blk);
      }
    }
    const bool moves = from_blk >= 0 && to_blk >= 0;
    const unsigned long long which = __ballot(moves);
    if (which == 0) continue;
    V v[R];
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (which >> j & 1) {
        const int64_t off = (int64_t)__builtin_amdgcn_readlane(from_blk, j) * at.block + (int64_t)__builtin_amdgcn_readlane(from_slot, j) * at.slot;
        if (has) v[j] = *(const V*)(at.base + off);
      }
#pragma unroll
    for (int j = 0; j < R; ++j)
      if (which >> j & 1) {
        const int64_t off = (int64_t)__builtin_amdgcn_readlane(to_blk, j) * at.block + (int64_t)__builtin_amdgcn_readlane(to_slot, j) * at.slot;
        if (has) *(V*)(at.base + off) = v[j];
      }
  }
}

// Workgroups of a layer and sequence: `groups` of 256 columns of K and V, then one for the scales.
template <int BYTES, int R>
__global__ __launch_bounds__(256) void fa_kv_keep_kernel(const KvRowsParams p, int groups) {
  const int layer = blockIdx.y, b = blockIdx.z;
  Place at = {nullptr, 0, 0};
  if ((int)blockIdx.x < groups) {
    const bool has = place_of<BYTES>(p, layer, blockIdx.x * 256 + threadIdx.x, at);
    keep_rows<BYTES, R>(p, b, has, at);
  } else {
    const bool has = scale_of(p, layer, (blockIdx.x - groups) * 256 + threadIdx.x, at);
    keep_rows<2, R>(p, b, has, at);
  }
}

template <int BYTES, int KMAX>
__device__ __forceinline__ void reorder_row(const KvRowsParams& p, int b, int full, int row, bool has, const Place& at) {
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
    if ((which >> k & 1) && has) v[k] = *(const V*)(to + (int64_t)__builtin_amdgcn_readlane(from, k) * at.block);
#pragma unroll
  for (int k = 0; k < KMAX; ++k)
    if ((which >> k & 1) && has) *(V*)(to + (int64_t)__builtin_amdgcn_readlane(own, k) * at.block) = v[k];
}

// Workgroups (x, y, z) = (columns of K and V, then scales; rows of a block for each layer; sequence), and
// behind the last layer's rows one that reorders the sequence's table.
template <int BYTES, int KMAX>
__global__ __launch_bounds__(256) void fa_kv_reorder_kernel(const KvRowsParams p, int groups) {
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
  Place at = {nullptr, 0, 0};
  if ((int)blockIdx.x < groups) {
    const bool has = place_of<BYTES>(p, layer, blockIdx.x * 256 + threadIdx.x, at);
    reorder_row<BYTES, KMAX>(p, b, full, row, has, at);
  } else {
    const bool has = scale_of(p, layer, (blockIdx.x - groups) * 256 + threadIdx.x, at);
    reorder_row<2, KMAX>(p, b, full, row, has, at);
  }
}

// Host entries used by the C ABI layer (arguments validated there).
template <int BYTES>
static int groups_of(const KvRowsParams& p) { return (2 * p.Hkv * (p.row_bytes / BYTES) + 255) / 256; }
static int scale_groups(const KvRowsParams& p) { return p.scales != nullptr ? (p.Hkv + 255) / 256 : 0; }

hipError_t kv_keep(const KvRowsParams& p, hipStream_t s) {
  if (p.width <= 32) {
    const int g = groups_of<16>(p);
    hipLaunchKernelGGL((fa_kv_keep_kernel<16, 16>), dim3(g + scale_groups(p), p.layers, p.B), dim3(256), 0, s, p, g);
  } else {
    const int g = groups_of<4>(p);
    hipLaunchKernelGGL((fa_kv_keep_kernel<4, 64>), dim3(g + scale_groups(p), p.layers, p.B), dim3(256), 0, s, p, g);
  }
  return hipGetLastError();
}
hipError_t kv_reorder(const KvRowsParams& p, hipStream_t s) {
  const unsigned rows = (unsigned)p.layers << p.block_shift;
  if (p.width <= 16) {
    const int g = groups_of<16>(p);
    hipLaunchKernelGGL((fa_kv_reorder_kernel<16, 16>), dim3(g + scale_groups(p), rows + 1, p.B), dim3(256), 0, s, p, g);
  } else {
    const int g = groups_of<4>(p);
    hipLaunchKernelGGL((fa_kv_reorder_kernel<4, 64>), dim3(g + scale_groups(p), rows + 1, p.B), dim3(256), 0, s, p, g);
  }
  return hipGetLastError();
}

}  // namespace lsfa
