// 8-bit paged KV cache for gfx950: K and V rows quantised to e4m3 as they are
// written, and read back.
//
// A row is the head_dim values of one token and KV head. With amax the largest
// magnitude of its finite values, the row's scale is s = 2^(e - 127), the least
// power of two with amax <= 448 s (448 is e4m3's largest value), 1 <= e <= 254,
// and the codes are e4m3(x / s), rounded to nearest even. e4m3 is a floating
// format, so a power of two costs no precision against amax / 448 (the
// relative step is the same; the subnormal range moves by at most one
// binade), and in return x / s is exact, codes do not depend on how a division
// rounds, a scale is one byte, and code * s is exact in bf16 and fp32. Where
// 256 s does not fit the rows' own type (the topmost binade), codes are held to
// 240, so that what a row stands for always fits the type that it came from.
// Infinities and NaN become NaN (e4m3 has no infinity).
//
// Codes lie as the 16-bit caches do, [num_blocks, block_size, Hkv, D]; the
// exponents e in [num_blocks, Hkv, block_size, 2] (K's, then V's), so that the
// attention kernels read the scales of four consecutive keys of a head, K's and
// V's, in one 8-byte access.
//
// Both kernels move every byte once and are bound by HBM (launch latency for a
// decode step): lane groups of D / 8 rounded up to 8 or 16 lanes take one row
// of K and the same of V, 8 values a lane, so a row is one contiguous access.
#include "fa_common.hpp"

namespace lsfa {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight values of a row as fp32, from 16-bit or 32-bit storage.
__device__ __forceinline__ void load8(const __bf16* p, float (&x)[8]) {
  const bf16x8 v = __builtin_bit_cast(bf16x8, __builtin_nontemporal_load((const u32x4*)p));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
__device__ __forceinline__ void load8(const _Float16* p, float (&x)[8]) {
  const f16x8 v = __builtin_bit_cast(f16x8, __builtin_nontemporal_load((const u32x4*)p));
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const f32x4 a = __builtin_nontemporal_load((const f32x4*)p), b = __builtin_nontemporal_load((const f32x4*)(p + 4));
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
__device__ __forceinline__ void store8(__bf16* p, const float (&x)[8]) {
  bf16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (__bf16)x[i];
  *(bf16x8*)p = v;
}
__device__ __forceinline__ void store8(_Float16* p, const float (&x)[8]) {
  f16x8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (_Float16)x[i];
  *(f16x8*)p = v;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *(f32x4*)p = f32x4{x[0], x[1], x[2], x[3]};
  *(f32x4*)(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
}

// Scale exponent from which a row's codes stop at 240 (256 s passes the type's largest value).
template <typename T> constexpr int kTopScale = 247;
template <> constexpr int kTopScale<_Float16> = 135;

// Codes of the lane's 8 values of a row that LPR adjacent lanes hold; e: the row's exponent.
template <typename T, int LPR>
__device__ __forceinline__ u32x2 quantise_row(const float (&x)[8], int& e) {
  // Magnitudes compare as integers; 0x7f800000 and up are infinities and NaN.
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t m = __float_as_uint(x[i]) & 0x7fffffffu;
    top = max(top, m < 0x7f800000u ? m : 0u);
  }
#pragma unroll
  for (int o = 1; o < LPR; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  // amax = 2^(E - 127) * 1.f: 448 = 1.75 * 2^8 holds it at E - 8 where 1.f <= 1.75, else at E - 7.
  e = max((int)(top >> 23) - ((top & 0x7fffffu) > 0x600000u ? 7 : 8), 1);
  const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
  const float most = e >= kTopScale<T> ? 240.f : 448.f;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(x[i] * inv, -most), most);
    y[i] = (__float_as_uint(x[i]) & 0x7fffffffu) < 0x7f800000u ? c : __uint_as_float(0x7fc00000u);
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  return u32x2{(uint32_t)lo, (uint32_t)hi};
}

// The values that 8 codes under a row's exponent stand for.
__device__ __forceinline__ void dequantise8(u32x2 c, uint32_t e, float (&x)[8]) {
  const float s = __uint_as_float(e << 23);
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[w], true);
    x[4 * w] = a[0] * s;
    x[4 * w + 1] = a[1] * s;
    x[4 * w + 2] = b[0] * s;
    x[4 * w + 3] = b[1] * s;
  }
}

// Sequence of packed token t by its offsets cu [B + 1], which the workgroup
// holds in LDS up to kCuStaged sequences (a search in memory waits out its
// latency log2(B) times); B where t lies past the last.
constexpr int kCuStaged = 1024;
__device__ __forceinline__ void stage_offsets(const int32_t* cu, int B, int32_t* s_cu) {
  if (cu != nullptr && B <= kCuStaged) {
    for (int i = threadIdx.x; i <= B; i += blockDim.x) s_cu[i] = cu[i];
    __syncthreads();
  }
}
__device__ __forceinline__ int sequence_of(const int32_t* cu, int B, int t) {
  int lo = 0, hi = B;  // the first b with cu[b + 1] > t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid + 1] > t) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

// Cache block and slot of position pos of sequence b; -1 where there is none.
__device__ __forceinline__ int block_of(const KvCacheParams& p, int b, int pos, int& slot) {
  const int i = pos >> p.block_shift;
  slot = pos & ((1 << p.block_shift) - 1);
  if (pos < 0 || i >= p.max_blocks) return -1;
  const int blk = p.block_tables[(int64_t)b * p.sbt + i];
  return (unsigned)blk < (unsigned)p.num_blocks ? blk : -1;
}

// One row a lane group, read and written once past the caches' usual order (nontemporal):
// 32768 rows of 8 heads of 128 in bf16 48.4 us, 4.2 TB/s (51.0 without the hints; two
// or four rows a lane group, their loads together, 59 and 66; the 2-byte scales cost 2 of
// it). Eight rows of a decode step take 4.0, a launch's own time.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void fa_kv_append_kernel(const KvCacheParams p) {
  __shared__ int32_t s_cu[kCuStaged + 1];
  stage_offsets(p.cu, p.B, s_cu);
  const int c = threadIdx.x % LPR;
  const int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
  const int t = (int)(row / p.Hkv), h = (int)(row - (int64_t)t * p.Hkv);
  if (t >= p.tokens) return;
  int b = t, pos;
  if (p.cu != nullptr) {
    const int32_t* cu = p.B <= kCuStaged ? s_cu : p.cu;
    b = sequence_of(cu, p.B, t);
    if (b >= p.B || t < cu[b]) return;  // rows of no sequence
    pos = p.seq_lens[b] - (cu[b + 1] - t);
  } else {
    pos = p.seq_lens[b] - 1;
  }
  int slot;
  const int blk = block_of(p, b, pos, slot);
  if (blk < 0) return;  // alike for the lanes of a row
  const bool has = 8 * c < p.D;
  float k[8] = {}, v[8] = {};
  if (has) {
    load8((const T*)p.k + (int64_t)t * p.sk[0] + (int64_t)h * p.sk[1] + 8 * c, k);
    load8((const T*)p.v + (int64_t)t * p.sv[0] + (int64_t)h * p.sv[1] + 8 * c, v);
  }
  int ke, ve;
  const u32x2 kq = quantise_row<T, LPR>(k, ke), vq = quantise_row<T, LPR>(v, ve);
  if (has) {
    __builtin_nontemporal_store(kq, (u32x2*)(p.kc + (int64_t)blk * p.skc[0] + (int64_t)slot * p.skc[1] + (int64_t)h * p.skc[2] + 8 * c));
    __builtin_nontemporal_store(vq, (u32x2*)(p.vc + (int64_t)blk * p.svc[0] + (int64_t)slot * p.svc[1] + (int64_t)h * p.svc[2] + 8 * c));
  }
  if (c == 0)
    *(uint16_t*)(p.scales + ((((int64_t)blk * p.Hkv + h) << p.block_shift) + slot) * 2) = (uint16_t)(ke | ve << 8);
}

template <typename T, int LPR, int U>
__global__ __launch_bounds__(256) void fa_kv_read_kernel(const KvCacheParams p) {
  __shared__ int32_t s_cu[kCuStaged + 1];
  stage_offsets(p.cu, p.B, s_cu);
  const int32_t* cu = p.B <= kCuStaged ? s_cu : p.cu;
  const int c = threadIdx.x % LPR;
  if (8 * c >= p.D) return;
  int t[U], h[U], blk[U], slot[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = ((int64_t)blockIdx.x * U + u) * (256 / LPR) + threadIdx.x / LPR;
    t[u] = (int)(row / p.Hkv), h[u] = (int)(row - (int64_t)t[u] * p.Hkv);
    blk[u] = -1;
    if (t[u] >= p.tokens) continue;
    const int b = sequence_of(cu, p.B, t[u]);
    if (b < p.B && t[u] >= cu[b]) blk[u] = block_of(p, b, t[u] - cu[b], slot[u]);
  }
  u32x2 kq[U], vq[U];
  uint32_t e[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    kq[u] = vq[u] = u32x2{0, 0};  // rows that no sequence or cache block holds are zeros
    e[u] = 0;
    if (blk[u] < 0) continue;
    e[u] = *(const uint16_t*)(p.scales + ((((int64_t)blk[u] * p.Hkv + h[u]) << p.block_shift) + slot[u]) * 2);
    kq[u] = *(const u32x2*)(p.kc + (int64_t)blk[u] * p.skc[0] + (int64_t)slot[u] * p.skc[1] + (int64_t)h[u] * p.skc[2] + 8 * c);
    vq[u] = *(const u32x2*)(p.vc + (int64_t)blk[u] * p.svc[0] + (int64_t)slot[u] * p.svc[1] + (int64_t)h[u] * p.svc[2] + 8 * c);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (t[u] >= p.tokens) continue;
    float x[8];
    dequantise8(kq[u], e[u] & 255u, x);
    store8((T*)p.k + (int64_t)t[u] * p.sk[0] + (int64_t)h[u] * p.sk[1] + 8 * c, x);
    dequantise8(vq[u], e[u] >> 8, x);
    store8((T*)p.v + (int64_t)t[u] * p.sv[0] + (int64_t)h[u] * p.sv[1] + 8 * c, x);
  }
}

template <typename T, int LPR>
static void launch_kv(const KvCacheParams& p, bool append, hipStream_t s) {
  const int64_t threads = (int64_t)p.tokens * p.Hkv * LPR;
  const dim3 grid((unsigned)((threads + 255) / 256)), half((unsigned)((threads + 511) / 512));
  // Reads take two rows a lane group where that leaves 2048 workgroups, 8 a CU (37000 rows of 8
  // heads 46.5 -> 40.0 us, 5.7 TB/s); fewer rows spread over the GPU (4096: 7.0 and 7.1).
  if (append) hipLaunchKernelGGL((fa_kv_append_kernel<T, LPR>), grid, dim3(256), 0, s, p);
  else if (threads >= 2 * 256 * 2048) hipLaunchKernelGGL((fa_kv_read_kernel<T, LPR, 2>), half, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((fa_kv_read_kernel<T, LPR, 1>), grid, dim3(256), 0, s, p);
}
template <typename T>
static void dispatch_kv(const KvCacheParams& p, bool append, hipStream_t s) {
  if (p.D <= 64) launch_kv<T, 8>(p, append, s);
  else launch_kv<T, 16>(p, append, s);
}

// Host entry used by the C ABI layer (arguments already validated).
hipError_t kv_cache_move(const KvCacheParams& p, int dtype, bool append, hipStream_t s) {
  if (dtype == 0) dispatch_kv<float>(p, append, s);
  else if (dtype == 1) dispatch_kv<_Float16>(p, append, s);
  else dispatch_kv<__bf16>(p, append, s);
  return hipGetLastError();
}

}  // namespace lsfa
