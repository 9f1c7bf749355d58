// The paged key / value cache: attention of one new token a row over it, new tokens' keys and values written into it,
// and pages copied within it.
//
// A cache's keys and values are two pools of pages, [pages, Hk, page size, D]; row b's position t lives in page
// table[b, t / page size] at offset t % page size. 8-bit pools hold e4m3 codes with one fp32 scale per token and head
// ([pages, Hk, page size]): a value is code * scale, scale = max(amax, 1e-12) / 448 of the D values (for D = 128 the
// block formats' 1 x 128 activation group).
#pragma once
#include "quant.cuh"

namespace b200 {
namespace paged {

// The larger value, NaN when either is NaN (fmaxf drops a NaN).
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen(uint8_t v) { return e4m3_to_float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }

struct AttendParams {
  const void* q;           // [rows, H, D], strides q_row, q_head elements
  int64_t q_row, q_head;
  const void* k;           // pools: element strides of a page, a head and a token
  const void* v;
  int64_t page_stride, head_stride, token_stride;
  const float* ks;         // scales (8-bit pools): strides of a page and a head, tokens contiguous
  const float* vs;
  int64_t s_page, s_head;
  int64_t pages;
  int page_size;
  const int32_t* table;    // [rows, width], row stride table_row
  int64_t table_row;
  int width;
  const int32_t* lengths;  // [rows]
  int rows, H, Hk;
  float scale;
  int window;              // 0: all; else the last `window` positions
  void* out;               // [rows, H, D]
};

// One new token's attention: o = sum_t p_t v_t / sum_t p_t, p_t = exp(scale q . k_t - max), over the row's positions
// first <= t < length. A CTA of 4 warps per (row, head); a warp takes every fourth position, a lane D / 32 dimensions,
// and keeps its running maximum, sum and weighted values in fp32; the warps' parts are joined in warp order.
template <typename TQ, typename TK, int D>
__global__ void __launch_bounds__(128) attend_simple_kernel(const AttendParams p) {
  pdl_wait();
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h = blockIdx.x, b = blockIdx.y, kvh = h / (p.H / p.Hk);
  const int64_t most = (int64_t)p.width * p.page_size;
  int n = max(p.lengths[b], 0);
  bool bad = n > most;
  if (bad) n = (int)most;
  const int first = p.window > 0 ? max(0, n - p.window) : 0;
  float q[E], o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = widen(static_cast<const TQ*>(p.q)[b * p.q_row + h * p.q_head + lane * E + e]);
    o[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int t = first + warp; t < n; t += 4) {
    const int page = p.table[b * p.table_row + t / p.page_size];
    if (page < 0 || page >= p.pages) {
      bad = true;
      continue;
    }
    const int off = t % p.page_size;
    const int64_t at = page * p.page_stride + kvh * p.head_stride + off * p.token_stride + lane * E;
    const int64_t sat = page * p.s_page + kvh * p.s_head + off;
    float z = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) z = fmaf(q[e], widen(static_cast<const TK*>(p.k)[at + e]), z);
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) z += __shfl_xor_sync(0xffffffffu, z, x);
    z *= p.scale;
    float sv = 1.0f;
    if (sizeof(TK) == 1) {
      z *= p.ks[sat];
      sv = p.vs[sat];
    }
    const float mn = max_nan(m, z), ref = mn == -INFINITY ? 0.0f : mn;
    const float a = expf(m - ref), w = expf(z - ref);
    l = l * a + w;
    m = mn;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * sv * widen(static_cast<const TK*>(p.v)[at + e]);
  }
  __shared__ float sm[4], sl[4], so[4][D];
  __shared__ int sbad;
  if (threadIdx.x == 0) sbad = 0;
  __syncthreads();
  if (bad) sbad = 1;
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) so[warp][lane * E + e] = o[e];
  __syncthreads();
  if (sbad && threadIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadPage);
  float top = -INFINITY;
  for (int w = 0; w < 4; ++w) top = max_nan(top, sm[w]);
  const float ref = top == -INFINITY ? 0.0f : top;
  for (int d = threadIdx.x; d < D; d += 128) {
    float total = 0.0f, acc = 0.0f;
    for (int w = 0; w < 4; ++w) {
      const float f = expf(sm[w] - ref);
      total += f * sl[w];
      acc += f * so[w][d];
    }
    float y = total == 0.0f ? 0.0f : acc / total;
    if (sbad) y = NAN;
    static_cast<TQ*>(p.out)[((int64_t)b * p.H + h) * D + d] = narrow<TQ>(y);
  }
  pdl_launch();
}

// ---------------------------------------------------------------------------------------------------------------
// New tokens into the pages: a warp per (row, token, head) of the keys and of the values, a lane D / 32 consecutive
// values. 16-bit pools take the values' bits; 8-bit pools their codes and the token's scale, by the activation
// quantiser's arithmetic (IEEE quotients, round to nearest even, saturation).
// ---------------------------------------------------------------------------------------------------------------
struct AppendParams {
  const void* src[2];      // keys, values: [rows, T, Hk, D], element strides below
  int64_t row[2], tok[2], head[2];
  void* pool[2];
  int64_t page_stride, head_stride, token_stride;
  float* scale[2];
  int64_t s_page, s_head;
  int64_t pages;
  int page_size;
  const int32_t* table;
  int64_t table_row;
  int width;
  const int32_t* start;    // [rows] the position of a row's token 0; negative: the row brings nothing
  const int32_t* count;    // [rows] tokens that a row brings (null: T)
  int rows, T, Hk;
};

template <int BYTES>
struct Vec;
template <>
struct Vec<2> { using type = uint16_t; };
template <>
struct Vec<4> { using type = uint32_t; };
template <>
struct Vec<8> { using type = uint2; };
template <>
struct Vec<16> { using type = uint4; };

template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  pdl_wait();
  constexpr int E = D / 32;
  using V = typename Vec<E * 2>::type;
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
  if (item < (int64_t)p.rows * p.T * p.Hk * 2) {  // warp-uniform
    const int which = (int)(item & 1);
    const int h = (int)((item >> 1) % p.Hk);
    const int64_t rt = (item >> 1) / p.Hk;
    const int t = (int)(rt % p.T), b = (int)(rt / p.T);
    const int start = p.start[b], count = p.count ? min(p.count[b], p.T) : p.T;
    if (start >= 0 && t < count) {
      const int64_t pos = (int64_t)start + t;
      const int64_t pi = pos / p.page_size;
      const int page = pi < p.width ? p.table[b * p.table_row + pi] : -1;
      if (page < 0 || page >= p.pages) {
        if (lane == 0) atomicOr(&g_fault, (unsigned)kFaultBadPage);
      } else {
        const int off = (int)(pos % p.page_size);
        const T* src = static_cast<const T*>(p.src[which]) + b * p.row[which] + t * p.tok[which] + h * p.head[which];
        const V raw = *reinterpret_cast<const V*>(src + lane * E);
        const int64_t at = page * p.page_stride + h * p.head_stride + off * p.token_stride + lane * E;
        if (!FP8) {
          *reinterpret_cast<V*>(static_cast<T*>(p.pool[which]) + at) = raw;
        } else {
          const T* x = reinterpret_cast<const T*>(&raw);
          float v[E], amax = 0.0f;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            v[e] = widen(x[e]);
            amax = max_nan(amax, fabsf(v[e]));
          }
#pragma unroll
          for (int o = 16; o >= 1; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float s = __fdiv_rn(max_nan(amax, 1e-12f), 448.0f);
          uint8_t c[E];
#pragma unroll
          for (int e = 0; e < E; ++e) c[e] = float_to_e4m3(__fdiv_rn(v[e], s));
          using W = typename std::conditional<E == 8, uint2, typename Vec<E == 8 ? 4 : E>::type>::type;
          *reinterpret_cast<W*>(static_cast<uint8_t*>(p.pool[which]) + at) = *reinterpret_cast<const W*>(c);
          if (lane == 0) p.scale[which][page * p.s_page + h * p.s_head + off] = s;
        }
      }
    }
  }
  pdl_launch();
}

// ---------------------------------------------------------------------------------------------------------------
// Pages copied within their pools: pool i holds layers[i] layers of pages, page_bytes[i] bytes each. The moves travel
// in the kernel's parameters (no device list to upload, none to outlive the call); the host has checked that no page
// is written twice or both read and written, so the order of the copies does not matter.
// ---------------------------------------------------------------------------------------------------------------
constexpr int kCopyPools = 8;

template <int N>
struct CopyParams {
  char* pool[kCopyPools];
  int64_t layer_bytes[kCopyPools], page_bytes[kCopyPools];
  int layers[kCopyPools];
  int n;
  int32_t src[N], dst[N];
};

// grid (move, layer, pool)
template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
  pdl_wait();
  const int pool = blockIdx.z;
  if ((int)blockIdx.y < p.layers[pool]) {
    const int64_t bytes = p.page_bytes[pool];
    char* base = p.pool[pool] + (int64_t)blockIdx.y * p.layer_bytes[pool];
    const char* s = base + p.src[blockIdx.x] * bytes;
    char* d = base + p.dst[blockIdx.x] * bytes;
    if (((reinterpret_cast<uintptr_t>(base) | (uintptr_t)bytes) & 15) == 0)
      for (int64_t i = threadIdx.x * 16; i < bytes; i += blockDim.x * 16)
        *reinterpret_cast<uint4*>(d + i) = *reinterpret_cast<const uint4*>(s + i);
    else
      for (int64_t i = threadIdx.x * 4; i < bytes; i += blockDim.x * 4)
        *reinterpret_cast<uint32_t*>(d + i) = *reinterpret_cast<const uint32_t*>(s + i);
  }
  pdl_launch();
}

}  // namespace paged
}  // namespace b200
