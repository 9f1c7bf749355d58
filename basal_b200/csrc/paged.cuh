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

// x / d for 0 <= x < 2^31 by a multiplication (Granlund and Montgomery 1994): shift = ceil(log2 d), mul =
// floor(2^32 (2^shift - d) / d) + 1, x / d = (mulhi(x, mul) + x) >> shift. Exact, and the sum stays below 2^32.
struct Divide {
  uint32_t mul, shift;
};
__device__ __forceinline__ int divide(int x, Divide d) {
  return (int)((__umulhi((uint32_t)x, d.mul) + (uint32_t)x) >> d.shift);
}

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

// ---------------------------------------------------------------------------------------------------------------
// New tokens into the pages: a CTA takes up to APPEND_TOKENS tokens of one row with all their heads, keys and values; where
// each token goes is looked up once. D / 8 lanes (D / 16 for 8-bit pages) take a token's head, its keys and its values.
// 16-bit pools take the values' bits; 8-bit pools their codes and the token's scale, by the activation quantiser's
// arithmetic (block_codes8: IEEE quotients, round to nearest even, saturation). 16 rows of up to 2048 tokens (4 heads of
// 128): bf16 18.6 us, 98 MB at 5.3 TB/s; 8-bit 23 us, bound by the quantiser's instructions (68% of the issue slots).
// ---------------------------------------------------------------------------------------------------------------
constexpr int APPEND_TOKENS = 16;

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

template <typename T>
struct Pair;
template <>
struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <>
struct Pair<__half> { using type = __half2; };

// grid (blocks of APPEND_TOKENS tokens, rows)
template <typename T, bool FP8, int D>
__global__ void __launch_bounds__(256, FP8 ? 5 : 1) append_kernel(const AppendParams p, const Divide by_head) {
  // 8-bit pages: 16 values a lane, so that a token's shuffles, quotient and reciprocal serve more of them, and the codes
  // are 16 bytes too
  constexpr int VALUES = FP8 ? 16 : 8, LANES = D / VALUES, UNROLL = FP8 ? 1 : 2, WORDS = VALUES / 8;
  __shared__ int64_t to[APPEND_TOKENS], scale_to[APPEND_TOKENS];  // element offsets of head 0; negative: nowhere
  pdl_wait();
  pdl_launch();
  const int b = blockIdx.y, t0 = blockIdx.x * APPEND_TOKENS;
  const int start = p.start[b];
  const int count = min(start < 0 ? 0 : p.count ? min(p.count[b], p.T) : p.T, t0 + APPEND_TOKENS) - t0;
  if (count <= 0) return;  // uniform
  if ((int)threadIdx.x < count) {
    const int64_t pos = (int64_t)start + t0 + threadIdx.x, pi = pos / p.page_size;
    const int off = (int)(pos - pi * p.page_size);
    const int page = pi < p.width ? p.table[b * p.table_row + pi] : -1;
    const bool fine = page >= 0 && page < p.pages;
    if (!fine) atomicOr(&g_fault, (unsigned)kFaultBadPage);
    to[threadIdx.x] = fine ? page * p.page_stride + off * p.token_stride : -1;
    scale_to[threadIdx.x] = page * p.s_page + off;
  }
  __syncthreads();
  const int l = threadIdx.x % LANES, items = count * p.Hk;  // item: a token's head, its keys and its values
  constexpr int STEP = 256 / LANES;
  const int rounds = (items + STEP * UNROLL - 1) / (STEP * UNROLL);  // the same for every thread: whole shuffles
  for (int round = 0; round < rounds; ++round) {
    uint4 raw[UNROLL][2][WORDS];
    int64_t at[UNROLL], sat[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = threadIdx.x / LANES + (round * UNROLL + u) * STEP;
      at[u] = -1;
#pragma unroll
      for (int j = 0; j < WORDS; ++j) raw[u][0][j] = raw[u][1][j] = make_uint4(0, 0, 0, 0);
      if (i < items) {
        const int t = divide(i, by_head), h = i - t * p.Hk;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(p.src[w]) + b * p.row[w] +
                                                            (t0 + t) * p.tok[w] + h * p.head[w] + l * VALUES);
#pragma unroll
          for (int j = 0; j < WORDS; ++j) raw[u][w][j] = src[j];
        }
        at[u] = to[t] < 0 ? -1 : to[t] + h * p.head_stride + l * VALUES;
        sat[u] = scale_to[t] + h * p.s_head;
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (!FP8) {
          if (at[u] >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.pool[w]) + at[u]) = raw[u][w][0];
        } else {
          using T2 = typename Pair<T>::type;
          T2 top = __habs2(reinterpret_cast<const T2*>(&raw[u][w][0])[0]);
#pragma unroll
          for (int j = 1; j < VALUES / 2; ++j)
            top = __hmax2_nan(top, __habs2(reinterpret_cast<const T2*>(&raw[u][w][0])[j]));
          float amax = max_nan(widen(top.x), widen(top.y));
#pragma unroll
          for (int o = LANES / 2; o >= 1; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          const float s = __fdiv_rn(max_nan(amax, 1e-12f), 448.0f);
          uint2 codes[2];
#pragma unroll
          for (int j = 0; j < WORDS; ++j) {
            const T* x = reinterpret_cast<const T*>(&raw[u][w][j]);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = widen(x[e]);
            codes[j] = block_codes8<false>(v, s);
          }
          if (at[u] >= 0) {
            *reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.pool[w]) + at[u]) =
                make_uint4(codes[0].x, codes[0].y, codes[1].x, codes[1].y);
            if (l == 0) p.scale[w][sat[u]] = s;
          }
        }
      }
    }
  }
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
  int chunks;  // CTAs of the largest page
  int32_t src[N], dst[N];
};

constexpr int COPY_BYTES = 16384;  // of a page, a CTA: four 16-byte loads a thread, all in flight

// grid (move * chunks + chunk, layer, pool)
template <int N>
__global__ void __launch_bounds__(256) copy_pages_kernel(const __grid_constant__ CopyParams<N> p) {
  pdl_wait();
  pdl_launch();
  const int pool = blockIdx.z, move = blockIdx.x / p.chunks, chunk = blockIdx.x - move * p.chunks;
  const int64_t bytes = p.page_bytes[pool], first = (int64_t)chunk * COPY_BYTES;
  if ((int)blockIdx.y >= p.layers[pool] || first >= bytes) return;
  char* base = p.pool[pool] + (int64_t)blockIdx.y * p.layer_bytes[pool];
  const char* s = base + p.src[move] * bytes + first;
  char* d = base + p.dst[move] * bytes + first;
  const int n = (int)min((int64_t)COPY_BYTES, bytes - first);
  if (((reinterpret_cast<uintptr_t>(base) | (uintptr_t)bytes) & 15) == 0) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (((int)threadIdx.x + u * 256) * 16 < n) v[u] = *reinterpret_cast<const uint4*>(s + (threadIdx.x + u * 256) * 16);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (((int)threadIdx.x + u * 256) * 16 < n) *reinterpret_cast<uint4*>(d + (threadIdx.x + u * 256) * 16) = v[u];
  } else {
    for (int i = threadIdx.x * 4; i < n; i += 256 * 4)
      *reinterpret_cast<uint32_t*>(d + i) = *reinterpret_cast<const uint32_t*>(s + i);
  }
}

}  // namespace paged
}  // namespace b200
