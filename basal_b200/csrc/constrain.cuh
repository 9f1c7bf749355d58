// A step's logits under penalties, biases and a grammar mask, in fp32:
//   z = logit; if the token occurs n > 0 times in the row's history: z = (z > 0 ? z / r : z r) - (f n + p);
//   z += the biases listed for the token; z = -inf where the mask's bit is 0.
// A CTA owns a slice of a row's vocabulary. It first streams the slice (-inf where the mask's bit is 0, without reading
// the logit; the logit elsewhere), which is all of the traffic, and then mends the few tokens that the history and the
// biases name: the history is short beside the vocabulary, so counting its tokens of the slice in shared memory (no
// counts are kept between steps) and rewriting those places costs less than a test at every token.
#pragma once
#include "quant.cuh"
#include "paged.cuh"

namespace b200 {
namespace constrain {

constexpr int NT = 512;         // threads
constexpr int HELD = 4;         // tokens of the history that a thread holds in registers
constexpr int SLICE = 16384;    // tokens of a slice at most (4 bytes of shared memory each)

struct Params {
  const void* logits;      // [rows, V], row stride ld
  int64_t ld;
  int rows, V;
  const uint32_t* mask;    // [rows or 1, ceil(V / 32)], row stride mask_row (0: shared); null: every token
  int64_t mask_row;
  const int32_t* past;     // [rows, T], row stride past_row; negative: nothing; null: no history
  int64_t past_row;
  int T;
  const float* repetition; // [rows], null: 1
  const float* presence;   // [rows], null: 0
  const float* frequency;  // [rows], null: 0
  const int32_t* ids;      // [rows, N], row stride bias_row; negative: nothing; null: no biases
  const float* values;
  int64_t bias_row;
  int N;
  float* out;              // [rows, V]
  int slice;               // tokens of a slice, a multiple of 32
};

template <typename T>
__device__ __forceinline__ float load_logit(const T* x) { return paged::widen(*x); }
__device__ __forceinline__ float load_logit(const float* x) { return *x; }

// 4 consecutive logits
template <typename T>
__device__ __forceinline__ float4 load4(const T* x) {
  const uint2 u = *reinterpret_cast<const uint2*>(x);
  const T* h = reinterpret_cast<const T*>(&u);
  return make_float4(paged::widen(h[0]), paged::widen(h[1]), paged::widen(h[2]), paged::widen(h[3]));
}
__device__ __forceinline__ float4 load4(const float* x) { return *reinterpret_cast<const float4*>(x); }

__device__ __forceinline__ bool allowed(const uint32_t* mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1); }

// grid (slice, row). VEC: rows of logits and of out start at multiples of 4 elements (8 or 16, and 16 bytes).
template <typename T, bool VEC>
__global__ void __launch_bounds__(NT) constrain_kernel(const Params p) {
  extern __shared__ int count[];
  pdl_wait();
  pdl_launch();
  const int b = blockIdx.y, v0 = blockIdx.x * p.slice, nv = min(p.slice, p.V - v0);
  const T* z = static_cast<const T*>(p.logits) + b * p.ld + v0;
  const uint32_t* mask = p.mask ? p.mask + b * p.mask_row + (v0 >> 5) : nullptr;
  float* out = p.out + (int64_t)b * p.V + v0;

  // the history's first tokens are asked for before the slice is streamed
  const int32_t* past = p.past + b * p.past_row;
  int ids[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) ids[k] = (int)threadIdx.x + k * NT < p.T ? past[threadIdx.x + k * NT] : -1;
  if (p.T > 0)
    for (int i = threadIdx.x; i < p.slice / 4; i += NT) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
  if constexpr (VEC) {
    constexpr int U = 4;  // loads in flight a thread
    int i = threadIdx.x * 4;
    for (; i + (U - 1) * NT * 4 + 4 <= nv; i += U * NT * 4) {
      uint32_t m[U];
      float4 x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int j = i + u * NT * 4;
        m[u] = mask ? mask[j >> 5] >> (j & 31) & 15u : 15u;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = m[u] ? load4(z + i + u * NT * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int u = 0; u < U; ++u)
        *reinterpret_cast<float4*>(out + i + u * NT * 4) =
            make_float4(m[u] & 1 ? x[u].x : -INFINITY, m[u] & 2 ? x[u].y : -INFINITY, m[u] & 4 ? x[u].z : -INFINITY,
                        m[u] & 8 ? x[u].w : -INFINITY);
    }
    for (; i < nv; i += NT * 4)
      for (int j = i; j < min(i + 4, nv); ++j) out[j] = allowed(mask, j) ? load_logit(z + j) : -INFINITY;
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += NT) out[i] = allowed(mask, i) ? load_logit(z + i) : -INFINITY;
  }

  if (p.T > 0) {
    auto tally = [&](int id) {
      if (id >= v0 && id - v0 < nv) atomicAdd(&count[id - v0], 1);
      if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
    };
    __syncthreads();
#pragma unroll
    for (int k = 0; k < HELD; ++k) tally(ids[k]);
    for (int i = threadIdx.x + HELD * NT; i < p.T; i += NT) tally(past[i]);
    __syncthreads();
    const float r = p.repetition ? p.repetition[b] : 1.0f, pr = p.presence ? p.presence[b] : 0.0f,
                f = p.frequency ? p.frequency[b] : 0.0f;
    auto mend = [&](int id) {
      const int v = id - v0;
      if (id >= v0 && v < nv && allowed(mask, v)) {
        const int n = atomicExch(&count[v], 0);  // whoever takes the count mends the place
        if (n > 0) {
          const float x = load_logit(z + v);
          out[v] = __fsub_rn(x > 0.0f ? __fdiv_rn(x, r) : __fmul_rn(x, r), __fadd_rn(__fmul_rn(f, (float)n), pr));
        }
      }
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) mend(ids[k]);
    for (int i = threadIdx.x + HELD * NT; i < p.T; i += NT) mend(past[i]);
  }
  if (p.N > 0) {
    __syncthreads();
    const int32_t* ids = p.ids + b * p.bias_row;
    for (int i = threadIdx.x; i < p.N; i += NT) {
      const int id = ids[i];
      if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
      if (id >= v0 && id - v0 < nv && allowed(mask, id - v0)) {
        // a token listed more than once gets its values in the list's order: the first of its places adds them all
        bool first = true;
        for (int j = 0; j < i; ++j) first &= ids[j] != id;
        if (first) {
          float y = out[id - v0];
          for (int j = i; j < p.N; ++j)
            if (ids[j] == id) y = __fadd_rn(y, p.values[b * p.bias_row + j]);
          out[id - v0] = y;
        }
      }
    }
  }
}

}  // namespace constrain
}  // namespace b200
