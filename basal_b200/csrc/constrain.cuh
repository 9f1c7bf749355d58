// A step's logits under penalties, biases and a grammar mask, in fp32:
//   z = logit; if the token occurs n > 0 times in the row's history: z = (z > 0 ? z / r : z r) - (f n + p);
//   z += the biases listed for the token; z = -inf where the mask's bit is 0.
// A token's occurrences are counted on the spot: a CTA owns a slice of the vocabulary and scans the row's history (a
// few KB, in L2) for the tokens of its slice, so no counts are kept between steps.
#pragma once
#include "quant.cuh"
#include "paged.cuh"

namespace b200 {
namespace constrain {

constexpr int SLICE = 2048;

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
};

template <typename T>
__device__ __forceinline__ float load_logit(const T* x) { return paged::widen(*x); }
__device__ __forceinline__ float load_logit(const float* x) { return *x; }

// grid (slice, row)
template <typename T>
__global__ void __launch_bounds__(256) constrain_kernel(const Params p) {
  pdl_wait();
  __shared__ int count[SLICE];
  __shared__ float bias[SLICE];
  const int b = blockIdx.y, v0 = blockIdx.x * SLICE, nv = min(SLICE, p.V - v0);
  for (int i = threadIdx.x; i < SLICE; i += blockDim.x) {
    count[i] = 0;
    bias[i] = 0.0f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < p.T; i += blockDim.x) {
    const int id = p.past[b * p.past_row + i];
    if (id >= v0 && id - v0 < nv) atomicAdd(&count[id - v0], 1);
    if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
  }
  // a token listed more than once gets its values in the list's order: the first of its places adds them all
  const int32_t* ids = p.ids + b * p.bias_row;
  for (int i = threadIdx.x; i < p.N; i += blockDim.x) {
    const int id = ids[i];
    if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
    if (id >= v0 && id - v0 < nv) {
      bool first = true;
      for (int j = 0; j < i; ++j) first &= ids[j] != id;
      if (first) {
        float s = 0.0f;
        for (int j = i; j < p.N; ++j)
          if (ids[j] == id) s = __fadd_rn(s, p.values[b * p.bias_row + j]);
        bias[id - v0] = s;
      }
    }
  }
  __syncthreads();
  const float r = p.repetition ? p.repetition[b] : 1.0f, pr = p.presence ? p.presence[b] : 0.0f,
              f = p.frequency ? p.frequency[b] : 0.0f;
  for (int i = threadIdx.x; i < nv; i += blockDim.x) {
    const int v = v0 + i;
    float z = -INFINITY;
    if (!p.mask || (p.mask[b * p.mask_row + (v >> 5)] >> (v & 31) & 1)) {
      z = load_logit(static_cast<const T*>(p.logits) + b * p.ld + v);
      const int n = count[i];
      if (n > 0)
        z = __fsub_rn(z > 0.0f ? __fdiv_rn(z, r) : __fmul_rn(z, r), __fadd_rn(__fmul_rn(f, (float)n), pr));
      z = __fadd_rn(z, bias[i]);
    }
    p.out[(int64_t)b * p.V + v] = z;
  }
  pdl_launch();
}

}  // namespace constrain
}  // namespace b200
