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

constexpr int NT = 512;         // threads, three CTAs an SM
constexpr int HELD = 4;         // tokens of the history that a thread holds in registers
constexpr int SLICE = 32768;    // tokens of a slice at most: 16-bit counts, 64 KB of shared memory
constexpr int MAX_PAST = 65535; // so that they hold

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

// 4 consecutive logits as they lie in memory, and in fp32
template <typename T>
struct Four {
  uint2 raw;
  __device__ __forceinline__ void load(const T* x) { raw = *reinterpret_cast<const uint2*>(x); }
  __device__ __forceinline__ void zero() { raw = make_uint2(0, 0); }
  __device__ __forceinline__ float get(int i) const { return paged::widen(reinterpret_cast<const T*>(&raw)[i]); }
};
template <>
struct Four<float> {
  float4 raw;
  __device__ __forceinline__ void load(const float* x) { raw = *reinterpret_cast<const float4*>(x); }
  __device__ __forceinline__ void zero() { raw = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
  __device__ __forceinline__ float get(int i) const { return reinterpret_cast<const float*>(&raw)[i]; }
};

__device__ __forceinline__ bool allowed(const uint32_t* mask, int v) { return !mask || (mask[v >> 5] >> (v & 31) & 1); }

// grid (slice, row)
template <typename T>
__global__ void __launch_bounds__(NT, 3) constrain_kernel(const Params p) {
  extern __shared__ uint32_t count[];  // two tokens a word
  pdl_wait();
  pdl_launch();
  const int b = blockIdx.y, v0 = blockIdx.x * p.slice, nv = min(p.slice, p.V - v0);
  const T* z = static_cast<const T*>(p.logits) + b * p.ld + v0;
  const uint32_t* mask = p.mask ? p.mask + b * p.mask_row + (v0 >> 5) : nullptr;
  float* out = p.out + (int64_t)b * p.V + v0;

  const int32_t* past = p.past + b * p.past_row;
  const int32_t* ids = p.ids + b * p.bias_row;
  const float* values = p.values + b * p.bias_row;
  // the biases' first NT places: this thread's token, whether it is of the slice and allowed, and who else names it
  __shared__ int named[NT];
  const int bias_id = (int)threadIdx.x < p.N ? ids[threadIdx.x] : -1;
  const float bias = (int)threadIdx.x < p.N ? values[threadIdx.x] : 0.0f;
  bool biased = bias_id >= v0 && bias_id - v0 < nv && allowed(mask, bias_id - v0), alone = p.N <= NT;
  if (p.N > 0) {
    if (bias_id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
    named[threadIdx.x] = bias_id;
    __syncthreads();
    if (biased)
      for (int j = 0; j < min(p.N, NT); ++j) alone &= named[j] != bias_id || j == (int)threadIdx.x;
  }

  // What the history makes of its tokens: counted before the slice is streamed, and for the first HELD * NT places the
  // new value too, so that only stores are left for afterwards.
  int held[HELD];
  float made[HELD];
  const float rep = p.T > 0 && p.repetition ? p.repetition[b] : 1.0f, pr = p.T > 0 && p.presence ? p.presence[b] : 0.0f,
              fr = p.T > 0 && p.frequency ? p.frequency[b] : 0.0f;
  auto take = [&](int id) {  // the token's count, given to one caller; 0 to the others and where there is nothing to do
    const int v = id - v0;
    if (id < v0 || v >= nv || !allowed(mask, v)) return 0;
    const int at = (v & 1) * 16;
    return (int)(atomicAnd(&count[v >> 1], ~(0xFFFFu << at)) >> at & 0xFFFFu);
  };
  auto penal = [&](int id, int n) {
    const float x = load_logit(z + id - v0);
    return __fsub_rn(x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep), __fadd_rn(__fmul_rn(fr, (float)n), pr));
  };
  if (p.T > 0) {
#pragma unroll
    for (int k = 0; k < HELD; ++k) held[k] = (int)threadIdx.x + k * NT < p.T ? past[threadIdx.x + k * NT] : -1;
    for (int i = threadIdx.x; i < p.slice / 8; i += NT) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    __syncthreads();
    auto tally = [&](int id) {
      if (id >= v0 && id - v0 < nv) atomicAdd(&count[(id - v0) >> 1], 1u << ((id - v0) & 1) * 16);
      if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) tally(held[k]);
    for (int i = threadIdx.x + HELD * NT; i < p.T; i += NT) tally(past[i]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < HELD; ++k) {
      const int n = take(held[k]);
      made[k] = n > 0 ? penal(held[k], n) : 0.0f;
      if (n <= 0) held[k] = -1;
    }
  }

  // The slice in groups of 4 from the first one whose stores are 16-byte aligned (rows of any V), where the logits'
  // groups are aligned too.
  const int head = min((int)(-(reinterpret_cast<intptr_t>(out) >> 2) & 3), nv);
  if (reinterpret_cast<uintptr_t>(z + head) % (4 * sizeof(T)) == 0) {
    constexpr int U = 4;  // loads in flight a thread
    if ((int)threadIdx.x < head)
      out[threadIdx.x] = allowed(mask, threadIdx.x) ? load_logit(z + threadIdx.x) : -INFINITY;
    auto four = [&](int i) -> uint32_t {  // the mask's bits i .. i + 3
      if (!mask) return 15u;
      const uint32_t lo = mask[i >> 5], hi = (i & 31) > 28 ? mask[(i >> 5) + 1] : 0u;
      return __funnelshift_r(lo, hi, i & 31) & 15u;
    };
    int i = head + threadIdx.x * 4;
    for (; i + (U - 1) * NT * 4 + 4 <= nv; i += U * NT * 4) {
      uint32_t m[U];
      Four<T> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) m[u] = four(i + u * NT * 4);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u].zero();
        if (m[u]) x[u].load(z + i + u * NT * 4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        *reinterpret_cast<float4*>(out + i + u * NT * 4) =
            make_float4(m[u] & 1 ? x[u].get(0) : -INFINITY, m[u] & 2 ? x[u].get(1) : -INFINITY,
                        m[u] & 4 ? x[u].get(2) : -INFINITY, m[u] & 8 ? x[u].get(3) : -INFINITY);
    }
    for (; i + 4 <= nv; i += NT * 4) {
      const uint32_t m = four(i);
      Four<T> x;
      x.zero();
      if (m) x.load(z + i);
      *reinterpret_cast<float4*>(out + i) = make_float4(m & 1 ? x.get(0) : -INFINITY, m & 2 ? x.get(1) : -INFINITY,
                                                        m & 4 ? x.get(2) : -INFINITY, m & 8 ? x.get(3) : -INFINITY);
    }
    for (int j = i; j < nv && j < i + 4; ++j) out[j] = allowed(mask, j) ? load_logit(z + j) : -INFINITY;
  } else {
#pragma unroll 8
    for (int i = threadIdx.x; i < nv; i += NT) out[i] = allowed(mask, i) ? load_logit(z + i) : -INFINITY;
  }

  if (p.T > 0) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (held[k] >= 0) out[held[k] - v0] = made[k];
    for (int i = threadIdx.x + HELD * NT; i < p.T; i += NT) {
      const int id = past[i], n = take(id);
      if (n > 0) out[id - v0] = penal(id, n);
    }
  }
  if (p.N > 0) {
    __syncthreads();
    if (biased && alone) {
      out[bias_id - v0] = __fadd_rn(out[bias_id - v0], bias);
      biased = false;
    }
    // the others: a token listed more than once gets its values in the list's order, the first of its places adds them all
    for (int i = threadIdx.x; i < p.N; i += NT) {
      const int id = i < NT ? bias_id : ids[i];
      if (i >= NT) {
        biased = id >= v0 && id - v0 < nv && allowed(mask, id - v0);
        if (id >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
      }
      if (biased) {
        bool first = true;
#pragma unroll 8
        for (int j = 0; j < i; ++j) first &= ids[j] != id;
        if (first) {
          float y = out[id - v0];
#pragma unroll 8
          for (int j = i; j < p.N; ++j)
            if (ids[j] == id) y = __fadd_rn(y, values[j]);
          out[id - v0] = y;
        }
      }
    }
  }
}

}  // namespace constrain
}  // namespace b200
