// A step's logits under penalties, biases and a grammar mask, in fp32:
//   z = logit; if the token occurs n > 0 times in the row's history: z = (z > 0 ? z / r : z r) - (f n + p);
//   z += the biases listed for the token; z = -inf where the mask's bit is 0.
// A CTA owns a slice of a row's vocabulary. Streaming the slice (-inf where the mask's bit is 0, without reading the
// logit; the logit elsewhere) is all of the traffic; the history is short beside the vocabulary, so a few of the CTA's
// warps count its tokens of the slice in shared memory meanwhile (no counts are kept between steps), and the few places
// that the history and the biases name are rewritten afterwards, which costs less than a test at every token. 256 rows of
// 151,936 bf16 logits: 39.5 us without lists (233 MB, 5.9 TB/s), 42.4 with a mask, 56.7 with 2000 tokens of history and
// 64 biases too: what is left over the traffic is the latency of the passes after the stream, 3 CTAs an SM. Measured and
// not kept: counting before the stream (63 us), smaller slices with more CTAs (59), more loads in flight a thread (57).
#pragma once
#include "quant.cuh"
#include "paged.cuh"

namespace b200 {
namespace constrain {

constexpr int NT = 512;         // threads, three CTAs an SM
constexpr int HELD = 4;         // tokens of the history that a thread holds in registers
constexpr int U = 4;            // groups of 4 tokens in flight a thread
constexpr int COUNTERS = 128;   // threads that count while the others stream
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
  extern __shared__ uint32_t count[];        // of the slice's tokens in the history, two a word
  __shared__ uint32_t words[SLICE / 32 + 1]; // the slice's mask
  __shared__ int named[NT];                  // the biases' first NT tokens
  pdl_wait();
  pdl_launch();
  const int b = blockIdx.y, v0 = blockIdx.x * p.slice, nv = min(p.slice, p.V - v0), tid = threadIdx.x;
  const T* z = static_cast<const T*>(p.logits) + b * p.ld + v0;
  float* out = p.out + (int64_t)b * p.V + v0;
  const int32_t* past = p.past + b * p.past_row;
  const int32_t* ids = p.ids + b * p.bias_row;
  const float* values = p.values + b * p.bias_row;

  // Asked for at once: the slice's mask (read from HBM: its latency ahead of every batch of logits cost 10 us at 256 x
  // 151936), the history's first tokens, the biases' first ones.
  int held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k) held[k] = tid + k * NT < p.T ? past[tid + k * NT] : -1;
  const int bias_id = tid < p.N ? ids[tid] : -1;
  const float bias = tid < p.N ? values[tid] : 0.0f;
  named[tid] = bias_id;
  const uint32_t* mask = p.mask ? words : nullptr;
  if (p.mask) {
    const uint32_t* from = p.mask + b * p.mask_row + (v0 >> 5);
    for (int i = tid; i < (nv + 31) >> 5; i += NT) words[i] = from[i];
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    bool wrong = bias_id >= p.V;
#pragma unroll
    for (int k = 0; k < HELD; ++k) wrong |= held[k] >= p.V;
    if (wrong) atomicOr(&g_fault, (unsigned)kFaultBadId);
  }

  // The first COUNTERS threads count the history's tokens of the slice while the others stream it.
  const bool counting = p.T > 0 && tid < COUNTERS;
  if (counting) {
    for (int i = tid; i < p.slice / 8; i += COUNTERS) reinterpret_cast<int4*>(count)[i] = make_int4(0, 0, 0, 0);
    named_barrier(1, COUNTERS);
#pragma unroll 8
    for (int i = tid; i < p.T; i += COUNTERS) {
      const int id = past[i];
      if (id >= v0 && id - v0 < nv) atomicAdd(&count[(id - v0) >> 1], 1u << ((id - v0) & 1) * 16);
    }
  } else {
    // In groups of 4 from the first one whose stores are 16-byte aligned (rows of any V), where the logits' groups are
    // aligned too.
    const int rank = p.T > 0 ? tid - COUNTERS : tid, step = (p.T > 0 ? NT - COUNTERS : NT) * 4;
    const int head = min((int)(-(reinterpret_cast<intptr_t>(out) >> 2) & 3), nv);
    if (reinterpret_cast<uintptr_t>(z + head) % (4 * sizeof(T)) == 0) {
      if (rank < head) out[rank] = allowed(mask, rank) ? load_logit(z + rank) : -INFINITY;
      auto four = [&](int i) -> uint32_t {  // the mask's bits i .. i + 3
        if (!mask) return 15u;
        return __funnelshift_r(mask[i >> 5], mask[(i >> 5) + 1], i & 31) & 15u;
      };
      const int whole = head + (nv - head) / 4 * 4;  // the end of the last whole group
      for (int i = head + rank * 4; i < whole; i += U * step) {
        uint32_t m[U];
        Four<T> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) m[u] = i + u * step < whole ? four(i + u * step) : 0u;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          x[u].zero();
          if (m[u]) x[u].load(z + i + u * step);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (i + u * step < whole)
            *reinterpret_cast<float4*>(out + i + u * step) =
                make_float4(m[u] & 1 ? x[u].get(0) : -INFINITY, m[u] & 2 ? x[u].get(1) : -INFINITY,
                            m[u] & 4 ? x[u].get(2) : -INFINITY, m[u] & 8 ? x[u].get(3) : -INFINITY);
      }
      const int last = whole + rank;
      if (last < nv) out[last] = allowed(mask, last) ? load_logit(z + last) : -INFINITY;
    } else {
#pragma unroll 8
      for (int i = rank; i < nv; i += step / 4) out[i] = allowed(mask, i) ? load_logit(z + i) : -INFINITY;
    }
  }

  if (p.T > 0) {
    __syncthreads();
    const float rep = p.repetition ? p.repetition[b] : 1.0f, pr = p.presence ? p.presence[b] : 0.0f,
                fr = p.frequency ? p.frequency[b] : 0.0f;
    auto mend = [&](int id) {
      const int v = id - v0, at = (v & 1) * 16;
      if (id < v0 || v >= nv || !allowed(mask, v)) return;
      const int n = atomicAnd(&count[v >> 1], ~(0xFFFFu << at)) >> at & 0xFFFFu;  // whoever takes the count mends the place
      if (n == 0) return;
      const float x = load_logit(z + v);
      out[v] = __fsub_rn(x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep), __fadd_rn(__fmul_rn(fr, (float)n), pr));
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k) mend(held[k]);
    for (int i = tid + HELD * NT; i < p.T; i += NT) {
      if (past[i] >= p.V && blockIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadId);
      mend(past[i]);
    }
  }
  if (p.N > 0) {
    bool biased = bias_id >= v0 && bias_id - v0 < nv && allowed(mask, bias_id - v0), alone = p.N <= NT;
    if (biased)
      for (int j = 0; j < min(p.N, NT); ++j) alone &= named[j] != bias_id || j == tid;
    __syncthreads();
    if (biased && alone) {
      out[bias_id - v0] = __fadd_rn(out[bias_id - v0], bias);
      biased = false;
    }
    // the others: a token listed more than once gets its values in the list's order, the first of its places adds them all
    for (int i = tid; i < p.N; i += NT) {
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
