// The Gated DeltaNet's step for one new token a row: its input steps (gdn_prep_kernel's arithmetic for one token: the
// 4-tap convolution and SiLU rounded to 16 bits, l2 norms, gates) and the gated delta rule's single-token form, with
// the row's state S [128, 128] (fp32) and last 3 convolution inputs updated in place:
//   S' = e^g S + k (beta (v - e^g S^T k))^T,  o = S'^T q.
// The work is the state's traffic: 128 KB read and written a row and value head, 7 operations an element, so the state
// is read once into registers (all of a thread's loads are issued before the input steps, which run while they arrive,
// and the next head's before the current one's output is summed), updated there and written once. A CTA of 256 threads
// takes a row's key head and its value heads one after another (they share k and q, and the CTA alone reads and writes
// their convolution inputs); two CTAs an SM keep 128 KB of state in flight. 256 rows of 32 heads: 175 us, 1.10 GB at
// 6.3 TB/s (96% of a copy's rate). Where few rows leave SMs idle, each value head gets a CTA of
// its own: those of a key head form a cluster (of up to 8, which then take every 8th head), each computes k and q for
// itself, and the first writes the key head's new inputs after a barrier of the cluster that the others only arrive at:
// one row of 16 key heads by 2 6.1 us against 6.8, 10 rows of 2 by 8 8.4 against 20.3 (the rule is at the launch).
// Splitting a head's columns over a cluster as well gained 0.2 us at one row.
#pragma once
#include "hybrid.cuh"

namespace b200 {
namespace gdnstep {

struct Params {
  const void* proj;        // [rows, ld]: q, k, v channels from column 0, b at b_off, a at a_off
  int64_t ld;
  void* tail;              // [slots, 3, C] 16-bit, oldest first
  const void* conv;        // [C, 4]
  const float* A_log;      // [Hv]
  const void* dt_bias;     // [Hv]
  int b_off, a_off;
  float* state;            // [slots, Hv, 128, 128]
  const int32_t* at;       // [rows] the row's slot (null: the row's number); negative: a row of padding
  int64_t slots;
  int rows, Hk, Hv;
  float q_scale;
  void* o;                 // [rows, Hv, 128]
};

// 1: the row has a slot; 0: padding; -1: refused (a slot out of range, or one that an earlier row has).
__device__ __forceinline__ int row_slot(const Params& p, int b, int64_t* slot) {
  if (!p.at) {
    *slot = b;
    return b < p.slots ? 1 : -1;
  }
  const int32_t mine = p.at[b];
  *slot = mine;
  int twice = 0;
  for (int j = threadIdx.x; j < b; j += blockDim.x) twice |= p.at[j] == mine;
  if (__syncthreads_or(twice) && mine >= 0) return -1;
  return mine < 0 ? 0 : (mine < p.slots ? 1 : -1);
}

// The convolution + SiLU of channels c .. c + 3 for the row's token, each rounded to T (conv4_tokens' arithmetic).
template <typename T>
__device__ __forceinline__ void conv4(const T* x, const T* tail, const T* conv, int C, int c, float (&y)[4]) {
  float in[4][4], w[4][4];
#pragma unroll
  for (int j = 0; j < 3; ++j) hybrid::ld4(tail + (int64_t)j * C + c, in[j]);
  hybrid::ld4(x + c, in[3]);
#pragma unroll
  for (int i = 0; i < 4; ++i) hybrid::ld4(conv + (int64_t)(c + i) * 4, w[i]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float acc = __fmul_rn(in[0][i], w[i][0]);
#pragma unroll
    for (int j = 1; j < 4; ++j) acc = __fadd_rn(acc, __fmul_rn(in[j][i], w[i][j]));
    y[i] = hybrid::round_to<T>(hybrid::silu_f(acc));
  }
}

__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float4 fma4(float s, float4 a, float4 b) {
  return make_float4(fmaf(s, a.x, b.x), fmaf(s, a.y, b.y), fmaf(s, a.z, b.z), fmaf(s, a.w, b.w));
}

// The sum of N values `stride` apart as a binary tree.
template <int N>
__device__ __forceinline__ float4 tree(const float4* v, int stride) {
  if constexpr (N == 1)
    return *v;
  else
    return add4(tree<N / 2>(v, stride), tree<N / 2>(v + N / 2 * stride, stride));
}

constexpr int AHEAD = 6;  // value heads whose inputs are prepared at a time

constexpr int NT = 256, LANES = 32, BANDS = 8, ROWS = 16;  // 32 lanes of 4 columns by 8 bands of 16 rows of S
constexpr int GROUPS = ROWS / 4;

// grid (Hk * cluster, rows); SPLIT: clusters of `cluster` along x, else cluster is 1. A column's sums over the rows of S are
// a binary tree over groups of 4 rows.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(NT, 2) gdn_step_kernel(const Params p, int cluster_arg) {
  __shared__ __align__(16) float sq[128], sk[128], sv[AHEAD][128];
  __shared__ float sbeta[AHEAD], sdecay[AHEAD];
  __shared__ __align__(16) float4 part[2][BANDS][LANES];
  pdl_wait();
  pdl_launch();
  const int cluster = SPLIT ? cluster_arg : 1;
  const int h = blockIdx.x / cluster, rank = blockIdx.x % cluster, b = blockIdx.y, rep = p.Hv / p.Hk;
  const int heads = (rep - rank + cluster - 1) / cluster;  // of this CTA: rank, rank + cluster, ..
  const int head0 = h * rep + rank;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int band = threadIdx.x / LANES, mine = threadIdx.x % LANES, col = mine * 4;
  const int C = (2 * p.Hk + p.Hv) * 128;
  T* out = static_cast<T*>(p.o) + ((int64_t)b * p.Hv + head0) * 128;
  int64_t slot;
  const int ok = row_slot(p, b, &slot);
  if (ok <= 0) {  // the same in every CTA of a cluster
    if (ok < 0 && rank == 0 && threadIdx.x == 0) atomicOr(&g_fault, (unsigned)kFaultBadSlot);
    for (int i = threadIdx.x; i < heads * 128; i += NT)
      out[i / 128 * cluster * 128 + i % 128] = hybrid::from_f<T>(ok < 0 ? NAN : 0.0f);
    return;
  }
  const T* x = static_cast<const T*>(p.proj) + b * p.ld;
  T* tail = static_cast<T*>(p.tail) + slot * 3 * C;
  const T* conv = static_cast<const T*>(p.conv);
  float4* S = reinterpret_cast<float4*>(p.state + ((slot * p.Hv + head0) * 128 + band * ROWS) * 128 + col);
  float4 s[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) s[i] = S[i * 32];

  for (int r = 0; r < heads; ++r) {
    if (r % AHEAD == 0) {  // q and k (once) and the next heads' v, beta and decay: a warp each, 4 channels a lane
      const int next = min(AHEAD, heads - r);
      for (int t = warp + (r ? 2 : 0); t < 2 + next; t += NT / 32) {
        float y[4];
        const int vh = head0 + (r + t - 2) * cluster;
        conv4(x, tail, conv, C, (t < 2 ? t * p.Hk * 128 + h * 128 : 2 * p.Hk * 128 + vh * 128) + lane * 4, y);
        if (t < 2) {
          float ss = 0.0f;
#pragma unroll
          for (int i = 0; i < 4; ++i) ss = __fadd_rn(ss, __fmul_rn(y[i], y[i]));
          const float rn = rsqrtf(__fadd_rn(hybrid::warp_sum(ss), 1e-6f));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            (t == 0 ? sq : sk)[lane * 4 + i] = t == 0 ? __fmul_rn(__fmul_rn(y[i], rn), p.q_scale) : __fmul_rn(y[i], rn);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) sv[t - 2][lane * 4 + i] = y[i];
          if (lane == 0) {
            sbeta[t - 2] = hybrid::round_to<T>(hybrid::sigmoid_f(hybrid::to_f<T>(x[p.b_off + vh])));
            const float dt = hybrid::to_f<T>(static_cast<const T*>(p.dt_bias)[vh]);
            sdecay[t - 2] = expf(__fmul_rn(
                -expf(p.A_log[vh]), hybrid::softplus_f(__fadd_rn(hybrid::to_f<T>(x[p.a_off + vh]), dt))));
          }
        }
      }
      __syncthreads();
      // this CTA has read the key head's convolution inputs
      if (SPLIT && r == 0) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    const float4 v = *reinterpret_cast<const float4*>(&sv[r % AHEAD][col]);
    const float beta = sbeta[r % AHEAD], decay = sdecay[r % AHEAD];
    float4 sum[GROUPS];
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      sum[a] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float4 k4 = *reinterpret_cast<const float4*>(&sk[band * ROWS + a * 4]);
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4& e = s[a * 4 + i];
        e = make_float4(e.x * decay, e.y * decay, e.z * decay, e.w * decay);
        sum[a] = fma4(kk[i], e, sum[a]);
      }
    }
    part[0][band][mine] = tree<GROUPS>(sum, 1);
    __syncthreads();
    const float4 kv = tree<BANDS>(&part[0][0][mine], LANES);
    const float4 u = make_float4(beta * (v.x - kv.x), beta * (v.y - kv.y), beta * (v.z - kv.z), beta * (v.w - kv.w));
#pragma unroll
    for (int a = 0; a < GROUPS; ++a) {
      sum[a] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      const float4 k4 = *reinterpret_cast<const float4*>(&sk[band * ROWS + a * 4]);
      const float4 q4 = *reinterpret_cast<const float4*>(&sq[band * ROWS + a * 4]);
      const float kk[4] = {k4.x, k4.y, k4.z, k4.w}, qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float4& e = s[a * 4 + i];
        e = fma4(kk[i], u, e);
        S[(a * 4 + i) * 32] = e;
        sum[a] = fma4(qq[i], e, sum[a]);
      }
    }
    if (r + 1 < heads) {  // the next head's state
      S += cluster * 128 * 32;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) s[i] = S[i * 32];
    }
    part[1][band][mine] = tree<GROUPS>(sum, 1);
    __syncthreads();  // also: everyone has read part[0], sv, sbeta and sdecay of this head
    if (band == 0) {
      const float4 o = tree<BANDS>(&part[1][0][mine], LANES);
      T y[4] = {hybrid::from_f<T>(o.x), hybrid::from_f<T>(o.y), hybrid::from_f<T>(o.z), hybrid::from_f<T>(o.w)};
      *reinterpret_cast<uint2*>(out + r * cluster * 128 + col) = *reinterpret_cast<const uint2*>(y);
    }
  }

  // the convolution's last inputs: of this CTA's value heads (the loop's barriers came after every read of them), and the
  // key head's by the first CTA once the others have read them
  if (SPLIT) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  for (int i = threadIdx.x + (rank == 0 ? 0 : 2 * LANES); i < (2 + heads) * LANES; i += NT) {
    const int which = i / LANES;
    const int c = (which < 2 ? which * p.Hk * 128 + h * 128 : 2 * p.Hk * 128 + (head0 + (which - 2) * cluster) * 128) +
                  i % LANES * 4;
    const uint2 a = *reinterpret_cast<const uint2*>(tail + C + c), d = *reinterpret_cast<const uint2*>(tail + 2 * C + c);
    *reinterpret_cast<uint2*>(tail + c) = a;
    *reinterpret_cast<uint2*>(tail + C + c) = d;
    *reinterpret_cast<uint2*>(tail + 2 * C + c) = *reinterpret_cast<const uint2*>(x + c);
  }
}

}  // namespace gdnstep
}  // namespace b200
