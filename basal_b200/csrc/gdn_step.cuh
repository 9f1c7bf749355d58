// The Gated DeltaNet's step for one new token a row: its input steps (gdn_prep_kernel's arithmetic for one token: the
// 4-tap convolution and SiLU rounded to 16 bits, l2 norms, gates) and the gated delta rule's single-token form, with
// the row's state S [128, 128] (fp32) and last 3 convolution inputs updated in place:
//   S' = e^g S + k (beta (v - e^g S^T k))^T,  o = S'^T q.
// The work is the state's traffic (128 KB read and written a row and value head, 7 operations an element).
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

// The convolution + SiLU of channel c for the row's token, rounded to T (conv4_tokens' arithmetic).
template <typename T>
__device__ __forceinline__ float conv_channel(const T* x, const T* tail, const T* conv, int C, int c) {
  using hybrid::to_f;
  float acc = __fmul_rn(to_f<T>(tail[c]), to_f<T>(conv[(int64_t)c * 4]));
  acc = __fadd_rn(acc, __fmul_rn(to_f<T>(tail[C + c]), to_f<T>(conv[(int64_t)c * 4 + 1])));
  acc = __fadd_rn(acc, __fmul_rn(to_f<T>(tail[2 * C + c]), to_f<T>(conv[(int64_t)c * 4 + 2])));
  acc = __fadd_rn(acc, __fmul_rn(to_f<T>(x[c]), to_f<T>(conv[(int64_t)c * 4 + 3])));
  return hybrid::round_to<T>(hybrid::silu_f(acc));
}

// A CTA of 128 threads per (key head, row), its value heads one after another; thread j owns column j of the state.
template <typename T>
__global__ void __launch_bounds__(128) gdn_step_kernel(const Params p) {
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y, j = threadIdx.x, rep = p.Hv / p.Hk;
  const int C = (2 * p.Hk + p.Hv) * 128;
  T* out = static_cast<T*>(p.o) + ((int64_t)b * p.Hv + h * rep) * 128;
  int64_t slot;
  const int ok = row_slot(p, b, &slot);
  if (ok <= 0) {
    if (ok < 0 && j == 0) atomicOr(&g_fault, (unsigned)kFaultBadSlot);
    for (int r = 0; r < rep; ++r) out[r * 128 + j] = hybrid::from_f<T>(ok < 0 ? NAN : 0.0f);
  } else {
    const T* x = static_cast<const T*>(p.proj) + b * p.ld;
    T* tail = static_cast<T*>(p.tail) + slot * 3 * C;
    const T* conv = static_cast<const T*>(p.conv);
    __shared__ float sq[128], sk[128], part[2][4];
    const int cq = h * 128 + j, ck = p.Hk * 128 + cq;
    const float yq = conv_channel(x, tail, conv, C, cq), yk = conv_channel(x, tail, conv, C, ck);
    const float ssq = hybrid::warp_sum(__fmul_rn(yq, yq)), ssk = hybrid::warp_sum(__fmul_rn(yk, yk));
    if ((j & 31) == 0) {
      part[0][j >> 5] = ssq;
      part[1][j >> 5] = ssk;
    }
    __syncthreads();
    const float nq = rsqrtf((part[0][0] + part[0][1]) + (part[0][2] + part[0][3]) + 1e-6f);
    const float nk = rsqrtf((part[1][0] + part[1][1]) + (part[1][2] + part[1][3]) + 1e-6f);
    sq[j] = __fmul_rn(__fmul_rn(yq, nq), p.q_scale);
    sk[j] = __fmul_rn(yk, nk);
    __syncthreads();
    for (int r = 0; r < rep; ++r) {
      const int vh = h * rep + r, cv = 2 * p.Hk * 128 + vh * 128 + j;
      const float v = conv_channel(x, tail, conv, C, cv);
      const float beta = hybrid::round_to<T>(hybrid::sigmoid_f(hybrid::to_f<T>(x[p.b_off + vh])));
      const float dt = hybrid::to_f<T>(static_cast<const T*>(p.dt_bias)[vh]);
      const float g = __fmul_rn(-expf(p.A_log[vh]),
                                hybrid::softplus_f(__fadd_rn(hybrid::to_f<T>(x[p.a_off + vh]), dt)));
      const float decay = expf(g);
      float* S = p.state + (slot * p.Hv + vh) * 16384 + j;
      float kv = 0.0f;
      for (int i = 0; i < 128; ++i) kv = fmaf(sk[i], decay * S[i * 128], kv);
      const float u = beta * (v - kv);
      float o = 0.0f;
      for (int i = 0; i < 128; ++i) {
        const float s = fmaf(sk[i], u, decay * S[i * 128]);
        S[i * 128] = s;
        o = fmaf(sq[i], s, o);
      }
      out[r * 128 + j] = hybrid::from_f<T>(o);
    }
    // the convolution's last inputs: every thread moves the channels that it alone read
    for (int r = 0; r < 2 + rep; ++r) {
      const int c = r == 0 ? cq : r == 1 ? ck : 2 * p.Hk * 128 + (h * rep + r - 2) * 128 + j;
      tail[c] = tail[C + c];
      tail[C + c] = tail[2 * C + c];
      tail[2 * C + c] = x[c];
    }
  }
  pdl_launch();
}

}  // namespace gdnstep
}  // namespace b200
