// Attention of one new token a row over a paged key / value cache (the layout is paged.cuh's):
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  first <= t < length,
// for the G = H / Hk query heads that share a key / value head. Every key and value is read once and used for up to 16 of
// them (8 at D = 256); more heads are groups of that many, each an item of its own that reads them again. 4 G D
// operations on 4 D bytes (16-bit), so up to G of about 16 the bound is the cache's bytes, and the kernel is built to keep
// enough of them in flight (96 KB an SM).
//
// Work. A row's positions are cut into tiles of 16 or 32 and the tiles into items (tiles_per_item: by the row's own length,
// so a row's sums are in the same order, and its bits the same, whatever else the call holds). A persistent CTA (of 4
// warps) takes every gridDim-th (row, item, key / value head); the warps take an item's tiles in turn. Each warp streams
// its tiles' keys and values through a ring of shared-memory stages of its own with cp.async, and the ring runs on
// across items: the warp that reads lengths, tables and the next item's first tiles is the one that computes the
// current ones, and no warp waits for another but where they join an item's result. An item that is a whole row is
// written at once; parts of longer rows go to the workspace and attend_join_kernel adds them up. Measured: 64 rows of up
// to 8192 (16 heads over 4 of 128, 543 MB) 94 us, 88% of a copy's rate, waiting for memory; 8-bit pages, 128 rows of up to
// 4001 (32 over 8, 541 MB) 112 us, 74%, by the latency of the warps' own chains (11.6 warps an SM, half of the issue slots
// and 38% of the ALU pipe in use); one row of 200 6.6 us, a warp's 1700 instructions one after another at 6.8 cycles each (of
// them 1.9 fixed latencies, 1.6 global memory, 0.9 shared memory, 0.9 instruction fetches).
//
// Arithmetic, per 16 tokens: S^T [16 tokens x 8 heads] = K Q^T and O^T [D x 8 heads] += V^T P^T on mma.sync m16n8k16 with
// fp32 accumulators (8 heads fill the n side; tcgen05 would want 64 rows or more of a tile that has G). 16-bit pages
// reach the MMA by ldmatrix (V transposed). 8-bit pages: codes become fp16 exactly; the products of a dot product may
// be taken in any order, so the k index of a step stands for the dimensions whose bytes a lane holds, the same for K
// and Q, and V's pairs of tokens are put together by byte permutes. P^T is moved into place by movmatrix, and split into
// two 16-bit values where one would show beside the output's own rounding (p = hi + lo: 2^-17 of p lost in bf16, 2^-22 in
// fp16 while p is within 2^-16 of the largest).
// Weights are 2^(z - ref) with z the logit times log2 e and ref a maximum that is raised only when some z passes it by
// more than 8 (2 for fp16 pages): a tile then costs one vote instead of a maximum across lanes and a rescaling of the sums,
// and the largest weight is 2^-8 to 1 (2^13 to 2^15), which changes no relative error (sums and outputs are fp32). An 8-bit
// key's scale multiplies its logit, a value's scale its weight; the query and those products are brought to fp16 by powers of
// two of their own, the head's largest query value and the largest product of a weight and a scale that it has seen
// (over_top), so that neither the largest nor what counts beside it leaves fp16's range: a product is off by its rounding
// (2^-11 under a bf16 output, 2^-22 split in two) or, below 2^-18 of the largest, by 2^-29 of the largest. Following the
// products costs 5 us of the 112; splitting them under bf16 outputs too would cost 20.
#pragma once
#include "paged.cuh"

namespace b200 {
namespace paged {

constexpr int MAX_PARTS = 256;  // items of one row and head, at most (the threads of attend_join_kernel)
constexpr int SMS = 148;        // of a B200; part of the rule below, so that it is the same wherever it runs

// Positions a tile: what a warp loads and computes at a time. 32 where a token's head is small (about 8 KB of keys and
// values a tile), with two independent halves in the computation; one m tile of the MMA where it is not, and where 16
// heads take the registers.
__host__ __device__ constexpr int tile_of(bool fp8, int D, int NG) {
  return D * (fp8 ? 1 : 2) <= 128 && !(D == 128 && NG == 2) ? 32 : 16;
}
// CTAs an SM, as the registers and the ring's shared memory allow, and warps a CTA.
__host__ __device__ constexpr int ctas_of(int D, int NG) { return D == 256 ? 1 : NG == 2 ? 2 : 3; }
__host__ __device__ constexpr int warps_of(bool fp8, int D) { return fp8 && D == 256 ? 8 : 4; }
// Tiles of an item, at least. An item costs a warp about 450 instructions beside its tiles' 260 each, so it should hold
// several tiles a warp; but a row's items are what spreads it over the SMs, and more parts are more to join. 256
// positions of 128 16-bit values (128 KB of keys and values), in proportion for others; more where an item costs more.
__host__ __device__ constexpr int item_tiles(bool fp8, int D, int NG) {
  return (D == 256 ? 512 * (fp8 ? 2 : 1) : 256 * 128 / D * (fp8 ? 2 : 1) * NG) / tile_of(fp8, D, NG);
}
// Parts that a row is cut into at most: its items then fill the resident CTAs once, so that a long row, alone or among a
// few, leaves none of them idle (of 1024 equal items 444 CTAs take 3 or 2 each: 65536 positions 34.4 us; cut into 111
// parts a head, 444 items, 30.7).
__host__ __device__ constexpr int parts_cap(int D, int NG, int units) {
  const int ctas = SMS * ctas_of(D, NG), n = ctas / units;
  return n < 1 ? 1 : n < MAX_PARTS ? n : MAX_PARTS;
}
__host__ __device__ __forceinline__ int tiles_per_item(int nt, int least, int cap) {
  const int c = (nt + cap - 1) / cap;
  return c < least ? least : c;
}
__host__ __device__ __forceinline__ int parts_of(int nt, int least, int cap) {
  const int c = tiles_per_item(nt, least, cap);
  return nt <= c ? 1 : (nt + c - 1) / c;
}
// Parts of any row of at most nt tiles.
__host__ __device__ __forceinline__ int most_parts(int64_t nt, int least, int cap) {
  const int64_t n = (nt + least - 1) / least;
  return n < 1 ? 1 : n < cap ? (int)n : cap;
}

// The query head that lane row r of an item's g-th eight heads reads: its own, or the item's first head, which is always
// there, where the item has no such head (the lane then drops what it read). An item has 1 to 8 NG heads, from head0.
__host__ __device__ constexpr int query_head(int head0, int heads, int g, int r) {
  return head0 + (g * 8 + r < heads ? g * 8 + r : 0);
}

struct Workspace {
  float* o;  // [rows, H, parts, D] sums of p v, relative to m
  float* m;  // [rows, H, parts] maximum, base 2; NaN: the row is refused
  float* l;  // [rows, H, parts] sum of p
  int parts; // the second-last dimension
  int cap;   // parts_cap
};

// A row's span of positions, from its length: n (clamped to the table), first, and whether it was too long.
__device__ __forceinline__ bool row_span(const AttendParams& p, int b, int* n, int* first) {
  const int len = p.lengths[b];
  const int most = p.width * p.page_size;  // <= 2^31 - 65, checked by the host
  const bool bad = len > most;
  *n = bad ? 0 : max(len, 0);
  *first = p.window > 0 ? max(0, *n - p.window) : 0;
  return bad;
}

template <int TT>
__device__ __forceinline__ int tiles_of(int n, int first) {
  return (n + TT - 1) / TT - first / TT;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ uint4 lds16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ float lds_f(uint32_t a) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}

// 2^x; -inf gives 0
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>  // the MMA's 16-bit type
struct Mma;
template <>
struct Mma<__nv_bfloat16> {
  static __device__ __forceinline__ void run(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u));
  }
};
template <>
struct Mma<__half> {
  static __device__ __forceinline__ void run(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  }
};

// Four 8 x 8 matrices of 16-bit values (lane l gives the address of row l % 8 of matrix l / 8); T: each transposed.
template <bool T>
__device__ __forceinline__ void ldmatrix4(uint32_t a, uint32_t (&v)[4]) {
  if (T)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}

// Four e4m3 codes as two pairs of fp16 values, exactly.
__device__ __forceinline__ void codes_f16(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(four));
}

// An 8 x 8 matrix of 16-bit values held by a warp (lane: row lane / 4, columns 2 (lane % 4) ..), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// The reference before any logit: finite, so that a difference with it is never NaN.
constexpr float NO_MAX = -3.0e38f;
// 8-bit values: a head's weights times their scales are handed to the MMA over a power of two near the largest such
// product that the head has seen, `top`: 2^4 to 2^5 is the largest one's size (below 2^15 for a scale of up to 2^10 times
// top, which is what is taken before top is raised: weights are below 1, the largest one 2^-8 or more). Only the product counts: a far larger scale under a weight
// that is next to nothing leaves the others what they are. top is kept from 2^-122 on, so that both powers exist.
constexpr float TOP_LEAST = 1.8807909613156600e-37f;  // 2^-122
__device__ __forceinline__ float over_top(float top) {  // 2^4 / 2^floor(log2 top)
  return __uint_as_float((258u << 23) - (__float_as_uint(top) & 0x7F800000u));
}
__device__ __forceinline__ float times_top(float top) {  // its inverse
  return __uint_as_float((__float_as_uint(top) & 0x7F800000u) - (4u << 23));
}

template <bool FP8, int D, int NG>
struct AttendShape {
  static constexpr int RB = D * (FP8 ? 1 : 2);          // bytes of a token's head
  static constexpr int CH = RB / 16;                    // 16-byte chunks of it
  static constexpr int TT = tile_of(FP8, D, NG);
  static constexpr int STAGE = 2 * TT * RB + (FP8 ? 2 * TT * 4 : 0);
  static constexpr int CTAS = ctas_of(D, NG), W = warps_of(FP8, D);
  static constexpr int JHEADS = NG == 2 ? 8 : 4;        // heads that the warps join at a time, as room allows
  static constexpr int JOIN = W * JHEADS * (D + 2) * 4;
  static constexpr int ROOM = (228 * 1024 / CTAS - 1024 - JOIN - 16) / W;  // a warp's share
  static constexpr int FIT = (ROOM - 32) / (STAGE + 32);
  static constexpr int STAGES = FIT < 6 ? FIT : 6;
  static constexpr int ITEMS = STAGES + 1;              // items that a warp may have begun to load
  static constexpr int RING = W * STAGES * STAGE;
  static constexpr int SMEM = RING + W * ITEMS * 32 + JOIN + 16;
  static_assert(STAGES >= 2 && SMEM <= 227 * 1024 && (SMEM + 1024) * CTAS <= 228 * 1024, "shared memory");

  // where a 16-byte chunk of token row `row` of a tile goes, so that the reads of a warp hit different banks
  static __host__ __device__ constexpr int k_chunk(int ch, int row) {
    return FP8 ? (CH >= 8 ? ch ^ ((row & 1) << 2) : ch) : ch ^ (row & 7);
  }
  static __host__ __device__ constexpr int v_chunk(int ch, int row) {
    return FP8 ? (CH >= 8 ? ch ^ (row & 6) : ch ^ ((row >> 1) & 3)) : ch ^ (row & 7);
  }
};

// An item as a warp's loading side leaves it for its computing side.
struct __align__(16) ItemInfo {
  int row, unit, part, parts;  // unit: key / value head * groups + group of heads; parts 0: there is no further item
  int n, first, tile, tile_end;  // the row's span, this warp's first tile (then every W-th) and the item's end
};

// The joins' state in shared memory, counted over the kernel's life: parts left by the warps, joins read by the warps that
// join, and whether a wait gave up. Waits are bounded (a caller that changes the lengths while the kernel reads them can
// make its warps disagree on the items): the kernel then records a fault bit, refuses the rows and ends.
struct JoinState {
  int left, read, gave_up;
};
__device__ __forceinline__ int load_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.cta.shared.s32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}
__device__ __forceinline__ void store_release(int* p, int v) {
  asm volatile("st.release.cta.shared.s32 [%0], %1;" ::"r"(smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ void add_release(int* p) {
  asm volatile("red.release.cta.shared.add.s32 [%0], 1;" ::"r"(smem_u32(p)) : "memory");
}
// Waits until *p >= want; false when this or another warp's wait gave up.
__device__ __forceinline__ bool wait_for(const int* p, int want, JoinState* js) {
  if (load_acquire(p) >= want) return true;
  const unsigned long long t0 = globaltimer();
  for (int n = 0;; ++n) {
    if (load_acquire(p) >= want) return true;
    if ((n & 255) == 255 && (load_acquire(&js->gave_up) || globaltimer() - t0 > kWaitLimitNs)) {
      store_release(&js->gave_up, 1);
      atomicOr(&g_fault, (unsigned)kFaultTimeoutEpilogue);
      return false;
    }
  }
}
// The same for a warp, whose lanes may have seen different answers: one for all of them.
__device__ __forceinline__ bool warp_wait(const int* p, int want, JoinState* js) {
  return __all_sync(0xffffffffu, wait_for(p, want, js));
}

// What a wait that gave up leaves behind: every row refused (NaN pairs `nan` in the output, NaN maxima of the parts), since
// it is not known which items its CTA has left. Lane `lane` of `lanes`.
__host__ __device__ inline void refuse_rows(uint32_t* out, int64_t pairs, uint32_t nan, float* m, int64_t parts, int lane,
                                            int lanes) {
  for (int64_t i = lane; i < pairs; i += lanes) out[i] = nan;
  for (int64_t i = lane; i < parts; i += lanes) m[i] = NAN;
}

template <typename TQ, bool FP8, int D, int NG>
__global__ void __launch_bounds__(warps_of(FP8, D) * 32, AttendShape<FP8, D, NG>::CTAS)
    attend_kernel(const AttendParams p, const Workspace ws, int groups, const Divide by_page, const Divide by_unit,
                  const Divide by_group, const Divide by_cap) {
  using Sh = AttendShape<FP8, D, NG>;
  using TM = typename std::conditional<FP8, __half, TQ>::type;
  using MM = Mma<TM>;
  constexpr int STAGES = Sh::STAGES, ITEMS = Sh::ITEMS, CH = Sh::CH, RB = Sh::RB, JHEADS = Sh::JHEADS;
  constexpr int W = Sh::W, TT = Sh::TT, SUB = TT / 16, LEAST = item_tiles(FP8, D, NG);
  // A weight in one 16-bit value is off by 2^-11 (fp16), which stays under a bf16 output's 2^-8 but not under an fp16
  // one's 2^-11, and by 2^-8 in bf16: those are split in two.
  constexpr bool SPLIT = !(FP8 && std::is_same<TQ, __nv_bfloat16>::value);
  // A head's reference is set LIFT below the largest logit and raised when one passes that by SLACK: weights reach
  // 2^(LIFT + SLACK), and the largest is at least 2^LIFT. They stay below 1, so that a sum of them times values near the
  // type's largest overflows only where the softmax's own terms would. Not so in fp16, whose smallest step is 2^-24 (and
  // whose values end at 2^16): the weights of a long row lie far below one token's that takes nearly all, so the largest is
  // put close to fp16's top: a weight down to 2^-27 of the largest keeps its 11 bits, a smaller one is held to 2^-38 of it.
  constexpr bool F16 = !FP8 && std::is_same<TQ, __half>::value;
  constexpr float LIFT = F16 ? 13.0f : -8.0f, SLACK = F16 ? 2.0f : 8.0f;
  constexpr int ROWS_STEP = 32 / CH;                 // token rows that one warp-wide load covers
  constexpr int JC = CH / 4 > 0 ? CH / 4 : 1;          // 8-bit: 16-byte chunks of a key that a lane feeds to the MMA
  constexpr int VB = RB / 8 < 16 ? RB / 8 : 16;      // 8-bit: bytes of a value load
  constexpr int NV = RB / 8 / VB;                    // of them a token
  constexpr int MT = D / 16;                         // m tiles of O^T
  constexpr int QW = D / 8;                          // query registers of 8 heads
  constexpr bool AHEAD = NG == 1 && D <= 128;        // registers left to load the next item's query early

  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3, r8 = lane & 7, mat = lane >> 3;
  const uint32_t ring = smem_u32(smem) + warp * STAGES * Sh::STAGE;
  ItemInfo* info = reinterpret_cast<ItemInfo*>(smem + Sh::RING) + warp * ITEMS;
  float* join_o = reinterpret_cast<float*>(smem + Sh::RING + W * ITEMS * 32);  // [warp][JHEADS][D]
  float* join_m = join_o + W * JHEADS * D;                                     // [warp][JHEADS]
  float* join_l = join_m + W * JHEADS;
  JoinState* js = reinterpret_cast<JoinState*>(join_l + W * JHEADS);
  if (threadIdx.x == 0) *js = {0, 0, 0};
  __syncthreads();

  pdl_wait();
  pdl_launch();  // every CTA is resident: what follows may take its place in the queue

  const int G = p.H / p.Hk;
  const int units = p.Hk * groups;

  // A lane's share of the query of an item's g-th eight heads: head g * 8 + r's, or zeros past the item's heads.
  auto load_q = [&](int row, int head0, int heads, int g, uint32_t (&w)[QW]) {
    const bool in = g * 8 + r < heads;
    const TQ* src = static_cast<const TQ*>(p.q) + row * p.q_row + query_head(head0, heads, g, r) * p.q_head;
    if constexpr (!FP8) {
#pragma unroll
      for (int j = 0; j < QW; ++j) {  // step j / 2: dimensions 8 j + 2c, 8 j + 2c + 1
        const uint32_t u = *reinterpret_cast<const uint32_t*>(src + j * 8 + 2 * c);
        w[j] = in ? u : 0u;
      }
    } else {
#pragma unroll
      for (int j = 0; j < QW / 4; ++j) {  // the dimensions of the 16 bytes of a key that the lane holds
        uint4 u = *reinterpret_cast<const uint4*>(src + ((j >> 1) * 4 + c) * 16 + (j & 1) * 8);
        if (!in) u = make_uint4(0, 0, 0, 0);
        w[j * 4] = u.x;
        w[j * 4 + 1] = u.y;
        w[j * 4 + 2] = u.z;
        w[j * 4 + 3] = u.w;
      }
    }
  };
  auto head0_of = [&](int unit, int* heads) {
    const int kvh = divide(unit, by_group), h0 = (unit - kvh * groups) * 8 * NG;
    *heads = min(8 * NG, G - h0);
    return kvh * G + h0;
  };

  // ---- the loading side: items in order, their tiles, one stage a call ----
  int64_t item = blockIdx.x, base = 0;
  int blk = -32, total = 0, incl = 0, row_n = 0, row_first = 0, row_parts = 0;
  bool row_bad = false;
  int begun = 0, it_row = 0, it_n = 0, it_first = 0, tile = 0, tile_end = 0;
  bool active = false, more = true;
  int page_at = 0, page_id = -1, page_lim = 0;  // page_id: table entry page_at + lane
  uint32_t qn[AHEAD ? QW : 1];
  int q_for = -1;

  constexpr int ES = FP8 ? 1 : 2;
  // a lane loads 16-byte chunk ch of token rows rr, rr + ROWS_STEP, ..
  const int ch = lane % CH, rr = lane / CH;
  const int64_t tok_bytes = p.token_stride * ES;
  const bool whole_subs = p.page_size % 16 == 0;    // 16 positions of a tile lie in one page
  const bool whole_pages = p.page_size % TT == 0;    // the tile does
  const char *kbase = nullptr, *vbase = nullptr;     // of the item's head
  const float* sbase = nullptr;                      // 8-bit: lanes 0 .. 15 keys' scales, 16 .. 31 values'

  auto next_item = [&](int done) {  // done: items that the computing side has begun
    while (item >= base + total) {
      base += total;
      blk += 32;
      if (blk >= p.rows) {
        more = false;
        if (lane == 0) info[begun % ITEMS].parts = 0;
        return;
      }
      const int b = blk + lane;
      row_n = row_first = row_parts = 0;
      row_bad = false;
      if (b < p.rows) {
        row_bad = row_span(p, b, &row_n, &row_first);
        row_parts = parts_of(tiles_of<TT>(row_n, row_first), LEAST, ws.cap);
      }
      incl = row_parts * units;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
      }
      total = __shfl_sync(0xffffffffu, incl, 31);
    }
    const int local = (int)(item - base);
    const int who = __popc(__ballot_sync(0xffffffffu, incl <= local));
    it_n = __shfl_sync(0xffffffffu, row_n, who);
    it_first = __shfl_sync(0xffffffffu, row_first, who);
    const int parts = __shfl_sync(0xffffffffu, row_parts, who);
    const bool bad = __shfl_sync(0xffffffffu, (int)row_bad, who);
    const int k = local - __shfl_sync(0xffffffffu, incl, who) + parts * units;
    const int part = divide(k, by_unit), unit = k - part * units;
    it_row = blk + who;
    const int nt = tiles_of<TT>(it_n, it_first), per = max(LEAST, divide(nt + ws.cap - 1, by_cap)), t0 = it_first / TT;
    tile = t0 + part * per + warp;
    tile_end = t0 + min(nt, (part + 1) * per);
    page_at = -64;
    page_lim = divide(it_n + p.page_size - 1, by_page);
    const int kvh = divide(unit, by_group);
    kbase = static_cast<const char*>(p.k) + kvh * p.head_stride * ES + ch * 16;
    vbase = static_cast<const char*>(p.v) + kvh * p.head_stride * ES + ch * 16;
    if (FP8) sbase = (lane < 16 ? p.ks : p.vs) + kvh * p.s_head;
    if (lane == 0) {
      int4* to = reinterpret_cast<int4*>(&info[begun % ITEMS]);
      to[0] = make_int4(it_row, unit, part, bad ? -parts : parts);  // negative: the row is refused
      to[1] = make_int4(it_n, it_first, tile, tile_end);
    }
    if constexpr (AHEAD) {
      if (q_for < done) {  // the query loaded early has been taken
        int heads;
        const int h0 = head0_of(unit, &heads);
        load_q(it_row, h0, heads, 0, qn);
        q_for = begun;
      }
    }
    ++begun;
    active = true;
    item += gridDim.x;
  };

  auto issue = [&](int slot, int done) {
    if (!active && more) next_item(done);
    if (active) {
      if (tile < tile_end) {
        const int pos0 = tile * TT;
        const uint32_t dst = ring + slot * Sh::STAGE;
        const int page_lo = divide(max(pos0, it_first), by_page);
        const int page_hi = whole_pages ? page_lo : divide(min(pos0 + TT, it_n) - 1, by_page);
        // the pages of the tile's positions: 32 table entries at a time, one a lane
        if (page_lo < page_at || page_hi >= page_at + 32) {
          page_at = page_lo;
          page_id = page_at + lane < page_lim ? p.table[it_row * p.table_row + page_at + lane] : -1;
        }
        int one = __shfl_sync(0xffffffffu, page_id, page_lo - page_at), at_page = page_lo;
        bool whole = whole_subs && pos0 >= it_first && pos0 + TT <= it_n && (uint32_t)one < (uint32_t)p.pages;
        if (SUB == 2 && whole && !whole_pages)
          whole = (uint32_t)__shfl_sync(0xffffffffu, page_id, page_hi - page_at) < (uint32_t)p.pages;
        if (whole) {
          // whole pages of 16 positions: rows a stride apart
#pragma unroll
          for (int s = 0; s < SUB; ++s) {
            if (s == 1 && !whole_pages) {  // the tile's second half may be in another page
              at_page = page_hi;
              one = __shfl_sync(0xffffffffu, page_id, page_hi - page_at);
            }
            const int off = pos0 + s * 16 - at_page * p.page_size;
            const int64_t at = one * p.page_stride * ES + (off + rr) * tok_bytes;
            const char *kp = kbase + at, *vp = vbase + at;
            const uint32_t to = dst + (s * 16 + rr) * RB;
            auto copy = [&](auto step) {
#pragma unroll
              for (int i = 0; i < 16 / ROWS_STEP; ++i) {
                const int row = i * ROWS_STEP + rr;
                cp_async16(to + i * ROWS_STEP * RB + (Sh::k_chunk(ch, row) << 4), kp + i * step);
                cp_async16(to + (TT + i * ROWS_STEP) * RB + (Sh::v_chunk(ch, row) << 4), vp + i * step);
              }
            };
            if (tok_bytes == RB)  // a head's tokens one after another: offsets known at compile time
              copy(std::integral_constant<int, ROWS_STEP * RB>{});
            else
              copy(tok_bytes * ROWS_STEP);
            if (FP8)  // lanes 0 .. 15 the keys', 16 .. 31 the values'
              cp_async4(dst + 2 * TT * RB + (s * 16 + (lane & 15) + (lane >> 4) * TT) * 4,
                        sbase + one * p.s_page + off + (lane & 15), true);
          }
        } else {
          // the row's ends, and pages that end elsewhere: each token's page on its own, zeros where there is none
          const int mine = pos0 + lane % TT;
          const bool live = mine >= it_first && mine < it_n;
          const int pi = live ? divide(mine, by_page) : page_lo;
          const int off = mine - pi * p.page_size;
          const int page = __shfl_sync(0xffffffffu, page_id, pi - page_at);
          const bool fine = live && page >= 0 && page < p.pages;
          if (__any_sync(0xffffffffu, live && !fine) && lane == 0) {
            int* parts = &info[(begun - 1) % ITEMS].parts;
            *parts = -abs(*parts);
          }
          const int64_t at = fine ? page * p.page_stride * ES + off * tok_bytes : -1;
          const int64_t sat = fine ? page * p.s_page + off : -1;
#pragma unroll 1
          for (int row = rr; row < TT; row += ROWS_STEP) {
            const int64_t a = __shfl_sync(0xffffffffu, at, row);
            const int64_t g = a >= 0 ? a : 0;
            cp_async16(dst + row * RB + (Sh::k_chunk(ch, row) << 4), kbase + g, a >= 0);
            cp_async16(dst + (TT + row) * RB + (Sh::v_chunk(ch, row) << 4), vbase + g, a >= 0);
          }
          if (FP8) {
#pragma unroll
            for (int s = 0; s < SUB; ++s) {
              const int64_t a = __shfl_sync(0xffffffffu, sat, s * 16 + (lane & 15));
              cp_async4(dst + 2 * TT * RB + (s * 16 + (lane & 15) + (lane >> 4) * TT) * 4, sbase + (a >= 0 ? a : 0),
                        a >= 0);
            }
          }
        }
      }
      tile += W;
      active = tile < tile_end;
    }
    cp_async_commit();
  };

  // ---- the computing side ----
  uint32_t q[NG][QW];
  float o[NG][MT][4], mx[NG][2], sum[NG][2], fac[NG][2];  // mx: the weights' reference, base 2
  float top_p[NG][2];                                     // 8-bit: the largest product of a weight and its value's scale
  int joined = 0;                                         // joins so far, the same in every warp
  bool alive = true;                                      // no wait has given up

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s, 0);
  int slot = 0;
  for (int now = 0; alive; ++now) {
    // the item's first stage (an empty one where this warp has no tile of it)
    issue(slot == 0 ? STAGES - 1 : slot - 1, now);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const ItemInfo* in = &info[now % ITEMS];
    if (in->parts == 0) break;
    const int row = in->row, unit = in->unit, n = in->n, first = in->first, end = in->tile_end;
    int tl = in->tile;
    int heads;
    const int head0 = head0_of(unit, &heads);

#pragma unroll
    for (int g = 0; g < NG; ++g) {
      uint32_t w[QW];
      bool have = false;
      if constexpr (AHEAD) {
        have = q_for == now;
        if (have) {
#pragma unroll
          for (int i = 0; i < QW; ++i) w[i] = qn[i];
        }
      }
      if (!have) load_q(row, head0, heads, g, w);
      float f = p.scale * 1.4426950408889634f;
      if constexpr (!FP8) {
#pragma unroll
        for (int i = 0; i < QW; ++i) q[g][i] = w[i];
        fac[g][0] = fac[g][1] = f;
      } else {
        // the head's query over a power of two near its largest value, in fp16 (what falls below fp16's smallest
        // values is under 2^-24 of the largest one)
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const float2 x = Mma<TQ>::unpack(w[i]);
          top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
        const float down = __uint_as_float((254u - e) << 23);
        f *= __uint_as_float(e << 23);
#pragma unroll
        for (int i = 0; i < QW; ++i) {
          const float2 x = Mma<TQ>::unpack(w[i]);
          q[g][i] = MM::pack(x.x * down, x.y * down);
        }
        fac[g][0] = __shfl_sync(0xffffffffu, f, c * 8);      // head 2c: lanes of row 2c
        fac[g][1] = __shfl_sync(0xffffffffu, f, c * 8 + 4);  // head 2c + 1
      }
      mx[g][0] = mx[g][1] = NO_MAX;
      top_p[g][0] = top_p[g][1] = TOP_LEAST;
      sum[g][0] = sum[g][1] = 0.0f;
#pragma unroll
      for (int t = 0; t < MT; ++t) o[g][t][0] = o[g][t][1] = o[g][t][2] = o[g][t][3] = 0.0f;
    }

    while (tl < end) {
      const int at = tl * TT;
      const uint32_t ks = ring + slot * Sh::STAGE, vs = ks + TT * RB;
      // per half u of the tile: two sums taken in turn (shorter chains of dependent MMAs)
      float s[SUB][NG][4], s2[SUB][NG][4];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[u][g][i] = s2[u][g][i] = 0.0f;
        if constexpr (!FP8) {
          const uint32_t a = (ks + (u * 16 + r8 + (mat & 1) * 8) * RB) + (((mat >> 1) ^ r8) << 4);
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            uint32_t k[4];
            ldmatrix4<false>(a ^ (j << 5), k);
#pragma unroll
            for (int g = 0; g < NG; ++g)
              MM::run(j & 1 ? s2[u][g] : s[u][g], k[0], k[1], k[2], k[3], q[g][2 * j], q[g][2 * j + 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < JC; ++j) {
            const int chunk = j * 4 + c;
            const uint4 a = lds16(ks + (u * 16 + r) * RB + (Sh::k_chunk(chunk, r) << 4)),
                        b = lds16(ks + (u * 16 + r + 8) * RB + (Sh::k_chunk(chunk, r) << 4));
            const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              uint32_t a0, a1, a2, a3;
              codes_f16(aw[w], a0, a2);
              codes_f16(bw[w], a1, a3);
#pragma unroll
              for (int g = 0; g < NG; ++g)
                MM::run(w & 1 ? s2[u][g] : s[u][g], a0, a1, a2, a3, q[g][j * 8 + 2 * w], q[g][j * 8 + 2 * w + 1]);
            }
          }
        }
      }
      // the logits, base 2: rows are tokens r and r + 8 of the half, columns heads 2c and 2c + 1
      float sk[SUB][2], sv[SUB][2], top_v = 0.0f;
      if (FP8) {
        const uint32_t sc = ks + 2 * TT * RB + r * 4;
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sk[u][i] = lds_f(sc + (u * 16 + i * 8) * 4);
            sv[u][i] = lds_f(sc + (TT + u * 16 + i * 8) * 4);
            top_v = fmaxf(top_v, fabsf(sv[u][i]));
          }
      }
      const bool edge = at < first || at + TT > n;
      float z[SUB][NG][4], hi[NG][2];
      bool up = false;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            z[u][g][i] = (s[u][g][i] + s2[u][g][i]) * fac[g][i & 1];
            if (FP8) z[u][g][i] *= sk[u][i >> 1];
          }
          if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int pos = at + u * 16 + r + (i < 2 ? 0 : 8);
              z[u][g][i] = pos >= first && pos < n ? z[u][g][i] : -INFINITY;
            }
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          hi[g][h] = fmaxf(z[0][g][h], z[0][g][h + 2]);
          if (SUB == 2) hi[g][h] = fmaxf(hi[g][h], fmaxf(z[SUB - 1][g][h], z[SUB - 1][g][h + 2]));
          up |= hi[g][h] > mx[g][h] + (LIFT + SLACK) || (FP8 && top_v > 1024.0f * top_p[g][h]);
        }
      }
      if (__any_sync(0xffffffffu, up)) {  // raise the references to what has been seen, and the sums with them
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float m = hi[g][h];
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            m = fmaxf(m - LIFT, mx[g][h]);
            float f = ex2(mx[g][h] - m);
            mx[g][h] = m;
            sum[g][h] *= f;
            if (FP8) {
              float t = 0.0f;
#pragma unroll
              for (int u = 0; u < SUB; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) t = fmaxf(t, ex2(z[u][g][h + 2 * i] - m) * fabsf(sv[u][i]));
#pragma unroll
              for (int x = 4; x <= 16; x <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, x));
              t = fmaxf(fmaxf(top_p[g][h] * f, t), TOP_LEAST);
              f = f * times_top(top_p[g][h]) * over_top(t);
              top_p[g][h] = t;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[g][i][h] *= f;
              o[g][i][h + 2] *= f;
            }
          }
      }
      uint32_t ph[SUB][NG][2], pl[SUB][NG][2];
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          float w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = ex2(z[u][g][i] - mx[g][i & 1]);
          sum[g][0] += w[0] + w[2];
          sum[g][1] += w[1] + w[3];
          if (FP8) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = w[i] * sv[u][i >> 1] * over_top(top_p[g][i & 1]);
          }
          const uint32_t h0 = MM::pack(w[0], w[1]), h1 = MM::pack(w[2], w[3]);
          ph[u][g][0] = transposed(h0);
          ph[u][g][1] = transposed(h1);
          if (SPLIT) {
            const float2 f0 = MM::unpack(h0), f1 = MM::unpack(h1);
            pl[u][g][0] = transposed(MM::pack(w[0] - f0.x, w[1] - f0.y));
            pl[u][g][1] = transposed(MM::pack(w[2] - f1.x, w[3] - f1.y));
          }
        }
      // O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        auto add = [&](int t, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            MM::run(o[g][t], a0, a1, a2, a3, ph[u][g][0], ph[u][g][1]);
            if (SPLIT) MM::run(o[g][t], a0, a1, a2, a3, pl[u][g][0], pl[u][g][1]);
          }
        };
        if constexpr (!FP8) {
          const uint32_t a = (vs + (u * 16 + r8 + (mat >> 1) * 8) * RB) + (((mat & 1) ^ r8) << 4);
#pragma unroll
          for (int j = 0; j < MT; ++j) {
            uint32_t v[4];
            ldmatrix4<true>(a ^ (j << 5), v);
            add(j, v[0], v[1], v[2], v[3]);
          }
        } else {
          // a lane takes piece i * 8 + r of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            uint32_t v[4][VB / 4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              const int tok = u * 16 + 2 * c + (t & 1) + (t >> 1) * 8;
              if constexpr (VB == 16) {
                const uint4 x = lds16(vs + tok * RB + (Sh::v_chunk(i * 8 + r, tok) << 4));
                v[t][0] = x.x;
                v[t][1] = x.y;
                v[t][2] = x.z;
                v[t][3] = x.w;
              } else {
                const uint2 x = lds8(vs + tok * RB + (Sh::v_chunk(r >> 1, tok) << 4) + (r & 1) * 8);
                v[t][0] = x.x;
                v[t][1] = x.y;
              }
            }
#pragma unroll
            for (int w = 0; w < VB / 4; ++w)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t sel = h ? 0x7362 : 0x5140;
                const uint32_t x = __byte_perm(v[0][w], v[1][w], sel), y = __byte_perm(v[2][w], v[3][w], sel);
                uint32_t a0, a1, a2, a3;
                codes_f16(x, a0, a1);
                codes_f16(y, a2, a3);
                add(i * (VB / 2) + w * 2 + h, a0, a1, a2, a3);
              }
          }
        }
      }
      tl += W;
      if (tl >= end) break;
      __syncwarp();  // the stage may be filled again
      slot = slot == STAGES - 1 ? 0 : slot + 1;
      issue(slot == 0 ? STAGES - 1 : slot - 1, now + 1);
      cp_async_wait<STAGES - 1>();
      __syncwarp();
    }

    // The four warps' parts of the item, JHEADS heads at a time. The warps take turns to join them, in warp order; the
    // others leave their parts and go on to the next item (they wait only where the last join still reads).
    const int parts = in->parts;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) sum[g][h] += __shfl_xor_sync(0xffffffffu, sum[g][h], x);
#pragma unroll
      for (int half = 0; half < 8 / JHEADS; ++half) {
        const int live = min(JHEADS, heads - g * 8 - half * JHEADS);
        if (live <= 0 || !alive) break;
        const int turn = joined % W;
        alive = warp_wait(&js->read, joined, js);  // the last join has been read
        if (!alive) break;
        if (JHEADS == 8 || c >> 1 == half) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float back = FP8 ? times_top(top_p[g][h]) : 1.0f;
            const int head = 2 * (c & (JHEADS / 2 - 1)) + h;
            if (r == 0) {
              join_m[warp * JHEADS + head] = parts < 0 ? NAN : mx[g][h];
              join_l[warp * JHEADS + head] = sum[g][h];
            }
            if (head < live) {
              float* to = join_o + (warp * JHEADS + head) * D;
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                // the rows r and r + 8 of m tile t; every two heads eight places aside: other banks
                const int d0 = FP8 ? (t / (VB / 2) * 8 + r) * VB + t % (VB / 2) * 2 : t * 16 + r;
                const int d1 = d0 + (FP8 ? 1 : 8);
                to[d0 ^ (head >> 1 << 3)] = o[g][t][h] * back;
                to[d1 ^ (head >> 1 << 3)] = o[g][t][h + 2] * back;
              }
            }
          }
        }
        ++joined;
        __syncwarp();
        if (lane == 0) add_release(&js->left);
        if (warp == turn) {
          alive = warp_wait(&js->left, joined * W, js);
          if (!alive) break;
#pragma unroll 2
          for (int e = lane; e < live * (D / 4); e += 32) {
            const int head = e / (D / 4), d = e % (D / 4) * 4;
            float f[W], top = join_m[head];
#pragma unroll
            for (int w = 1; w < W; ++w) top = max_nan(top, join_m[w * JHEADS + head]);
            float l = 0.0f;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; ++w) f[w] = ex2(join_m[w * JHEADS + head] - top);
#pragma unroll
            for (int w = 0; w < W; ++w) {
              const float4 v =
                  *reinterpret_cast<const float4*>(join_o + (w * JHEADS + head) * D + (d ^ (head >> 1 << 3)));
              l = fmaf(join_l[w * JHEADS + head], f[w], l);
              y.x = fmaf(v.x, f[w], y.x);
              y.y = fmaf(v.y, f[w], y.y);
              y.z = fmaf(v.z, f[w], y.z);
              y.w = fmaf(v.w, f[w], y.w);
            }
            const int64_t rh = (int64_t)row * p.H + head0 + g * 8 + half * JHEADS + head;
            if (abs(parts) == 1) {
              const float inv = l == 0.0f ? 0.0f : 1.0f / l;
              *reinterpret_cast<uint2*>(static_cast<TQ*>(p.out) + rh * D + d) =
                  make_uint2(Mma<TQ>::pack(y.x * inv, y.y * inv), Mma<TQ>::pack(y.z * inv, y.w * inv));
            } else {
              const int64_t at2 = rh * ws.parts + in->part;
              *reinterpret_cast<float4*>(ws.o + at2 * D + d) = y;
              if (d == 0) {
                ws.m[at2] = top;
                ws.l[at2] = l;
              }
            }
          }
          __syncwarp();
          if (lane == 0) store_release(&js->read, joined);
        }
      }
    }
    if (parts < 0 && lane == 0) atomicOr(&g_fault, (unsigned)kFaultBadPage);
    __syncwarp();  // the stage and the item's entry may be filled again
    slot = slot == STAGES - 1 ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  if (!alive)
    refuse_rows(static_cast<uint32_t*>(p.out), (int64_t)p.rows * p.H * (D / 2), Mma<TQ>::pack(NAN, NAN), ws.m,
                ws.m ? (int64_t)p.rows * p.H * ws.parts : 0, lane, 32);
}

// Joins the parts of a row and head that has several: grid (H, rows), 256 threads; D / 4 threads a part, 1024 / D parts
// at a time, added in a fixed order.
template <typename TQ, int D, int TT>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendParams p, const Workspace ws, int least) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float weight[MAX_PARTS], red[16];
  __shared__ float4 acc[GROUPS][LANES];
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y;
  int n, first;
  row_span(p, b, &n, &first);
  const int parts = parts_of(tiles_of<TT>(n, first), least, ws.cap);
  if (parts > 1) {
    const int64_t rh = (int64_t)b * p.H + h;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float m = (int)threadIdx.x < parts ? ws.m[rh * ws.parts + threadIdx.x] : NO_MAX;
    const float l = (int)threadIdx.x < parts ? ws.l[rh * ws.parts + threadIdx.x] : 0.0f;
    float top = m;
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, x));
    if (lane == 0) red[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = max_nan(top, red[w]);
    const float f = ex2(m - top);
    weight[threadIdx.x] = f;
    float total = f * l;
#pragma unroll
    for (int x = 16; x >= 1; x >>= 1) total += __shfl_xor_sync(0xffffffffu, total, x);
    if (lane == 0) red[8 + warp] = total;
    __syncthreads();
    total = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) total += red[8 + w];
    const int g = threadIdx.x / LANES, t = threadIdx.x % LANES;
    const float4* src = reinterpret_cast<const float4*>(ws.o + rh * ws.parts * D) + t;
    float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int i = g; i < parts; i += GROUPS) {
      const float4 v = src[(int64_t)i * LANES];
      const float w = weight[i];
      a.x = fmaf(w, v.x, a.x);
      a.y = fmaf(w, v.y, a.y);
      a.z = fmaf(w, v.z, a.z);
      a.w = fmaf(w, v.w, a.w);
    }
    acc[g][t] = a;
    __syncthreads();
    if (g == 0) {
#pragma unroll
      for (int i = 1; i < GROUPS; ++i) {
        const float4 v = acc[i][t];
        a.x += v.x;
        a.y += v.y;
        a.z += v.z;
        a.w += v.w;
      }
      const float inv = total == 0.0f ? 0.0f : 1.0f / total;
      const uint2 u = make_uint2(Mma<TQ>::pack(a.x * inv, a.y * inv), Mma<TQ>::pack(a.z * inv, a.w * inv));
      *reinterpret_cast<uint2*>(static_cast<TQ*>(p.out) + rh * D + t * 4) = u;
    }
  }
  pdl_launch();
}

}  // namespace paged
}  // namespace b200
