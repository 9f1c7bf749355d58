// Attention of one new token a row over a paged key / value cache (the layout is paged.cuh's):
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - max),  first <= t < length,
// for the G = H / Hk query heads that share a key / value head. Every key and value is read once and used for G heads:
// 4 G D operations on 4 D bytes (16-bit), so up to G of about 16 the bound is the cache's bytes, and the kernel is
// built to keep enough of them in flight.
//
// Work. A row's positions are cut into tiles of 16 and the tiles into items (tiles_per_item: by the row's own length,
// so a row's sums are in the same order, and its bits the same, whatever else the call holds). A persistent CTA of 4
// warps takes every gridDim-th (row, item, key / value head); the warps take an item's tiles in turn. Each warp streams
// its tiles' keys and values through a ring of shared-memory stages of its own with cp.async, and the ring runs on
// across items: the warp that reads lengths, tables and the next item's first tiles is the one that computes the
// current ones, and no warp waits for another but where the four join an item's result. An item that is a whole row is
// written at once; parts of longer rows go to the workspace and attend_join_kernel adds them up.
//
// Arithmetic, per tile: S^T [16 tokens x 8 heads] = K Q^T and O^T [D x 8 heads] += V^T P^T on mma.sync m16n8k16 with
// fp32 accumulators (8 heads fill the n side; tcgen05 would want 64 rows or more of a tile that has G). 16-bit pages
// reach the MMA by ldmatrix (V transposed). 8-bit pages: codes become fp16 exactly; the products of a dot product may
// be taken in any order, so the k index of a step stands for the dimensions whose bytes a lane holds, the same for K
// and Q, and V's pairs of tokens are put together by byte permutes. P^T is moved into place by movmatrix, and split into
// two 16-bit values (p = hi + lo, 2^-17 of p lost), so the rounding of p does not show beside the output's own.
// Weights are 2^(z - ref) with z the logit times log2 e and ref a maximum that is raised only when some z passes it by
// more than 8: a tile then costs one vote instead of a maximum across lanes and a rescaling of the sums, and weights
// stay below 2^8, which changes no relative error (sums and outputs are fp32). An 8-bit key's scale multiplies its
// logit, a value's scale its weight, relative to a power of two that follows the largest scale seen; the query is
// brought to fp16 by a power of two of its own; so neither can leave fp16's range.
#pragma once
#include "paged.cuh"

namespace b200 {
namespace paged {

constexpr int TILE = 16;       // positions a tile
constexpr int AWARPS = 4;      // warps a CTA
constexpr int MAX_PARTS = 256; // items of one row and head, at most

// Tiles of an item for a row of nt tiles: 16 (256 positions, 4 tiles a warp), more where that would give a row more
// than 256 parts. Fewer positions an item spread a short row over more SMs but cost more parts to write and join.
__host__ __device__ __forceinline__ int tiles_per_item(int nt) {
  const int c = (nt + MAX_PARTS - 1) / MAX_PARTS;
  return c < 16 ? 16 : c;
}
__host__ __device__ __forceinline__ int parts_of(int nt) {
  const int c = tiles_per_item(nt);
  return nt <= c ? 1 : (nt + c - 1) / c;
}
// Parts of any row of at most nt tiles.
__host__ __device__ __forceinline__ int most_parts(int nt) {
  return nt <= 16 ? 1 : nt <= 16 * MAX_PARTS ? (nt + 15) / 16 : MAX_PARTS;
}

struct Workspace {
  float* o;  // [rows, H, parts, D] sums of p v, relative to m
  float* m;  // [rows, H, parts] maximum, base 2; NaN: the row is refused
  float* l;  // [rows, H, parts] sum of p
  int parts; // the second-last dimension
};

// x / d for 0 <= x < 2^31 by a multiplication (Granlund and Montgomery 1994): shift = ceil(log2 d), mul =
// floor(2^32 (2^shift - d) / d) + 1, x / d = (mulhi(x, mul) + x) >> shift. Exact, and the sum stays below 2^32.
struct Divide {
  uint32_t mul, shift;
};
__device__ __forceinline__ int divide(int x, Divide d) {
  return (int)((__umulhi((uint32_t)x, d.mul) + (uint32_t)x) >> d.shift);
}

// A row's span of positions, from its length: n (clamped to the table), first, and whether it was too long.
__device__ __forceinline__ bool row_span(const AttendParams& p, int b, int* n, int* first) {
  const int len = p.lengths[b];
  const int most = p.width * p.page_size;  // <= 2^31 - 65, checked by the host
  const bool bad = len > most;
  *n = bad ? 0 : max(len, 0);
  *first = p.window > 0 ? max(0, *n - p.window) : 0;
  return bad;
}

__device__ __forceinline__ int tiles_of(int n, int first) { return (n + TILE - 1) / TILE - first / TILE; }

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

// Two e4m3 codes (the low 16 bits) as two fp16 values, exactly.
__device__ __forceinline__ uint32_t codes_f16(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(two & 0xFFFFu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}

// An 8 x 8 matrix of 16-bit values held by a warp (lane: row lane / 4, columns 2 (lane % 4) ..), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

template <bool FP8, int D, int NG>
struct AttendShape {
  static constexpr int RB = D * (FP8 ? 1 : 2);          // bytes of a token's head
  static constexpr int CH = RB / 16;                    // 16-byte chunks of it
  static constexpr int STAGE = 2 * TILE * RB + (FP8 ? 2 * TILE * 4 : 0);
  // stages a warp: about 24 KB for each of 8 warps on an SM (two CTAs), 48 KB for each of 4 where D is 256
  static constexpr int STAGES = (D == 256 ? 49152 : 24576 + 512) / STAGE < 8 ? (D == 256 ? 49152 : 24576 + 512) / STAGE : 8;
  // where a 16-byte chunk of token row `row` of a tile goes, so that the reads of a warp hit different banks
  static __host__ __device__ constexpr int k_chunk(int ch, int row) {
    return FP8 ? (CH >= 8 ? ch ^ ((row & 1) << 2) : ch) : ch ^ (row & 7);
  }
  static __host__ __device__ constexpr int v_chunk(int ch, int row) {
    return FP8 ? (CH >= 8 ? ch ^ (row & 6) : ch ^ ((row >> 1) & 3)) : ch ^ (row & 7);
  }
  static constexpr int JOIN = AWARPS * 8 * (D + 2) * 4 + 16;  // the warps' parts of 8 heads
  static constexpr int RING = AWARPS * STAGES * STAGE;
  static constexpr int META = AWARPS * STAGES * 32;
  static constexpr int SMEM = RING + META + JOIN;
  static constexpr int PER_SM = SMEM <= 115712 ? 2 : 1;
};

// What a stage holds, written by lane 0 of its warp.
struct StageMeta {
  int row, unit, part;   // unit: key / value head * groups + group of heads
  int flags;             // kHas: the stage counts; kFirst, kLast tile of this warp in the item; kTile: it holds a tile
  int at, n, first;      // the tile's first position, and the row's span
  int parts;             // items of the row
};
// The reference before any logit: finite, so that a difference with it is never NaN.
constexpr float NO_MAX = -3.0e38f;
constexpr float SLACK = 8.0f;
enum { kHas = 1, kFirst = 2, kLast = 4, kTile = 8, kBad = 16 };

template <typename TQ, bool FP8, int D, int NG>
__global__ void __launch_bounds__(AWARPS * 32, AttendShape<FP8, D, NG>::PER_SM)
    attend_kernel(const AttendParams p, const Workspace ws, int groups, const Divide by_page,
                  const Divide by_unit) {
  using Sh = AttendShape<FP8, D, NG>;
  using TM = typename std::conditional<FP8, __half, TQ>::type;
  using MM = Mma<TM>;
  constexpr int STAGES = Sh::STAGES, CH = Sh::CH, RB = Sh::RB;
  constexpr int ROWS_STEP = 32 / CH;                 // token rows that one warp-wide load covers
  constexpr int JC = CH / 4;                         // 8-bit: 16-byte chunks of a key that a lane feeds to the MMA
  constexpr int VB = RB / 8 < 16 ? RB / 8 : 16;      // 8-bit: bytes of a value load
  constexpr int NV = RB / 8 / VB;                    // of them a token
  constexpr int MT = D / 16;                         // m tiles of O^T

  extern __shared__ __align__(1024) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = lane >> 2, c = lane & 3, r8 = lane & 7, mat = lane >> 3;
  uint8_t* ring = smem + warp * STAGES * Sh::STAGE;
  StageMeta* meta = reinterpret_cast<StageMeta*>(smem + Sh::RING) + warp * STAGES;
  float* join_o = reinterpret_cast<float*>(smem + Sh::RING + Sh::META);  // [warp][8][D]
  float* join_m = join_o + AWARPS * 8 * D;                               // [warp][8]
  float* join_l = join_m + AWARPS * 8;

  pdl_wait();
  pdl_launch();  // every CTA is resident: what follows may take its place in the queue

  const int G = p.H / p.Hk;
  const int units = p.Hk * groups;

  // ---- the loading side: items in order, their tiles, one stage a call ----
  int64_t item = blockIdx.x, base = 0;
  int blk = -32, total = 0, incl = 0, row_n = 0, row_first = 0, row_parts = 0;
  bool row_bad = false;
  int it_row = 0, it_unit = 0, it_part = 0, it_parts = 0, it_n = 0, it_first = 0, tile = 0, tile_end = 0;
  bool it_bad = false, active = false, fresh = false;
  int page_at = 0, page_id = -1, page_lim = 0;  // page_id: table entry page_at + lane

  constexpr int ES = FP8 ? 1 : 2;
  // a lane loads 16-byte chunk ch of token rows rr, rr + ROWS_STEP, ..
  const int ch = lane % CH, rr = lane / CH;
  const int64_t tok_bytes = p.token_stride * ES, step_bytes = tok_bytes * ROWS_STEP;
  const char* const kbase = static_cast<const char*>(p.k) + ch * 16;
  const char* const vbase = static_cast<const char*>(p.v) + ch * 16;
  const bool whole_pages = p.page_size % TILE == 0;  // a tile lies in one page
  int64_t head_bytes = 0, head_scales = 0;

  auto next_item = [&]() -> bool {
    while (item >= base + total) {
      base += total;
      blk += 32;
      if (blk >= p.rows) {
        total = 0;
        item = INT64_MAX;
        return false;
      }
      const int b = blk + lane;
      row_n = row_first = row_parts = 0;
      row_bad = false;
      if (b < p.rows) {
        row_bad = row_span(p, b, &row_n, &row_first);
        row_parts = parts_of(tiles_of(row_n, row_first));
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
    it_bad = __shfl_sync(0xffffffffu, (int)row_bad, who);
    const int before = who ? __shfl_sync(0xffffffffu, incl, who - 1) : 0;
    const int k = local - before;
    it_row = blk + who;
    it_part = divide(k, by_unit);
    it_unit = k - it_part * units;
    const int nt = tiles_of(it_n, it_first);
    it_parts = __shfl_sync(0xffffffffu, row_parts, who);
    const int per = tiles_per_item(nt), t0 = it_first / TILE;
    tile = t0 + it_part * per + warp;
    tile_end = t0 + min(nt, (it_part + 1) * per);
    page_at = -64;
    page_lim = divide(it_n + p.page_size - 1, by_page);
    head_bytes = (it_unit / groups) * p.head_stride * ES;
    head_scales = (it_unit / groups) * p.s_head;
    item += gridDim.x;
    return true;
  };

  auto issue = [&](int slot) {
    if (!active) {
      active = next_item();
      fresh = true;
    }
    StageMeta m;
    m.flags = 0;
    if (active) {
      const bool has = tile < tile_end;
      m.row = it_row;
      m.unit = it_unit;
      m.part = it_part;
      m.parts = it_parts;
      m.n = it_n;
      m.first = it_first;
      m.at = tile * TILE;
      m.flags = kHas | (fresh ? kFirst : 0) | (tile + AWARPS >= tile_end ? kLast : 0) | (has ? kTile : 0) |
                (it_bad ? kBad : 0);
      if (has) {
        const int pos0 = tile * TILE;
        const int lo_pos = max(pos0, it_first), hi_pos = min(pos0 + TILE, it_n) - 1;
        const int need_lo = divide(lo_pos, by_page), need_hi = whole_pages ? need_lo : divide(hi_pos, by_page);
        // the pages of the tile's positions: 32 table entries at a time, one a lane
        if (need_lo < page_at || need_hi >= page_at + 32) {
          page_at = need_lo;
          page_id = page_at + lane < page_lim ? p.table[it_row * p.table_row + page_at + lane] : -1;
        }
        const uint32_t dst = smem_u32(ring + slot * Sh::STAGE);
        const int one = __shfl_sync(0xffffffffu, page_id, need_lo - page_at);
        if (whole_pages && lo_pos == pos0 && hi_pos == pos0 + TILE - 1 && one >= 0 && one < p.pages) {
          // a whole tile in one page: the same copies with the rows a stride apart
          const int off = pos0 - need_lo * p.page_size;
          const int64_t at = one * p.page_stride * ES + head_bytes + (off + rr) * tok_bytes;
          const char *kp = kbase + at, *vp = vbase + at;
          const uint32_t to = dst + rr * RB;
          auto copy = [&](auto step) {
#pragma unroll
            for (int i = 0; i < TILE / ROWS_STEP; ++i) {
              const int row = i * ROWS_STEP + rr;
              cp_async16(to + i * ROWS_STEP * RB + (Sh::k_chunk(ch, row) << 4), kp + i * step);
              cp_async16(to + (TILE + i * ROWS_STEP) * RB + (Sh::v_chunk(ch, row) << 4), vp + i * step);
            }
          };
          if (tok_bytes == RB)  // a head's tokens one after another: offsets known at compile time
            copy(std::integral_constant<int, ROWS_STEP * RB>{});
          else
            copy(step_bytes);
          if (FP8) {
            const int64_t s = one * p.s_page + head_scales + off + (lane & 15);
            cp_async4(dst + 2 * TILE * RB + lane * 4, (lane < 16 ? p.ks : p.vs) + s, true);
          }
        } else {
          // the row's ends, and tiles that cross pages: each token's page on its own, zeros where there is none
          const int mine = pos0 + (lane & 15);
          const bool live = mine >= it_first && mine < it_n;
          const int pi = live ? divide(mine, by_page) : need_lo;
          const int off = mine - pi * p.page_size;
          const int page = __shfl_sync(0xffffffffu, page_id, pi - page_at);
          const bool fine = live && page >= 0 && page < p.pages;
          if (__any_sync(0xffffffffu, live && !fine)) m.flags |= kBad;
          const int64_t at = fine ? page * p.page_stride * ES + head_bytes + off * tok_bytes : -1;
#pragma unroll 1
          for (int row = rr; row < TILE; row += ROWS_STEP) {
            const int64_t a = __shfl_sync(0xffffffffu, at, row);
            const int64_t g = a >= 0 ? a : 0;
            cp_async16(dst + row * RB + (Sh::k_chunk(ch, row) << 4), kbase + g, a >= 0);
            cp_async16(dst + (TILE + row) * RB + (Sh::v_chunk(ch, row) << 4), vbase + g, a >= 0);
          }
          if (FP8) {
            const int64_t s = fine ? page * p.s_page + head_scales + off : 0;
            cp_async4(dst + 2 * TILE * RB + lane * 4, (lane < 16 ? p.ks : p.vs) + s, fine);
          }
        }
      }
      fresh = false;
      if (tile + AWARPS >= tile_end) active = false;
      tile += AWARPS;
    }
    if (lane == 0) meta[slot] = m;
    cp_async_commit();
  };

  // ---- the computing side ----
  uint32_t q[NG][D / 8];
  float o[NG][MT][4], mx[NG][2], sum[NG][2], fac[NG][2];  // mx: the weights' reference, base 2
  float ref_v = 0.0f;  // 8-bit: the power of two that the values' scales are relative to
  bool refused = false;

#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) issue(s);
  int slot = 0;
  while (true) {
    issue(slot == 0 ? STAGES - 1 : slot - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const int4 m0 = *reinterpret_cast<const int4*>(&meta[slot]);
    const int4 m1 = *(reinterpret_cast<const int4*>(&meta[slot]) + 1);
    const int row = m0.x, unit = m0.y, part = m0.z, flags = m0.w, at = m1.x, n = m1.y, first = m1.z, parts = m1.w;
    if (!(flags & kHas)) break;
    const int kvh = unit / groups, head0 = kvh * G + (unit - kvh * groups) * 8 * NG;  // of this item
    const int heads = min(8 * NG, kvh * G + G - head0);

    if (flags & kFirst) {
      refused = false;
      ref_v = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const bool live = g * 8 + r < heads;
        const TQ* src = static_cast<const TQ*>(p.q) + row * p.q_row + (head0 + (live ? g * 8 + r : 0)) * p.q_head;
        float f = p.scale * 1.4426950408889634f;
        if constexpr (!FP8) {
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {  // step j / 2: dimensions 8 j + 2c, 8 j + 2c + 1
            const uint32_t u = *reinterpret_cast<const uint32_t*>(src + j * 8 + 2 * c);
            q[g][j] = live ? u : 0u;
          }
        } else {
          // the head's query over a power of two near its largest value, in fp16 (what falls below fp16's smallest
          // values is under 2^-24 of the largest one)
          uint32_t raw[JC * 8];
          float top = 0.0f;
#pragma unroll
          for (int j = 0; j < JC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint4 u = *reinterpret_cast<const uint4*>(src + (j * 4 + c) * 16 + h * 8);
              if (!live) u = make_uint4(0, 0, 0, 0);
              const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                raw[j * 8 + h * 4 + i] = w[i];
                const float2 x = Mma<TQ>::unpack(w[i]);
                top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
              }
            }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const uint32_t e = min(max(__float_as_uint(top) >> 23, 1u), 253u);
          const float down = __uint_as_float((254u - e) << 23);
          f *= __uint_as_float(e << 23);
#pragma unroll
          for (int i = 0; i < JC * 8; ++i) {
            const float2 x = Mma<TQ>::unpack(raw[i]);
            q[g][i] = MM::pack(x.x * down, x.y * down);
          }
        }
        fac[g][0] = __shfl_sync(0xffffffffu, f, c * 8);      // head 2c: lanes of row 2c
        fac[g][1] = __shfl_sync(0xffffffffu, f, c * 8 + 4);  // head 2c + 1
        mx[g][0] = mx[g][1] = NO_MAX;
        sum[g][0] = sum[g][1] = 0.0f;
#pragma unroll
        for (int t = 0; t < MT; ++t) o[g][t][0] = o[g][t][1] = o[g][t][2] = o[g][t][3] = 0.0f;
      }
    }
    refused |= (flags & kBad) != 0;

    if (flags & kTile) {
      const uint32_t ks = smem_u32(ring + slot * Sh::STAGE), vs = ks + TILE * RB;
      float s[NG][4], s2[NG][4];  // two sums, taken in turn: shorter chains of dependent MMAs
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[g][i] = s2[g][i] = 0.0f;
      if constexpr (!FP8) {
        const uint32_t a = (ks + (r8 + (mat & 1) * 8) * RB) + (((mat >> 1) ^ r8) << 4);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t k[4];
          ldmatrix4<false>(a ^ (j << 5), k);
#pragma unroll
          for (int g = 0; g < NG; ++g)
            MM::run(j & 1 ? s2[g] : s[g], k[0], k[1], k[2], k[3], q[g][2 * j], q[g][2 * j + 1]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < JC; ++j) {
          const int chunk = j * 4 + c;
          const uint4 a = lds16(ks + r * RB + (Sh::k_chunk(chunk, r) << 4)),
                      b = lds16(ks + (r + 8) * RB + (Sh::k_chunk(chunk, r) << 4));
          const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t a0 = codes_f16(aw[w]), a1 = codes_f16(bw[w]), a2 = codes_f16(aw[w] >> 16),
                           a3 = codes_f16(bw[w] >> 16);
#pragma unroll
            for (int g = 0; g < NG; ++g)
              MM::run(w & 1 ? s2[g] : s[g], a0, a1, a2, a3, q[g][j * 8 + 2 * w], q[g][j * 8 + 2 * w + 1]);
          }
        }
      }
      // the logits, base 2: rows are tokens at + r and at + r + 8, columns heads 2c and 2c + 1
      float k0 = 1.0f, k1 = 1.0f, v0 = 1.0f, v1 = 1.0f, top_v = 0.0f;
      if (FP8) {
        const uint32_t sc = ks + 2 * TILE * RB;
        k0 = lds_f(sc + r * 4);
        k1 = lds_f(sc + r * 4 + 32);
        v0 = lds_f(sc + 64 + r * 4);
        v1 = lds_f(sc + 64 + r * 4 + 32);
        top_v = fmaxf(fabsf(v0), fabsf(v1));
      }
      const bool edge = at < first || at + TILE > n;
      float z[NG][4];
      bool up = FP8 && top_v > ref_v;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          z[g][i] = (s[g][i] + s2[g][i]) * fac[g][i & 1];
          if (FP8) z[g][i] *= i < 2 ? k0 : k1;
        }
        if (edge) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = at + r + (i < 2 ? 0 : 8);
            z[g][i] = pos >= first && pos < n ? z[g][i] : -INFINITY;
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) up |= fmaxf(z[g][h], z[g][h + 2]) > mx[g][h] + SLACK;
      }
      if (__any_sync(0xffffffffu, up)) {  // raise the references to what has been seen, and the sums with them
        float grow = 1.0f;
        if (FP8) {
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) top_v = fmaxf(top_v, __shfl_xor_sync(0xffffffffu, top_v, x));
          if (top_v > ref_v) {
            const uint32_t e = min((__float_as_uint(top_v) >> 23) + 2u, 253u);
            grow = ref_v * __uint_as_float((254u - e) << 23);
            ref_v = __uint_as_float(e << 23);
          }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float m = fmaxf(z[g][h], z[g][h + 2]);
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
            m = fmaxf(m, mx[g][h]);
            float f = ex2(mx[g][h] - m);
            mx[g][h] = m;
            sum[g][h] *= f;
            f *= grow;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              o[g][i][h] *= f;
              o[g][i][h + 2] *= f;
            }
          }
      }
      if (FP8) {
        const float inv = ref_v > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(ref_v)) : 0.0f;
        v0 *= inv;
        v1 *= inv;
      }
      uint32_t ph[NG][2], pl[NG][2];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = ex2(z[g][i] - mx[g][i & 1]);
        sum[g][0] += w[0] + w[2];
        sum[g][1] += w[1] + w[3];
        if (FP8) {
          w[0] *= v0;
          w[1] *= v0;
          w[2] *= v1;
          w[3] *= v1;
        }
        const uint32_t h0 = MM::pack(w[0], w[1]), h1 = MM::pack(w[2], w[3]);
        const float2 f0 = MM::unpack(h0), f1 = MM::unpack(h1);
        ph[g][0] = transposed(h0);
        ph[g][1] = transposed(h1);
        pl[g][0] = transposed(MM::pack(w[0] - f0.x, w[1] - f0.y));
        pl[g][1] = transposed(MM::pack(w[2] - f1.x, w[3] - f1.y));
      }
      // O^T += V^T P^T
      if constexpr (!FP8) {
        const uint32_t a = (vs + (r8 + (mat >> 1) * 8) * RB) + (((mat & 1) ^ r8) << 4);
#pragma unroll
        for (int j = 0; j < MT; ++j) {
          uint32_t v[4];
          ldmatrix4<true>(a ^ (j << 5), v);
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            MM::run(o[g][j], v[0], v[1], v[2], v[3], ph[g][0], ph[g][1]);
            MM::run(o[g][j], v[0], v[1], v[2], v[3], pl[g][0], pl[g][1]);
          }
        }
      } else {
        // a lane takes piece i * 8 + r of tokens 2c, 2c + 1, 2c + 8, 2c + 9
#pragma unroll
        for (int i = 0; i < NV; ++i) {
          uint32_t v[4][VB / 4];
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int tok = 2 * c + (t & 1) + (t >> 1) * 8;
            if constexpr (VB == 16) {
              const uint4 u = lds16(vs + tok * RB + (Sh::v_chunk(i * 8 + r, tok) << 4));
              v[t][0] = u.x;
              v[t][1] = u.y;
              v[t][2] = u.z;
              v[t][3] = u.w;
            } else {
              const uint2 u = lds8(vs + tok * RB + (Sh::v_chunk(r >> 1, tok) << 4) + (r & 1) * 8);
              v[t][0] = u.x;
              v[t][1] = u.y;
            }
          }
#pragma unroll
          for (int w = 0; w < VB / 4; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t sel = h ? 0x7362 : 0x5140;
              const uint32_t x = __byte_perm(v[0][w], v[1][w], sel), y = __byte_perm(v[2][w], v[3][w], sel);
              const uint32_t a0 = codes_f16(x), a1 = codes_f16(x >> 16), a2 = codes_f16(y), a3 = codes_f16(y >> 16);
#pragma unroll
              for (int g = 0; g < NG; ++g) {
                MM::run(o[g][i * (VB / 2) + w * 2 + h], a0, a1, a2, a3, ph[g][0], ph[g][1]);
                MM::run(o[g][i * (VB / 2) + w * 2 + h], a0, a1, a2, a3, pl[g][0], pl[g][1]);
              }
            }
        }
      }
    }

    if (flags & kLast) {
      // the four warps' parts of the item, 8 heads at a time, joined in warp order
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int live = min(8, heads - g * 8);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int x = 4; x <= 16; x <<= 1) sum[g][h] += __shfl_xor_sync(0xffffffffu, sum[g][h], x);
          const int head = 2 * c + h;
          if (r == 0) {
            join_m[warp * 8 + head] = refused ? NAN : mx[g][h];
            join_l[warp * 8 + head] = sum[g][h];
          }
          const float back = FP8 ? ref_v : 1.0f;
          if (head < live) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              // the rows r and r + 8 of m tile t
              const int d0 = FP8 ? (t / (VB / 2) * 8 + r) * VB + t % (VB / 2) * 2 : t * 16 + r, d1 = d0 + (FP8 ? 1 : 8);
              float* to = join_o + (warp * 8 + head) * D;
              to[d0 ^ (c << 3)] = o[g][t][h] * back;  // c = head / 2: other banks for the other heads
              to[d1 ^ (c << 3)] = o[g][t][h + 2] * back;
            }
          }
        }
        __syncthreads();
        for (int e = threadIdx.x; e < live * (D / 2); e += AWARPS * 32) {
          const int head = e / (D / 2), d = e % (D / 2) * 2;
          float top = join_m[head];
#pragma unroll
          for (int w = 1; w < AWARPS; ++w) top = max_nan(top, join_m[w * 8 + head]);
          float l = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
          for (int w = 0; w < AWARPS; ++w) {
            const float f = ex2(join_m[w * 8 + head] - top);
            const float2 v = *reinterpret_cast<const float2*>(join_o + (w * 8 + head) * D + (d ^ (head >> 1 << 3)));
            l = fmaf(join_l[w * 8 + head], f, l);
            x = fmaf(v.x, f, x);
            y = fmaf(v.y, f, y);
          }
          const int64_t rh = (int64_t)row * p.H + head0 + g * 8 + head;
          if (parts == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const uint32_t u = Mma<TQ>::pack(x * inv, y * inv);
            *reinterpret_cast<uint32_t*>(static_cast<TQ*>(p.out) + rh * D + d) = u;
          } else {
            const int64_t at2 = rh * ws.parts + part;
            *reinterpret_cast<float2*>(ws.o + at2 * D + d) = make_float2(x, y);
            if (d == 0) {
              ws.m[at2] = top;
              ws.l[at2] = l;
            }
          }
        }
        __syncthreads();
      }
      if (refused && lane == 0) atomicOr(&g_fault, (unsigned)kFaultBadPage);
    }
    __syncwarp();  // the stage may be filled again
    slot = slot == STAGES - 1 ? 0 : slot + 1;
  }
  cp_async_wait<0>();
}

// Joins the parts of a row and head that has several: grid (H, rows), 256 threads; D / 4 threads a part, 1024 / D parts
// at a time, added in a fixed order.
template <typename TQ, int D>
__global__ void __launch_bounds__(256) attend_join_kernel(const AttendParams p, const Workspace ws) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float weight[MAX_PARTS], red[16];
  __shared__ float4 acc[GROUPS][LANES];
  pdl_wait();
  const int h = blockIdx.x, b = blockIdx.y;
  int n, first;
  row_span(p, b, &n, &first);
  const int parts = parts_of(tiles_of(n, first));
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
