// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out[t, c] = y[t, c] + s * (x[t] A[i, p]^T) B[i, c]^T      i = index[t] (negative: no adapter), p the part of the output that c is in
//
// Mathematics: two products with a small inner size r, one after the other, so what bounds them is the traffic of x, y
// and out (or, with a token or two per adapter, of A and B), not arithmetic: at r = 16 a byte of x or y brings 16 products.
//
// Three forms. Few rows (or rows that no 16-byte access fits, or fp32): one launch, a cluster of CTAs per adapter and chunk of rows, which
// keeps u = x A^T in shared memory. Many rows: a launch that reduces x to u and one that expands u onto y, each of which only
// streams. Gradients of A and B: a launch that contracts over rows. Long contractions run on tcgen05 with copies in flight that no
// register waits for; where only a few ranks are contracted, and with few rows, warp-level `mma.sync` is enough.
// Which rows go together is found by each CTA from the indexes of its rows, so a captured graph follows the indexes of the step and nothing
// is sorted, counted or copied by the host.
//
// Precision: sums are fp32. u enters the second product (and the gradients) as two bf16 parts, off by 2^-16 of it at most, which a bf16 result does
// not show but in single roundings; three where the result is fp32, which hold all of it. fp32 operands enter as three bf16 parts each. The tensor
// cores cut their sums off, so fp32 results take the products of 16 columns, ranks or rows at a time from them and add those up outside, where
// sums are rounded: 4096 to 4096 columns, rank 16, off by 1.3e-7 of the result (2.0e-6 in the accumulators; fp32 library products 1.1e-6). Only fp32
// results beside many bf16 rows do not (14336 columns, rank 64: 2e-6; the second product would take 7 % longer).
#include <cooperative_groups.h>

#include <atomic>

#include "common.cuh"

namespace edl {
namespace cg = cooperative_groups;

namespace {

constexpr int LORA_THREADS = 256, LORA_WARPS = 8, LORA_MAX_WARPS = 10;
constexpr int LORA_ROWS = 256;       // rows whose adapters a cluster looks through
constexpr int LORA_SEGS = 8;

// ---------------------------------------------------------------------------------------------------------- registers
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t turn(uint32_t v) {      // 8 x 8 transpose over the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// Two values as sums of `S` bf16 values each, in packed pairs, rounded to nearest: a remainder is exact and at most 2^-8 of what it remains of.
// Three parts hold an fp32 value's 24 bits, two are off by 2^-16 of it at most. (Parts cut off towards zero are off by twice that, and all remainders
// then have the value's sign: products of the lower parts, which `mma_parts` leaves out, add up instead of cancelling.) What would round to
// infinity stays finite in the first part; an infinity has infinite or undefined later parts. Two at a time take one conversion per part:
// 4096 rows of fp32, 4096 columns to 4096, rank 16: 79 us, 108 value by value.
template <int S>
__device__ __forceinline__ void split(float lo, float hi, uint32_t (&p)[S]) {
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s == 0) asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(p[s]) : "f"(hi), "f"(lo));
    else p[s] = pack_bf16x2(lo, hi);
    lo -= __uint_as_float(p[s] << 16);
    hi -= __uint_as_float(p[s] & 0xffff0000u);
  }
}

template <typename T> constexpr int PARTS = sizeof(T) == 4 ? 3 : 1;

// N neighbouring elements from `p` as packed pairs of each part; elements from `valid` on are zero.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void load_pairs(const T* p, int valid, uint32_t (&q)[PARTS<T>][N / 2]) {
  if constexpr (sizeof(T) == 2) {
    if constexpr (WIDE) {
      if constexpr (N == 8) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (valid >= 8) v = *reinterpret_cast<const uint4*>(p);
        q[0][0] = v.x; q[0][1] = v.y; q[0][2] = v.z; q[0][3] = v.w;
      } else {
        uint2 v = make_uint2(0, 0);
        if (valid >= 4) v = *reinterpret_cast<const uint2*>(p);
        q[0][0] = v.x; q[0][1] = v.y;
      }
    } else {
      const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const uint32_t lo = 2 * i < valid ? s[2 * i] : 0, hi = 2 * i + 1 < valid ? s[2 * i + 1] : 0;
        q[0][i] = lo | (hi << 16);
      }
    }
  } else {
    float f[N];
    if constexpr (WIDE) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (valid >= i + 4) v = *reinterpret_cast<const float4*>(p + i);
        f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = i < valid ? p[i] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      uint32_t v[3];
      split<3>(f[2 * i], f[2 * i + 1], v);
#pragma unroll
      for (int s = 0; s < 3; ++s) q[s][i] = v[s];
    }
  }
}

// Eight neighbouring values of a row as fp32; those from `ok` on are zero (WIDE: all or none).
template <typename TY>
__device__ __forceinline__ void unpack_row(const uint4 (&v)[sizeof(TY) / 2], float (&f)[8]) {
  const uint32_t q[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[sizeof(TY) / 2 - 1].x, v[sizeof(TY) / 2 - 1].y, v[sizeof(TY) / 2 - 1].z, v[sizeof(TY) / 2 - 1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if constexpr (sizeof(TY) == 2) f[e] = __uint_as_float(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16);
    else f[e] = __uint_as_float(q[e]);
  }
}
template <typename TY, bool WIDE>
__device__ __forceinline__ void load_row(const TY* src, int ok, float (&f)[8]) {
  if constexpr (WIDE) {
    uint4 v[sizeof(TY) / 2];
#pragma unroll
    for (int q = 0; q < (int)sizeof(TY) / 2; ++q) v[q] = ok >= 8 ? reinterpret_cast<const uint4*>(src)[q] : make_uint4(0, 0, 0, 0);
    unpack_row<TY>(v, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < ok ? (float)src[e] : 0.f;
  }
}
template <typename TY, bool WIDE>
__device__ __forceinline__ void store_row(TY* dst, int ok, const float (&f)[8]) {
  if constexpr (WIDE) {
    if (ok < 8) return;
    if constexpr (sizeof(TY) == 2) {
      *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
    } else {
      *reinterpret_cast<float4*>(dst) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(dst + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < ok) {
        if constexpr (sizeof(TY) == 2) dst[e] = __float2bfloat16_rn(f[e]);
        else dst[e] = f[e];
      }
  }
}

// d += a b over the parts of both operands whose product is above the rounding of fp32: the second part is at most 2^-8 of its value, the third 2^-17,
// so what is left out of nine products is at most 2^-24 of theirs, of either sign.
// Where `F32` results need sums that are rounded, the products are added up by themselves first.
template <bool F32, int PA, int PB>
__device__ __forceinline__ void mma_parts(float (&d)[4], const uint32_t (&a)[PA][4], const uint32_t (&b)[PB][2]) {
  constexpr int TOP = PA > PB ? PA : PB;
  float few[4];
  bool first = F32;
#pragma unroll
  for (int o = TOP - 1; o >= 0; --o)      // small products first
#pragma unroll
    for (int i = 0; i < PA; ++i) {
      if (o - i < 0 || o - i >= PB) continue;
      if (!F32) mma_bf16(d, a[i][0], a[i][1], a[i][2], a[i][3], b[o - i][0], b[o - i][1]);
      else if (first) mma_bf16_first(few, a[i][0], a[i][1], a[i][2], a[i][3], b[o - i][0], b[o - i][1]);
      else mma_bf16(few, a[i][0], a[i][1], a[i][2], a[i][3], b[o - i][0], b[o - i][1]);
      first = false;
    }
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 4; ++e) d[e] += few[e];
  }
}

// A kernel that was launched to start early waits here until the one before it, and with that all before, has ended and its results are there;
// the one before says from where on the next may take the SMs that its blocks leave.
__device__ __forceinline__ void wait_for_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Sum of the values at `addr` (shared memory) of the CTAs of a cluster, in rank order; all are asked for before the first is used.
__device__ __forceinline__ float cluster_sum(uint32_t addr, int C) {
  float v[8], sum = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    v[k] = 0.f;
    if (k < C) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v[k]) : "r"(mapa_shared(addr, k)) : "memory");
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) sum += v[k];
  return sum;
}

__device__ __forceinline__ void cluster_sum4(uint32_t addr, int C, float (&sum)[4]) {      // four neighbours
  float v[8][4];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[k][i] = 0.f;
    if (k < C)
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[k][0]), "=f"(v[k][1]), "=f"(v[k][2]), "=f"(v[k][3])
                   : "r"(mapa_shared(addr, k)) : "memory");
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += v[k][i];
}

// ---------------------------------------------------------------------------------------------------------- which rows
struct LoraSeg {
  int c0, c1;       // columns of the matrix this side works on
  int u0, ru;       // ranks: first one, count
};

// Weights of the second product for 32 output columns from n0 on and ranks kc .. kc + 15: [column tile][part][register]. A lane's columns are
// the eight from n0 + 8 * (lane & 3) on, two of each tile. UP_T: they lie [ranks][columns].
template <typename T, bool UP_T, bool WIDE>
__device__ __forceinline__ void load_up(const T* wu, long long ld, int n0, const LoraSeg& seg, int kc, uint32_t (&wb)[4][PARTS<T>][2]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  if constexpr (!UP_T) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
      uint32_t v[PARTS<T>][2];
      load_pairs<T, 4, WIDE>(wu + (long long)n * ld + kc + 4 * t4, n < seg.c1 ? seg.ru - kc - 4 * t4 : 0, v);
#pragma unroll
      for (int s = 0; s < PARTS<T>; ++s) {
        wb[j][s][0] = v[s][0];
        wb[j][s][1] = v[s][1];
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rank = kc + 4 * (g >> 1) + (g & 1) + 2 * h, col = n0 + 8 * t4;
      uint32_t v[PARTS<T>][4];
      load_pairs<T, 8, WIDE>(wu + (long long)rank * ld + col, rank < seg.ru ? seg.c1 - col : 0, v);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int s = 0; s < PARTS<T>; ++s) wb[j][s][h] = turn(v[s][j]);
    }
  }
}

struct LoraArgs {
  const void* x;
  const void* y;
  void* out;
  const void* down;      // contracted with x
  const void* up;        // expanded to out
  long long ldx, ldy, ldo, down_adapter, ld_down, up_adapter, ld_up;
  const int* index;
  const float* scale;
  unsigned short* u;     // [parts of u][T][ucols] scaled, bf16; may be null in the one-launch form
  int* status;
  float scale_all;
  int T, n, rtot, ucols, groups, splits, down_segs, up_segs, copy;
  int* mixed;            // [blocks of rows] written by the kernel that reduces, read by the one-launch form, which then takes mixed blocks alone
  LoraSeg down_seg[LORA_SEGS], up_seg[LORA_SEGS];
};

__host__ __device__ constexpr int round16(int v) { return (v + 15) & ~15; }
__host__ __device__ constexpr int u_stride(int cols) { return cols % 32 ? cols : cols + 16; }      // 8-byte reads without conflicts

// Rows of a block in the order of their adapters, cut into units of at most `chunk` rows of one adapter.
struct RowUnits {
  int idx0, total;
  bool mixed;                                                   // rows of more than MIXED adapters
  short order[LORA_ROWS], base[LORA_ROWS], rows[LORA_ROWS];     // row of a place; first place and rows of a unit
  int ad[LORA_ROWS];
  int scan[LORA_MAX_WARPS];
};
// What finding them takes: lies where the kernels have their stages later, two of which then fit an SM.
constexpr int UNIT_SLOTS = 2 * LORA_ROWS;
struct UnitTable {
  int key[UNIT_SLOTS];                              // adapters by a hash of their number
  uint8_t count[UNIT_SLOTS][LORA_ROWS / 32];        // rows of a slot's adapter in each warp
  short place[UNIT_SLOTS];                          // of its first row in `order`
};

// Among many rows, a block of LORA_ROWS rows of more adapters than this (the single tokens of a step) goes to the one-launch kernel, whose
// clusters take a few rows of an adapter each; the streaming kernels take the others. Every kernel of a call decides so for itself.
// 3900 rows, 4096 columns to 4096, rank 16, 256 of them single tokens of 16 (64) adapters: 56 (67) us; 169 (531) where the streaming kernels took
// all of them. Where there is nothing to take, the third launch costs 4 us.
constexpr int MIXED = 4;

// Exclusive sum over the CTA's threads; `total` gets the sum of all.
__device__ __forceinline__ int cta_scan(int v, int* scan, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int at = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += t;
  }
  if (lane == 31) scan[w] = at;
  __syncthreads();
  total = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) {
    if (i < w) at += scan[i];
    total += scan[i];
  }
  __syncthreads();
  return at - v;
}

// All threads of the CTA. Rows without an adapter form units (adapter -1) where they have to be copied. Most blocks of a prompt or a
// training batch belong to one request: those take no look-up. Else rows of one adapter find each other within their warp (`match`) and
// across warps through a slot of a hash table, whose place decides nothing: units are numbered by their first rows.
// 256 rows of 64 adapters: 2.7 us from the launch on; 4.9 us when every row compared itself with all others.
__device__ __forceinline__ void find_units(RowUnits& u, void* scratch, const LoraArgs& a, long long row0, int rows, int chunk) {
  UnitTable& t = *reinterpret_cast<UnitTable*>(scratch);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  int id = -2;
  if (tid < rows) {
    id = a.index ? a.index[row0 + tid] : 0;
    if (id >= a.n && a.status) atomicCAS(a.status, 0, EDL_BAD_INDEX);
    if (id < 0 || id >= a.n) id = -1;
  }
  if (tid == 0) u.idx0 = id;
  if (tid < LORA_ROWS) {
    u.order[tid] = (short)tid;
#pragma unroll
    for (int i = 0; i < UNIT_SLOTS / LORA_ROWS; ++i) {
      t.key[tid + i * LORA_ROWS] = -3;
      *reinterpret_cast<uint2*>(t.count[tid + i * LORA_ROWS]) = make_uint2(0, 0);
    }
  }
  __syncthreads();
  if (!a.index || __syncthreads_and(tid >= rows || id == u.idx0)) {
    const int all = u.idx0 >= 0 || a.copy ? (rows + chunk - 1) / chunk : 0;
    if (tid < all) {
      u.base[tid] = (short)(tid * chunk);
      u.rows[tid] = (short)min(chunk, rows - tid * chunk);
      u.ad[tid] = u.idx0;
    }
    if (tid == 0) {
      u.total = all;
      u.mixed = false;
    }
    __syncthreads();
    return;
  }
  int slot = 0, lower = 0;
  if (tid < LORA_ROWS) {
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int leader = __ffs(same) - 1;
    lower = __popc(same & ((1u << lane) - 1));
    if (lane == leader && id >= -1) {
      slot = (uint32_t)(id * 0x9e3779b1u) >> 23;      // the top 9 bits: UNIT_SLOTS
      for (int found; (found = atomicCAS(&t.key[slot], -3, id)) != -3 && found != id;) slot = (slot + 1) & (UNIT_SLOTS - 1);
      t.count[slot][w] = (uint8_t)__popc(same);
    }
    slot = __shfl_sync(0xffffffffu, slot, leader);
  }
  __syncthreads();
  int before = lower, count = 0;
#pragma unroll
  for (int i = 0; i < LORA_ROWS / 32; ++i) {
    const int v = t.count[slot][i];
    count += v;
    before += i < w ? v : 0;
  }
  // first rows: their adapter's rows, units and one adapter, summed in one word
  const bool any = tid < rows && before == 0, taken = tid < rows && (id >= 0 || a.copy), first = taken && before == 0;
  const int nu = (count + chunk - 1) / chunk;
  int all;
  const int at = cta_scan((first ? count | nu << 10 : 0) | (any ? 1 << 20 : 0), u.scan, all);
  const int place = at & 1023, unit = at >> 10 & 1023;
  if (first) {
    t.place[slot] = (short)place;
    for (int q = 0; q < nu; ++q) {
      u.base[unit + q] = (short)(place + q * chunk);
      u.rows[unit + q] = (short)min(chunk, count - q * chunk);
      u.ad[unit + q] = id;
    }
  }
  if (tid == 0) {
    u.total = all >> 10 & 1023;
    u.mixed = (all >> 20) > MIXED;
  }
  __syncthreads();
  if (taken) u.order[t.place[slot] + before] = (short)tid;
  __syncthreads();      // the table makes way
}

// --------------------------------------------------------------------------------------------------- one launch, few rows
// A cluster of CTAs takes up to 16 rows of one adapter: each CTA contracts its share of the columns of x (spread over its warps), the
// CTAs add up their parts of u through each other's shared memory (in rank order, so results repeat), and each
// expands its share of the output's columns. Every `groups`-th unit of a block of 256 rows belongs to a cluster.
// Operands come straight from global memory: the contraction index of a product may be permuted as long as both operands agree, so a lane
// takes eight neighbouring elements with one 16-byte load and calls them the four register pairs of two m16n8k16 products; the same
// holds for output columns. Weights that are needed across their rows (the backward pass) are turned in registers (`movmatrix`).
// DOWN_T: the weights of the first product lie [columns][ranks] (B in the backward pass) and those of the second [ranks][columns].
//
// One row, 4096 columns to 4096, rank 16: 8 us (start 1.3, contraction 1.8, cluster 0.7, u 0.8, expansion 2); 48 rows of 32 adapters to 6144
// columns in three parts: 16 us; 256 rows of 64 adapters, 14336 to 4096, rank 32: 33 us, 2.5 TB/s of 83 MB (all cold). What bounds the last: an SM
// has two CTAs or one (252 of 296 places), a warp's loads of a step follow the last step's products, and the expansion reads its weights
// after the cluster has met. Weights copied ahead into rings in shared memory, or asked for before the cluster met, gained nothing.
// 4096 rows of fp32, 4096 to 4096: 79 us against 31 of traffic: the weights are read and cut into their parts again for every 16 rows, and every
// element of x is cut in registers, between loads that wait for the products of the step before.
template <typename T, typename TY, int RT, bool DOWN_T, bool WIDE>
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_kernel(const __grid_constant__ LoraArgs a) {
  constexpr int NT = 2, CHUNK = 8 * NT;
  constexpr int P = PARTS<T>;                           // parts of x and of the weights
  constexpr int S = sizeof(TY) == 4 ? 3 : 2;            // parts of u
  constexpr int RSTRIDE = 16 * RT + 4;
  __shared__ RowUnits units;
  extern __shared__ __align__(16) uint8_t dyn[];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int r16 = a.up_segs ? round16(a.up_seg[0].ru) : 0, ucols = a.ucols, ustride = u_stride(ucols);
  const int pstride = a.rtot;
  float* part = reinterpret_cast<float*>(dyn);                                      // [CHUNK][rtot]: this CTA's share of u
  uint8_t* second = dyn + ((CHUNK * pstride * 4 + 15) & ~15);
  float* red = reinterpret_cast<float*>(second);                                    // [warps][CHUNK][RSTRIDE], then
  unsigned short* su = reinterpret_cast<unsigned short*>(second);                   // [S][CHUNK][ustride]: scaled u in parts

  // groups of 32 columns: neighbouring ones belong to a CTA, so that its weights lie together
  int all_groups = 0;
  for (int p = 0; p < a.up_segs; ++p) all_groups += (a.up_seg[p].c1 - a.up_seg[p].c0 + 31) / 32;
  const int g0 = (int)((long long)all_groups * c / C), g1 = (int)((long long)all_groups * (c + 1) / C);
  auto column_of = [&](int grp) {      // first column of a group, its part
    int p = 0;
    for (int have; grp >= (have = (a.up_seg[p].c1 - a.up_seg[p].c0 + 31) / 32); ++p) grp -= have;
    return make_int2(a.up_seg[p].c0 + 32 * grp, p);
  };
  // a cluster works on one block of rows, or, where only mixed ones are left, on its share of each of those
  const int cid = blockIdx.x / C, nblocks = (int)(((long long)a.T + LORA_ROWS - 1) / LORA_ROWS);
  bool pending = false;
  for (int block = a.mixed ? 0 : cid / a.groups, step = a.mixed ? 1 : nblocks; block < nblocks; block += step) {
  if (a.mixed) {      // on to the next one, 32 at a look (one at a time took 4 us for 15)
    const uint32_t found = __ballot_sync(0xffffffffu, block + lane < nblocks && a.mixed[block + lane]);
    if (!found) {
      block += 31;
      continue;
    }
    block += __ffs(found) - 1;
  }
  const long long row0 = (long long)block * LORA_ROWS;
  // (not where `part` lies: other CTAs may still read that of the last unit)
  find_units(units, second, a, row0, (int)min((long long)LORA_ROWS, a.T - row0), CHUNK);
  for (int unit = cid % a.groups; unit < units.total; unit += a.groups) {
    const int ad = units.ad[unit], m = units.rows[unit];
    const short* order = units.order + units.base[unit];

    if (ad >= 0) {
      // ---- this CTA's share of u: ranks are the rows of the product, tokens its columns
      const T* wd = reinterpret_cast<const T*>(a.down) + (long long)ad * a.down_adapter;
      const T* xr[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int tok = i * 8 + g;
        xr[i] = tok < m ? reinterpret_cast<const T*>(a.x) + (row0 + order[tok]) * a.ldx : nullptr;
      }
      if (pending) {
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // every CTA has read the last unit's parts
        pending = false;
      }
      for (int sg = 0; sg < a.down_segs; ++sg) {
        const LoraSeg seg = a.down_seg[sg];
        for (int r0 = 0; r0 < seg.ru; r0 += 16 * RT) {
          float acc[RT][NT][4];
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
          // a warp takes whole lines of 128 bytes: 64 columns (32 of fp32)
          constexpr int HALVES = P == 1 ? 2 : 1;
          for (int k2 = seg.c0 + 32 * HALVES * (c * LORA_WARPS + w); k2 < seg.c1; k2 += 32 * HALVES * C * LORA_WARPS)
#pragma unroll(RT <= 2 ? HALVES : 1)
          for (int half = 0; half < HALVES; ++half) {
            const int k = k2 + 32 * half;
            uint32_t wa[RT][2][P][4];      // [rank tile][k16][part][register]
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              if constexpr (!DOWN_T) {
                uint32_t lo[P][4], hi[P][4];
                const int rank = r0 + 16 * i + g;
                load_pairs<T, 8, WIDE>(wd + (long long)(seg.u0 + rank) * a.ld_down + k + 8 * t4, rank < seg.ru ? seg.c1 - k - 8 * t4 : 0, lo);
                load_pairs<T, 8, WIDE>(wd + (long long)(seg.u0 + rank + 8) * a.ld_down + k + 8 * t4,
                                       rank + 8 < seg.ru ? seg.c1 - k - 8 * t4 : 0, hi);
#pragma unroll
                for (int p = 0; p < P; ++p)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    wa[i][h][p][0] = lo[p][2 * h];
                    wa[i][h][p][1] = hi[p][2 * h];
                    wa[i][h][p][2] = lo[p][2 * h + 1];
                    wa[i][h][p][3] = hi[p][2 * h + 1];
                  }
              } else {
                const int rank = r0 + 16 * i + 4 * t4;
#pragma unroll
                for (int mq = 0; mq < 4; ++mq) {
                  uint32_t v[P][2];
                  const int kk = k + 8 * (g >> 1) + (g & 1) + 2 * mq;
                  load_pairs<T, 4, WIDE>(wd + (long long)kk * a.ld_down + rank, kk < seg.c1 ? seg.ru - rank : 0, v);
#pragma unroll
                  for (int p = 0; p < P; ++p) {
                    wa[i][mq >> 1][p][2 * (mq & 1)] = turn(v[p][0]);
                    wa[i][mq >> 1][p][2 * (mq & 1) + 1] = turn(v[p][1]);
                  }
                }
              }
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              uint32_t v[P][4], b[2][P][2];
              load_pairs<T, 8, WIDE>(xr[j] + k + 8 * t4, xr[j] ? seg.c1 - k - 8 * t4 : 0, v);
#pragma unroll
              for (int p = 0; p < P; ++p) {
                b[0][p][0] = v[p][0]; b[0][p][1] = v[p][1];
                b[1][p][0] = v[p][2]; b[1][p][1] = v[p][3];
              }
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                mma_parts<S == 3, P, P>(acc[i][j], wa[i][0], b[0]);
                mma_parts<S == 3, P, P>(acc[i][j], wa[i][1], b[1]);
              }
            }
          }
          // sum over the warps
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int tok = j * 8 + 2 * t4;
              const int lo = 16 * i + (DOWN_T ? 4 * (g >> 1) + (g & 1) : g), hi = lo + (DOWN_T ? 2 : 8);
              float* dst = red + (w * CHUNK + tok) * RSTRIDE;
              dst[lo] = acc[i][j][0];
              dst[RSTRIDE + lo] = acc[i][j][1];
              dst[hi] = acc[i][j][2];
              dst[RSTRIDE + hi] = acc[i][j][3];
            }
          __syncthreads();
          for (int e = tid; e < m * 16 * RT; e += LORA_THREADS) {
            const int tok = e / (16 * RT), rank = e % (16 * RT);
            if (r0 + rank >= seg.ru) continue;
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < LORA_WARPS; ++k) sum += red[(k * CHUNK + tok) * RSTRIDE + rank];
            part[tok * pstride + seg.u0 + r0 + rank] = sum;
          }
          __syncthreads();
        }
      }
      // ---- u of all CTAs, scaled, as bf16 parts
      cluster_sync_all();
      const float s = a.scale ? a.scale[ad] : a.scale_all;
      for (int e = tid; e < CHUNK * ucols; e += LORA_THREADS) {
        const int tok = e / ucols, col = e - tok * ucols;
        const int p = a.up_segs > 1 ? col / r16 : 0, rank = col - p * r16;
        float v = 0.f;
        if (tok < m && rank < a.up_seg[p].ru) v = cluster_sum(smem_u32(part + tok * pstride + a.up_seg[p].u0 + rank), C) * s;
        uint32_t parts[S];
        split<S>(v, 0.f, parts);
#pragma unroll
        for (int k = 0; k < S; ++k) {
          su[(k * CHUNK + tok) * ustride + col] = (unsigned short)parts[k];
          if (a.u && c == 0 && tok < m) a.u[((long long)k * a.T + row0 + order[tok]) * ucols + col] = (unsigned short)parts[k];
        }
      }
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      pending = true;
      __syncthreads();
    }

    // ---- out = y + u B^T over this CTA's share of the columns: two times 32 per warp and turn
    const T* wu = reinterpret_cast<const T*>(a.up) + (long long)(ad < 0 ? 0 : ad) * a.up_adapter;
    for (int grp = g0 + w; a.out && grp < g1; grp += 2 * LORA_WARPS) {
      int2 at[2];      // first column, part
      float acc[2][4][4];
      long long row[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) row[h] = 8 * h + g < m ? row0 + order[8 * h + g] : -1;
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        at[d] = grp + d * LORA_WARPS < g1 ? column_of(grp + d * LORA_WARPS) : make_int2(0, -1);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[d][j][e] = 0.f;
      }
      if (ad >= 0) {
        for (int kc = 0; kc < r16; kc += 16) {
          uint32_t wb[2][4][P][2];
#pragma unroll
          for (int d = 0; d < 2; ++d)
            load_up<T, DOWN_T, WIDE>(wu, a.ld_up, at[d].x, at[d].y < 0 ? LoraSeg{0, 0, 0, 0} : a.up_seg[at[d].y], kc, wb[d]);
#pragma unroll
          for (int d = 0; d < 2; ++d) {
            uint32_t ua[S][4];
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint2 v = *reinterpret_cast<const uint2*>(su + (s * CHUNK + 8 * h + g) * ustride + max(at[d].y, 0) * r16 + kc + 4 * t4);
                ua[s][h] = v.x;
                ua[s][2 + h] = v.y;
              }
#pragma unroll
            for (int j = 0; j < 4; ++j) mma_parts<S == 3, S, P>(acc[d][j], ua, wb[d][j]);
          }
        }
      }
#pragma unroll
      for (int d = 0; d < 2; ++d) {
        if (at[d].y < 0) continue;
        const int col = at[d].x + 8 * t4, ok = a.up_seg[at[d].y].c1 - col;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[8];
          load_row<TY, WIDE>(reinterpret_cast<const TY*>(a.y) + row[h] * a.ldy + col, a.y && row[h] >= 0 ? ok : 0, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += acc[d][e >> 1][2 * h + (e & 1)];
          store_row<TY, WIDE>(reinterpret_cast<TY*>(a.out) + row[h] * a.ldo + col, row[h] >= 0 ? ok : 0, v);
        }
      }
    }
    __syncthreads();      // parts of u make way for the next unit
  }
  }
  if (pending) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // no CTA leaves while its parts are read
}

// --------------------------------------------------------------------------------------------------- many rows: x to u
template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src, bool ok) {      // zeros where not ok
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(ok ? 8 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A ring of shared-memory stages (rows of 128 bytes, swizzled) that one lane feeds to `tcgen05.mma`. Rows that lie one after the other in
// memory come by TMA; others are gathered by all threads with `cp.async`, which costs instructions for every piece. A stage is filled
// again once its products are done.
constexpr int RING_STAGES = 4;
struct Ring {
  uint32_t base, done, all, full, tmem;      // stages; barriers: a stage's products, all products, a stage's copies; accumulators
  int bytes, used, passes;                   // of a stage; stages fed so far; passes finished
  volatile int* abort_flag;
  int* status;
  __device__ __forceinline__ void wait(uint32_t bar, uint32_t parity, int code) { mbar_wait(bar, parity, abort_flag, status, code); }
  __device__ __forceinline__ int at(int step) const { return (used + step) % RING_STAGES; }
  // until the stage that `step` takes is free
  __device__ __forceinline__ uint32_t free_stage(int step) {
    const int use = used + step;
    if (use >= RING_STAGES) wait(done + 8 * at(step), (use / RING_STAGES - 1) & 1, EDL_TIMEOUT_PRODUCER);
    return base + at(step) * bytes;
  }
  __device__ __forceinline__ void finish(int steps) {
    used += steps;
    wait(all, passes++ & 1, EDL_TIMEOUT_MMA);
    tc_fence_after();
  }
};
struct RingShared {
  uint64_t bars[2 * RING_STAGES + 1];
  uint32_t tmem;
  int abort_flag;
};
// All threads. Waits that run out leave their code in the status word; everything after them goes on, without meaning.
__device__ __forceinline__ Ring ring_start(RingShared& sh, const uint8_t* stages, int bytes, int tmem_cols, int* status) {
  if (threadIdx.x == 0) {
    for (int i = 0; i <= 2 * RING_STAGES; ++i) mbar_init(smem_u32(&sh.bars[i]), 1);
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (threadIdx.x >> 5 == 1) {
    tmem_alloc(smem_u32(&sh.tmem), tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t bars = smem_u32(sh.bars);
  return Ring{smem_u32(stages), bars, bars + 8 * RING_STAGES, bars + 8 * (RING_STAGES + 1), sh.tmem, bytes, 0, 0, &sh.abort_flag, status};
}
// Both return once all products are done and visible in tensor memory. `feed(stage address, step)` issues a stage's products (one lane).
// `fill(stage address, step)`: every thread copies its share.
template <typename Fill, typename Feed>
__device__ __forceinline__ void ring_gather(Ring& r, int steps, Fill fill, Feed feed) {
  if (!steps) return;
#pragma unroll
  for (int i = 0; i < RING_STAGES - 1; ++i) {
    if (i < steps) fill(r.free_stage(i), i);
    cp_commit();
  }
  for (int step = 0; step < steps; ++step) {
    cp_wait<RING_STAGES - 2>();
    fence_proxy_async_smem();
    __syncthreads();
    if (threadIdx.x < 32) {
      const bool leader = elect_one();
      tc_fence_after();
      if (leader) {
        feed(r.base + r.at(step) * r.bytes, step);
        tc_commit(r.done + 8 * r.at(step));
        mbar_arrive(r.full + 8 * r.at(step));      // keeps step with the copies by TMA
        if (step == steps - 1) tc_commit(r.all);
      }
      __syncwarp();
    }
    if (step + RING_STAGES - 1 < steps) fill(r.free_stage(step + RING_STAGES - 1), step + RING_STAGES - 1);
    cp_commit();
  }
  cp_wait<0>();
  r.finish(steps);
}
// `load(stage address, barrier, step)`: one lane of warp 0 issues copies of `bytes` bytes.
template <typename Load, typename Feed>
__device__ __forceinline__ void ring_tma(Ring& r, int steps, int bytes, Load load, Feed feed) {
  if (!steps) return;
  fence_proxy_async_smem();      // what lay in the stages before
  __syncthreads();
  const int w = threadIdx.x >> 5;
  if (w == 0) {
    if (elect_one()) {
      for (int step = 0; step < steps; ++step) {
        const uint32_t dst = r.free_stage(step), bar = r.full + 8 * r.at(step);
        mbar_expect_tx(bar, bytes);
        load(dst, bar, step);
      }
    }
    __syncwarp();
  } else if (w == 1) {
    const bool leader = elect_one();
    for (int step = 0; step < steps; ++step) {
      r.wait(r.full + 8 * r.at(step), ((r.used + step) / RING_STAGES) & 1, EDL_TIMEOUT_MMA);
      tc_fence_after();
      if (leader) {
        feed(r.base + r.at(step) * r.bytes, step);
        tc_commit(r.done + 8 * r.at(step));
        if (step == steps - 1) tc_commit(r.all);
      }
    }
    __syncwarp();
  }
  r.finish(steps);
}
__device__ __forceinline__ void ring_end(Ring& r, int tmem_cols) {
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x >> 5 == 1) tmem_dealloc(r.tmem, tmem_cols);
}

// u of up to 128 rows of one adapter (the M side; ranks are the N side): columns in steps of 64 through the ring, cut over the CTAs of a
// cluster where there are few rows. Passes (up to 64 ranks of a part) run one after the other into columns of their own of tensor memory,
// up to 128 at a time, before the CTAs' sums are added, in a fixed order.
// 8192 rows: 4096 columns, rank 16: 22 us, 67 MB at 3.0 TB/s; 14336 columns, rank 64: 57 us, 4.1 TB/s. It is bound by the stream of x while that
// lasts (15 of the 22 us); the rest is its start and the sums' way through the cluster.
constexpr int DOWN_ROWS = 128, DOWN_K = 64, DOWN_X = DOWN_ROWS * DOWN_K * 2, DOWN_RANKS = 64, DOWN_COLS = 128;
__host__ __device__ constexpr int down_stage(int np, bool down_t) { return DOWN_X + (down_t ? DOWN_K : np) * 128; }

template <bool DOWN_T>
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_down_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ CUtensorMap map_x,
                                                                  const __grid_constant__ CUtensorMap map_w, int tma, int parts, int np) {
  __shared__ RowUnits units;
  __shared__ RingShared shared;
  extern __shared__ uint8_t raw[];
  uint8_t* dyn = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  float* part = reinterpret_cast<float*>(dyn);      // [128][pstride], where the stages were
  constexpr int pstride = DOWN_COLS + 4;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int cid = blockIdx.x / C;
  const long long row0 = (long long)(cid / a.groups) * LORA_ROWS;
  const __nv_bfloat16* x = reinterpret_cast<const __nv_bfloat16*>(a.x);
  Ring ring = ring_start(shared, dyn, down_stage(np, DOWN_T), DOWN_COLS, a.status);
  find_units(units, dyn, a, row0, (int)min((long long)LORA_ROWS, a.T - row0), DOWN_ROWS);
  let_next_start();
  if (a.mixed && tid == 0) a.mixed[row0 / LORA_ROWS] = units.mixed;
  const uint32_t idesc = umma_idesc_bf16(128, np, 0, DOWN_T);
  // passes: `each` of a part's ranks in all parts; `at_once` of them fit tensor memory
  const int each = (a.down_seg[0].ru + np - 1) / np, passes = a.down_segs * each, at_once = DOWN_COLS / np;
  struct Pass {
    int c0, c1, r0, k0, steps, lo, hi;      // columns of the part; first rank in it; first column and steps of this CTA; ranks in u
  };
  auto pass_of = [&](int i) {
    const LoraSeg& seg = a.down_seg[i / each];
    const int r0 = i % each * np, all = (seg.c1 - seg.c0 + DOWN_K - 1) / DOWN_K, per = (all + C - 1) / C, first = min(all, c * per);
    return Pass{seg.c0, seg.c1, r0, seg.c0 + first * DOWN_K, min(all, first + per) - first, seg.u0 + r0, min(seg.u0 + r0 + np, seg.u0 + seg.ru)};
  };
  bool pending = false;
  for (int unit = cid % a.groups; unit < (units.mixed ? 0 : units.total); unit += a.groups) {
    const int ad = units.ad[unit], m = units.rows[unit];
    if (ad < 0) continue;
    const short* order = units.order + units.base[unit];
    const __nv_bfloat16* wd = reinterpret_cast<const __nv_bfloat16*>(a.down) + (long long)ad * a.down_adapter;
    const float s = a.scale ? a.scale[ad] : a.scale_all;
    const bool line = tma && order[m - 1] - order[0] == m - 1;      // neighbouring rows; those behind the unit's come along and are not looked at
    for (int pass0 = 0; pass0 < passes; pass0 += at_once) {
      const int pass1 = min(passes, pass0 + at_once);
      int steps = 0;
      for (int i = pass0; i < pass1; ++i) steps += pass_of(i).steps;
      // the pass that a step belongs to (steps come in order)
      struct At {
        Pass p;
        int i, base;
      };
      const At start{pass_of(pass0), pass0, 0};
      auto go = [&](At& at, int step) {
        while (step - at.base >= at.p.steps) {
          at.base += at.p.steps;
          at.p = pass_of(++at.i);
        }
        return step - at.base;
      };
      At fed = start, loaded = start;
      if (pending) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // every CTA has read the last parts
      pending = false;
      auto feed = [&](uint32_t src, int step) {
        step = go(fed, step);
#pragma unroll
        for (int q = 0; q < DOWN_K / 16; ++q)
          umma_f16_ss(ring.tmem + (fed.i - pass0) * np, umma_smem_desc_sw128(src + 32 * q, 16, 1024),
                      umma_smem_desc_sw128(src + DOWN_X + (DOWN_T ? 2048 : 32) * q, DOWN_T ? 8192 : 16, 1024), idesc, step || q);
      };
      if (line) {
        const int at_row = (int)row0 + order[0];
        auto load = [&](uint32_t dst, uint32_t bar, int step) {
          const int k = go(loaded, step) * DOWN_K + loaded.p.k0;
          const Pass& p = loaded.p;
          tma_load_2d(dst, &map_x, bar, k, at_row);
          if constexpr (!DOWN_T) tma_load_3d(dst + DOWN_X, &map_w, bar, k, p.r0, ad);
          else tma_load_3d(dst + DOWN_X, &map_w, bar, p.r0, k, ad);
        };
        ring_tma(ring, steps, down_stage(np, DOWN_T), load, feed);
      } else {
        const __nv_bfloat16* xr[4];      // a thread copies the same piece of four rows in every step
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = (tid >> 3) + 32 * i;
          xr[i] = tok < m ? x + (row0 + order[tok]) * a.ldx + 8 * (tid & 7) : nullptr;
        }
        const uint32_t piece = 16 * ((tid & 7) ^ ((tid >> 3) & 7));
        auto fill = [&](uint32_t dst, int step) {
          const int k = go(loaded, step) * DOWN_K + loaded.p.k0, ru = loaded.p.hi - loaded.p.lo;
          const Pass& p = loaded.p;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            cp_async<16>(dst + ((tid >> 3) + 32 * i) * 128 + piece, xr[i] ? xr[i] + k : x, xr[i] && k + 8 * (tid & 7) < p.c1);
          const uint32_t wdst = dst + DOWN_X;
          if constexpr (!DOWN_T) {
            for (int i = tid; i < np * 8; i += LORA_THREADS) {
              const int rank = i >> 3, col = k + 8 * (i & 7);
              const bool ok = rank < ru && col < p.c1;
              cp_async<16>(wdst + rank * 128 + 16 * ((i & 7) ^ (rank & 7)), ok ? wd + (long long)(p.r0 + rank) * a.ld_down + col : wd, ok);
            }
          } else {
            for (int i = tid; i < DOWN_K * 16; i += LORA_THREADS) {
              const int kk = i >> 4, rank = 4 * (i & 15);
              const bool ok = k + kk < p.c1 && rank < ru;
              cp_async<8>(wdst + kk * 128 + 16 * ((rank >> 3) ^ (kk & 7)) + 2 * (rank & 7),
                          ok ? wd + (long long)(k + kk) * a.ld_down + p.r0 + rank : wd, ok);
            }
          }
        };
        ring_gather(ring, steps, fill, feed);
      }
      __syncthreads();      // part takes the stages' place
      if (w < 4) {
        float* dst = part + (32 * w + lane) * pstride;
        for (int i = pass0; i < pass1; ++i) {
          const bool any = pass_of(i).steps;
          for (int r = (i - pass0) * np; r < (i - pass0 + 1) * np; r += 16) {
            uint32_t v[16];
            tmem_ld_32x32b_x16(ring.tmem + (uint32_t(32 * w) << 16) + r, v);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < 16; j += 4)
              *reinterpret_cast<uint4*>(dst + r + j) = any ? make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]) : make_uint4(0, 0, 0, 0);
          }
        }
        tc_fence_before();
      }
      cluster_sync_all();
      tc_fence_after();
      // ---- each CTA adds up and writes its share
      const int r16 = round16(a.up_seg[0].ru), lo = pass_of(pass0).lo, hi = pass_of(pass1 - 1).hi;
      // (four ranks at a time: r is a multiple of 4 here, so they belong to one part and one pass)
      const int quads = a.ucols / 4;
      for (int e = c * LORA_THREADS + tid; e < m * quads; e += C * LORA_THREADS) {
        const int tok = e / quads, col = 4 * (e - tok * quads);
        const int p = a.up_segs > 1 ? col / r16 : 0, j = col - p * r16, rank = a.up_seg[p].u0 + j;
        const bool pad = j >= a.up_seg[p].ru;
        if (pad ? pass0 > 0 : rank < lo || rank >= hi) continue;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (!pad) {
          const int of = a.down_segs > 1 ? rank / a.down_seg[0].ru : 0, in = rank - of * a.down_seg[0].ru;      // part and rank in it
          cluster_sum4(smem_u32(part + tok * pstride + (of * each - pass0) * np + in), C, v);
        }
        unsigned short* dst = a.u + (row0 + order[tok]) * a.ucols + col;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = pad ? 0.f : v[i] * s;
        uint32_t q[2][3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (parts == 2) {
            uint32_t two[2];
            split<2>(v[2 * h], v[2 * h + 1], two);
            q[h][0] = two[0];
            q[h][1] = two[1];
          } else {
            split<3>(v[2 * h], v[2 * h + 1], q[h]);
          }
        }
#pragma unroll
        for (int k = 0; k < 3; ++k)
          if (k < parts) *reinterpret_cast<uint2*>(dst + (long long)k * a.T * a.ucols) = make_uint2(q[0][k], q[1][k]);
      }
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      pending = true;
    }
  }
  if (pending) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
  ring_end(ring, DOWN_COLS);
}

// --------------------------------------------------------------------------------------------------- many rows: u onto y
// What no TMA box fits or tensor memory holds (fp32 outputs, ranks that are no multiple of 8 or above 64), on `mma.sync`. A CTA takes 256
// columns of one part (32 per warp) of some of a block's units of 16 rows. The rows' u goes to shared memory once, the weights of
// a warp's columns stay in registers for all rows of an adapter (up to 16 KC ranks); what remains per 16 rows is to read y, asked for
// two turns ahead, and to write out. 4096 rows, 4096 columns: rank 12 27 us (67 MB at 2.4 TB/s), fp32 rank 16 35 us (134 MB at 3.8 TB/s): traffic;
// rank 128 72 us: `mma.sync`, 20 clocks a product and scheduler, and weights that are read again for every 16 rows.
constexpr int UP_COLS = 32 * LORA_WARPS;
template <typename TY, int KC, bool UP_T>
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_up_any_kernel(const __grid_constant__ LoraArgs a) {
  constexpr int S = sizeof(TY) == 4 ? 3 : 2;
  __shared__ RowUnits units;
  extern __shared__ __align__(16) uint8_t dyn[];
  unsigned short* su = reinterpret_cast<unsigned short*>(dyn);      // [S][own rows][ustride], in the units' order
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const long long row0 = (long long)(blockIdx.x / (a.groups * a.splits)) * LORA_ROWS;
  int p = 0, tile = blockIdx.x % a.groups;
  for (; tile >= (a.up_seg[p].c1 - a.up_seg[p].c0 + UP_COLS - 1) / UP_COLS; ++p) tile -= (a.up_seg[p].c1 - a.up_seg[p].c0 + UP_COLS - 1) / UP_COLS;
  const LoraSeg seg = a.up_seg[p];
  const int n0 = seg.c0 + tile * UP_COLS + 32 * w, col = n0 + 8 * t4, r16 = round16(seg.ru), ustride = u_stride(r16);
  const bool ok = col < seg.c1;
  find_units(units, dyn, a, row0, (int)min((long long)LORA_ROWS, a.T - row0), 16);
  const int share = (units.total + a.splits - 1) / a.splits, unit0 = min(units.total, (int)(blockIdx.x / a.groups % a.splits) * share);
  const int total = min(units.total, unit0 + share);
  if (units.mixed || unit0 >= total) return;
  const int place0 = units.base[unit0], places = units.base[total - 1] + units.rows[total - 1] - place0;
  const TY* y = reinterpret_cast<const TY*>(a.y) + col;
  TY* out = reinterpret_cast<TY*>(a.out) + col;
  constexpr int W = sizeof(TY) / 2;      // 16-byte pieces of eight values
  uint4 ring[2][2][W];
  long long rows[2][2];      // of the units asked for
  auto ask = [&](int unit, uint4 (&into)[2][W], long long (&row)[2]) {
    const int m = unit < total ? units.rows[unit] : 0;
    const short* order = units.order + (m ? units.base[unit] : 0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[h] = 8 * h + g < m ? row0 + order[8 * h + g] : -1;
      const bool read = a.y && ok && row[h] >= 0;
#pragma unroll
      for (int q = 0; q < W; ++q) {
        into[h][q] = make_uint4(0, 0, 0, 0);
        if (read) into[h][q] = reinterpret_cast<const uint4*>(y + row[h] * a.ldy)[q];
      }
    }
  };
  {
    const int per = r16 / 8;
    for (int i = tid; i < S * places * per; i += LORA_THREADS) {
      const int q = i % per, place = (i / per) % places, s = i / (per * places);
      cp_async<16>(smem_u32(su + (s * places + place) * ustride + 8 * q),
                   a.u + ((long long)s * a.T + row0 + units.order[place0 + place]) * a.ucols + p * r16 + 8 * q, true);
    }
    cp_commit();
  }
  ask(unit0, ring[0], rows[0]);
  ask(unit0 + 1, ring[1], rows[1]);
  cp_wait<0>();
  __syncthreads();
  int have = -1;
  uint32_t wb[KC][4][1][2];
  auto turn_of = [&](int unit, uint4 (&yq)[2][W], long long (&row)[2]) {
    const int ad = units.ad[unit], base = units.base[unit] - place0;
    // [column tile][row half, column]: y and what is added to it. The tensor cores cut sums off, so 32-bit results add y to the sum of products.
    float acc[4][4], yv[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      unpack_row<TY>(yq[h], yv[h]);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e >> 1][2 * h + (e & 1)] = S == 3 ? 0.f : yv[h][e];
    }
    TY* dst[2] = {row[0] >= 0 ? out + row[0] * a.ldo : nullptr, row[1] >= 0 ? out + row[1] * a.ldo : nullptr};
    ask(unit + 2, yq, row);
    if (ad >= 0) {
      // places behind the unit's rows: whatever lies there goes into rows that are not written
      const unsigned short* su0 = su + min(base + g, places - 1) * ustride + 4 * t4;
      const unsigned short* su1 = su + min(base + 8 + g, places - 1) * ustride + 4 * t4;
      for (int kc0 = 0; kc0 < r16; kc0 += 16 * KC) {
        if (ad != have || r16 > 16 * KC) {
          const __nv_bfloat16* wu = reinterpret_cast<const __nv_bfloat16*>(a.up) + (long long)ad * a.up_adapter;
#pragma unroll
          for (int i = 0; i < KC; ++i) load_up<__nv_bfloat16, UP_T, true>(wu, a.ld_up, n0, seg, kc0 + 16 * i, wb[i]);
          have = ad;
        }
#pragma unroll
        for (int i = 0; i < KC; ++i) {
          if (KC > 1 && kc0 + 16 * i >= r16) break;
          uint32_t ua[S][4];
#pragma unroll
          for (int s = 0; s < S; ++s) {
            const int at = s * places * ustride + kc0 + 16 * i;
            const uint2 v0 = *reinterpret_cast<const uint2*>(su0 + at), v1 = *reinterpret_cast<const uint2*>(su1 + at);
            ua[s][0] = v0.x; ua[s][1] = v1.x;
            ua[s][2] = v0.y; ua[s][3] = v1.y;
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) mma_parts<false, S, 1>(acc[j], ua, wb[i][j]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = acc[e >> 1][2 * h + (e & 1)] + (S == 3 ? yv[h][e] : 0.f);
      store_row<TY, true>(dst[h], ok && dst[h] ? 8 : 0, v);
    }
  };
  for (int unit = unit0; unit < total; unit += 2) {
    turn_of(unit, ring[0], rows[0]);
    if (unit + 1 < total) turn_of(unit + 1, ring[1], rows[1]);
  }
}

// 64 bytes of a row: two 32-byte stores where rows start on 32 bytes, so that every sector is written once.
__device__ __forceinline__ void store_64(void* p, const uint32_t (&v)[16], bool wide) {
  uint4* q = reinterpret_cast<uint4*>(p);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t* r = v + 8 * i;
    if (wide) {
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(q + 2 * i), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                   "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
    } else {
      q[2 * i] = make_uint4(r[0], r[1], r[2], r[3]);
      q[2 * i + 1] = make_uint4(r[4], r[5], r[6], r[7]);
    }
  }
}

// The same on tcgen05: 128 rows of one adapter are the M side, 64 columns at a time the N side, the ranks of both parts of u the inner index.
// A lane loads tiles of y and of the weights ahead (TMA), a lane of the second warp issues the products into one of two accumulators, and
// two times four warps, a row per lane, add every other tile to y where it lies and send it out as boxes of 32 rows (TMA). What bounds it is
// the traffic of y and out. Rows of y that lanes asked for themselves, two tiles ahead, took a third longer than by TMA.
// 8192 rows, 4096 columns: 27 us, 134 MB at 5.0 TB/s; 3900 rows of 8 requests, 28672 columns: 95 us, 447 MB at 4.7 TB/s; without y (the backward
// pass), 14336 columns: 59 us, 235 MB at 4.0 TB/s.
constexpr int UP_THREADS = 320, UP_ROWS = 128, UP_TILE = 64, UP_STAGES = 3;
constexpr int UP_Y = UP_ROWS * UP_TILE * 2, UP_W = 64 * 128, UP_STAGE = UP_Y + UP_W, UP_U = UP_ROWS * 128;
constexpr int UP_SMEM = UP_STAGES * UP_STAGE + 2 * UP_U + 1024;

template <bool UP_T>
__global__ void __launch_bounds__(UP_THREADS, 2) lora_up_kernel(const __grid_constant__ LoraArgs a, const __grid_constant__ CUtensorMap map_y,
                                                               const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_u,
                                                               const __grid_constant__ CUtensorMap map_out) {
  __shared__ RowUnits units;
  __shared__ uint64_t s_bars[2 * UP_STAGES + 7];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  extern __shared__ uint8_t raw[];
  uint8_t* dyn = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const uint32_t stages = smem_u32(dyn), su = stages + UP_STAGES * UP_STAGE;
  const uint32_t full = smem_u32(s_bars), empty = full + 8 * UP_STAGES, dfull = empty + 8 * UP_STAGES, dempty = dfull + 16, ufull = dempty + 16,
                 ufree = ufull + 8, ugo = ufree + 8;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const long long row0 = (long long)(blockIdx.x / a.splits) * LORA_ROWS;
  if (tid == 0) {
    for (int i = 0; i < UP_STAGES; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 5);      // the products and four warps
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(dfull + 8 * i, 1);
      mbar_init(dempty + 8 * i, 4);
    }
    mbar_init(ufull, 1);
    mbar_init(ufree, 1);
    mbar_init(ugo, 1);
    s_abort = 0;
    fence_mbar_init();
  }
  if (w == 1) {
    tmem_alloc(smem_u32(&s_tmem), 2 * UP_TILE);
    tmem_relinquish();
  }
  tc_fence_before();
  find_units(units, dyn, a, row0, (int)min((long long)LORA_ROWS, a.T - row0), UP_ROWS);
  fence_proxy_async_smem();      // the table makes way for copies
  wait_for_last();
  let_next_start();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  const int r16 = round16(a.up_seg[0].ru), share = (a.groups + a.splits - 1) / a.splits;      // column tiles: all, of a CTA
  const int tile0 = min(a.groups, (int)(blockIdx.x % a.splits) * share), tile1 = min(a.groups, tile0 + share);
  volatile int* abort_flag = &s_abort;
  auto wait = [&](uint32_t bar, int use, int code) { mbar_wait(bar, use & 1, abort_flag, a.status, code); };

  // Every role walks the same runs: a unit's tiles within one part, whose u they share. Rows without an adapter are copied by the eight
  // warps alone. A wait by parity tells a phase from its neighbours alone, so whoever waits on a barrier waits for each of its phases: the lane
  // that loads is the only one that waits until the last run's products have read their u (`ufree`, a phase per run; the next one's products need
  // weights that it has not asked for yet), and passes that on to the eight warps where they bring u themselves (`ugo`, a phase per such run).
  struct Run {
    int ad, m, p, n0, count, run, tile;      // first column, tiles; number of this run and of its first tile
    const short* order;
  };
  auto walk = [&](auto f) {
    Run r{};
    for (int unit = 0; unit < (units.mixed ? 0 : units.total); ++unit) {
      r.ad = units.ad[unit];
      r.m = units.rows[unit];
      r.order = units.order + units.base[unit];
      int first = 0;      // of part p's tiles
      for (r.p = 0; r.p < a.up_segs; ++r.p) {
        const int c0 = a.up_seg[r.p].c0, last = first + (a.up_seg[r.p].c1 - c0 + UP_TILE - 1) / UP_TILE;
        const int lo = max(first, tile0);
        r.count = min(last, tile1) - lo;
        r.n0 = c0 + (lo - first) * UP_TILE;
        first = last;
        if (r.count <= 0) continue;
        f(r);
        if (r.ad >= 0) {
          ++r.run;
          r.tile += r.count;
        }
      }
    }
  };
  auto line = [](const Run& r) { return r.order[r.m - 1] - r.order[0] == r.m - 1; };      // neighbouring rows
  if (w == 0) {
    if (elect_one()) {
      walk([&](const Run& r) {
        if (r.ad < 0) return;
        if (r.run) wait(ufree, r.run - 1, EDL_TIMEOUT_PRODUCER);
        if (line(r)) {
          mbar_expect_tx(ufull, 2 * UP_U);
          for (int s = 0; s < 2; ++s) tma_load_3d(su + s * UP_U, &map_u, ufull, r.p * r16, (int)row0 + r.order[0], s);
        } else {
          mbar_arrive(ugo);
        }
        for (int t = 0; t < r.count; ++t) {
          const int tile = r.tile + t, at = tile % UP_STAGES, use = tile / UP_STAGES;
          if (use) wait(empty + 8 * at, use - 1, EDL_TIMEOUT_PRODUCER);
          const uint32_t dst = stages + at * UP_STAGE, bar = full + 8 * at;
          const bool read = a.y && line(r);
          mbar_expect_tx(bar, (UP_T ? r16 * 128 : UP_W) + (read ? UP_Y : 0));
          if (read) tma_load_2d(dst, &map_y, bar, r.n0 + t * UP_TILE, (int)row0 + r.order[0]);
          if constexpr (UP_T) tma_load_3d(dst + UP_Y, &map_w, bar, r.n0 + t * UP_TILE, 0, r.ad);
          else tma_load_3d(dst + UP_Y, &map_w, bar, 0, r.n0 + t * UP_TILE, r.ad);
        }
      });
    }
    __syncwarp();
  } else if (w == 1) {
    const bool leader = elect_one();
    const uint32_t idesc = umma_idesc_bf16(UP_ROWS, UP_TILE, 0, UP_T);
    walk([&](const Run& r) {
      if (r.ad < 0) return;
      wait(ufull, r.run, EDL_TIMEOUT_MMA);
      for (int t = 0; t < r.count; ++t) {
        const int tile = r.tile + t, at = tile % UP_STAGES, buf = tile & 1;
        wait(full + 8 * at, tile / UP_STAGES, EDL_TIMEOUT_MMA);
        if (tile > 1) wait(dempty + 8 * buf, tile / 2 - 1, EDL_TIMEOUT_MMA);
        tc_fence_after();
        if (leader) {
          const uint32_t src = stages + at * UP_STAGE + UP_Y;
          for (int s = 1; s >= 0; --s)
            for (int k = 0; k < r16 / 16; ++k)
              umma_f16_ss(tmem + buf * UP_TILE, umma_smem_desc_sw128(su + s * UP_U + 32 * k, 16, 1024),
                          umma_smem_desc_sw128(src + (UP_T ? 2048 : 32) * k, UP_T ? 8192 : 16, 1024), idesc, s == 0 || k);
          tc_commit(empty + 8 * at);
          tc_commit(dfull + 8 * buf);
          if (t == r.count - 1) tc_commit(ufree);
        }
      }
    });
    __syncwarp();
  } else {
    const int q = w & 3, half = (w - 2) >> 2, i = 32 * q + lane;      // this lane's row of a unit; its four warps take every other tile
    const bool wide = a.ldo % 16 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
    int gathered = 0;
    walk([&](const Run& r) {
      if (r.ad >= 0 && !line(r)) {      // u of rows that are no neighbours
        wait(ugo, gathered++, EDL_TIMEOUT_EPILOGUE);
        for (int e = tid - 64; e < 2 * UP_ROWS * (r16 / 8); e += 256) {
          const int j = e % (r16 / 8), tok = e / (r16 / 8) % UP_ROWS, s = e / (r16 / 8 * UP_ROWS);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (tok < r.m) v = *reinterpret_cast<const uint4*>(a.u + ((long long)s * a.T + row0 + r.order[tok]) * a.ucols + r.p * r16 + 8 * j);
          *reinterpret_cast<uint4*>(dyn + UP_STAGES * UP_STAGE + s * UP_U + tok * 128 + 16 * (j ^ (tok & 7))) = v;
        }
        fence_proxy_async_smem();
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (tid == 64) mbar_arrive(ufull);
      }
      const bool neighbours = line(r), boxed = a.y && r.ad >= 0 && neighbours;
      const long long row = row0 + (i < r.m ? r.order[i] : 0);
      const __nv_bfloat16* y = reinterpret_cast<const __nv_bfloat16*>(a.y) + row * a.ldy;
      __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out) + row * a.ldo;
      for (int t = (r.tile ^ half) & 1; t < r.count; t += 2) {
        const int tile = r.tile + t, at = tile % UP_STAGES, n0 = r.n0 + t * UP_TILE, left = a.up_seg[r.p].c1 - n0;
        uint8_t* box = dyn + at * UP_STAGE + i * 128;
        // 32 whole rows of a whole tile leave as one box from where y lay; others from registers
        const bool whole = r.ad >= 0 && neighbours && 32 * q + 32 <= r.m && left >= UP_TILE;
        if (r.ad >= 0) {
          wait(full + 8 * at, tile / UP_STAGES, EDL_TIMEOUT_EPILOGUE);
          wait(dfull + 8 * half, tile / 2, EDL_TIMEOUT_EPILOGUE);
          tc_fence_after();
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int have = left - 32 * h;
          uint32_t v[16];      // y, then out
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (boxed) x = *reinterpret_cast<const uint4*>(box + 16 * ((4 * h + e) ^ (i & 7)));
            else if (a.y && i < r.m && have > 8 * e) x = *reinterpret_cast<const uint4*>(y + n0 + 32 * h + 8 * e);
            v[4 * e] = x.x; v[4 * e + 1] = x.y; v[4 * e + 2] = x.z; v[4 * e + 3] = x.w;
          }
          if (r.ad >= 0) {
            uint32_t d[32];
            tmem_ld_32x32b_x32(tmem + (uint32_t(32 * q) << 16) + half * UP_TILE + 32 * h, d);
            tc_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
              v[e] = pack_bf16x2(__uint_as_float(v[e] << 16) + __uint_as_float(d[2 * e]), __uint_as_float(v[e] & 0xffff0000u) + __uint_as_float(d[2 * e + 1]));
          }
          if (whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<uint4*>(box + 16 * ((4 * h + e) ^ (i & 7))) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          } else if (i < r.m) {
            if (have >= 32) {
              store_64(out + n0 + 32 * h, v, wide && (n0 & 15) == 0);
            } else {      // the last columns of a part
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (have > 8 * e) *reinterpret_cast<uint4*>(out + n0 + 32 * h + 8 * e) = make_uint4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
            }
          }
        }
        if (r.ad >= 0) {
          tc_fence_before();
          if (whole) fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(dempty + 8 * half);
            if (whole) {
              tma_store_2d(&map_out, smem_u32(dyn + at * UP_STAGE + 32 * q * 128), n0, (int)row0 + r.order[0] + 32 * q);
              tma_store_commit();
              tma_store_wait_read<0>();
            }
            mbar_arrive(empty + 8 * at);
          }
          __syncwarp();
        }
      }
    });
  }
  tma_store_wait<0>();
  tc_fence_before();
  __syncthreads();
  if (w == 1) tmem_dealloc(tmem, 2 * UP_TILE);
}

// Raises a kernel's limit of dynamic shared memory on the current device, once per thread. The limit belongs to all threads and a call may lower it, so
// it is always the most that the device allows beside the kernel's static part, whatever this launch takes.
int shared_memory(const void* kernel, const char* what) {
  struct Known {
    const void* kernel;
    int dev;
  };
  static thread_local Known known[64] = {};
  int dev = 0, most = 0;
  if (check_cuda(cudaGetDevice(&dev), what)) return -1;
  Known* slot = known;
  for (; slot < known + 64 && slot->kernel; ++slot)
    if (slot->kernel == kernel && slot->dev == dev) return 0;
  cudaFuncAttributes attr{};
  if (check_cuda(cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, dev), what) || check_cuda(cudaFuncGetAttributes(&attr, kernel), what) ||
      check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most - (int)attr.sharedSizeBytes), what))
    return -1;
  if (slot < known + 64) *slot = Known{kernel, dev};
  return 0;
}

// `early`: the kernel may start while the one before it ends (it waits by itself, see `wait_for_last`).
template <typename... E, typename... A>
int launch_sized(void (*k)(E...), dim3 grid, int threads, int cluster, bool early, int smem, cudaStream_t stream, const char* what, const A&... args) {
  if (smem > 40 * 1024 && shared_memory(reinterpret_cast<const void*>(k), what)) return -1;      // 48 KB with the static part
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k, args...), what);
}

template <typename... E, typename... A>
int launch_cluster(void (*k)(E...), dim3 grid, int cluster, int smem, cudaStream_t stream, const char* what, const A&... args) {
  return launch_sized(k, grid, LORA_THREADS, cluster, false, smem, stream, what, args...);
}

// ------------------------------------------------------------------------------------------------------------- gradients
struct GradJob {
  const void* z;               // [T, *] rows: x for dA, dy for dB
  const unsigned short* p;     // parts of g for dA, of u for dB: [parts][T][pcols]
  void* out;
  long long ldz, out_adapter, ld_out;
  int c0, c1, u0, ru;          // columns of z, ranks
  int pcols, p0;               // columns of p, the first one of these ranks
  int tiles;                   // column tiles x rank passes
  int across;                  // out lies [column][rank] (dB) instead of [rank][column] (dA)
};

struct GradArgs {
  const int* index;
  int* status;
  int T, n, jobs, out_f32, accumulate;
  GradJob job[LORA_SEGS + 1];
};

constexpr int GRAD_COLS = 256, GRAD_LIST = 1024, GRAD_STRIDE = GRAD_COLS + 4;

// Rows of adapter `ad` among `len` rows from `at` on, in order; returns how many (all of them without an index: the list stays empty).
__device__ __forceinline__ int list_rows(const GradArgs& a, int ad, long long at, int len, int* rows, int* scan) {
  if (!a.index) return len;
  const int tid = threadIdx.x;
  int mine[GRAD_LIST / LORA_THREADS], cnt = 0, found;
#pragma unroll
  for (int i = 0; i < GRAD_LIST / LORA_THREADS; ++i) {
    const int t = tid * (GRAD_LIST / LORA_THREADS) + i;
    mine[i] = t < len && a.index[at + t] == ad;
    cnt += mine[i];
  }
  int pos = cta_scan(cnt, scan, found);
#pragma unroll
  for (int i = 0; i < GRAD_LIST / LORA_THREADS; ++i)
    if (mine[i]) rows[pos++] = (int)(at + tid * (GRAD_LIST / LORA_THREADS) + i);
  __syncthreads();
  return found;
}

struct GradTile {
  GradJob job;
  int r0, col0;      // first rank and column of the tile
  long long lo, hi;  // rows of this CTA
};
__device__ __forceinline__ GradTile grad_tile(const GradArgs& a, int tile, int ranks, int C, int c) {
  int jb = 0;
  while (jb + 1 < a.jobs && tile >= a.job[jb].tiles) tile -= a.job[jb++].tiles;
  GradTile t;
  t.job = a.job[jb];
  const int passes = (t.job.ru + ranks - 1) / ranks;
  t.r0 = (tile % passes) * ranks;
  t.col0 = t.job.c0 + (tile / passes) * GRAD_COLS;
  const long long per = (((long long)a.T + C - 1) / C + 31) / 32 * 32;
  t.lo = min((long long)a.T, per * c);
  t.hi = min((long long)a.T, t.lo + per);
  return t;
}

// Adds up the CTAs' tiles [ranks][GRAD_STRIDE] through each other's shared memory, in order; each writes its share, four columns of a rank at a
// time (one by one it took 15 us longer for 72 tiles of 64 ranks).
__device__ __forceinline__ void write_grad(cg::cluster_group& cluster, const GradArgs& a, const GradTile& t, float* tile, int ranks, int ad) {
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const GradJob& job = t.job;
  cluster_sync_all();
  constexpr int QUADS = GRAD_COLS / 4;
  const int all = ranks * QUADS, share = (all + C - 1) / C;
  for (int e = c * share + threadIdx.x; e < min(all, (c + 1) * share); e += LORA_THREADS) {
    const int rank = job.across ? e % ranks : e / QUADS, col = 4 * (job.across ? e / ranks : e % QUADS), have = job.c1 - t.col0 - col;
    if (t.r0 + rank >= job.ru || have <= 0) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    cluster_sum4(smem_u32(tile + rank * GRAD_STRIDE + col), C, v);
    const long long next = job.across ? job.ld_out : 1;      // from one of the four to the next
    const long long pos = (long long)ad * job.out_adapter + (job.across ? (long long)(t.col0 + col) * job.ld_out + t.r0 + rank
                                                                         : (long long)(job.u0 + t.r0 + rank) * job.ld_out + t.col0 + col);
    if (a.out_f32) {
      float* o = reinterpret_cast<float*>(job.out) + pos;
      if (!job.across && have >= 4 && (reinterpret_cast<uintptr_t>(o) & 15) == 0) {
        float4 b = a.accumulate ? *reinterpret_cast<const float4*>(o) : make_float4(0.f, 0.f, 0.f, 0.f);
        *reinterpret_cast<float4*>(o) = make_float4(b.x + v[0], b.y + v[1], b.z + v[2], b.w + v[3]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < have) o[i * next] = a.accumulate ? o[i * next] + v[i] : v[i];
      }
    } else {
      __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(job.out) + pos;
      if (!job.across && have >= 4 && (reinterpret_cast<uintptr_t>(o) & 7) == 0) {
        *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (i < have) o[i * next] = __float2bfloat16_rn(v[i]);
      }
    }
  }
  cluster_sync_all();      // no CTA leaves while its tile is read
}

// out[rank, col] (+)= sum over the adapter's rows t of p[t, rank] z[t, col]: ranks x 256 columns per cluster, the rows cut over its CTAs.
// This form takes rows of any alignment and fp32 ones: 16 ranks at a time, operands along their rows from global memory, turned in registers.
// Warps 0-3 and 4-7 take every other 16 rows. 1000 rows, 1023 and 1021 columns, rank 5: 12 us; 4096 rows of fp32, 4096 and 4096 columns, rank 16:
// 89 us, 134 MB at 1.5 TB/s: elements are cut into parts in registers, between loads that wait for the products of the rows before.
template <typename T, int S, bool WIDE>
__global__ void __launch_bounds__(LORA_THREADS, 1) lora_grad_any_kernel(const __grid_constant__ GradArgs a) {
  constexpr int P = PARTS<T>;
  __shared__ int s_rows[GRAD_LIST];
  __shared__ int s_scan[LORA_WARPS];
  extern __shared__ __align__(16) uint8_t dyn[];
  float* tile = reinterpret_cast<float*>(dyn);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
  const int ad = blockIdx.y, cw = w & 3, half = w >> 2;
  const GradTile t = grad_tile(a, blockIdx.x / C, 16, C, c);
  const GradJob& job = t.job;
  const T* z = reinterpret_cast<const T*>(job.z);
  const int colw = t.col0 + cw * 64;

  float acc[8][4];
#pragma unroll
  for (int j = 0; j < 8; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
  for (long long at = t.lo; at < t.hi; at += GRAD_LIST) {
    const int found = list_rows(a, ad, at, (int)min((long long)GRAD_LIST, t.hi - at), s_rows, s_scan);
    for (int t0 = 16 * half; t0 < found; t0 += 32) {
      long long row[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = t0 + 8 * h + g;
        row[h] = i < found ? (a.index ? (long long)s_rows[i] : at + i) : -1;
      }
      uint32_t zb[8][P][2];      // [column tile][part][register]
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t v[P][4];
          const int col = colw + 32 * q + 8 * t4;
          load_pairs<T, 8, WIDE>(z + (row[h] < 0 ? 0 : row[h]) * job.ldz + col, row[h] < 0 ? 0 : job.c1 - col, v);
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int s = 0; s < P; ++s) zb[4 * q + j][s][h] = turn(v[s][j]);
        }
      uint32_t pa[S][4];      // rows of the product: ranks; its inner index: tokens
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t v = 0;
            if (row[k] >= 0) v = *reinterpret_cast<const uint32_t*>(job.p + ((long long)s * a.T + row[k]) * job.pcols + job.p0 + t.r0 + 8 * h + 2 * t4);
            pa[s][h + 2 * k] = turn(v);
          }
#pragma unroll
      for (int j = 0; j < 8; ++j) mma_parts<S == 3, S, P>(acc[j], pa, zb[j]);
    }
    if (a.index) __syncthreads();
  }
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f((g + (e >> 1) * 8) * GRAD_STRIDE + cw * 64 + 32 * (j >> 2) + 8 * t4 + 2 * (j & 3) + (e & 1), acc[j][e]);
  };
  if (half == 1) each([&](int at, float v) { tile[at] = v; });
  __syncthreads();
  if (half == 0) each([&](int at, float v) { tile[at] += v; });
  write_grad(cluster, a, t, tile, 16, ad);
}

// The same for bf16 rows that 16-byte copies fit: 32 rows at a time through the ring. z's columns are the M side (128 at a time), both parts of
// p side by side the N side, and the rows the inner index of the products; both operands lie along M and N. 8192 rows: 4096 and 4096 columns,
// rank 16: 35 us, 134 MB at 3.8 TB/s; 14336 and 4096 columns, rank 64: 72 us, 302 MB at 4.2 TB/s. Its stream bounds it: without the products
// both take 4 us less, without the reads of p 2 us less.
constexpr int GRAD_ROWS = 32, GRAD_Z = GRAD_ROWS * GRAD_COLS * 2, GRAD_BOX = GRAD_ROWS * 128, GRAD_STAGE = GRAD_Z + 2 * GRAD_BOX;
struct GradMaps {
  CUtensorMap z[2], p[2];      // of dA's and dB's inputs
};
__global__ void __launch_bounds__(LORA_THREADS, 2) lora_grad_kernel(const __grid_constant__ GradArgs a, const __grid_constant__ GradMaps maps,
                                                                    int rp) {
  __shared__ int s_rows[GRAD_LIST];
  __shared__ int s_scan[LORA_WARPS];
  __shared__ RingShared shared;
  extern __shared__ uint8_t raw[];
  uint8_t* dyn = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int ad = blockIdx.y;
  const GradTile t = grad_tile(a, blockIdx.x / C, rp, C, c);
  const GradJob& job = t.job;
  const __nv_bfloat16* z = reinterpret_cast<const __nv_bfloat16*>(job.z);
  const int r16 = round16(job.ru) - t.r0;      // ranks that p has from r0 on
  const int tmem_cols = 4 * rp;
  Ring ring = ring_start(shared, dyn, GRAD_STAGE, tmem_cols, a.status);
  // both parts of p in one product where they fill their boxes
  const int merged = rp == 64 ? 2 : 1;
  const uint32_t idesc = umma_idesc_bf16(128, merged * rp, 1, 1);
  wait_for_last();
  bool any = false;
  const int at_once = a.index ? GRAD_LIST : a.T;      // without a list the ring runs dry only once
  for (long long at = t.lo; at < t.hi; at += at_once) {
    const int found = list_rows(a, ad, at, (int)min((long long)at_once, t.hi - at), s_rows, s_scan);
    auto row_of = [&](int k) -> long long { return k < found ? (a.index ? (long long)s_rows[k] : at + k) : 0; };
    auto fill = [&](uint32_t dst, int step) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {      // a warp copies whole rows
        const int r = w + 8 * i, k = step * GRAD_ROWS + r, col = t.col0 + 8 * lane;
        const bool ok = k < found && col < job.c1;
        cp_async<16>(dst + (lane >> 3) * GRAD_BOX + r * 128 + 16 * ((lane & 7) ^ (r & 7)), ok ? z + row_of(k) * job.ldz + col : z, ok);
      }
      for (int i = tid; i < GRAD_ROWS * 16; i += LORA_THREADS) {
        const int r = i >> 4, s = (i >> 3) & 1, j = i & 7, k = step * GRAD_ROWS + r;
        const bool ok = k < found && 8 * j < r16;
        cp_async<16>(dst + GRAD_Z + s * GRAD_BOX + r * 128 + 16 * (j ^ (r & 7)),
                     ok ? job.p + ((long long)s * a.T + row_of(k)) * job.pcols + job.p0 + t.r0 + 8 * j : job.p, ok);
      }
    };
    const bool start = !any;
    auto feed = [&](uint32_t src, int step) {
#pragma unroll
      for (int q = 0; q < GRAD_ROWS / 16; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          for (int s = 0; s < 2; s += merged)
            umma_f16_ss(ring.tmem + rp * (2 * h + s), umma_smem_desc_sw128(src + 2 * h * GRAD_BOX + 2048 * q, GRAD_BOX, 1024),
                        umma_smem_desc_sw128(src + GRAD_Z + s * GRAD_BOX + 2048 * q, GRAD_BOX, 1024), idesc, !start || step || q);
    };
    // whole steps of neighbouring rows by TMA (behind the last row of all there are zeros), the rest row by row
    const long long first = found ? (a.index ? (long long)s_rows[0] : at) : 0;
    const bool run = found && (!a.index || s_rows[found - 1] - s_rows[0] == found - 1);
    const int steps = (found + GRAD_ROWS - 1) / GRAD_ROWS, whole = !run ? 0 : first + found == a.T ? steps : found / GRAD_ROWS;
    auto load = [&](uint32_t dst, uint32_t bar, int step) {
      const int row = (int)first + step * GRAD_ROWS;
#pragma unroll
      for (int i = 0; i < 4; ++i) tma_load_2d(dst + i * GRAD_BOX, &maps.z[job.across], bar, t.col0 + 64 * i, row);
#pragma unroll
      for (int s = 0; s < 2; ++s) tma_load_3d(dst + GRAD_Z + s * GRAD_BOX, &maps.p[job.across], bar, job.p0 + t.r0, row, s);
    };
    ring_tma(ring, whole, GRAD_STAGE, load, feed);
    ring_gather(ring, steps - whole, [&](uint32_t dst, int step) { fill(dst, whole + step); }, [&](uint32_t src, int step) { feed(src, whole + step); });
    any = any || steps;
    __syncthreads();      // the list makes way
  }
  float* tile = reinterpret_cast<float*>(dyn);      // [rp][GRAD_STRIDE], where the stages were
  for (int r = 0; r < rp; r += 16) {
    uint32_t hi[16], lo[16];
    const uint32_t src = ring.tmem + (uint32_t(32 * (w & 3)) << 16) + 2 * rp * (w >> 2) + r;
    tmem_ld_32x32b_x16(src, hi);
    tmem_ld_32x32b_x16(src + rp, lo);
    tc_wait_ld();
#pragma unroll
    for (int j = 0; j < 16; ++j) tile[(r + j) * GRAD_STRIDE + 32 * w + lane] = any ? __uint_as_float(hi[j]) + __uint_as_float(lo[j]) : 0.f;
  }
  write_grad(cluster, a, t, tile, rp, ad);
  ring_end(ring, tmem_cols);
}

// Clusters of `size` CTAs of the gradient kernel that the current device runs at once (asked for once per size): the runtime counts one CTA to an
// SM, two fit.
int grad_clusters(int size, int smem) {
  static std::atomic<int> known[64][9] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (!known[dev][size]) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(size);
    cfg.blockDim = dim3(LORA_THREADS);
    cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = size;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (shared_memory(reinterpret_cast<const void*>(lora_grad_kernel), "lora gradient shared memory") ||
        cudaOccupancyMaxActiveClusters(&clusters, lora_grad_kernel, &cfg) != cudaSuccess) {
      cudaGetLastError();
      clusters = sm_count() / size * 7 / 8;
    }
    known[dev][size] = clusters > 0 ? 2 * clusters : -1;
  }
  return known[dev][size];
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

}  // namespace
}  // namespace edl

using namespace edl;

// Rows that one launch takes: up to 512, or 256 of a wide output that all belong to one adapter, whose weights are read again for every 16 rows.
// 4096 columns to 4096, rank 16: 512 rows of one adapter take 16.4 us against 25.6 in two launches, of eight 18.5 against 42, 768 rows 22-25
// against 42. To 28672 columns: 512 rows of one adapter 43 against 34, of eight 46 against 50.
static bool few_rows(int T, int cols, bool index) { return T <= 256 || (T <= 512 && (index || cols <= 8192)); }

// Sizes of a call: strides in elements, `widths` columns of the `parts` parts of N. x_f32: x and the weights are fp32 (then y and out
// too), else bf16; y_f32: type of y and out.
struct edl_lora_shape {
  long long ldx, ldy, ldo, a_adapter, lda, b_adapter, ldb;
  int T, K, N, n, r, parts, x_f32, y_f32, backward, widths[8];
};

// x [T, K], y and out [T, N] (y null: the adapters' part alone; y == out: in place). a: [n][parts * r][K], b: [n][N][r].
// backward = 0: out = y + s (x a^T) b^T. backward = 1: x is dy [T, N], out dx [T, K] (null: u alone), y null. u: s x a^T or s dy b
// in bf16 parts (2 for bf16 results, 3 for fp32 ones), [parts][T][columns] with parts * r rounded up to 16 per part (forward) or as a
// whole (backward); asked for with many rows (see `few_rows`) of bf16, else it may be null. mixed: a flag per 256 rows, scratch; asked for
// with many rows of bf16 and an index. index [T] int32 or null (adapter 0 everywhere), scale [n] fp32 or null (scale_all). Indexes from n on set the status
// word and count as none.
EDL_HOST_API int edl_lora_apply(const edl_lora_shape* shape, const void* x, const void* y, void* out, const void* a, const void* b,
                                const int* index, const float* scale, float scale_all, void* u, long long u_size, int* mixed,
                                int* status, void* stream) {
  const long long ldx = shape->ldx, ldy = shape->ldy, ldo = shape->ldo, a_adapter = shape->a_adapter, lda = shape->lda, b_adapter = shape->b_adapter,
                  ldb = shape->ldb;
  const int T = shape->T, K = shape->K, N = shape->N, n = shape->n, r = shape->r, parts = shape->parts, x_f32 = shape->x_f32, y_f32 = shape->y_f32,
            backward = shape->backward;
  const int* widths = shape->widths;
  if (T <= 0) return 0;
  if (K <= 0 || N <= 0 || n <= 0 || r <= 0 || parts < 1 || parts > LORA_SEGS || r > 512 / parts) {
    set_last_error("edl_lora_apply: needs sizes above 0, up to %d parts and parts x rank up to 512", LORA_SEGS);
    return -1;
  }
  if ((x_f32 && !y_f32) || (backward && x_f32 != y_f32) || (backward && y) || (!out && !(backward && u))) {
    set_last_error("edl_lora_apply: fp32 inputs give fp32 results; the backward form takes one type and no y");
    return -1;
  }
  LoraArgs g{};
  g.x = x; g.ldx = ldx; g.y = y; g.ldy = ldy; g.out = out; g.ldo = ldo;
  g.index = index; g.scale = scale; g.scale_all = scale_all; g.u = (unsigned short*)u; g.status = status;
  g.T = T; g.n = n; g.rtot = parts * r;
  g.copy = out && out != y;
  int c0 = 0;
  bool wide = r % 4 == 0 && K % 8 == 0 && N % 8 == 0;
  LoraSeg seg[LORA_SEGS];
  for (int p = 0; p < parts; ++p) {
    if (widths[p] <= 0) {
      set_last_error("edl_lora_apply: a part has no columns");
      return -1;
    }
    seg[p] = LoraSeg{c0, c0 + widths[p], p * r, r};
    c0 += widths[p];
    wide = wide && widths[p] % 8 == 0;
  }
  if (c0 != N) {
    set_last_error("edl_lora_apply: the parts have %d columns, the output %d", c0, N);
    return -1;
  }
  const LoraSeg whole{0, K, 0, parts * r};
  if (!backward) {
    g.down = a; g.down_adapter = a_adapter; g.ld_down = lda;
    g.up = b; g.up_adapter = b_adapter; g.ld_up = ldb;
    g.down_segs = 1;
    g.down_seg[0] = whole;
    g.up_segs = parts;
    for (int p = 0; p < parts; ++p) g.up_seg[p] = seg[p];
  } else {
    g.down = b; g.down_adapter = b_adapter; g.ld_down = ldb;
    g.up = a; g.up_adapter = a_adapter; g.ld_up = lda;
    g.down_segs = parts;
    for (int p = 0; p < parts; ++p) g.down_seg[p] = seg[p];
    g.up_segs = 1;
    g.up_seg[0] = whole;
  }
  g.ucols = g.up_segs * round16(g.up_seg[0].ru);
  const int s = y_f32 ? 3 : 2;
  if (u && (u_size < (long long)s * T * g.ucols || !aligned(u, 16))) {
    set_last_error("edl_lora_apply: u needs %lld elements from a 16-byte boundary on", (long long)s * T * g.ucols);
    return -1;
  }
  const int va = x_f32 ? 4 : 8, vy = y_f32 ? 4 : 8;      // elements in 16 bytes
  wide = wide && ldx % va == 0 && aligned(x, 16) && aligned(a, 16) && lda % va == 0 && a_adapter % va == 0 && aligned(b, x_f32 ? 16 : 8) &&
         ldb % 4 == 0 && b_adapter % 4 == 0 && (!y || (ldy % vy == 0 && aligned(y, 16))) && (!out || (ldo % vy == 0 && aligned(out, 16)));
  cudaStream_t st = (cudaStream_t)stream;
  const int blocks = (int)(((long long)T + LORA_ROWS - 1) / LORA_ROWS), in_block = T < LORA_ROWS ? T : LORA_ROWS, sms = sm_count();
  // clusters for a block's units: as many as it can have, or fewer that take turns once there are enough for the GPU
  auto groups_of = [&](int chunk) {
    const long long most = index ? (long long)(n < in_block ? n + 1 : in_block) + in_block / chunk : (in_block + chunk - 1) / chunk;
    int groups = 128 / blocks;
    if (groups < LORA_ROWS / chunk) groups = LORA_ROWS / chunk;
    if (groups > most) groups = (int)most;
    return groups > in_block ? in_block : groups;
  };

  if (wide && !x_f32 && !few_rows(T, backward ? K : N, index)) {
    if (!u) {
      set_last_error("edl_lora_apply: %d rows need u", T);
      return -1;
    }
    const bool may_mix = index && n + 1 > MIXED;      // rows without an adapter count as one
    if (may_mix && !mixed) {
      set_last_error("edl_lora_apply: %d rows of %d adapters need a flag per block of rows", T, n);
      return -1;
    }
    g.mixed = may_mix ? mixed : nullptr;
    // a block has two units, one more for each end of a request within it; a third cluster takes most of those (six, most of them idle,
    // took 4 us longer for 3900 rows)
    g.groups = groups_of(DOWN_ROWS);
    if (g.groups > 3) g.groups = 3;
    int ru = 0, cols = 0;
    for (int i = 0; i < g.down_segs; ++i) {
      ru = g.down_seg[i].ru > ru ? g.down_seg[i].ru : ru;
      cols += g.down_seg[i].c1 - g.down_seg[i].c0;
    }
    const int np = ru < DOWN_RANKS ? round16(ru) : DOWN_RANKS;
    // as many CTAs as run at once (two per SM), each with at least four steps of columns
    int cluster = 1;
    while (cluster < 8 && (long long)blocks * g.groups * cluster * 2 <= 2 * sms && cols >= 2 * cluster * 4 * DOWN_K) cluster *= 2;
    const dim3 grid((unsigned)((long long)blocks * g.groups * cluster));
    const int ring = RING_STAGES * down_stage(np, backward), part = DOWN_ROWS * (DOWN_COLS + 4) * 4, down_smem = (ring > part ? ring : part) + 1024;
    // TMA takes weights whose rows start on 16 bytes; a box of the backward pass must not reach into the next part's columns
    bool tma = !backward || (r % 8 == 0 && ldb % 8 == 0 && b_adapter % 8 == 0 && aligned(b, 16));
    for (int p = 0; backward && p + 1 < parts; ++p) tma = tma && widths[p] % DOWN_K == 0;
    CUtensorMap map_x{}, map_w{};
    if (tma) {
      if (make_tmap_2d_16b(&map_x, x, T, backward ? N : K, ldx, DOWN_ROWS, DOWN_K)) return -1;
      if (backward ? make_tmap_3d_16b(&map_w, b, r, N, n, ldb, b_adapter, 64, DOWN_K, 1, 3)
                   : make_tmap_3d_16b(&map_w, a, K, parts * r, n, lda, a_adapter, DOWN_K, np, 1, 3))
        return -1;
    }
    if (backward ? launch_cluster(lora_down_kernel<true>, grid, cluster, down_smem, st, "lora down launch", g, map_x, map_w, (int)tma, s, np)
                 : launch_cluster(lora_down_kernel<false>, grid, cluster, down_smem, st, "lora down launch", g, map_x, map_w, (int)tma, s, np))
      return -1;
    if (out) {
      const int r16 = round16(g.up_seg[0].ru);
      const bool tiles = r16 <= 64 && !y_f32 && (backward || (r % 8 == 0 && ldb % 8 == 0 && b_adapter % 8 == 0 && aligned(b, 16)));
      const int width = tiles ? UP_TILE : UP_COLS;
      g.groups = 0;
      for (int i = 0; i < g.up_segs; ++i) g.groups += (g.up_seg[i].c1 - g.up_seg[i].c0 + width - 1) / width;
      if (tiles) {
        // a block's columns are cut into as many CTAs as run at once (two per SM), or three times that where blocks may have more
        // units than others, of at least four tiles. 28672 columns, 3900 rows of 8 requests: 128 us, 164 without the three times; 4096
        // columns, 8192 rows without an index: 52 us, 56 with them.
        const int ctas = (index ? 6 : 2) * sms / blocks;
        g.splits = ctas < g.groups / 4 ? ctas : g.groups / 4;
        if (g.splits < 1) g.splits = 1;
        g.splits = (g.groups + (g.groups + g.splits - 1) / g.splits - 1) / ((g.groups + g.splits - 1) / g.splits);
        CUtensorMap map_y{}, map_u{}, map_out{};
        if (make_tmap_2d_16b(&map_out, out, T, backward ? K : N, ldo, 32, UP_TILE)) return -1;
        if (y && make_tmap_2d_16b(&map_y, y, T, backward ? K : N, ldy, UP_ROWS, UP_TILE)) return -1;
        if (make_tmap_3d_16b(&map_u, u, g.ucols, T, 2, g.ucols, (uint64_t)T * g.ucols, 64, UP_ROWS, 1, 3)) return -1;
        if (backward ? make_tmap_3d_16b(&map_w, a, K, parts * r, n, lda, a_adapter, UP_TILE, r16, 1, 3)
                     : make_tmap_3d_16b(&map_w, b, r, N, n, ldb, b_adapter, 64, UP_TILE, 1, 3))
          return -1;
        const dim3 up((unsigned)((long long)blocks * g.splits));
        if (backward ? launch_sized(lora_up_kernel<true>, up, UP_THREADS, 1, true, UP_SMEM, st, "lora up launch", g, map_y, map_w, map_u, map_out)
                     : launch_sized(lora_up_kernel<false>, up, UP_THREADS, 1, true, UP_SMEM, st, "lora up launch", g, map_y, map_w, map_u, map_out))
          return -1;
      } else {
        // a block that is not mixed has at most 16 + MIXED units: they are shared out where there are few CTAs, or where u takes much memory
        const int row_bytes = s * u_stride(r16) * 2, units = LORA_ROWS / 16 + MIXED;
        auto own = [&](int splits) { return max((int)sizeof(UnitTable), ((units + splits - 1) / splits) * 16 * row_bytes); };
        g.splits = 1;
        while (g.splits < 8 && (own(g.splits) > 56 * 1024 || (g.splits < 4 && (long long)g.groups * blocks * g.splits < 4LL * sms))) g.splits *= 2;
        const long long ctas = (long long)g.groups * blocks * g.splits;
        if (ctas > 0x7fffffffLL) {
          set_last_error("edl_lora_apply: too many rows for one launch");
          return -1;
        }
        const int kc = r16 / 16;
#define EDL_LORA_UP_OF(TO, KC, BW) launch_cluster(lora_up_any_kernel<TO, KC, BW>, dim3((unsigned)ctas), 1, own(g.splits), st, "lora up launch", g)
#define EDL_LORA_UP(TO) (kc == 1 ? EDL_LORA_UP_OF(TO, 1, false) : kc == 2 ? EDL_LORA_UP_OF(TO, 2, false) : EDL_LORA_UP_OF(TO, 4, false))
        // (the backward pass comes here with more than 64 ranks alone)
        if (backward ? EDL_LORA_UP_OF(__nv_bfloat16, 4, true) : y_f32 ? EDL_LORA_UP(float) : EDL_LORA_UP(__nv_bfloat16)) return -1;
#undef EDL_LORA_UP_OF
#undef EDL_LORA_UP
      }
    }
    if (!g.mixed) return 0;      // what is left: blocks of single tokens
  }

  const int ranks = backward ? r : parts * r;      // that one pass over x can take
  // (fp32 takes 32 at a time at most: 3000 rows, 2816 to 1024, rank 64 127 us, 147 with 16 at a time; 64 of three parts do not fit registers)
  const int rt = !wide || ranks <= 16 ? 1 : ranks <= 32 || x_f32 ? 2 : 4;
  // clusters of eight while they all fit the GPU twice, then smaller ones
  int cluster = 8;
  g.groups = g.mixed ? 2 * sms / cluster : groups_of(16);
  const long long grid_blocks = g.mixed ? 1 : blocks;
  while (cluster > 2 && grid_blocks * g.groups * cluster > 4LL * sms) cluster /= 2;
  const int red = LORA_WARPS * 16 * (16 * rt + 4) * 4, su = s * 16 * u_stride(g.ucols) * 2;
  static_assert(LORA_WARPS * 16 * 20 * 4 >= sizeof(UnitTable) && UP_SMEM >= sizeof(UnitTable), "the table of units lies in the kernels' stages");
  const int smem = ((16 * g.rtot * 4 + 15) & ~15) + (red > su ? red : su);
  const dim3 grid((unsigned)(grid_blocks * g.groups * cluster));
#define EDL_LORA(TX, TO, RTV, BW, W) return launch_cluster(lora_kernel<TX, TO, RTV, BW, W>, grid, cluster, smem, st, "lora launch", g)
#define EDL_LORA_BF(TO, BW)                                    \
  {                                                            \
    if (!wide) EDL_LORA(__nv_bfloat16, TO, 1, BW, false);      \
    if (rt == 4) EDL_LORA(__nv_bfloat16, TO, 4, BW, true);     \
    if (rt == 2) EDL_LORA(__nv_bfloat16, TO, 2, BW, true);     \
    EDL_LORA(__nv_bfloat16, TO, 1, BW, true);                  \
  }
#define EDL_LORA_F32(BW)                               \
  {                                                    \
    if (!wide) EDL_LORA(float, float, 1, BW, false);   \
    if (rt == 2) EDL_LORA(float, float, 2, BW, true);  \
    EDL_LORA(float, float, 1, BW, true);               \
  }
  if (x_f32) {
    if (backward) EDL_LORA_F32(true) else EDL_LORA_F32(false)
  }
  if (backward) EDL_LORA_BF(__nv_bfloat16, true)
  if (y_f32) EDL_LORA_BF(float, false)
  EDL_LORA_BF(__nv_bfloat16, false)
#undef EDL_LORA
#undef EDL_LORA_BF
#undef EDL_LORA_F32
}

// da [n][parts * r][K] (+)= g^T x and db [n][N][r] (+)= dy^T u over each adapter's rows (either may be null); the strides of a and b in `shape`
// are theirs, ldy dy's. g (for da), u (for db): what edl_lora_apply left of the backward and the forward call. out_f32: type of da and
// db; accumulate (fp32 only): add to them. Adapters without rows get zeros.
static int lora_grads(const edl_lora_shape* shape, const void* x, const void* dy, const void* g, const void* u, const int* index,
                                void* da, void* db, int out_f32, int accumulate, int* status, void* stream) {
  const long long ldx = shape->ldx, ldy = shape->ldy, da_adapter = shape->a_adapter, ld_da = shape->lda, db_adapter = shape->b_adapter, ld_db = shape->ldb;
  const int T = shape->T, K = shape->K, N = shape->N, n = shape->n, r = shape->r, parts = shape->parts, in_f32 = shape->x_f32;
  const int* widths = shape->widths;
  if (K <= 0 || N <= 0 || n <= 0 || r <= 0 || parts < 1 || parts > LORA_SEGS || r > 512 / parts || n > 65535 || (!index && n != 1 && T > 0)) {
    set_last_error("edl_lora_backward: needs sizes above 0, up to %d parts, parts x rank up to 512, up to 65535 adapters, one without an index", LORA_SEGS);
    return -1;
  }
  if ((in_f32 && !out_f32) || (accumulate && !out_f32)) {
    set_last_error("edl_lora_backward: fp32 inputs give fp32 gradients, and only those are accumulated into");
    return -1;
  }
  GradArgs a{};
  a.index = index; a.status = status; a.T = T < 0 ? 0 : T; a.n = n; a.out_f32 = out_f32; a.accumulate = accumulate;
  const int va = in_f32 ? 4 : 8;
  bool wide = true;
  int most = 0;
  if (da) {
    a.job[a.jobs++] = GradJob{x, (const unsigned short*)g, da, ldx, da_adapter, ld_da, 0, K, 0, parts * r, round16(parts * r), 0, 0, 0};
    wide = wide && K % 8 == 0 && ldx % va == 0 && aligned(x, 16);
    most = parts * r;
  }
  if (db) {
    int c0 = 0;
    for (int p = 0; p < parts; ++p) {
      a.job[a.jobs++] = GradJob{dy, (const unsigned short*)u, db, ldy, db_adapter, ld_db, c0, c0 + widths[p], p * r, r, parts * round16(r),
                                p * round16(r), 0, 1};
      c0 += widths[p];
      wide = wide && widths[p] % 8 == 0;
    }
    if (c0 != N) {
      set_last_error("edl_lora_backward: the parts have %d columns, the output %d", c0, N);
      return -1;
    }
    wide = wide && ldy % va == 0 && aligned(dy, 16);
    most = r > most ? r : most;
  }
  if (!a.jobs) return 0;
  const bool fast = wide && !in_f32;
  const int rp = !fast || most <= 16 ? 16 : most <= 32 ? 32 : 64;      // ranks of a pass over the rows
  int tiles = 0;
  for (int j = 0; j < a.jobs; ++j) {
    GradJob& job = a.job[j];
    job.tiles = ((job.c1 - job.c0 + GRAD_COLS - 1) / GRAD_COLS) * ((job.ru + rp - 1) / rp);
    tiles += job.tiles;
  }
  // Rows are cut over the CTAs of a cluster, of the size that takes the least: a turn of all clusters that run at once takes its steps of 32 rows
  // and about as long as 6 more to start and to add up. A training step of 8192 rows, 32 tiles: 130 us in sixes (the choice), 138 in fours,
  // 166 in twos; 72 tiles: 242 us in threes (the choice), 248 in twos, 263 in fours.
  const int ring_bytes = fast ? RING_STAGES * GRAD_STAGE + 1024 : 16 * GRAD_STRIDE * 4;
  int cluster = 1;
  long long best = 0;
  for (int c = 1; c <= 8; ++c) {
    const int at_once = fast ? grad_clusters(c, ring_bytes) : 2 * sm_count() / c;
    if (at_once < 1) continue;
    const long long cost = (((long long)tiles * n + at_once - 1) / at_once) * (6 + (a.T + 32LL * c - 1) / (32LL * c));
    if (!best || cost < best) {
      best = cost;
      cluster = c;
    }
  }
  cudaStream_t st = (cudaStream_t)stream;
  const dim3 grid((unsigned)(tiles * cluster), (unsigned)n);
  const char* what = "lora gradient launch";
  if (fast) {
    GradMaps maps{};
    if (a.T && da && (make_tmap_2d_16b(&maps.z[0], x, a.T, K, ldx, GRAD_ROWS, 64) ||
                      make_tmap_3d_16b(&maps.p[0], g, round16(parts * r), a.T, 2, round16(parts * r), (uint64_t)a.T * round16(parts * r), 64, GRAD_ROWS, 1, 3)))
      return -1;
    if (a.T && db && (make_tmap_2d_16b(&maps.z[1], dy, a.T, N, ldy, GRAD_ROWS, 64) ||
                      make_tmap_3d_16b(&maps.p[1], u, parts * round16(r), a.T, 2, parts * round16(r), (uint64_t)a.T * parts * round16(r), 64, GRAD_ROWS, 1, 3)))
      return -1;
    return launch_sized(lora_grad_kernel, grid, LORA_THREADS, cluster, true, ring_bytes, st, what, a, maps, rp);
  }
  const int smem = ring_bytes;
  if (in_f32) return wide ? launch_cluster(lora_grad_any_kernel<float, 3, true>, grid, cluster, smem, st, what, a)
                          : launch_cluster(lora_grad_any_kernel<float, 3, false>, grid, cluster, smem, st, what, a);
  return launch_cluster(lora_grad_any_kernel<__nv_bfloat16, 2, false>, grid, cluster, smem, st, what, a);
}

// The backward pass: edl_lora_apply's backward form (`back` null: not wanted, or done by an earlier call), then the gradients of the weights.
EDL_HOST_API int edl_lora_backward(const edl_lora_shape* back, const edl_lora_shape* shape, const void* x, const void* dy, const void* a, const void* b,
                                   const int* index, const float* scale, float scale_all, void* g, long long g_size, int* mixed, void* dx,
                                   const void* u, void* da, void* db, int out_f32, int accumulate, int* status, void* stream) {
  if (back && edl_lora_apply(back, dy, nullptr, dx, a, b, index, scale, scale_all, g, g_size, mixed, status, stream)) return -1;
  return da || db ? lora_grads(shape, x, dy, g, u, index, da, db, out_f32, accumulate, status, stream) : 0;
}
