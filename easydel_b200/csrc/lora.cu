// Low-rank adapters of many requests beside a shared projection, and their gradients.
//
//   out[t, c] = y[t, c] + s * (x[t] A[i, p]^T) B[i, c]^T      i = index[t] (negative: no adapter), p the part of the output that c is in
//
// Mathematics of both kernels: two products with a small inner size r, one after the other, so what bounds them is the traffic of x, y
// and out (or, with a token or two per adapter, of A and B), not arithmetic: at r = 16 a byte of x or y brings 16 products.
// That is why they issue warp-level `mma.sync` on registers filled straight from global memory and leave tensor memory alone: nothing is
// reused often enough to be worth a trip through it.
//
// Operand layout: the contraction index of a product may be permuted as long as both operands agree, so a lane takes
// eight neighbouring elements with one 16-byte load and calls them the four register pairs of two m16n8k16 products. The same holds for
// output columns: a lane ends up with eight neighbouring columns. Weights that are needed across their rows (the backward pass) are loaded
// along their rows and turned in registers (`movmatrix`).
//
// Precision: sums are fp32. The intermediate x A^T enters the second product as two bf16 parts (three where the result is fp32), so it
// keeps 16 (24) bits; fp32 operands enter as three bf16 parts each.
#include <cooperative_groups.h>

#include "common.cuh"

namespace edl {
namespace cg = cooperative_groups;

namespace {

constexpr int LORA_THREADS = 256, LORA_WARPS = 8;
constexpr int LORA_ROWS = 256;       // rows whose adapters a cluster looks through
constexpr int LORA_SEGS = 8;
constexpr int LORA_MAX_CHUNK = 64;

// ---------------------------------------------------------------------------------------------------------- registers
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn(uint32_t v) {      // 8 x 8 transpose over the warp
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// v as the sum of `S` bf16 values (upper halves), each cut off towards zero, so that nothing overflows and the remainder is
// exact. Values that are not finite keep to the first part.
template <int S>
__device__ __forceinline__ void split(float v, uint32_t (&p)[S]) {
  const uint32_t u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    p[0] = (u & 0x7fffffu) ? 0x7fc0u : u >> 16;
#pragma unroll
    for (int s = 1; s < S; ++s) p[s] = 0;
    return;
  }
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (s + 1 < S) {
      const uint32_t h = __float_as_uint(v) & 0xffff0000u;
      p[s] = h >> 16;
      v -= __uint_as_float(h);
    } else {
      p[s] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
    }
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
      uint32_t a[3], b[3];
      split<3>(f[2 * i], a);
      split<3>(f[2 * i + 1], b);
#pragma unroll
      for (int s = 0; s < 3; ++s) q[s][i] = a[s] | (b[s] << 16);
    }
  }
}

// d += a b over the parts of both operands whose product is above the rounding of fp32 (part i has the bits from 8 i on).
template <int PA, int PB>
__device__ __forceinline__ void mma_parts(float (&d)[4], const uint32_t (&a)[PA][4], const uint32_t (&b)[PB][2]) {
  constexpr int TOP = PA > PB ? PA : PB;
#pragma unroll
  for (int o = TOP - 1; o >= 0; --o)      // small products first
#pragma unroll
    for (int i = 0; i < PA; ++i)
      if (o - i >= 0 && o - i < PB) mma_bf16(d, a[i][0], a[i][1], a[i][2], a[i][3], b[o - i][0], b[o - i][1]);
}

// ------------------------------------------------------------------------------------------------------------- apply
struct LoraSeg {
  int c0, c1;       // columns of the matrix this side works on
  int u0, ru;       // ranks: first column in u, count
};

struct LoraArgs {
  const void* x;
  const void* y;
  void* out;
  const void* down;      // contracted with x
  const void* up;        // expanded to out
  long long ldx, ldy, ldo, down_adapter, ld_down, up_adapter, ld_up;
  const int* index;
  const float* scale;
  float* u_out;
  int* status;
  float scale_all;
  int T, n, rtot, groups, down_segs, up_segs, copy;
  LoraSeg down_seg[LORA_SEGS], up_seg[LORA_SEGS];
};

__host__ __device__ constexpr int round16(int v) { return (v + 15) & ~15; }
__host__ __device__ constexpr int u_stride(int cols) { return cols % 32 ? cols : cols + 16; }      // 8-byte reads without conflicts

// One launch, no workspace. A cluster of CTAs takes up to CHUNK rows of one adapter: each CTA contracts its share of the columns of x
// (spread over its warps), the CTAs add up their parts of u = x A^T through each other's shared memory (in rank order, so results
// repeat), and each expands its share of the output's columns. Rows are grouped on the device: a cluster looks through
// the indexes of its 256 rows, lists the (adapter, chunk) pairs among them and takes every `groups`-th pair, so that a captured graph
// follows the indexes of the step and nothing is sorted, counted or copied by the host.
// DOWN_T: the weights of the first product lie [columns][ranks] (B in the backward pass) and those of the second [ranks][columns].
template <typename T, typename TY, int RT, int NT, bool DOWN_T, bool WIDE>
__global__ void __launch_bounds__(LORA_THREADS, RT == 1 ? 2 : 1) lora_kernel(const LoraArgs a, int tgroups) {
  constexpr int P = PARTS<T>;                           // parts of x and of the weights
  constexpr int S = sizeof(TY) == 4 ? 3 : 2;            // parts of u
  constexpr int RSTRIDE = 16 * RT + 4;
  __shared__ __align__(16) int s_idx[LORA_ROWS];
  __shared__ short s_count[LORA_ROWS], s_first[LORA_ROWS], s_chunk[LORA_ROWS];
  __shared__ int s_rows[LORA_MAX_CHUNK];
  __shared__ int s_scan[LORA_WARPS];
  extern __shared__ __align__(16) uint8_t dyn[];

  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int cid = blockIdx.x / C, row0 = (cid / a.groups) * LORA_ROWS;
  const int chunk = 8 * NT * tgroups, kwarps = LORA_WARPS / tgroups;
  const int r16 = a.up_segs ? round16(a.up_seg[0].ru) : 0, ucols = a.up_segs * r16, ustride = u_stride(ucols);
  const int pstride = a.rtot;
  float* part = reinterpret_cast<float*>(dyn);                                      // [chunk][rtot]: this CTA's share of u
  uint8_t* second = dyn + ((chunk * pstride * 4 + 15) & ~15);
  float* red = reinterpret_cast<float*>(second);                                    // [kwarps][chunk][RSTRIDE], then
  unsigned short* su = reinterpret_cast<unsigned short*>(second);                   // [S][chunk][ustride]: scaled u in parts

  // ---- which rows go together
  const int rows = min(LORA_ROWS, a.T - row0);
  int id = -2, before = 0, count = 0;
  if (tid < rows) {
    id = a.index ? a.index[row0 + tid] : 0;
    if (id >= a.n && a.status && c == 0) atomicCAS(a.status, 0, EDL_BAD_INDEX);
    if (id < 0 || id >= a.n) id = -1;
  }
  s_idx[tid] = id;
  __syncthreads();
  if (!a.index) {
    before = tid;
    count = rows;
  } else {
    for (int j = 0; j < rows; j += 4) {
      const int4 v = *reinterpret_cast<const int4*>(s_idx + j);      // indexes behind the last row are -2
      const int e0 = v.x == id, e1 = v.y == id, e2 = v.z == id, e3 = v.w == id;
      count += e0 + e1 + e2 + e3;
      before += (j < tid && e0) + (j + 1 < tid && e1) + (j + 2 < tid && e2) + (j + 3 < tid && e3);
    }
  }
  int units = 0;
  if (tid < rows && before == 0 && (id >= 0 || a.copy)) units = (count + chunk - 1) / chunk;
  int at = units;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += v;
  }
  if (lane == 31) s_scan[w] = at;
  __syncthreads();
  int total = 0;
  for (int i = 0; i < LORA_WARPS; ++i) {
    if (i < w) at += s_scan[i];
    total += s_scan[i];
  }
  for (int q = 0; q < units; ++q) {
    s_first[at - units + q] = (short)tid;
    s_chunk[at - units + q] = (short)q;
  }
  s_count[tid] = (short)count;
  __syncthreads();

  const int tg = w % tgroups, kw = w / tgroups;
  bool pending = false;
  for (int unit = cid % a.groups; unit < total; unit += a.groups) {
    const int first = s_first[unit], q0 = s_chunk[unit] * chunk, ad = s_idx[first], m = min(chunk, s_count[first] - q0);
    if (id == ad && before >= q0 && before < q0 + chunk) s_rows[before - q0] = row0 + tid;
    __syncthreads();

    if (ad >= 0) {
      // ---- this CTA's share of u: ranks are the rows of the product, tokens its columns
      const T* wd = reinterpret_cast<const T*>(a.down) + (long long)ad * a.down_adapter;
      const T* xr[NT];
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int tok = (tg * NT + i) * 8 + g;
        xr[i] = tok < m ? reinterpret_cast<const T*>(a.x) + (long long)s_rows[tok] * a.ldx : nullptr;
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
#pragma unroll(P == 1 ? 2 : 1)
          for (int k = seg.c0 + 32 * (c * kwarps + kw); k < seg.c1; k += 32 * C * kwarps) {
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
                mma_parts<P, P>(acc[i][j], wa[i][0], b[0]);
                mma_parts<P, P>(acc[i][j], wa[i][1], b[1]);
              }
            }
          }
          // sum over the warps
#pragma unroll
          for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              const int tok = (tg * NT + j) * 8 + 2 * t4;
              const int lo = 16 * i + (DOWN_T ? 4 * (g >> 1) + (g & 1) : g), hi = lo + (DOWN_T ? 2 : 8);
              float* dst = red + (kw * chunk + tok) * RSTRIDE;
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
            for (int k = 0; k < kwarps; ++k) sum += red[(k * chunk + tok) * RSTRIDE + rank];
            part[tok * pstride + seg.u0 + r0 + rank] = sum;
          }
          __syncthreads();
        }
      }
      // ---- u of all CTAs, scaled, as bf16 parts
      cluster_sync_all();
      const float s = a.scale ? a.scale[ad] : a.scale_all;
      for (int e = tid; e < chunk * ucols; e += LORA_THREADS) {
        const int tok = e / ucols, col = e - tok * ucols, p = col / r16, rank = col - p * r16;
        float v = 0.f;
        if (tok < m && rank < a.up_seg[p].ru) {
          const int pos = tok * pstride + a.up_seg[p].u0 + rank;
          for (int k = 0; k < C; ++k) v += cluster.map_shared_rank(part, k)[pos];
          v *= s;
          if (a.u_out && c == 0) a.u_out[(long long)s_rows[tok] * a.rtot + a.up_seg[p].u0 + rank] = v;
        }
        uint32_t parts[S];
        split<S>(v, parts);
#pragma unroll
        for (int k = 0; k < S; ++k) su[(k * chunk + tok) * ustride + col] = (unsigned short)parts[k];
      }
      if (!a.up_segs && c == 0) {      // only u is asked for
        for (int e = tid; e < m * a.rtot; e += LORA_THREADS) {
          float v = 0.f;
          for (int k = 0; k < C; ++k) v += cluster.map_shared_rank(part, k)[e];
          a.u_out[(long long)s_rows[e / a.rtot] * a.rtot + e % a.rtot] = v * s;
        }
      }
      asm volatile("barrier.cluster.arrive.release;" ::: "memory");
      pending = true;
      __syncthreads();
    }

    // ---- out = y + u B^T over this CTA's share of the columns, 32 per warp and turn
    const T* wu = reinterpret_cast<const T*>(a.up) + (long long)(ad < 0 ? 0 : ad) * a.up_adapter;
    const int kcs = r16 / 16;
    for (int grp = c * LORA_WARPS + w;; grp += C * LORA_WARPS) {
      int p = 0, gi = grp;
      while (p < a.up_segs) {
        const int have = (a.up_seg[p].c1 - a.up_seg[p].c0 + 31) / 32;
        if (gi < have) break;
        gi -= have;
        ++p;
      }
      if (p >= a.up_segs) break;
      const LoraSeg seg = a.up_seg[p];
      const int n0 = seg.c0 + 32 * gi, col = n0 + 8 * t4, ok = seg.c1 - col;      // this lane's eight columns
      uint32_t wb[RT][4][P][2];                                                 // [k16][column tile][part][register]
      for (int tt = 0; tt < m; tt += 16) {
        float acc[4][4];
        float yv[2][8];
        int row[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int tok = tt + 8 * h + g;
          row[h] = tok < m ? s_rows[tok] : -1;
#pragma unroll
          for (int e = 0; e < 8; ++e) yv[h][e] = 0.f;
          if (a.y && row[h] >= 0) {
            const TY* src = reinterpret_cast<const TY*>(a.y) + (long long)row[h] * a.ldy + col;
            if constexpr (WIDE) {
              if (ok >= 8) {
                if constexpr (sizeof(TY) == 2) {
                  const uint4 v = *reinterpret_cast<const uint4*>(src);
                  const uint32_t q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack_bf16x2(q[e]);
                    yv[h][2 * e] = f.x;
                    yv[h][2 * e + 1] = f.y;
                  }
                } else {
                  const float4 v0 = *reinterpret_cast<const float4*>(src), v1 = *reinterpret_cast<const float4*>(src + 4);
                  yv[h][0] = v0.x; yv[h][1] = v0.y; yv[h][2] = v0.z; yv[h][3] = v0.w;
                  yv[h][4] = v1.x; yv[h][5] = v1.y; yv[h][6] = v1.z; yv[h][7] = v1.w;
                }
              }
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e)
                if (e < ok) yv[h][e] = (float)src[e];
            }
          }
        }
        if (ad >= 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
          for (int k0 = 0; k0 < kcs; k0 += RT) {
            if (tt == 0 || kcs > RT) {      // up to RT steps of ranks stay in registers for all rows
#pragma unroll
              for (int i = 0; i < RT; ++i) {
                const int kc = 16 * (k0 + i);
                if constexpr (!DOWN_T) {
#pragma unroll
                  for (int j = 0; j < 4; ++j) {
                    const int n = n0 + 8 * (g >> 1) + 2 * j + (g & 1);
                    uint32_t v[P][2];
                    load_pairs<T, 4, WIDE>(wu + (long long)n * a.ld_up + kc + 4 * t4, n < seg.c1 ? seg.ru - kc - 4 * t4 : 0, v);
#pragma unroll
                    for (int s = 0; s < P; ++s) {
                      wb[i][j][s][0] = v[s][0];
                      wb[i][j][s][1] = v[s][1];
                    }
                  }
                } else {
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const int rank = kc + 4 * (g >> 1) + (g & 1) + 2 * h;
                    uint32_t v[P][4];
                    load_pairs<T, 8, WIDE>(wu + (long long)rank * a.ld_up + col, rank < seg.ru ? ok : 0, v);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                      for (int s = 0; s < P; ++s) wb[i][j][s][h] = turn(v[s][j]);
                  }
                }
              }
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              if (k0 + i >= kcs) break;
              uint32_t ua[S][4];
#pragma unroll
              for (int s = 0; s < S; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  // rows behind the chunk (chunks of 8) repeat its first ones: their products go nowhere
                  const int tok = (tt + 8 * h + g) & (chunk - 1);
                  const uint2 v = *reinterpret_cast<const uint2*>(su + (s * chunk + tok) * ustride + p * r16 + 16 * (k0 + i) + 4 * t4);
                  ua[s][h] = v.x;
                  ua[s][2 + h] = v.y;
                }
#pragma unroll
              for (int j = 0; j < 4; ++j) mma_parts<S, P>(acc[j], ua, wb[i][j]);
            }
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            yv[0][2 * j] += acc[j][0];
            yv[0][2 * j + 1] += acc[j][1];
            yv[1][2 * j] += acc[j][2];
            yv[1][2 * j + 1] += acc[j][3];
          }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (row[h] < 0) continue;
          TY* dst = reinterpret_cast<TY*>(a.out) + (long long)row[h] * a.ldo + col;
          if constexpr (WIDE) {
            if (ok >= 8) {
              if constexpr (sizeof(TY) == 2) {
                *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(yv[h][0], yv[h][1]), pack_bf16x2(yv[h][2], yv[h][3]),
                                                            pack_bf16x2(yv[h][4], yv[h][5]), pack_bf16x2(yv[h][6], yv[h][7]));
              } else {
                *reinterpret_cast<float4*>(dst) = make_float4(yv[h][0], yv[h][1], yv[h][2], yv[h][3]);
                *reinterpret_cast<float4*>(dst + 4) = make_float4(yv[h][4], yv[h][5], yv[h][6], yv[h][7]);
              }
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (e < ok) {
                if constexpr (sizeof(TY) == 2) dst[e] = __float2bfloat16_rn(yv[h][e]);
                else dst[e] = yv[h][e];
              }
          }
        }
      }
    }
    __syncthreads();      // rows and parts of u make way for the next unit
  }
  if (pending) asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // no CTA leaves while its parts are read
}

template <typename T, typename TY, int RT, int NT, bool DOWN_T, bool WIDE>
int launch_lora(const LoraArgs& a, int cluster, int tgroups, int smem, cudaStream_t stream) {
  auto* k = lora_kernel<T, TY, RT, NT, DOWN_T, WIDE>;
  if (smem > 48 * 1024 && check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "lora shared memory")) return -1;
  cudaLaunchConfig_t cfg{};
  const long long blocks = (a.T + LORA_ROWS - 1) / LORA_ROWS;
  cfg.gridDim = dim3((unsigned)(blocks * a.groups * cluster));
  cfg.blockDim = dim3(LORA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k, a, tgroups), "lora launch");
}

// ------------------------------------------------------------------------------------------------------------- gradients
struct GradJob {
  const void* z;         // [T, *] rows: x for dA, dy for dB
  const float* p;        // [T, rtot]: g for dA, scaled u for dB
  void* out;
  long long ldz, out_adapter, ld_out;
  int c0, c1, u0, ru;    // columns of z, ranks
  int tiles;             // column tiles x rank passes
  int across;            // out lies [column][rank] (dB) instead of [rank][column] (dA)
};

struct GradArgs {
  const int* index;
  int T, n, rtot, jobs, out_f32, accumulate;
  GradJob job[LORA_SEGS + 1];
};

constexpr int GRAD_COLS = 256, GRAD_LIST = 1024;

// out[rank, col] (+)= sum over the adapter's rows t of p[t, rank] z[t, col]: rank x 256 columns per cluster, the rows cut over its
// CTAs. z is read once, along its rows, and turned in registers, as is p. A CTA's two row halves (warps 0-3, 4-7) are
// added through shared memory, the CTAs' sums through each other's, both in a fixed order; each CTA writes its share of the tile.
template <typename T, int S, int RT, bool WIDE>
__global__ void __launch_bounds__(LORA_THREADS, 1) lora_grad_kernel(const GradArgs a) {
  constexpr int P = PARTS<T>;
  constexpr int GSTRIDE = GRAD_COLS + 4;
  __shared__ int s_rows[GRAD_LIST];
  __shared__ int s_scan[LORA_WARPS];
  extern __shared__ __align__(16) float tile[];      // [16 RT][GSTRIDE]
  cg::cluster_group cluster = cg::this_cluster();
  const int C = cluster.num_blocks(), c = cluster.block_rank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, g = lane >> 2, t4 = lane & 3;
  const int cid = blockIdx.x / C, ad = blockIdx.y;
  int jb = 0, ti = cid;
  while (jb + 1 < a.jobs && ti >= a.job[jb].tiles) ti -= a.job[jb++].tiles;
  const GradJob job = a.job[jb];
  const int passes = (job.ru + 16 * RT - 1) / (16 * RT);
  const int r0 = (ti % passes) * 16 * RT, col0 = job.c0 + (ti / passes) * GRAD_COLS;
  const int cw = w & 3, half = w >> 2, colw = col0 + cw * 64;
  const T* z = reinterpret_cast<const T*>(job.z);

  float acc[RT][8][4];
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;

  const long long per = (((long long)a.T + C - 1) / C + 15) / 16 * 16, lo = min((long long)a.T, per * c), hi = min((long long)a.T, lo + per);
  for (long long at = lo; at < hi; at += GRAD_LIST) {
    const int len = (int)min((long long)GRAD_LIST, hi - at);
    int found = len;
    if (a.index) {      // the adapter's rows among these, in order
      int mine[4], cnt = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = tid * 4 + i;
        mine[i] = t < len && a.index[at + t] == ad;
        cnt += mine[i];
      }
      int pos = cnt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, pos, o);
        if (lane >= o) pos += v;
      }
      if (lane == 31) s_scan[w] = pos;
      __syncthreads();
      found = 0;
      for (int i = 0; i < LORA_WARPS; ++i) {
        if (i < w) pos += s_scan[i];
        found += s_scan[i];
      }
      pos -= cnt;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (mine[i]) s_rows[pos++] = (int)(at + tid * 4 + i);
      __syncthreads();
    }
#pragma unroll(P == 1 && RT == 1 ? 2 : 1)
    for (int t0 = 16 * half; t0 < found; t0 += 32) {
      long long row[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int t = t0 + 8 * h + g;
        row[h] = t < found ? (a.index ? (long long)s_rows[t] : at + t) : -1;
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
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        uint32_t pa[S][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)          // rows of the product: ranks; its inner index: tokens
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int rank = r0 + 16 * i + 8 * h + 2 * t4;
            float f0 = 0.f, f1 = 0.f;
            if (row[k] >= 0) {
              const float* src = job.p + row[k] * a.rtot + job.u0 + rank;
              if (rank < job.ru) f0 = src[0];
              if (rank + 1 < job.ru) f1 = src[1];
            }
            uint32_t p0[S], p1[S];
            split<S>(f0, p0);
            split<S>(f1, p1);
#pragma unroll
            for (int s = 0; s < S; ++s) pa[s][h + 2 * k] = turn(p0[s] | (p1[s] << 16));
          }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (S == 3) {      // the tensor cores cut sums off: 32-bit results take a few products at a time and round the sum
            float few[4] = {0.f, 0.f, 0.f, 0.f};
            mma_parts<S, P>(few, pa, zb[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] += few[e];
          } else {
            mma_parts<S, P>(acc[i][j], pa, zb[j]);
          }
        }
      }
    }
    if (a.index) __syncthreads();
  }

  // ---- sums over the halves and the CTAs
  auto place = [&](int i, int j, int e) {      // position of accumulator e in the tile
    const int rank = 16 * i + g + (e >> 1) * 8;
    const int col = cw * 64 + 32 * (j >> 2) + 8 * t4 + 2 * (j & 3) + (e & 1);
    return rank * GSTRIDE + col;
  };
  if (half == 1)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[place(i, j, e)] = acc[i][j][e];
  __syncthreads();
  if (half == 0)
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) tile[place(i, j, e)] += acc[i][j][e];
  cluster_sync_all();
  const int all = 16 * RT * GRAD_COLS, share = (all + C - 1) / C;
  for (int e = c * share + tid; e < min(all, (c + 1) * share); e += LORA_THREADS) {
    const int rank = job.across ? e % (16 * RT) : e / GRAD_COLS, col = job.across ? e / (16 * RT) : e % GRAD_COLS;
    if (r0 + rank >= job.ru || col0 + col >= job.c1) continue;
    float v = 0.f;
    for (int k = 0; k < C; ++k) v += cluster.map_shared_rank(tile, k)[rank * GSTRIDE + col];
    const long long pos = (long long)ad * job.out_adapter + (job.across ? (long long)(col0 + col) * job.ld_out + r0 + rank
                                                                         : (long long)(job.u0 + r0 + rank) * job.ld_out + col0 + col);
    if (a.out_f32) {
      float* o = reinterpret_cast<float*>(job.out) + pos;
      *o = a.accumulate ? *o + v : v;
    } else {
      reinterpret_cast<__nv_bfloat16*>(job.out)[pos] = __float2bfloat16_rn(v);
    }
  }
  cluster_sync_all();      // no CTA leaves while its tile is read
}

template <typename T, int S, int RT, bool WIDE>
int launch_grad(const GradArgs& a, int tiles, int cluster, cudaStream_t stream) {
  auto* k = lora_grad_kernel<T, S, RT, WIDE>;
  const int smem = 16 * RT * (GRAD_COLS + 4) * 4;
  if (smem > 48 * 1024 && check_cuda(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem), "lora gradient shared memory"))
    return -1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)a.n);
  cfg.blockDim = dim3(LORA_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, k, a), "lora gradient launch");
}

bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

}  // namespace
}  // namespace edl

using namespace edl;

// x [T, K], y and out [T, N] (y null: the adapters' part alone; y == out: in place), row strides in elements. widths: columns of the
// `parts` parts of N. a: [n][parts * r][K], b: [n][N][r] with strides. backward = 0: out = y + s (x a^T) b^T, u_out [T, parts * r] (may
// be null) takes s x a^T. backward = 1: x is dy [T, N], out dx [T, K] (null: u_out alone), y null; u_out takes s dy b.
// index [T] int32 or null (adapter 0 everywhere), scale [n] fp32 or null (scale_all). x_f32: x and the weights are fp32 (then
// y and out too), else bf16; y_f32: type of y and out. Indexes from n on set the status word and count as none.
EDL_HOST_API int edl_lora_apply(const void* x, long long ldx, const void* y, long long ldy, void* out, long long ldo, const void* a,
                                long long a_adapter, long long lda, const void* b, long long b_adapter, long long ldb,
                                const int* index, const float* scale, float scale_all, float* u_out, int T, int K, int N, int n, int r,
                                int parts, const int* widths, int x_f32, int y_f32, int backward, int* status, void* stream) {
  if (T <= 0) return 0;
  if (K <= 0 || N <= 0 || n <= 0 || r <= 0 || parts < 1 || parts > LORA_SEGS || r > 512 / parts) {
    set_last_error("edl_lora_apply: needs sizes above 0, up to %d parts and parts x rank up to 512", LORA_SEGS);
    return -1;
  }
  if ((x_f32 && !y_f32) || (backward && x_f32 != y_f32) || (backward && y) || (!out && !(backward && u_out))) {
    set_last_error("edl_lora_apply: fp32 inputs give fp32 results; the backward form takes one type and no y");
    return -1;
  }
  LoraArgs g{};
  g.x = x; g.ldx = ldx; g.y = y; g.ldy = ldy; g.out = out; g.ldo = ldo;
  g.index = index; g.scale = scale; g.scale_all = scale_all; g.u_out = u_out; g.status = status;
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
    g.up_segs = out ? 1 : 0;
    g.up_seg[0] = whole;
  }
  const int va = x_f32 ? 4 : 8, vy = y_f32 ? 4 : 8;      // elements in 16 bytes
  wide = wide && ldx % va == 0 && aligned(x, 16) && aligned(a, 16) && lda % va == 0 && a_adapter % va == 0 && aligned(b, x_f32 ? 16 : 8) &&
         ldb % 4 == 0 && b_adapter % 4 == 0 && (!y || (ldy % vy == 0 && aligned(y, 16))) && (!out || (ldo % vy == 0 && aligned(out, 16)));

  // Chunks of 8 rows while the rows of a step fit one look (few rows per adapter, many clusters), of 64 above; wide ranks keep
  // less so that u fits shared memory.
  const int rt = wide && !x_f32 && (backward ? (r > 16 || parts * r > 16) : parts * r > 16) ? 4 : 1;
  int nt = 1, tgroups = 1;
  if (T > LORA_ROWS && g.rtot <= 256) {
    nt = 4;
    tgroups = g.rtot <= 128 ? 2 : 1;
  }
  const int chunk = 8 * nt * tgroups, cluster = 8;
  const int in_block = T < LORA_ROWS ? T : LORA_ROWS;
  const long long most = (long long)(index ? (n < in_block ? n + 1 : in_block) : 1) + in_block / chunk;      // pairs among a block's rows
  const int blocks = (T + LORA_ROWS - 1) / LORA_ROWS;
  int groups = 128 / blocks;
  if (groups < LORA_ROWS / chunk) groups = LORA_ROWS / chunk;
  if (groups > most) groups = (int)most;
  if (groups > in_block) groups = in_block;
  g.groups = groups;
  const int s = y_f32 ? 3 : 2;
  int ucols = g.up_segs ? g.up_segs * round16(g.up_seg[0].ru) : 0;
  const int red = (LORA_WARPS / tgroups) * chunk * (16 * rt + 4) * 4, su = s * chunk * u_stride(ucols) * 2;
  const int smem = ((chunk * g.rtot * 4 + 15) & ~15) + (red > su ? red : su);
  cudaStream_t st = (cudaStream_t)stream;
#define EDL_LORA_NT(TX, TO, RTV, BW, W)                                                     \
  return nt == 1 ? launch_lora<TX, TO, RTV, 1, BW, W>(g, cluster, tgroups, smem, st)        \
                 : launch_lora<TX, TO, RTV, 4, BW, W>(g, cluster, tgroups, smem, st)
#define EDL_LORA_BF(TO, BW)                                             \
  {                                                                     \
    if (!wide) { EDL_LORA_NT(__nv_bfloat16, TO, 1, BW, false); }        \
    if (rt == 4) { EDL_LORA_NT(__nv_bfloat16, TO, 4, BW, true); }       \
    EDL_LORA_NT(__nv_bfloat16, TO, 1, BW, true);                        \
  }
#define EDL_LORA_F32(BW)                                        \
  {                                                             \
    if (!wide) { EDL_LORA_NT(float, float, 1, BW, false); }     \
    EDL_LORA_NT(float, float, 1, BW, true);                     \
  }
  if (x_f32) {
    if (backward) EDL_LORA_F32(true) else EDL_LORA_F32(false)
  }
  if (backward) EDL_LORA_BF(__nv_bfloat16, true)
  if (y_f32) EDL_LORA_BF(float, false)
  EDL_LORA_BF(__nv_bfloat16, false)
#undef EDL_LORA_NT
#undef EDL_LORA_BF
#undef EDL_LORA_F32
}

// da [n][parts * r][K] (+)= g^T x and db [n][N][r] (+)= dy^T u over each adapter's rows (either may be null). g, u: fp32 [T, parts * r]
// as edl_lora_apply leaves them. out_f32: type of da and db; accumulate (fp32 only): add to them. Adapters without rows get zeros.
EDL_HOST_API int edl_lora_grads(const void* x, long long ldx, const void* dy, long long ldy, const float* g, const float* u,
                                const int* index, void* da, long long da_adapter, long long ld_da, void* db, long long db_adapter,
                                long long ld_db, int T, int K, int N, int n, int r, int parts, const int* widths, int in_f32,
                                int out_f32, int accumulate, void* stream) {
  if (K <= 0 || N <= 0 || n <= 0 || r <= 0 || parts < 1 || parts > LORA_SEGS || r > 512 / parts || n > 65535 || (!index && n != 1 && T > 0)) {
    set_last_error("edl_lora_grads: needs sizes above 0, up to %d parts, parts x rank up to 512, up to 65535 adapters, one without an index", LORA_SEGS);
    return -1;
  }
  if ((in_f32 && !out_f32) || (accumulate && !out_f32)) {
    set_last_error("edl_lora_grads: fp32 inputs give fp32 gradients, and only those are accumulated into");
    return -1;
  }
  GradArgs a{};
  a.index = index; a.T = T < 0 ? 0 : T; a.n = n; a.rtot = parts * r; a.out_f32 = out_f32; a.accumulate = accumulate;
  const int va = in_f32 ? 4 : 8;
  bool wide = true;
  const int rt = in_f32 || (da ? parts * r : r) <= 16 ? 1 : 4;      // ranks that one pass over the rows takes
  auto tiles_of = [&](int cols, int ru) { return ((cols + GRAD_COLS - 1) / GRAD_COLS) * ((ru + 16 * rt - 1) / (16 * rt)); };
  int tiles = 0;
  if (da) {
    a.job[a.jobs++] = GradJob{x, g, da, ldx, da_adapter, ld_da, 0, K, 0, parts * r, tiles_of(K, parts * r), 0};
    wide = wide && K % 8 == 0 && ldx % va == 0 && aligned(x, 16);
  }
  if (db) {
    int c0 = 0;
    for (int p = 0; p < parts; ++p) {
      a.job[a.jobs++] = GradJob{dy, u, db, ldy, db_adapter, ld_db, c0, c0 + widths[p], p * r, r, tiles_of(widths[p], r), 1};
      c0 += widths[p];
      wide = wide && widths[p] % 8 == 0;
    }
    if (c0 != N) {
      set_last_error("edl_lora_grads: the parts have %d columns, the output %d", c0, N);
      return -1;
    }
    wide = wide && ldy % va == 0 && aligned(dy, 16);
  }
  if (!a.jobs) return 0;
  for (int j = 0; j < a.jobs; ++j) tiles += a.job[j].tiles;
  int cluster = 8;      // rows of a cluster are cut into as many shares; short inputs need fewer
  while (cluster > 1 && a.T < cluster * 32) cluster /= 2;
  cudaStream_t st = (cudaStream_t)stream;
  if (in_f32) return wide ? launch_grad<float, 3, 1, true>(a, tiles, cluster, st) : launch_grad<float, 3, 1, false>(a, tiles, cluster, st);
#define EDL_LORA_GRAD(SV)                                                                        \
  {                                                                                              \
    if (rt == 4) return wide ? launch_grad<__nv_bfloat16, SV, 4, true>(a, tiles, cluster, st)    \
                             : launch_grad<__nv_bfloat16, SV, 4, false>(a, tiles, cluster, st);  \
    return wide ? launch_grad<__nv_bfloat16, SV, 1, true>(a, tiles, cluster, st)                 \
                : launch_grad<__nv_bfloat16, SV, 1, false>(a, tiles, cluster, st);               \
  }
  if (out_f32) EDL_LORA_GRAD(3)
  EDL_LORA_GRAD(2)
#undef EDL_LORA_GRAD
}
