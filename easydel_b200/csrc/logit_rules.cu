// Rules for the next token, applied to the logits of a step's rows in one pass: penalties for tokens that were seen, biases of single
// tokens, grammar masks of one bit per token.
//
//   z = logit;  count c > 0:  z = (z > 0 ? z / repetition : z * repetition) - presence - frequency * c
//   z += sum of the row's biases for the token (a sum of minus infinity forbids the token, whatever z is)
//   z = minus infinity where the row's mask has no bit (whatever z is)
//
// What bounds it is traffic: two or four bytes in, four out, four of counts where a row has penalties. A row is cut into slices, a CTA
// each, and a thread asks for all it needs of one or two groups of eight values before it uses any of it. Groups that the mask forbids
// entirely are written without being read (of a grammar's states most allow a few tokens). Biases are few: a CTA looks through
// its row's list once, and drops what falls into its slice into shared memory behind a bit per value. Groups without counts, biases or
// forbidden tokens skip those steps.
//
// One row of 32000: 3.2 us, 7 rows of 50257 with counts: 5 us (launch and one round of loads); 64 rows of 128256, half of them with counts and
// half with masks: 20 us, 66 MB at 3.3 TB/s (rounds of CTAs of unlike work, each of which waits for its mask, then its values, then its
// biases; biases asked for before the values took registers and were no faster); 256 fp32 rows of 151936: 75 us, 436 MB at 5.8 TB/s.
#include "common.cuh"

namespace edl {
namespace {

constexpr int RULE_THREADS = 128;      // 256: 64 x 128256 bf16 21.1 us (20.3), 256 x 151936 fp32 76.3 us (75)

struct RuleArgs {
  const void* logits;
  void* out;
  long long ld, ldo;
  int V, slices;
  const int* counts;
  long long ld_counts;
  const int* count_rows;
  int slots;
  const float *presence, *frequency, *repetition;
  const int* bias_ptr;
  const int* bias_ids;
  const float* bias_values;
  int bias_n;
  const uint32_t* bits;
  long long ld_bits;
  const int* mask_rows;
  int masks;
  int* status;
};

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  if constexpr (sizeof(T) == 2) return __bfloat162float(v);
  else return v;
}

// WIDE: a thread's eight values are neighbours that start on 16 bytes, in rows of any length (`shift` values of a row's first group belong
// to the row before it); else they lie a CTA's threads apart, so that rows of any alignment are read in whole lines.
template <typename T, typename TO, bool WIDE, int GROUPS>
__global__ void __launch_bounds__(RULE_THREADS) rules_kernel(const RuleArgs a) {
  constexpr int SLICE = RULE_THREADS * GROUPS * 8;
  extern __shared__ __align__(16) float s_add[];                                  // [SLICE], set where the bit is
  uint32_t* s_bit = reinterpret_cast<uint32_t*>(s_add + SLICE);                   // [SLICE / 32]
  const int row = blockIdx.x / a.slices, tid = threadIdx.x;
  const T* src = reinterpret_cast<const T*>(a.logits) + row * a.ld;
  TO* dst = reinterpret_cast<TO*>(a.out) + row * a.ldo;
  const int shift = WIDE ? (int)(row * a.ld & 7) : 0;
  const int v0 = (int)(blockIdx.x % a.slices) * SLICE - shift;

  int mrow = a.mask_rows ? a.mask_rows[row] : a.bits ? row : -1;
  int slot = !a.counts ? -1 : a.count_rows ? a.count_rows[row] : row;
  const float pres = a.presence ? a.presence[row] : 0.f, freq = a.frequency ? a.frequency[row] : 0.f;
  const float rep = a.repetition ? a.repetition[row] : 1.f;
  if (mrow >= a.masks || slot >= a.slots) {
    if (a.status && tid == 0) atomicCAS(a.status, 0, EDL_BAD_INDEX);
    if (mrow >= a.masks) mrow = -1;
    if (slot >= a.slots) slot = -1;
  }
  const int* cnt = slot >= 0 && (pres != 0.f || freq != 0.f || rep != 1.f) ? a.counts + (long long)slot * a.ld_counts : nullptr;
  const uint8_t* bits = mrow >= 0 ? reinterpret_cast<const uint8_t*>(a.bits + (long long)mrow * a.ld_bits) : nullptr;
  const bool cnt_wide = WIDE && cnt && (reinterpret_cast<uintptr_t>(cnt - shift) & 15) == 0;

  auto index = [&](int grp, int j) { return WIDE ? v0 + (grp * RULE_THREADS + tid) * 8 + j : v0 + (grp * 8 + j) * RULE_THREADS + tid; };
  uint32_t allow[GROUPS], valid[GROUPS];      // of a group's values: allowed, in the row
#pragma unroll
  for (int q = 0; q < GROUPS; ++q) {
    const int v = index(q, 0);
    valid[q] = 0;
    if (WIDE && v >= 0 && v + 8 <= a.V) {
      valid[q] = allow[q] = 0xff;
      if (bits) {
        allow[q] = bits[v >> 3];
        if (shift) allow[q] = (allow[q] | (uint32_t)bits[(v + 7) >> 3] << 8) >> (v & 7) & 0xff;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) valid[q] |= (index(q, j) >= 0 && index(q, j) < a.V ? 1u : 0u) << j;
      allow[q] = valid[q];
      if (bits) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (valid[q] >> j & 1) allow[q] &= ~((~(uint32_t)bits[index(q, j) >> 3] >> (index(q, j) & 7) & 1) << j);
      }
    }
  }
  float z[GROUPS][8];
  int seen[GROUPS][8];
#pragma unroll
  for (int q = 0; q < GROUPS; ++q) {
    const int v = index(q, 0);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      z[q][j] = 0.f;
      seen[q][j] = 0;
    }
    if (WIDE && valid[q] == 0xff) {
      if (allow[q]) {
        if constexpr (sizeof(T) == 2) {
          const uint4 x = *reinterpret_cast<const uint4*>(src + v);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack_bf16x2(w[j]);
            z[q][2 * j] = f.x;
            z[q][2 * j + 1] = f.y;
          }
        } else {
          const float4 x = *reinterpret_cast<const float4*>(src + v), y = *reinterpret_cast<const float4*>(src + v + 4);
          z[q][0] = x.x; z[q][1] = x.y; z[q][2] = x.z; z[q][3] = x.w;
          z[q][4] = y.x; z[q][5] = y.y; z[q][6] = y.z; z[q][7] = y.w;
        }
        if (cnt_wide) {
          const int4 x = *reinterpret_cast<const int4*>(cnt + v), y = *reinterpret_cast<const int4*>(cnt + v + 4);
          seen[q][0] = x.x; seen[q][1] = x.y; seen[q][2] = x.z; seen[q][3] = x.w;
          seen[q][4] = y.x; seen[q][5] = y.y; seen[q][6] = y.z; seen[q][7] = y.w;
        } else if (cnt) {
#pragma unroll
          for (int j = 0; j < 8; ++j) seen[q][j] = cnt[v + j];
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (allow[q] >> j & 1) {
          z[q][j] = to_float(src[index(q, j)]);
          if (cnt) seen[q][j] = cnt[index(q, j)];
        }
    }
  }

  if (a.bias_ptr) {
    for (int i = tid; i < SLICE / 32; i += RULE_THREADS) s_bit[i] = 0;
    __syncthreads();
    int lo = a.bias_ptr[row], hi = a.bias_ptr[row + 1];
    if (lo < 0 || hi > a.bias_n || lo > hi) {
      if (a.status && tid == 0) atomicCAS(a.status, 0, EDL_BAD_INDEX);
      lo = hi = 0;
    }
    for (int e = lo + tid; e < hi; e += RULE_THREADS) {
      const int id = a.bias_ids[e];
      if (id < 0 || id >= a.V) {
        if (a.status) atomicCAS(a.status, 0, EDL_BAD_INDEX);
        continue;
      }
      if (id < v0 || id >= v0 + SLICE || (e > lo && a.bias_ids[e - 1] == id)) continue;
      float sum = a.bias_values[e];                                       // the first of a token's entries adds up the rest, in order
      for (int f = e + 1; f < hi && a.bias_ids[f] == id; ++f) sum += a.bias_values[f];
      s_add[id - v0] = sum;
      atomicOr(&s_bit[(id - v0) >> 5], 1u << ((id - v0) & 31));
    }
    __syncthreads();
  }

#pragma unroll
  for (int q = 0; q < GROUPS; ++q) {
    if (cnt) {
      int any = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) any = max(any, seen[q][j]);
      if (any > 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (seen[q][j] > 0) {
            float x = z[q][j];
            if (rep != 1.f) x = x > 0.f ? x / rep : x * rep;
            z[q][j] = x - (pres + freq * (float)seen[q][j]);
          }
      }
    }
    if (a.bias_ptr) {
      uint32_t touched = 0;
      if constexpr (WIDE) {
        const int at = index(q, 0) - v0;
        touched = s_bit[at >> 5] >> (at & 31) & 0xff;
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) touched |= (s_bit[(index(q, j) - v0) >> 5] >> ((index(q, j) - v0) & 31) & 1) << j;
      }
      if (touched) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (touched >> j & 1) {
            const float add = s_add[index(q, j) - v0];
            z[q][j] = add == -INFINITY ? add : z[q][j] + add;
          }
      }
    }
    if (allow[q] != 0xff) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (!(allow[q] >> j & 1)) z[q][j] = -INFINITY;
    }
    if (WIDE && valid[q] == 0xff) {
      const int v = index(q, 0);
      if constexpr (sizeof(TO) == 2) {
        *reinterpret_cast<uint4*>(dst + v) = make_uint4(pack_bf16x2(z[q][0], z[q][1]), pack_bf16x2(z[q][2], z[q][3]),
                                                        pack_bf16x2(z[q][4], z[q][5]), pack_bf16x2(z[q][6], z[q][7]));
      } else {
        *reinterpret_cast<float4*>(dst + v) = make_float4(z[q][0], z[q][1], z[q][2], z[q][3]);
        *reinterpret_cast<float4*>(dst + v + 4) = make_float4(z[q][4], z[q][5], z[q][6], z[q][7]);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (valid[q] >> j & 1) {
          if constexpr (sizeof(TO) == 2) dst[index(q, j)] = __float2bfloat16_rn(z[q][j]);
          else dst[index(q, j)] = z[q][j];
        }
    }
  }
}

}  // namespace
}  // namespace edl

using namespace edl;

// logits, out: [R, V] (bf16 or fp32 each; the same memory for in place). counts [slots, *] int32 with a row per entry of count_rows (negative:
// no penalties; null: row r), presence / frequency / repetition fp32 [R] or null. bias_ptr [R + 1], ids (sorted within a row) and values
// of bias_n entries, or null. bits: [masks, ld_bits] words, mask_rows [R] (negative: no mask; null: row r).
EDL_HOST_API int edl_adjust_logits(const void* logits, int in_f32, long long ld, void* out, int out_f32, long long ldo, int R, int V,
                                   const int* counts, long long ld_counts, int slots, const int* count_rows, const float* presence,
                                   const float* frequency, const float* repetition, const int* bias_ptr, const int* bias_ids,
                                   const float* bias_values, int bias_n, const void* bits, long long ld_bits, int masks,
                                   const int* mask_rows, int* status, void* stream) {
  if (R <= 0 || V <= 0) return 0;
  if (logits == out && (in_f32 != out_f32 || ld != ldo)) {
    set_last_error("edl_adjust_logits: in place needs one type and one stride");
    return -1;
  }
  auto odd = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; };
  // rows of both sides start at the same place within a group of eight
  const bool wide = ld % 8 == ldo % 8 && !odd(logits) && !odd(out);
  // two groups per thread while that leaves eight CTAs per SM, else one (and one where values lie apart, which takes more registers):
  // 256 x 151936 fp32 79 us with two, 85 with one; 1 x 32000 bf16 2.5 us with two, 2.2 with one (both in CTAs of 256)
  const int groups = wide && (long long)R * ((V + 2047) / 2048) >= 8LL * sm_count() ? 2 : 1, slice = RULE_THREADS * groups * 8;
  RuleArgs a{logits, out, ld, ldo, V, (int)(((long long)V + (wide ? 7 : 0) + slice - 1) / slice), counts, ld_counts, count_rows, slots, presence, frequency,
             repetition, bias_ptr, bias_ids, bias_values, bias_n, (const uint32_t*)bits, ld_bits, bits ? mask_rows : nullptr, masks, status};
  const long long ctas = (long long)R * a.slices;
  if (ctas > 0x7fffffffLL) {
    set_last_error("edl_adjust_logits: too many values for one launch");
    return -1;
  }
  const int smem = bias_ptr ? slice * 4 + slice / 8 : 0;
  cudaStream_t st = (cudaStream_t)stream;
#define EDL_RULES(TI, TO)                                                                                     \
  {                                                                                                           \
    if (!wide) rules_kernel<TI, TO, false, 1><<<(unsigned)ctas, RULE_THREADS, smem, st>>>(a);                 \
    else if (groups == 1) rules_kernel<TI, TO, true, 1><<<(unsigned)ctas, RULE_THREADS, smem, st>>>(a);       \
    else rules_kernel<TI, TO, true, 2><<<(unsigned)ctas, RULE_THREADS, smem, st>>>(a);                        \
  }
  if (in_f32 && out_f32) EDL_RULES(float, float)
  else if (in_f32) EDL_RULES(float, __nv_bfloat16)
  else if (out_f32) EDL_RULES(__nv_bfloat16, float)
  else EDL_RULES(__nv_bfloat16, __nv_bfloat16)
#undef EDL_RULES
  return check_cuda(cudaGetLastError(), "adjust_logits launch");
}
