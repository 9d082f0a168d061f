// One score row per thread: the row's extreme, its exponentials into TMEM, the
// rescaling of its output row. Shared by the tensor-memory attention kernels.
#pragma once

#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

#include "sm100_ptx.cuh"

namespace fa {

constexpr int BN = 128;  // keys per K/V tile = columns of a score row

// Max over the valid columns [lo, nvalid) of a raw score row (min when the scale is
// negative), so that extreme * scale is the row max of the scaled scores.
__device__ __forceinline__ float row_extreme(const uint32_t* s, int nvalid, bool full, bool pos, int lo = 0) {
  if (full) {
    float a0 = __uint_as_float(s[0]), a1 = __uint_as_float(s[1]);
    float a2 = __uint_as_float(s[2]), a3 = __uint_as_float(s[3]);
    if (pos) {
#pragma unroll
      for (int c = 4; c < BN; c += 8) {
        a0 = fmax3(a0, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
        a1 = fmax3(a1, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
        if (c + 4 < BN) {
          a2 = fmax3(a2, __uint_as_float(s[c + 4]), __uint_as_float(s[c + 5]));
          a3 = fmax3(a3, __uint_as_float(s[c + 6]), __uint_as_float(s[c + 7]));
        }
      }
      return fmax3(fmaxf(a0, a1), a2, a3);
    }
#pragma unroll
    for (int c = 4; c < BN; c += 8) {
      a0 = fmin3(a0, __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
      a1 = fmin3(a1, __uint_as_float(s[c + 2]), __uint_as_float(s[c + 3]));
      if (c + 4 < BN) {
        a2 = fmin3(a2, __uint_as_float(s[c + 4]), __uint_as_float(s[c + 5]));
        a3 = fmin3(a3, __uint_as_float(s[c + 6]), __uint_as_float(s[c + 7]));
      }
    }
    return fmin3(fminf(a0, a1), a2, a3);
  }
  float a0 = pos ? -INFINITY : INFINITY;
#pragma unroll
  for (int c = 0; c < BN; ++c) {
    const float x = __uint_as_float(s[c]);
    if (c >= lo && c < nvalid) a0 = pos ? fmaxf(a0, x) : fminf(a0, x);
  }
  return a0;
}

// P = exp2(s * sl2 + neg_m) for one 128-column score row, rounded to fp16 and
// stored into TMEM columns [tS, tS + 64) (two fp16 per column); returns the
// fp32 row sum in two partial sums. EMU_PAIRS of every 4 column pairs use the
// FMA-pipe polynomial, the rest MUFU (balances the two pipes). MASK zeroes columns outside [lo,
// nvalid) (last key tile).
// TWO_STEPS rounds the product before neg_m is added, as a maximum that was
// computed by itself was rounded.
// When half_bar is non-zero, the first half of P (keys 0..63) is published on
// it as soon as it is stored (after before_half() has run), so the tensor core
// can start on those keys while the second half is computed. before_store()
// runs once, after the first half's exponentials and before any of P is stored.
template <int EMU_PAIRS, bool MASK, bool TWO_STEPS = false, typename BeforeHalf, typename BeforeStore>
__device__ __forceinline__ void row_exp_store(const uint32_t* s, float sl2, float neg_m, int nvalid,
                                              uint32_t tS, float& sum0, float& sum1, uint32_t half_bar,
                                              BeforeHalf&& before_half, BeforeStore&& before_store, int lo = 0) {
  const uint64_t sl2x2 = f2_pack(sl2, sl2);
  const uint64_t negm2 = f2_pack(neg_m, neg_m);
  uint64_t acc0 = f2_pack(0.f, 0.f), acc1 = acc0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t pk[32];
#pragma unroll
    for (int c2 = 0; c2 < 32; ++c2) {
      const int c = h * 64 + 2 * c2;
      float x0, x1, e0, e1;
      if (TWO_STEPS) {
        x0 = __fadd_rn(__fmul_rn(__uint_as_float(s[c]), sl2), neg_m);
        x1 = __fadd_rn(__fmul_rn(__uint_as_float(s[c + 1]), sl2), neg_m);
      } else {
        f2_unpack(f2_fma(f2_pack(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), sl2x2, negm2), x0, x1);
      }
      if ((c2 & 3) < EMU_PAIRS) {
        exp2_poly3_x2(x0, x1, e0, e1);
      } else {
        e0 = ex2_approx(x0);
        e1 = ex2_approx(x1);
      }
      if (MASK) {
        e0 = (c >= lo && c < nvalid) ? e0 : 0.f;
        e1 = (c + 1 >= lo && c + 1 < nvalid) ? e1 : 0.f;
      }
      if (c2 & 1)
        acc1 = f2_add(acc1, f2_pack(e0, e1));
      else
        acc0 = f2_add(acc0, f2_pack(e0, e1));
      pk[c2] = pack_half2(e0, e1);
    }
    if (h == 0) before_store();
    tmem_st32(tS + 32 * h, pk);
    if (h == 0 && half_bar) {
      before_half();
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(half_bar);
    }
  }
  float a, b, c, d;
  f2_unpack(acc0, a, b);
  f2_unpack(acc1, c, d);
  sum0 = a + c;
  sum1 = b + d;
}

// Multiply this thread's TMEM row of O (DP fp32 columns at tO) by factor when
// do_it (warp-uniform).
template <int DP>
__device__ __forceinline__ void rescale_rows(uint32_t tO, bool do_it, float factor) {
  if (!do_it) return;
#pragma unroll
  for (int c = 0; c < DP / 16; ++c) {
    uint32_t o[16];
    tmem_ld16(tO + 16 * c, o);
    tmem_wait_ld();
    reg_fence16(o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
    tmem_st16(tO + 16 * c, o);
  }
}

}  // namespace fa
