// The paged 4-bit key/value cache: byte layout of a page and the conversions
// between its numbers and 16-bit ones. Shared by the kernels that write, read
// and attend to the cache.
//
// A value is code * scale * factor: the code is an e2m1 number (4 bits), the
// scale an e4m3 number shared by 16 neighbouring channels of one token, the
// factor one 32-bit number per kv head. code * scale has at most six
// significant bits and lies in [2^-10, 2688] or is zero, so it is exact in
// fp16: the attention kernels multiply codes by scales in fp16 without a
// rounding and apply the factors in 32 bits (to the scores and the output).
//
// A page holds PAGE = 64 tokens of one kv head in four blocks of 16 tokens.
// Block (D = head dim, all offsets in bytes): K codes [0, 8D), K scales
// [8D, 9D), V codes [9D, 17D), V scales [17D, 18D). A block is contiguous, so
// any run of blocks of a page is one contiguous copy. Inside a block the bytes
// are ordered for the 32 lanes (n = lane / 4, c = lane % 4) of the warp that
// multiplies it with m16n8k16 matrix instructions, so that every shared-memory
// read is one conflict-free 32-lane access and feeds the A fragments directly:
//  * K codes: token t's row of D/2 bytes at t * D/2, channels in order. Lane
//    (n, c) holds channels [c D/4, (c+1) D/4) of tokens n and n + 8.
//  * K scales of token t, group g: with gpl = D/64 groups per lane, byte
//    (t % 8 * 4 + g / gpl) * 2 gpl + t / 8 * gpl + g % gpl.
//  * V codes: channels [n D/8, (n+1) D/8) of token t are D/16 bytes at
//    t/8 * 4D + (n * 4 + t % 8 / 2) * D/8 + t % 2 * D/16: lane (n, c) finds
//    tokens 2c and 2c + 1 of each half block side by side.
//  * V scales of token t, group g: byte (g * 4 + t % 8 / 2) * 4 + t / 8 * 2 + t % 2.
// The low four bits of a code byte are the even channel.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace c4 {

constexpr int PAGE = 64;   // tokens of a page
constexpr int BLOCK = 16;  // tokens of a block

template <int D>
struct Layout {
  static constexpr int KC = 0;
  static constexpr int KS = 8 * D;
  static constexpr int VC = 9 * D;
  static constexpr int VS = 17 * D;
  static constexpr int BLOCK_BYTES = 18 * D;
  static constexpr int PAGE_BYTES = 72 * D;
  static constexpr int GROUPS = D / 16;
  static constexpr int GPL = D / 64;  // K scale groups per lane

  // token t of 16, 16-channel group g
  __host__ __device__ static constexpr int k_code(int t, int g) { return KC + t * (D / 2) + g * 8; }
  __host__ __device__ static constexpr int k_scale(int t, int g) {
    return KS + (t % 8 * 4 + g / GPL) * 2 * GPL + t / 8 * GPL + g % GPL;
  }
  // the D/16 bytes of channels [n D/8, (n+1) D/8)
  __host__ __device__ static constexpr int v_code(int t, int n) {
    return VC + t / 8 * 4 * D + (n * 4 + t % 8 / 2) * (D / 8) + t % 2 * (D / 16);
  }
  __host__ __device__ static constexpr int v_scale(int t, int g) {
    return VS + (g * 4 + t % 8 / 2) * 4 + t / 8 * 2 + t % 2;
  }
};

// Four bytes of codes -> four pairs of fp16 (low code of a byte in the low half).
__device__ __forceinline__ void codes_to_half2(uint32_t w, uint32_t* o) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(o[0]), "=r"(o[1]), "=r"(o[2]), "=r"(o[3])
      : "r"(w));
}
// Two e4m3 scales in the low 16 bits of w -> a pair of fp16.
__device__ __forceinline__ uint32_t scales_to_half2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
// Nearest e4m3 of x (ties to even, |x| <= 448), as its byte.
__device__ __forceinline__ uint32_t to_e4m3(float x) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %1, %2;\n\tcvt.u32.u16 %0, h;\n\t}"
      : "=r"(r)
      : "f"(0.f), "f"(x));
  return r;
}
// Nearest e2m1 codes of two numbers (ties to even, saturating at 6), lo in bits [0, 4).
__device__ __forceinline__ uint32_t to_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
      : "=r"(r)
      : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ float2 half2_to_float2(uint32_t h) {
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
__device__ __forceinline__ float2 bf162_to_float2(uint32_t h) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&h));
}
// A pair of 16-bit numbers of the caller's type, as floats and back.
template <bool BF16>
__device__ __forceinline__ float2 pair_to_float2(uint32_t h) {
  return BF16 ? bf162_to_float2(h) : half2_to_float2(h);
}
template <bool BF16>
__device__ __forceinline__ uint32_t float2_to_pair(float lo, float hi) {
  if (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

}  // namespace c4
