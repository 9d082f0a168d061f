// Parameters shared by the attention kernels over the 4-bit cache.
#pragma once

#include <stdint.h>

namespace c4 {

struct AttnParams {
  const uint16_t* q;  // fp16 or bf16
  uint16_t* o;
  const uint8_t* cache;
  const int* tables;
  const int* lengths;
  const int* query_start;
  const float* k_scale;
  const float* v_scale;
  long long q_stride_t, q_stride_h, o_stride_t, o_stride_h;
  int tokens, kv_heads, group, pages, requests, width;
  int causal, zero_rest;
  float scale_log2;  // scale * log2(e)
  unsigned group_magic;  // ceil(2^32 / group) where rows / group is its high product, else 0

  // Of query row `row` of a request (token * group + head of the group): its token.
  __device__ __forceinline__ int token_of(int row) const {
    return group_magic ? static_cast<int>(__umulhi(static_cast<unsigned>(row), group_magic)) : row / group;
  }
};

// The product's error is below row * group / 2^32 of a token.
inline unsigned group_magic(long long rows, int group) {
  return group > 1 && rows * group < (1ll << 32) ? static_cast<unsigned>(((1ll << 32) + group - 1) / group) : 0u;
}

// Rows of bf16 are divided by a power of two that brings their largest number to
// [1, 2) and then fit fp16; this is its exponent field, from that of the largest.
// The first power stands for subnormal rows too, the last but one for the largest
// rows, whose own reciprocal would be subnormal. Rows that hold an infinity or NaN
// stay as they are (127: a power of one).
__device__ __forceinline__ uint32_t row_exponent(float largest) {
  const uint32_t ex = (__float_as_uint(largest) >> 23) & 255u;
  return ex == 255u ? 127u : min(max(ex, 1u), 253u);
}

// Query rows of request r: first token and number of tokens, whatever the
// array holds (it comes from the caller's device memory).
struct Rows {
  int first, n;
};
__device__ __forceinline__ Rows rows_of(const AttnParams& p, int r) {
  const int a = min(max(p.query_start[r], 0), p.tokens), b = min(max(p.query_start[r + 1], 0), p.tokens);
  return {a, max(b - a, 0)};
}
__device__ __forceinline__ int length_of(const AttnParams& p, int r) {
  const long long most = static_cast<long long>(p.width) * 64;
  const int n = max(p.lengths[r], 0);
  return n < most ? n : static_cast<int>(most);
}

}  // namespace c4
