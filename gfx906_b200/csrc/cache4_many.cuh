// The kernel for requests with many query rows, as its caller sees it.
#pragma once

#include <cuda_runtime.h>

#include "cache4_attn.cuh"

namespace c4 {

struct ManyParams {
  AttnParams a;
  int min_rows;     // requests with at most this many query rows are another kernel's
  int max_blocks;   // blocks of 256 query rows of all requests, at most
  int pieces;       // runs that each unit's keys are cut into
  float* part_o;    // [blocks * kv_heads * pieces][D / 4][256][4], pieces > 1
  float* part_ml;   // [blocks * kv_heads * pieces][256][2]
  unsigned long long timeout_ns;
};
struct ManyPlan {
  int max_blocks, pieces;  // max_blocks 0: too large a call
  size_t ml_off, bytes;    // workspace
};
ManyPlan many_plan(int tokens, int requests, int group, int kv_heads, int D, int sms);
int launch_many(const ManyParams& p, int D, int dtype, cudaStream_t stream);

}  // namespace c4
