// The kernel for requests with many query rows, as its caller sees it.
#pragma once

#include <cuda_runtime.h>

#include "cache4_attn.cuh"

namespace c4 {

struct ManyParams {
  AttnParams a;
  int min_rows;      // requests with at most this many query rows are another kernel's
  int max_units;     // units of 256 query rows and a kv head, at most
  int sms;
  // a slot for every piece that there can be, at most CUT_CTAS * sms
  float* part_o;     // [slots][D / 4][256][4]
  float* part_ml;    // [slots][256][2]
  // [sms][2] pieces of a cut unit that are in the workspace, for each of its query
  // tiles, tagged with the launch as in the other kernel. A CTA whose wait ran out
  // counts its piece too, as LOST: the unit is not joined then, and its word is
  // none again for a replay of the launch, which has the same tag.
  unsigned long long* done;
  unsigned long long epoch;
  unsigned long long timeout_ns;
};
struct ManyPlan {
  bool fits;      // false: too large a call
  int max_units;
  size_t ml_off, done_off, bytes;  // workspace
};
ManyPlan many_plan(int tokens, int requests, int group, int kv_heads, int D, int sms);
int launch_many(const ManyParams& p, int D, int dtype, cudaStream_t stream);

}  // namespace c4
