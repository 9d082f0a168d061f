// Page plan, writes and reads of the paged 4-bit key/value cache (cache4.cuh).
#include <limits.h>

#include "cache4.cuh"
#include "cache4_host.cuh"
#include "sm100_ptx.cuh"

namespace c4 {

// -------------------------------------------------------------------- plan
// One launch without any exchange between blocks: every block scans all
// requests by itself (their lengths and counts are a few KB, from L2) and then
// does its share of the requests' pages and of the tokens. No block reads what
// another writes: pages granted are looked up where they come from -- the
// stack below the old top, or, above it, the row of the ended request that
// returns them -- and not where the call puts them.
constexpr int PLAN_THREADS = 256;
constexpr int PLAN_MAX_REQUESTS = 8192;  // five ints of shared memory each

struct PlanParams {
  int* tables;
  const int* lengths;
  const int* counts;
  int* free_pages;
  const int* free_count;
  int requests, width, free_pages_size, tokens;
  int* query_start;
  int* lengths_out;
  int* added;
  int* slots;
  int* positions;
  int* free_count_out;
};

__device__ __forceinline__ long long warp_inclusive(long long x, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  return x;
}
// Exclusive prefix of x over the block's threads; total over all of them.
__device__ __forceinline__ long long block_exclusive(long long x, long long* part, long long* total) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long inc = warp_inclusive(x, lane);
  __syncthreads();
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 32; ++w) {
    if (w < warp) before += part[w];
    all += part[w];
  }
  *total = all;
  return before + inc - x;
}
__device__ __forceinline__ int clamp_int(long long x) { return x > INT_MAX ? INT_MAX : static_cast<int>(x); }
__device__ __forceinline__ int pages_of(long long tokens) { return static_cast<int>((tokens + PAGE - 1) / PAGE); }

__global__ void __launch_bounds__(PLAN_THREADS) cache4_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  __shared__ long long part[PLAN_THREADS / 32];
  const int R = p.requests;
  int* len = plan_smem;          // tokens held, clamped to what the table row can hold
  int* cnt = len + R;            // tokens to add; -1: ended
  int* start = cnt + R;          // first token (query_start)
  int* back = start + R;         // pages returned by the requests before
  int* need = back + R;          // pages needed by the requests before; -1 - that: refused
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();
  const long long row_tokens = static_cast<long long>(p.width) * PAGE;
  for (int r = threadIdx.x; r < R; r += PLAN_THREADS) {
    const long long n = p.lengths[r];
    len[r] = static_cast<int>(n < 0 ? 0 : (n > row_tokens ? row_tokens : n));
    const int c = p.counts[r];
    cnt[r] = c < 0 ? -1 : c;
  }
  const int old_free = min(max(*p.free_count, 0), p.free_pages_size);
  __syncthreads();

  // each thread scans a run of requests
  const int per = (R + PLAN_THREADS - 1) / PLAN_THREADS;
  const int r0 = min(R, static_cast<int>(threadIdx.x) * per), r1 = min(R, r0 + per);
  long long tokens = 0, returned = 0, total_tokens, total_back, total_need;
  for (int r = r0; r < r1; ++r) {
    tokens += max(cnt[r], 0);
    returned += cnt[r] < 0 ? pages_of(len[r]) : 0;
  }
  tokens = block_exclusive(tokens, part, &total_tokens);
  returned = block_exclusive(returned, part, &total_back);
  long long wanted = 0;
  for (int r = r0; r < r1; ++r) {
    start[r] = clamp_int(tokens);
    back[r] = clamp_int(returned);
    const int n = max(cnt[r], 0);
    tokens += n;
    returned += cnt[r] < 0 ? pages_of(len[r]) : 0;
    const bool fits = cnt[r] >= 0 && static_cast<long long>(len[r]) + n <= row_tokens && tokens <= p.tokens;
    need[r] = fits ? pages_of(static_cast<long long>(len[r]) + n) - pages_of(len[r]) : -1;
    wanted += max(need[r], 0);
  }
  const long long free_now = min(old_free + total_back, static_cast<long long>(p.free_pages_size));
  wanted = block_exclusive(wanted, part, &total_need);
  long long taken = 0;
  for (int r = r0; r < r1; ++r) {
    const int k = need[r];
    const bool granted = k == 0 || (k > 0 && wanted + k <= free_now);
    const int before = clamp_int(wanted);
    wanted += max(k, 0);
    taken += granted ? k : 0;
    need[r] = granted ? before : -1 - before;
  }
  long long total_taken;
  (void)block_exclusive(taken, part, &total_taken);
  __syncthreads();

  // page `i` below the top of the stack after the returns
  auto page_at = [&](int i) -> int {
    const int at = static_cast<int>(free_now) - 1 - i;
    if (at < old_free) return p.free_pages[at];
    const int want = at - old_free;  // among the pages returned by this call
    int lo = 0, hi = R - 1;          // last request with back[r] <= want that returned pages
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (back[mid] <= want)
        lo = mid;
      else
        hi = mid - 1;
    }
    return p.tables[static_cast<long long>(lo) * p.width + want - back[lo]];
  };

  const int blocks = gridDim.x;
  for (int r = blockIdx.x * PLAN_THREADS + threadIdx.x; r < R; r += blocks * PLAN_THREADS) {
    const int n = need[r] >= 0 ? max(cnt[r], 0) : 0;
    p.query_start[r] = start[r];
    p.lengths_out[r] = cnt[r] < 0 ? 0 : len[r] + n;
    p.added[r] = n;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.query_start[R] = clamp_int(total_tokens);
    *p.free_count_out = static_cast<int>(free_now - total_taken);
  }
  // pages: a warp per request
  const int lane = threadIdx.x % 32;
  for (int r = blockIdx.x + blocks * (threadIdx.x / 32); r < R; r += blocks * (PLAN_THREADS / 32)) {
    int* row = p.tables + static_cast<long long>(r) * p.width;
    const int held = pages_of(len[r]);
    if (cnt[r] < 0) {
      for (int i = lane; i < held; i += 32) {
        const long long at = static_cast<long long>(old_free) + back[r] + i;
        if (at < p.free_pages_size) p.free_pages[at] = row[i];
      }
    } else if (need[r] >= 0) {
      const int k = pages_of(static_cast<long long>(len[r]) + cnt[r]) - held;
      for (int i = lane; i < k; i += 32) row[held + i] = page_at(need[r] + i);
    }
  }
  // tokens
  for (int t = blockIdx.x * PLAN_THREADS + threadIdx.x; t < p.tokens; t += blocks * PLAN_THREADS) {
    int slot = -1, position = -1;
    if (t < total_tokens) {
      int lo = 0, hi = R - 1;  // last request that starts at or before t: the one that holds it
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (start[mid] <= t)
          lo = mid;
        else
          hi = mid - 1;
      }
      if (need[lo] >= 0) {
        position = len[lo] + t - start[lo];
        const int held = pages_of(len[lo]), at = position / PAGE;
        const int page = at < held ? p.tables[static_cast<long long>(lo) * p.width + at] : page_at(need[lo] + at - held);
        slot = page * PAGE + position % PAGE;
      }
    }
    p.slots[t] = slot;
    p.positions[t] = position;
  }
}

// ------------------------------------------------------------------- write
struct WriteParams {
  const void* x[2];           // K, V
  long long stride_t[2], stride_h[2];
  const float* factor[2];
  uint8_t* cache;
  const int* slots;
  int tokens, heads, pages;
};

// A thread turns 16 channels (one scale group) of one token of K
// (blockIdx.y == 0) or V into 8 bytes of codes and a scale.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) cache4_write_kernel(const WriteParams p) {
  using L = Layout<D>;
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int g = static_cast<int>(i % L::GROUPS);
  const long long th = i / L::GROUPS;
  const int h = static_cast<int>(th % p.heads);
  const long long t = th / p.heads;
  if (t >= p.tokens) return;
  const int slot = p.slots[t];
  if (slot < 0 || slot / PAGE >= p.pages) return;
  const int kv = blockIdx.y;
  const uint4* src = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x[kv]) + t * p.stride_t[kv] +
                                                    h * p.stride_h[kv] + g * 16);
  const uint4 a = __ldcs(src), b = __ldcs(src + 1);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  float x[16];
  float most = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 f = pair_to_float2<BF16>(w[e]);
    x[2 * e] = f.x == f.x ? f.x : 0.f;  // NaN is held as zero
    x[2 * e + 1] = f.y == f.y ? f.y : 0.f;
    most = fmaxf(most, fmaxf(fabsf(x[2 * e]), fabsf(x[2 * e + 1])));
  }
  const float factor = p.factor[kv] ? p.factor[kv][h] : 1.f;
  // the scale is rounded once, from the 32-bit quotient, and never zero
  const uint32_t scale = to_e4m3(fminf(fmaxf(most / (6.f * factor), 0.001953125f), 448.f));
  const float step = half2_to_float2(scales_to_half2(scale)).x * factor;
  uint32_t codes[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    codes[e] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      codes[e] |= to_e2m1x2(x[8 * e + 2 * j] / step, x[8 * e + 2 * j + 1] / step) << (8 * j);
  }
  const int at = slot % PAGE, bt = at % BLOCK;
  uint8_t* block = p.cache + (static_cast<long long>(slot / PAGE) * p.heads + h) * L::PAGE_BYTES +
                   at / BLOCK * L::BLOCK_BYTES;
  if (kv == 0) {
    *reinterpret_cast<uint2*>(block + L::k_code(bt, g)) = make_uint2(codes[0], codes[1]);
    block[L::k_scale(bt, g)] = static_cast<uint8_t>(scale);
  } else {
    if (D == 128) {
      *reinterpret_cast<uint2*>(block + L::v_code(bt, g)) = make_uint2(codes[0], codes[1]);
    } else {
      *reinterpret_cast<uint32_t*>(block + L::v_code(bt, 2 * g)) = codes[0];
      *reinterpret_cast<uint32_t*>(block + L::v_code(bt, 2 * g + 1)) = codes[1];
    }
    block[L::v_scale(bt, g)] = static_cast<uint8_t>(scale);
  }
}

// -------------------------------------------------------------------- read
struct ReadParams {
  const uint8_t* cache;
  const int* slots;
  const float* factor[2];
  void* x[2];
  int tokens, heads, pages;
};

// A thread reads 16 channels of one token of K (blockIdx.y == 0) or V.
// OUT: 0 = fp16, 1 = bf16, 2 = fp32.
template <int D, int OUT>
__global__ void __launch_bounds__(256) cache4_read_kernel(const ReadParams p) {
  using L = Layout<D>;
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int g = static_cast<int>(i % L::GROUPS);
  const long long th = i / L::GROUPS;
  const int h = static_cast<int>(th % p.heads);
  const long long t = th / p.heads;
  if (t >= p.tokens) return;
  const int slot = p.slots[t];
  const int kv = blockIdx.y;
  float x[16];
  if (slot < 0 || slot / PAGE >= p.pages) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = 0.f;
  } else {
    const int at = slot % PAGE, bt = at % BLOCK;
    const uint8_t* block = p.cache + (static_cast<long long>(slot / PAGE) * p.heads + h) * L::PAGE_BYTES +
                           at / BLOCK * L::BLOCK_BYTES;
    uint32_t codes[2], scale;
    if (kv == 0 || D == 128) {
      const uint2 c = *reinterpret_cast<const uint2*>(block + (kv == 0 ? L::k_code(bt, g) : L::v_code(bt, g)));
      codes[0] = c.x;
      codes[1] = c.y;
    } else {
      codes[0] = *reinterpret_cast<const uint32_t*>(block + L::v_code(bt, 2 * g));
      codes[1] = *reinterpret_cast<const uint32_t*>(block + L::v_code(bt, 2 * g + 1));
    }
    scale = block[kv == 0 ? L::k_scale(bt, g) : L::v_scale(bt, g)];
    const float step = half2_to_float2(scales_to_half2(scale)).x * (p.factor[kv] ? p.factor[kv][h] : 1.f);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      uint32_t pair[4];
      codes_to_half2(codes[e], pair);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = half2_to_float2(pair[j]);
        x[8 * e + 2 * j] = f.x * step;
        x[8 * e + 2 * j + 1] = f.y * step;
      }
    }
  }
  const long long to = (t * p.heads + h) * D + g * 16;
  if (OUT == 2) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.x[kv]) + to);
#pragma unroll
    for (int e = 0; e < 4; ++e) __stcs(dst + e, make_float4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]));
  } else {
    uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.x[kv]) + to);
#pragma unroll
    for (int e = 0; e < 2; ++e)
      __stcs(dst + e, make_uint4(float2_to_pair<OUT == 1>(x[8 * e], x[8 * e + 1]),
                                 float2_to_pair<OUT == 1>(x[8 * e + 2], x[8 * e + 3]),
                                 float2_to_pair<OUT == 1>(x[8 * e + 4], x[8 * e + 5]),
                                 float2_to_pair<OUT == 1>(x[8 * e + 6], x[8 * e + 7])));
  }
}

// -------------------------------------------------------------------- host
static int plan(const PlanParams& p, cudaStream_t stream) {
  int sms = 0;
  const int rc = gfx906_b200_internal_device(&sms);
  if (rc != GFX906_B200_OK) return rc;
  static SmemAttribute smem;
  if (!smem.set(cache4_plan_kernel, PLAN_MAX_REQUESTS * 5 * static_cast<int>(sizeof(int)))) return GFX906_B200_ECUDA;
  // a block for every 1024 tokens or 32 requests
  const int blocks = min(sms, 1 + max(p.tokens / 1024, p.requests / 32));
  return launch(cache4_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), static_cast<size_t>(p.requests) * 5 * sizeof(int),
                stream, p);
}

static int blocks_of(int tokens, int heads, int D, unsigned* blocks) {
  const long long n = (static_cast<long long>(tokens) * heads * (D / 16) + 255) / 256;
  if (n > INT_MAX) return GFX906_B200_EINVAL;
  *blocks = static_cast<unsigned>(n);
  return GFX906_B200_OK;
}

static int write(const WriteParams& p, int dtype, int D, cudaStream_t stream) {
  int sms = 0, rc = gfx906_b200_internal_device(&sms);
  unsigned blocks = 0;
  if (rc == GFX906_B200_OK) rc = blocks_of(p.tokens, p.heads, D, &blocks);
  if (rc != GFX906_B200_OK) return rc;
  const dim3 grid(blocks, 2), block(256);
  if (D == 128)
    return dtype ? launch(cache4_write_kernel<128, true>, grid, block, 0, stream, p)
                 : launch(cache4_write_kernel<128, false>, grid, block, 0, stream, p);
  return dtype ? launch(cache4_write_kernel<64, true>, grid, block, 0, stream, p)
               : launch(cache4_write_kernel<64, false>, grid, block, 0, stream, p);
}

template <int D>
static int read_d(const ReadParams& p, int dtype, unsigned blocks, cudaStream_t stream) {
  const dim3 grid(blocks, 2), block(256);
  if (dtype == 0) return launch(cache4_read_kernel<D, 0>, grid, block, 0, stream, p);
  if (dtype == 1) return launch(cache4_read_kernel<D, 1>, grid, block, 0, stream, p);
  return launch(cache4_read_kernel<D, 2>, grid, block, 0, stream, p);
}

static int read(const ReadParams& p, int dtype, int D, cudaStream_t stream) {
  int sms = 0, rc = gfx906_b200_internal_device(&sms);
  unsigned blocks = 0;
  if (rc == GFX906_B200_OK) rc = blocks_of(p.tokens, p.heads, D, &blocks);
  if (rc != GFX906_B200_OK) return rc;
  return D == 128 ? read_d<128>(p, dtype, blocks, stream) : read_d<64>(p, dtype, blocks, stream);
}

}  // namespace c4

extern "C" {

int gfx906_b200_cache4_page_bytes(int D) { return c4::head_dim_ok(D) ? 72 * D : 0; }

int gfx906_b200_cache4_plan(int* tables, const int* lengths, const int* counts, int* free_pages, const int* free_count,
                            int requests, int width, int free_pages_size, int tokens, int* query_start,
                            int* lengths_out, int* added, int* slots, int* positions, int* free_count_out,
                            cudaStream_t stream) {
  if (requests < 0 || requests > c4::PLAN_MAX_REQUESTS || width < 0 || width > INT_MAX / c4::PAGE ||
      free_pages_size < 0 || tokens < 0 || static_cast<long long>(requests) * width > INT_MAX || !query_start ||
      !free_count || !free_count_out || (requests && (!lengths || !counts || !lengths_out || !added)) ||
      (static_cast<long long>(requests) * width && !tables) || (free_pages_size && !free_pages) ||
      (tokens && (!slots || !positions)))
    return c4::done(GFX906_B200_EINVAL);
  c4::PlanParams p{tables, lengths, counts, free_pages, free_count, requests, width, free_pages_size, tokens,
                   query_start, lengths_out, added, slots, positions, free_count_out};
  return c4::done(c4::plan(p, stream));
}

int gfx906_b200_cache4_write(const void* k, const void* v, int dtype, long long k_stride_t, long long k_stride_h,
                             long long v_stride_t, long long v_stride_h, int tokens, int kv_heads, int D, void* cache,
                             int pages, const int* slots, const float* k_scale, const float* v_scale,
                             cudaStream_t stream) {
  if (!c4::head_dim_ok(D)) return c4::done(GFX906_B200_EHEADDIM);
  if (dtype < 0 || dtype > 1 || tokens < 0 || kv_heads < 0 || pages < 0) return c4::done(GFX906_B200_EINVAL);
  if (tokens == 0 || kv_heads == 0 || pages == 0) return c4::done(GFX906_B200_OK);
  if (!k || !v || !cache || !slots) return c4::done(GFX906_B200_EINVAL);
  if (!c4::aligned16(k) || !c4::aligned16(v) || !c4::aligned16(cache) ||
      ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 7))
    return c4::done(GFX906_B200_EALIGN);
  c4::WriteParams p{{k, v}, {k_stride_t, v_stride_t}, {k_stride_h, v_stride_h}, {k_scale, v_scale},
                    static_cast<uint8_t*>(cache), slots, tokens, kv_heads, pages};
  return c4::done(c4::write(p, dtype, D, stream));
}

int gfx906_b200_cache4_read(const void* cache, int pages, const int* slots, const float* k_scale, const float* v_scale,
                            int tokens, int kv_heads, int D, void* k, void* v, int dtype, cudaStream_t stream) {
  if (!c4::head_dim_ok(D)) return c4::done(GFX906_B200_EHEADDIM);
  if (dtype < 0 || dtype > 2 || tokens < 0 || kv_heads < 0 || pages < 0) return c4::done(GFX906_B200_EINVAL);
  if (tokens == 0 || kv_heads == 0) return c4::done(GFX906_B200_OK);
  if (!k || !v || (pages && !cache) || !slots) return c4::done(GFX906_B200_EINVAL);
  if (!c4::aligned16(k) || !c4::aligned16(v) || !c4::aligned16(cache)) return c4::done(GFX906_B200_EALIGN);
  c4::ReadParams p{static_cast<const uint8_t*>(cache), slots, {k_scale, v_scale}, {k, v}, tokens, kv_heads, pages};
  return c4::done(c4::read(p, dtype, D, stream));
}

}  // extern "C"
