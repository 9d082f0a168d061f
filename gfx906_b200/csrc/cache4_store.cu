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
// returns them -- and not where the call puts them. Bound by latency: 64 requests
// 3.1 us of GPU time, 1000 requests with 18000 tokens and 437 ended ones 5.8 us.
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

template <typename T>
__device__ __forceinline__ T warp_inclusive(T x, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const T y = __shfl_up_sync(0xffffffffu, x, d);
    if (lane >= d) x += y;
  }
  return x;
}
// Exclusive prefixes of x and y over the block's threads, and their totals.
struct Prefix {
  long long x, y, all_x, all_y;
};
__device__ __forceinline__ Prefix block_prefix(long long x, int y, long long* part_x, int* part_y) {
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const long long ix = warp_inclusive(x, lane);
  const int iy = warp_inclusive(y, lane);
  if (lane == 31) {
    part_x[warp] = ix;
    part_y[warp] = iy;
  }
  __syncthreads();
  Prefix p{ix - x, iy - y, 0, 0};
#pragma unroll
  for (int w = 0; w < PLAN_THREADS / 32; ++w) {
    if (w < warp) {
      p.x += part_x[w];
      p.y += part_y[w];
    }
    p.all_x += part_x[w];
    p.all_y += part_y[w];
  }
  return p;
}
__device__ __forceinline__ int clamp_int(long long x) { return x > INT_MAX ? INT_MAX : static_cast<int>(x); }
__device__ __forceinline__ int pages_of(long long tokens) { return static_cast<int>((tokens + PAGE - 1) / PAGE); }

__global__ void __launch_bounds__(PLAN_THREADS) cache4_plan_kernel(const PlanParams p) {
  extern __shared__ int plan_smem[];
  __shared__ long long part[2][PLAN_THREADS / 32];
  __shared__ int part_pages[2][PLAN_THREADS / 32];
  __shared__ int taken;
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
  if (threadIdx.x == 0) taken = 0;
  __syncthreads();

  // each thread scans a run of requests; pages are counted in 32 bits (the
  // tables hold no more), tokens in 64
  const int per = (R + PLAN_THREADS - 1) / PLAN_THREADS;
  const int r0 = min(R, static_cast<int>(threadIdx.x) * per), r1 = min(R, r0 + per);
  long long tokens = 0;
  int returned = 0;
  for (int r = r0; r < r1; ++r) {
    tokens += max(cnt[r], 0);
    returned += cnt[r] < 0 ? pages_of(len[r]) : 0;
  }
  Prefix before = block_prefix(tokens, returned, part[0], part_pages[0]);
  const long long total_tokens = before.all_x;
  const long long free_now = min(old_free + before.all_y, static_cast<long long>(p.free_pages_size));
  tokens = before.x;
  returned = static_cast<int>(before.y);
  int wanted = 0;
  for (int r = r0; r < r1; ++r) {
    start[r] = clamp_int(tokens);
    back[r] = returned;
    const int n = max(cnt[r], 0);
    tokens += n;
    returned += cnt[r] < 0 ? pages_of(len[r]) : 0;
    const bool fits = cnt[r] >= 0 && static_cast<long long>(len[r]) + n <= row_tokens && tokens <= p.tokens;
    need[r] = fits ? pages_of(static_cast<long long>(len[r]) + n) - pages_of(len[r]) : -1;
    wanted += max(need[r], 0);
  }
  before = block_prefix(0, wanted, part[1], part_pages[1]);
  wanted = static_cast<int>(before.y);
  int last = 0;  // pages granted up to here
  for (int r = r0; r < r1; ++r) {
    const int k = need[r];
    const bool granted = k == 0 || (k > 0 && wanted + k <= free_now);
    need[r] = granted ? wanted : -1 - wanted;
    wanted += max(k, 0);
    if (granted && k > 0) last = wanted;
  }
  last = __reduce_max_sync(0xffffffffu, last);
  if (threadIdx.x % 32 == 0 && last > 0) atomicMax(&taken, last);
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
    *p.free_count_out = static_cast<int>(free_now - taken);
  }
  // pages: a warp per request
  const int lane = threadIdx.x % 32;
  for (int r = blockIdx.x + blocks * (threadIdx.x / 32); r < R; r += blocks * (PLAN_THREADS / 32)) {
    int* row = p.tables + static_cast<long long>(r) * p.width;
    const int held = pages_of(len[r]);
    if (cnt[r] < 0) {
      for (int i0 = lane; i0 < held; i0 += 32 * 8) {  // eight loads in flight
        int page[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) page[i] = i0 + 32 * i < held ? row[i0 + 32 * i] : 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const long long at = static_cast<long long>(old_free) + back[r] + i0 + 32 * i;
          if (i0 + 32 * i < held && at < p.free_pages_size) p.free_pages[at] = page[i];
        }
      }
    } else if (need[r] >= 0) {
      const int k = pages_of(static_cast<long long>(len[r]) + cnt[r]) - held;
      for (int i = lane; i < k; i += 32) row[held + i] = page_at(need[r] + i);
    }
  }
  // tokens; a step behind the last one may leave 31 bits
  for (unsigned next = blockIdx.x * PLAN_THREADS + threadIdx.x; next < static_cast<unsigned>(p.tokens);
       next += blocks * PLAN_THREADS) {
    const int t = static_cast<int>(next);
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
        // a slot has 31 bits: page ids that have none are no page of any cache
        if (page >= 0 && page <= INT_MAX / PAGE) slot = page * PAGE + position % PAGE;
      }
    }
    p.slots[t] = slot;
    p.positions[t] = position;
  }
}

// ---------------------------------------------------------- write and read
// A warp handles TOKENS tokens of one kv head, K and V: a lane has 16 channels
// (one scale group) of two of them at 32 bytes an access, so that a warp moves
// whole 128-byte lines of 16-bit numbers and, for neighbouring slots, whole
// sectors of the cache. Reading is bound by memory: 32768 tokens of 8 heads of 128
// into bf16 take 29 us, 5.9 TB/s (16-byte accesses, one group a lane: 59 us);
// 16411 tokens into fp32 25 us, 6.1 TB/s. Writing is bound by its instructions:
// 16411 tokens of bf16 take 21.8 us, 3.95 TB/s, with the ALU pipe busy 61% and the
// issue slots 65% of the time, DRAM 34%.
template <int D>
struct Lanes {
  static constexpr int ROW = D / 16;          // lanes of a token
  static constexpr int AT_ONCE = 32 / ROW;    // tokens of one access of the warp
  static constexpr int TURNS = 2;
  static constexpr int TOKENS = AT_ONCE * TURNS;
};

__device__ __forceinline__ void load32(const void* src, uint32_t* w) {
  asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(src));
}
__device__ __forceinline__ void store32(void* dst, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

struct WriteParams {
  const uint16_t *k, *v;
  long long k_stride_t, k_stride_h, v_stride_t, v_stride_h;
  const float *k_factor, *v_factor;
  uint8_t* cache;
  const int* slots;
  int tokens, heads, pages;
  bool wide;  // rows start on 32 bytes
};

// 16 numbers (eight pairs of 16 bits) -> two words of codes, and their scale.
//
// codes = e2m1(x / step), the quotient rounded to 32 bits. A division per number
// would bound the kernel by its instructions (about 300 of a warp for 16 numbers
// a lane, where the memory's pace allows 170), so the quotient is
// corrected from the reciprocal r = 1 / step, which the 16 share: q0 = x r,
// q = q0 + (x - q0 step) r (Markstein, "Computation of elementary functions on
// the IBM RISC System/6000", 1990). Steps and groups for which a product could
// overflow or lose its low bits, and groups that hold a NaN, are divided.
template <bool BF16>
__device__ __forceinline__ uint32_t quantise16(const uint32_t* w, float factor, uint32_t* codes) {
  uint32_t most2 = 0;  // largest magnitudes of the even and the odd numbers, as bits
#pragma unroll
  for (int e = 0; e < 8; ++e) most2 = __vmaxu2(most2, w[e] & 0x7fff7fffu);
  const uint32_t most_bits = max(most2 & 0xffffu, most2 >> 16);
  const bool finite = most_bits < (BF16 ? 0x7f80u : 0x7c00u);
  float x[16], most = pair_to_float2<BF16>(most_bits).x;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float2 f = pair_to_float2<BF16>(w[e]);
    x[2 * e] = f.x;
    x[2 * e + 1] = f.y;
  }
  if (!finite) {  // NaN is held as zero
    most = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      x[e] = x[e] == x[e] ? x[e] : 0.f;
      most = fmaxf(most, fabsf(x[e]));
    }
  }
  // the scale is rounded once, from the 32-bit quotient, and never zero
  const float wanted = most / (6.f * factor);
  const uint32_t scale = to_e4m3(fminf(fmaxf(wanted, 0.001953125f), 448.f));
  const float step = half2_to_float2(scales_to_half2(scale)).x * factor;
  float y[16];
  if (finite && wanted <= 448.f && step > 1e-18f && step < 1e18f) {
    const float r = 1.f / step;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float q = x[e] * r;
      y[e] = copysignf(fmaf(fmaf(-q, step, x[e]), r, q), x[e]);  // zeros keep their sign
    }
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e) y[e] = x[e] / step;
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    codes[e] = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) codes[e] |= to_e2m1x2(y[8 * e + 2 * j], y[8 * e + 2 * j + 1]) << (8 * j);
  }
  return scale;
}

template <int D, bool BF16>
__global__ void __launch_bounds__(256) cache4_write_kernel(const WriteParams p) {
  using L = Layout<D>;
  using N = Lanes<D>;
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();
  const int lane = threadIdx.x % 32, g = lane % N::ROW;
  const unsigned warp = blockIdx.x * 8 + threadIdx.x / 32;
  const int h = warp % p.heads;
  const long long t0 = static_cast<long long>(warp / p.heads) * N::TOKENS + lane / N::ROW;
  int slot[N::TURNS];
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    const long long t = t0 + i * N::AT_ONCE;
    slot[i] = t < p.tokens ? p.slots[t] : -1;
    if (slot[i] < 0 || slot[i] / PAGE >= p.pages) slot[i] = -1;
  }
  uint32_t w[N::TURNS][2][8];
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    if (slot[i] < 0) continue;
    const long long t = t0 + i * N::AT_ONCE;
    const uint16_t* k = p.k + t * p.k_stride_t + h * p.k_stride_h + g * 16;
    const uint16_t* v = p.v + t * p.v_stride_t + h * p.v_stride_h + g * 16;
    if (p.wide) {
      load32(k, w[i][0]);
      load32(v, w[i][1]);
    } else {
      *reinterpret_cast<uint4*>(w[i][0]) = __ldcs(reinterpret_cast<const uint4*>(k));
      *reinterpret_cast<uint4*>(w[i][0] + 4) = __ldcs(reinterpret_cast<const uint4*>(k) + 1);
      *reinterpret_cast<uint4*>(w[i][1]) = __ldcs(reinterpret_cast<const uint4*>(v));
      *reinterpret_cast<uint4*>(w[i][1] + 4) = __ldcs(reinterpret_cast<const uint4*>(v) + 1);
    }
  }
  const float kf = p.k_factor ? p.k_factor[h] : 1.f, vf = p.v_factor ? p.v_factor[h] : 1.f;
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    if (slot[i] < 0) continue;
    const int at = slot[i] % PAGE, bt = at % BLOCK;
    uint8_t* block = p.cache + (static_cast<long long>(slot[i] / PAGE) * p.heads + h) * L::PAGE_BYTES +
                     at / BLOCK * L::BLOCK_BYTES;
    uint32_t codes[2];
    uint32_t scale = quantise16<BF16>(w[i][0], kf, codes);
    *reinterpret_cast<uint2*>(block + L::k_code(bt, g)) = make_uint2(codes[0], codes[1]);
    block[L::k_scale(bt, g)] = static_cast<uint8_t>(scale);
    scale = quantise16<BF16>(w[i][1], vf, codes);
    if (D == 128) {
      *reinterpret_cast<uint2*>(block + L::v_code(bt, g)) = make_uint2(codes[0], codes[1]);
    } else {
      *reinterpret_cast<uint32_t*>(block + L::v_code(bt, 2 * g)) = codes[0];
      *reinterpret_cast<uint32_t*>(block + L::v_code(bt, 2 * g + 1)) = codes[1];
    }
    block[L::v_scale(bt, g)] = static_cast<uint8_t>(scale);
  }
}

struct ReadParams {
  const uint8_t* cache;
  const int* slots;
  const float *k_factor, *v_factor;
  void *k, *v;
  int tokens, heads, pages;
  bool wide;  // outputs start on 32 bytes
};

// 16 numbers of the caller's type (OUT: 0 = fp16, 1 = bf16, 2 = fp32) at dst.
template <int OUT>
__device__ __forceinline__ void write16(void* dst, const uint32_t* codes, float step, bool wide) {
  uint32_t w[16];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    uint32_t pair[4];
    codes_to_half2(codes[e], pair);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = half2_to_float2(pair[j]);
      if (OUT == 2) {
        w[8 * e + 2 * j] = __float_as_uint(f.x * step);
        w[8 * e + 2 * j + 1] = __float_as_uint(f.y * step);
      } else {
        w[4 * e + j] = float2_to_pair<OUT == 1>(f.x * step, f.y * step);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < (OUT == 2 ? 2 : 1); ++i) {
    if (wide) {
      store32(static_cast<uint8_t*>(dst) + 32 * i, w + 8 * i);
    } else {
      uint4* to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(dst) + 32 * i);
      to[0] = make_uint4(w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3]);
      to[1] = make_uint4(w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]);
    }
  }
}

template <int D, int OUT>
__global__ void __launch_bounds__(256) cache4_read_kernel(const ReadParams p) {
  using L = Layout<D>;
  using N = Lanes<D>;
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();
  const int lane = threadIdx.x % 32, g = lane % N::ROW;
  const unsigned warp = blockIdx.x * 8 + threadIdx.x / 32;
  const int h = warp % p.heads;
  const long long t0 = static_cast<long long>(warp / p.heads) * N::TOKENS + lane / N::ROW;
  int slot[N::TURNS];
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    const long long t = t0 + i * N::AT_ONCE;
    slot[i] = t < p.tokens ? p.slots[t] : -1;
    if (slot[i] < 0 || slot[i] / PAGE >= p.pages) slot[i] = -1;
  }
  uint32_t codes[N::TURNS][2][2], scale[N::TURNS][2];
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    codes[i][0][0] = codes[i][0][1] = codes[i][1][0] = codes[i][1][1] = scale[i][0] = scale[i][1] = 0;
    if (slot[i] < 0) continue;
    const int at = slot[i] % PAGE, bt = at % BLOCK;
    const uint8_t* block = p.cache + (static_cast<long long>(slot[i] / PAGE) * p.heads + h) * L::PAGE_BYTES +
                           at / BLOCK * L::BLOCK_BYTES;
    const uint2 k = *reinterpret_cast<const uint2*>(block + L::k_code(bt, g));
    codes[i][0][0] = k.x;
    codes[i][0][1] = k.y;
    if (D == 128) {
      const uint2 v = *reinterpret_cast<const uint2*>(block + L::v_code(bt, g));
      codes[i][1][0] = v.x;
      codes[i][1][1] = v.y;
    } else {
      codes[i][1][0] = *reinterpret_cast<const uint32_t*>(block + L::v_code(bt, 2 * g));
      codes[i][1][1] = *reinterpret_cast<const uint32_t*>(block + L::v_code(bt, 2 * g + 1));
    }
    scale[i][0] = block[L::k_scale(bt, g)];
    scale[i][1] = block[L::v_scale(bt, g)];
  }
  const float kf = p.k_factor ? p.k_factor[h] : 1.f, vf = p.v_factor ? p.v_factor[h] : 1.f;
  constexpr int BYTES = OUT == 2 ? 4 : 2;
#pragma unroll
  for (int i = 0; i < N::TURNS; ++i) {
    const long long t = t0 + i * N::AT_ONCE;
    if (t >= p.tokens) continue;
    const long long to = ((t * p.heads + h) * D + g * 16) * BYTES;
    write16<OUT>(static_cast<uint8_t*>(p.k) + to, codes[i][0], half2_to_float2(scales_to_half2(scale[i][0])).x * kf, p.wide);
    write16<OUT>(static_cast<uint8_t*>(p.v) + to, codes[i][1], half2_to_float2(scales_to_half2(scale[i][1])).x * vf, p.wide);
  }
}

// -------------------------------------------------------------------- host
static int plan(const PlanParams& p, cudaStream_t stream) {
  int sms = 0;
  const int rc = gfx906_b200_internal_device(&sms);
  if (rc != GFX906_B200_OK) return rc;
  static SmemAttribute smem;
  if (!smem.set(cache4_plan_kernel, PLAN_MAX_REQUESTS * 5 * static_cast<int>(sizeof(int)))) return GFX906_B200_ECUDA;
  // a thread for every token, a warp for every request, as far as one wave goes
  const int blocks = min(sms, 1 + max(p.tokens / PLAN_THREADS, p.requests / (PLAN_THREADS / 32)));
  return launch(cache4_plan_kernel, dim3(blocks), dim3(PLAN_THREADS), static_cast<size_t>(p.requests) * 5 * sizeof(int),
                stream, p);
}

template <int D>
static int blocks_of(int tokens, int heads, unsigned* blocks) {
  const long long warps = (static_cast<long long>(tokens) + Lanes<D>::TOKENS - 1) / Lanes<D>::TOKENS * heads;
  if (warps > INT_MAX) return GFX906_B200_EINVAL;
  *blocks = static_cast<unsigned>((warps + 7) / 8);
  return GFX906_B200_OK;
}

template <int D>
static int write_d(const WriteParams& p, int dtype, cudaStream_t stream) {
  int sms = 0, rc = gfx906_b200_internal_device(&sms);
  unsigned blocks = 0;
  if (rc == GFX906_B200_OK) rc = blocks_of<D>(p.tokens, p.heads, &blocks);
  if (rc != GFX906_B200_OK) return rc;
  return dtype ? launch(cache4_write_kernel<D, true>, dim3(blocks), dim3(256), 0, stream, p)
               : launch(cache4_write_kernel<D, false>, dim3(blocks), dim3(256), 0, stream, p);
}

template <int D>
static int read_d(const ReadParams& p, int dtype, cudaStream_t stream) {
  int sms = 0, rc = gfx906_b200_internal_device(&sms);
  unsigned blocks = 0;
  if (rc == GFX906_B200_OK) rc = blocks_of<D>(p.tokens, p.heads, &blocks);
  if (rc != GFX906_B200_OK) return rc;
  if (dtype == 0) return launch(cache4_read_kernel<D, 0>, dim3(blocks), dim3(256), 0, stream, p);
  if (dtype == 1) return launch(cache4_read_kernel<D, 1>, dim3(blocks), dim3(256), 0, stream, p);
  return launch(cache4_read_kernel<D, 2>, dim3(blocks), dim3(256), 0, stream, p);
}

static bool aligned32(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 31u) == 0;
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
  const bool wide = c4::aligned32(k, v) && ((k_stride_t | k_stride_h | v_stride_t | v_stride_h) & 15) == 0;
  c4::WriteParams p{static_cast<const uint16_t*>(k), static_cast<const uint16_t*>(v), k_stride_t, k_stride_h, v_stride_t,
                    v_stride_h, k_scale, v_scale, static_cast<uint8_t*>(cache), slots, tokens, kv_heads, pages, wide};
  return c4::done(D == 128 ? c4::write_d<128>(p, dtype, stream) : c4::write_d<64>(p, dtype, stream));
}

int gfx906_b200_cache4_read(const void* cache, int pages, const int* slots, const float* k_scale, const float* v_scale,
                            int tokens, int kv_heads, int D, void* k, void* v, int dtype, cudaStream_t stream) {
  if (!c4::head_dim_ok(D)) return c4::done(GFX906_B200_EHEADDIM);
  if (dtype < 0 || dtype > 2 || tokens < 0 || kv_heads < 0 || pages < 0) return c4::done(GFX906_B200_EINVAL);
  if (tokens == 0 || kv_heads == 0) return c4::done(GFX906_B200_OK);
  if (!k || !v || (pages && !cache) || !slots) return c4::done(GFX906_B200_EINVAL);
  if (!c4::aligned16(k) || !c4::aligned16(v) || !c4::aligned16(cache)) return c4::done(GFX906_B200_EALIGN);
  c4::ReadParams p{static_cast<const uint8_t*>(cache), slots, k_scale, v_scale, k, v, tokens, kv_heads, pages,
                   c4::aligned32(k, v)};
  return c4::done(D == 128 ? c4::read_d<128>(p, dtype, stream) : c4::read_d<64>(p, dtype, stream));
}

}  // extern "C"
