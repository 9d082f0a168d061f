// Attention of a few new tokens per request against the paged 4-bit cache
// (cache4.cuh): O = softmax(scale * q K^T) V over a request's pages.
//
// Work is the list of units (request, row tile, kv head): a row tile is 8 * NT
// query rows of the request, a row being one (token, head of the group), so
// that all query heads of a kv head share one read of its keys and values. A
// unit's key range is cut into steps of 32 tokens (half a page, one contiguous
// copy of 36 D bytes). The steps of all units form one line that the blocks
// share evenly, whatever the requests' lengths; a unit that is cut at a block's
// end leaves partial sums (m, l, unnormalised O, 32 bits) in the workspace,
// joined by the block that finishes its last piece. Every unit counts one step more than it has
// keys for, so that units without any key have an owner that writes their
// zeros, and as the price of starting a unit. Where tables are so wide that the
// line could leave 31 bits, it counts grains of 2^k steps, a unit's last one
// partly filled.
//
// Inside a block four warps take the steps in turn, each with its own ring of
// copies in flight and its own running maximum m, sum l and accumulator; they
// meet once per unit. A warp computes S^T = K Q^T and O^T = V^T P^T: the keys
// and channels fill the 16 rows of m16n8k16 and the query rows are its n, so
// eight rows (all heads of a group for one token) leave no half of the
// instruction empty. Codes become fp16 by one conversion and one exact product
// per pair, in registers.
//
// Measured (B200, D = 128, 8 kv heads of 4 query heads): 32 requests of up to
// 16384 tokens 78 us in a captured graph, 4.7 TB/s of cache (84 us called with
// other inputs each time); 131072 tokens of one request 41 us, 3.6 TB/s. No unit
// is full (ALU pipe 53%, issue slots 59%, DRAM 53% of the time, 14 warps on an SM):
// 3.5 warps a scheduler do not overlap copies with arithmetic. With the arithmetic
// taken out the copies still take 69 and 35 us, with the copies taken out the
// arithmetic 74 and 40 (about 580 instructions of a warp per step, 270 of them on
// the ALU pipe); 8 us pass before the first step and behind the last.
#include <limits.h>
#include <math.h>

#include "cache4.cuh"
#include "cache4_attn.cuh"
#include "cache4_host.cuh"
#include "cache4_many.cuh"
#include "sm100_ptx.cuh"

namespace c4 {

// Requests with more query rows (tokens times heads of a group) go to the
// tensor-memory kernel of cache4_many.cu, which takes 256 rows at the price of
// one. Measured, us here and there for 48, 64, 96, 128 rows a request:
// D = 128: 1 x 8192 keys, 8 kv heads: 29, 31, 34, 38 and 38, 39, 39, 40; 8 x 4096,
// 8: 50, 60, 81, 101 and 48, 48, 48, 49; 32 x 2048, 8: 87, 111, 154, 196 and 122,
// 123, 125, 128; 4 x 32768, 2: 49, 56, 74, 93 and 72, 73, 74, 75.
// D = 64: 23, 25, 25, 27 and 30, 30, 30, 31; 34, 39, 50, 64 and 42, 42, 42, 42; 56,
// 70, 95, 121 and 92, 92, 92, 93; 34, 38, 49, 60 and 59, 60, 60, 61.
constexpr int FEW_ROWS = 64;

constexpr int MAX_REQUESTS = 8192;
constexpr int STEP = 32;                // tokens of a step
constexpr unsigned long long DRAIN_NS = 100000000ull;  // see the kernel's waits
// Log2 units, see step(): P of a row's largest score is 2^HEAD when the row's
// reference is set, and stays below 2^REACH, which fp16 holds.
constexpr float HEAD = 7.f;
constexpr float REACH = 15.f;
constexpr float LARGE = 4194304.f;  // 2^22: half a 32-bit step is 1/4 log2 unit

struct FewParams {
  AttnParams a;
  int max_rows;       // requests with more query rows are another kernel's
  int shift;          // a grain of the line is 2^shift steps
  float* part_o;      // [blocks][2][8 NT][D]
  float* part_ml;     // [blocks][2][8 NT][2]
  // [blocks] pieces in the workspace of the cut unit that the block starts,
  // tagged with the launch: (epoch << 16) | pieces. Whoever comes first to a
  // word with another tag sets it to none, so the workspace needs no clearing;
  // whoever joins a unit sets its word to none again, for a replay of the launch.
  unsigned long long* done;
  unsigned long long epoch;
  unsigned long long timeout_ns;
};

template <int D, int NT>
struct Few {
  using L = Layout<D>;
  // Four warps to a block. Eight, in half as many blocks, join fewer pieces of
  // one long context (131072 keys: 38 us, not 40) but wait longer at each unit's
  // end (ragged batch of 32: 82 us, not 79; drafts for 16 requests: 49, not 43).
  static constexpr int WARPS = 4;
  static constexpr int THREADS = WARPS * 32;
  static constexpr int PER_SM = NT == 1 ? 4 : 3;  // blocks that share an SM, by registers
  static constexpr int MAX_CHUNKS = (MAX_REQUESTS + THREADS - 1) / THREADS;
  // Steps of a unit that are worth a block of their own: one for each warp (two:
  // 8 heads x 1000 keys 10.2 us, not 9.7).
  static constexpr int MIN_STEPS = WARPS;
  static constexpr int ROWS = 8 * NT;
  static constexpr int STEP_BYTES = 2 * L::BLOCK_BYTES;
  static constexpr int STAGES = NT == 1 ? 2 : 3;  // four or three blocks share an SM
  static constexpr int LD = D + 4;  // floats of a row in the merge buffer
  static constexpr int RING = STAGES * STEP_BYTES;
  static constexpr int Q_OFF = WARPS * RING;
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int ML_OFF = Q_OFF + Q_BYTES;          // [WARPS][ROWS] (m, l)
  static constexpr int ROWF_OFF = ML_OFF + WARPS * ROWS * 8;  // [ROWS] factors of the rows of q
  static constexpr int SMEM = ROWF_OFF + ROWS * 4;
  static_assert(PER_SM >= 1 && ROWS * LD * 4 <= RING, "a warp's merge buffer is its ring");
};

__device__ unsigned int g_cache4_few_status = 0;  // 1: a wait for a copy ran out

// Contiguous copy global -> shared (16-byte aligned, bytes a multiple of 16),
// counted on `bar`.
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Whole warp: waits at most `limit_ns` for the phase of that parity.
__device__ __forceinline__ bool wait_copy(uint32_t bar, uint32_t parity, unsigned long long limit_ns) {
  bool ok = fa::mbar_try_wait(bar, parity);
  if (!ok) {
    const uint64_t t0 = fa::globaltimer_ns();
    uint32_t n = 0;
    while (!(ok = fa::mbar_try_wait(bar, parity))) {
      if ((++n & 31u) == 0u && (fa::globaltimer_ns() - t0 > limit_ns || n > (1u << 24))) {
        atomicOr(&g_cache4_few_status, 1u);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}
// W words at a, W = 2 or 4.
template <int W>
__device__ __forceinline__ void lds(const uint8_t* a, uint32_t* v) {
  if (W == 4)
    *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(a);
  else
    *reinterpret_cast<uint2*>(v) = *reinterpret_cast<const uint2*>(a);
}
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}

// One request's part of the line.
struct Share {
  int first, rows, len;  // first token; query rows (0: not this kernel's); keys
  int units, grains;     // units; grains of one unit's steps, with the one extra
};
__device__ __forceinline__ int steps_of(int len) { return (len + STEP - 1) / STEP + 1; }
template <int ROWS>
__device__ __forceinline__ Share share_of(const FewParams& p, int r) {
  const Rows t = rows_of(p.a, r);
  const int len = length_of(p.a, r), rows = t.n * p.a.group;
  if (rows > p.max_rows) return {t.first, 0, len, 0, 0};
  return {t.first, rows, len, (rows + ROWS - 1) / ROWS * p.a.kv_heads,
          rows ? (steps_of(len) + (1 << p.shift) - 1) >> p.shift : 0};
}

// Per-thread state of one warp's share of a unit.
template <int D, int NT>
struct Acc {
  float o[D / 16][NT][4];  // O^T: channels n D/8 + 2t (+1), query rows 2c, 2c + 1 of tile nt
  float m[NT][2], l[NT][2];
  bool large;  // some row of the warp has |m| > LARGE
};

// One step of 32 tokens (two blocks at `blk`): scores, running softmax, sums.
// MASK: tokens key0 + 0..31 may lie behind the last one a row sees
// (limit[nt][i], exclusive) or behind the request's length (`len`): those keys
// take no part, and their values -- whatever the page holds there -- are zeroed.
//
// A row's m is a reference that its scores may exceed by REACH (log2 units), not
// their maximum: P then stays below 2^REACH, O and l carry the same factor, and
// the maximum across the warp, with the products that follow from it, is taken
// only in the few steps where a vote finds a score beyond reach. The reference is
// set HEAD below the maximum, so that P uses all of fp16's range: weights down to
// 2^-21 of the largest are rounded to 2^-11 of themselves, smaller ones by 2^-32
// of the largest at most (without HEAD 2^-25: a long context's small weights
// beside one large one would count in l and be lost in O).
//
// m comes from a rounded product. Rows whose m is beyond LARGE round every score
// as m was, or the largest would lie half a step of m off it, out of reach or out
// of sight; the others take the difference unrounded. So equal keys weigh the
// same whichever steps they are in.
template <int D, int NT, bool MASK>
__device__ __forceinline__ void step(Acc<D, NT>& acc, const uint8_t* blk, const uint8_t* sq, int lane,
                                     const float (&factor)[NT][2], int key0, int len, const int (&limit)[NT][2]) {
  using L = Layout<D>;
  constexpr int W = D / 32;  // words of K codes of a lane and token
  const int n = lane >> 2, c = lane & 3;
  float s[2][NT][4];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[b][nt][e] = 0.f;
  // ---- S^T = K Q^T
  {
    uint32_t k[2][2][W];        // block, tokens n and n + 8
    uint32_t f[2][2][L::GPL];   // their scales, in both halves
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint8_t* base = blk + b * L::BLOCK_BYTES;
      lds<W>(base + L::KC + lane * (D / 8), k[b][0]);
      lds<W>(base + L::KC + 4 * D + lane * (D / 8), k[b][1]);
      if (L::GPL == 2) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(base + L::KS + lane * 4);
        const uint32_t x = scales_to_half2(w), y = scales_to_half2(w >> 16);
        f[b][0][0] = __byte_perm(x, x, 0x1010);
        f[b][0][L::GPL - 1] = __byte_perm(x, x, 0x3232);
        f[b][1][0] = __byte_perm(y, y, 0x1010);
        f[b][1][L::GPL - 1] = __byte_perm(y, y, 0x3232);
      } else {
        const uint32_t x = scales_to_half2(*reinterpret_cast<const uint16_t*>(base + L::KS + lane * 2));
        f[b][0][0] = __byte_perm(x, x, 0x1010);
        f[b][1][0] = __byte_perm(x, x, 0x3232);
      }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {  // two k-steps of 16 channels for each word
      uint32_t q[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) lds<4>(sq + ((nt * W + j) * 32 + lane) * 16, q[nt]);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        uint32_t x0[4], x1[4];
        codes_to_half2(k[b][0][j], x0);
        codes_to_half2(k[b][1][j], x1);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x0[e] = mul_half2(x0[e], f[b][0][j / 2]);
          x1[e] = mul_half2(x1[e], f[b][1][j / 2]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816(s[b][nt], x0[0], x1[0], x0[1], x1[1], q[nt][0], q[nt][1]);
          mma16816(s[b][nt], x0[2], x1[2], x0[3], x1[3], q[nt][2], q[nt][3]);
        }
      }
    }
  }
  // ---- running softmax; s[b][nt]: tokens 16 b + n (+ 8), rows 2c, 2c + 1
  auto hidden = [&](int b, int nt, int e) { return MASK && key0 + 16 * b + 8 * (e >> 1) + n >= limit[nt][e & 1]; };
  float y[2][NT][4];
  float far = -INFINITY;
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[b][nt][e] = hidden(b, nt, e) ? -INFINITY : fmaf(s[b][nt][e], factor[nt][e & 1], -acc.m[nt][e & 1]);
        far = fmaxf(far, y[b][nt][e]);
      }
  if (__any_sync(0xffffffffu, far > REACH) || acc.large) {
    bool large = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = i; e < 4; e += 2)
            if (!hidden(b, nt, e)) mx = fmaxf(mx, __fmul_rn(s[b][nt][e], factor[nt][i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mx = __fsub_rn(mx, HEAD);
        if (mx > acc.m[nt][i]) {
          const float alpha = fa::ex2_approx(acc.m[nt][i] - mx);
          acc.m[nt][i] = mx;
          acc.l[nt][i] *= alpha;
#pragma unroll
          for (int t = 0; t < D / 16; ++t) {
            acc.o[t][nt][i] *= alpha;
            acc.o[t][nt][2 + i] *= alpha;
          }
        }
        const float m_use = acc.m[nt][i] == -INFINITY ? 0.f : acc.m[nt][i];
        const bool rounded = fabsf(m_use) > LARGE;
        large |= rounded;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int e = i; e < 4; e += 2) {
            const float x = rounded ? __fsub_rn(__fmul_rn(s[b][nt][e], factor[nt][i]), m_use)
                                    : fmaf(s[b][nt][e], factor[nt][i], -m_use);
            y[b][nt][e] = hidden(b, nt, e) ? -INFINITY : x;
          }
      }
    acc.large = __any_sync(0xffffffffu, large);
  }
  // P in fp16 (the sum keeps 32 bits), transposed into B fragments
  uint32_t pb[2][NT][2];
#pragma unroll
  for (int b = 0; b < 2; ++b)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p0 = fa::ex2_approx(y[b][nt][2 * h]), p1 = fa::ex2_approx(y[b][nt][2 * h + 1]);
        acc.l[nt][0] += p0;
        acc.l[nt][1] += p1;
        pb[b][nt][h] = transpose8x8(fa::pack_half2(p0, p1));
      }
  // ---- O^T += V^T P^T
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const uint8_t* base = blk + b * L::BLOCK_BYTES;
    constexpr int W2 = D / 64;      // words of V codes of a lane and token
    uint32_t v0[2 * W2], v1[2 * W2];  // tokens 2c, 2c + 1; tokens 2c + 8, 2c + 9
    lds<2 * W2>(base + L::VC + lane * (D / 8), v0);
    lds<2 * W2>(base + L::VC + 4 * D + lane * (D / 8), v1);
    uint32_t w = *reinterpret_cast<const uint32_t*>(base + L::VS + (D == 128 ? lane : (n / 2) * 4 + c) * 4);
    if (MASK) {
      const int k = key0 + 16 * b + 2 * c;
      if (k >= len) w &= 0xffffff00u;
      if (k + 1 >= len) w &= 0xffff00ffu;
      if (k + 8 >= len) w &= 0xff00ffffu;
      if (k + 9 >= len) w &= 0x00ffffffu;
    }
    const uint32_t f0 = scales_to_half2(w), f1 = scales_to_half2(w >> 16);
#pragma unroll
    for (int j = 0; j < W2; ++j) {
      // bytes of one channel's codes of two tokens: even channels, odd channels
      const uint32_t m = 0x0f0f0f0fu;
      uint32_t e0[4], o0[4], e1[4], o1[4];
      codes_to_half2((v0[j] & m) | ((v0[W2 + j] << 4) & ~m), e0);
      codes_to_half2(((v0[j] >> 4) & m) | (v0[W2 + j] & ~m), o0);
      codes_to_half2((v1[j] & m) | ((v1[W2 + j] << 4) & ~m), e1);
      codes_to_half2(((v1[j] >> 4) & m) | (v1[W2 + j] & ~m), o1);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t a0 = mul_half2(e0[t], f0), a1 = mul_half2(o0[t], f0);
        const uint32_t a2 = mul_half2(e1[t], f1), a3 = mul_half2(o1[t], f1);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma16816(acc.o[4 * j + t][nt], a0, a1, a2, a3, pb[b][nt][0], pb[b][nt][1]);
      }
    }
  }
}

// The line of `total` grains in `blocks` runs: run c starts at total * c / blocks,
// so that equal units which the blocks divide evenly are cut where they end.
struct Split {
  int total, blocks, per, more;
  __device__ __forceinline__ Split(int total_, int blocks_)
      : total(total_), blocks(blocks_), per(total_ / blocks_), more(total_ - per * blocks_) {}
  __device__ __forceinline__ int start(int c) const { return c * per + c * more / blocks; }
  // the run that holds grain `at`
  __device__ __forceinline__ int owner(int at) const {
    int c = min(blocks - 1, static_cast<int>(static_cast<float>(at) * blocks / total));  // off by one or two
    while (c > 0 && start(c) > at) --c;
    while (c + 1 < blocks && start(c + 1) <= at) ++c;
    return c;
  }
};

template <bool BF16>
__device__ __forceinline__ void store4(uint16_t* dst, float4 x) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(float2_to_pair<BF16>(x.x, x.y), float2_to_pair<BF16>(x.z, x.w));
}

// Joins the pieces of a unit: the second slot of the block that starts it and
// the first slots of those after it. Whole block; `red` is free shared memory.
template <int D, int NT, bool BF16>
__device__ __forceinline__ void join(const FewParams& p, float* red, int first_block, int pieces, int first, int row0,
                                     int nrows, int head, float vf) {
  constexpr int ROWS = 8 * NT, V = D / 32;  // V channels of a lane
  constexpr int WARPS = Few<D, NT>::WARPS;
  const AttnParams& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // a warp per row and turn; where warps would be left over, several share a row's pieces
  int parts = 1;
  while (parts * 2 * nrows <= WARPS) parts *= 2;
  const int part = warp % parts;
  auto slot_row = [&](int k, int row) -> long long {
    return (k == 0 ? first_block * 2ll + 1 : (static_cast<long long>(first_block) + k) * 2) * ROWS + row;
  };
  for (int row = warp / parts; row < (parts > 1 ? WARPS / parts : nrows); row += WARPS / parts) {
    const bool there = row < nrows;
    float m = -INFINITY, l = 0.f, x[V];
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = 0.f;
    // the pieces of this warp, 32 at a time and 16 at once: lane i has the
    // (m, l) of the i-th, which is loaded together with the first 16 sums
    for (int k0 = part; there && k0 < pieces; k0 += 32 * parts) {
      const int here = min(32, (pieces - k0 + parts - 1) / parts);
      float2 u = make_float2(-INFINITY, 0.f);
      if (lane < here) u = __ldcg(reinterpret_cast<const float2*>(p.part_ml + slot_row(k0 + lane * parts, row) * 2));
      float w = 0.f;
      for (int i0 = 0; i0 < here; i0 += 16) {
        float y[16][V];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float* src = p.part_o + slot_row(k0 + min(i0 + i, here - 1) * parts, row) * D + lane * V;
          if (V == 4)
            *reinterpret_cast<float4*>(y[i]) = __ldcg(reinterpret_cast<const float4*>(src));
          else
            *reinterpret_cast<float2*>(y[i]) = __ldcg(reinterpret_cast<const float2*>(src));
        }
        if (i0 == 0) {
          float mx = u.x;
#pragma unroll
          for (int d = 16; d > 0; d /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          if (mx > m) {
            const float alpha = fa::ex2_approx(m - mx);
            l *= alpha;
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] *= alpha;
            m = mx;
          }
          w = u.x == -INFINITY ? 0.f : fa::ex2_approx(u.x - m);
          l += u.y * w;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float f = __shfl_sync(0xffffffffu, w, i0 + i);
          if (i0 + i < here) {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] += y[i][e] * f;
          }
        }
      }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
    if (parts > 1) {  // one turn, all warps
#pragma unroll
      for (int e = 0; e < V; ++e) red[warp * (D + 2) + lane * V + e] = x[e];
      if (lane == 0) {
        red[warp * (D + 2) + D] = m;
        red[warp * (D + 2) + D + 1] = l;
      }
      __syncthreads();
      if (part == 0) {
        float all = m;
        for (int k = 1; k < parts; ++k) all = fmaxf(all, red[(warp + k) * (D + 2) + D]);
        const float f0 = m == -INFINITY ? 0.f : fa::ex2_approx(m - all);
        l *= f0;
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] *= f0;
        m = all;
        for (int k = 1; k < parts; ++k) {
          const float* from = red + (warp + k) * (D + 2);
          const float f = from[D] == -INFINITY ? 0.f : fa::ex2_approx(from[D] - all);
          l += from[D + 1] * f;
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] += from[lane * V + e] * f;
        }
      }
    }
    if (there && part == 0) {
      const float inv = m == -INFINITY ? 0.f : vf / l;
      const int t = a.token_of(row0 + row), g = row0 + row - t * a.group;
      uint16_t* dst = a.o + (first + t) * a.o_stride_t + (static_cast<long long>(head) * a.group + g) * a.o_stride_h +
                      lane * V;
#pragma unroll
      for (int e = 0; e < V; e += 2)
        *reinterpret_cast<uint32_t*>(dst + e) = float2_to_pair<BF16>(x[e] * inv, x[e + 1] * inv);
    }
  }
}

template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(Few<D, NT>::THREADS, Few<D, NT>::PER_SM) cache4_few_kernel(const FewParams p) {
  using C = Few<D, NT>;
  using L = Layout<D>;
  constexpr int WARPS = C::WARPS, THREADS = C::THREADS;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int chunk_before[C::MAX_CHUNKS];
  __shared__ int weight_part[WARPS], unit_part[WARPS], weight_high[WARPS];
  __shared__ Share found;
  __shared__ int found_base, found_r;
  __shared__ bool joins;
  __shared__ __align__(8) unsigned long long copied_bars[WARPS][C::STAGES];
  const AttnParams& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int n = lane >> 2, c = lane & 3;
  const uint32_t s0 = fa::smem_u32(smem);
  const uint32_t ring = s0 + warp * C::RING;
  const uint8_t* ring_at = smem + warp * C::RING;
  float2* ml = reinterpret_cast<float2*>(smem + C::ML_OFF);
  float* rowf = reinterpret_cast<float*>(smem + C::ROWF_OFF);
  // this warp's stages: a barrier for each, and the parity of its next phase
  const uint32_t copied = fa::smem_u32(copied_bars[warp]);
  uint32_t phases = 0;
  bool late = false;
  if (lane == 0) {
    for (int i = 0; i < C::STAGES; ++i) fa::mbar_init(copied + 8 * i, 1);
    fa::fence_barrier_init();
    fa::fence_proxy_async_smem();
  }
  __syncwarp();
  fa::griddep_wait();
  if (threadIdx.x == 0) fa::griddep_launch_dependents();

  // ---- this block's part [pos, end) of the line
  const int chunks = (a.requests + THREADS - 1) / THREADS;
  long long total64 = 0;
  int units = 0;
  Share mine{};
  for (int k = 0; k < chunks; ++k) {
    const int r = k * THREADS + threadIdx.x;
    mine = Share{};
    if (r < a.requests) mine = share_of<C::ROWS>(p, r);
    // a request's weight fits 31 bits (the host sees to it), their sum may not,
    // if query_start decreases somewhere: it is added up in two halves
    const unsigned weight = static_cast<unsigned>(mine.units) * mine.grains;
    const unsigned low = __reduce_add_sync(0xffffffffu, weight & 0xffffu);
    const unsigned high = __reduce_add_sync(0xffffffffu, weight >> 16);
    const unsigned u = __reduce_add_sync(0xffffffffu, static_cast<unsigned>(mine.units));
    if (lane == 0) {
      weight_part[warp] = low;
      weight_high[warp] = high;
      unit_part[warp] = u;
    }
    __syncthreads();
    if (threadIdx.x == 0) chunk_before[k] = static_cast<int>(total64);
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      total64 += (static_cast<long long>(weight_high[i]) << 16) + weight_part[i];
      units += unit_part[i];
    }
    __syncthreads();
  }
  if (total64 > INT_MAX) total64 = 0;
  const int total = static_cast<int>(total64);
  // as many blocks as there are, or as many for each unit as its steps are
  // worth: equal units are then cut into equal pieces, or not at all
  int blocks = gridDim.x;
  const int least_run = max(1, C::MIN_STEPS >> p.shift);
  if (total < blocks * least_run) blocks = total ? min(blocks, units * max(1, total / units / least_run)) : 0;
  const Split split(total, max(blocks, 1));
  int pos = 0, end = 0;
  if (static_cast<int>(blockIdx.x) < blocks) {
    pos = split.start(blockIdx.x);
    end = split.start(blockIdx.x + 1);
  }
  int r = 0, base = 0;
  Share sh{};
  if (pos < end) {
    int k = 0;
    while (k + 1 < chunks && chunk_before[k + 1] <= pos) ++k;
    r = k * THREADS + threadIdx.x;
    if (chunks > 1) mine = r < a.requests ? share_of<C::ROWS>(p, r) : Share{};
    const int w = mine.units * mine.grains;
    int inc = w;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) unit_part[warp] = inc;
    __syncthreads();
    int before = chunk_before[k] + inc - w;
    for (int i = 0; i < warp; ++i) before += unit_part[i];
    if (before <= pos && pos - before < w) {
      found = mine;
      found_base = before;
      found_r = r;
    }
    __syncthreads();
    sh = found;
    base = found_base;
    r = found_r;
  }

  while (pos < end) {
    if (pos - base >= sh.units * sh.grains) {  // the next request (the line ends with the last one's units)
      base += sh.units * sh.grains;
      ++r;
      sh = share_of<C::ROWS>(p, r);
      continue;
    }
    const int unit = (pos - base) / sh.grains;
    const int off = pos - base - unit * sh.grains;
    const int stop = min(sh.grains, off + end - pos);
    const int head = unit % a.kv_heads;
    const int row0 = unit / a.kv_heads * C::ROWS;
    const int nrows = min(C::ROWS, sh.rows - row0);
    const int len = sh.len, tokens = a.token_of(sh.rows);
    // steps that hold keys
    const int k_begin = max(off << p.shift, 1) - 1, k_end = min(stop << p.shift, steps_of(len)) - 1;
    const int* table = a.tables + static_cast<long long>(r) * a.width;
    const bool starts = off == 0, ends = stop == sh.grains;
    const int first_block = starts ? static_cast<int>(blockIdx.x) : split.owner(pos - off);
    const float kf = a.scale_log2 * (a.k_scale ? a.k_scale[head] : 1.f);
    const float vf = a.v_scale ? a.v_scale[head] : 1.f;
    unsigned long long* count = p.done + first_block;
    // the unit's count is looked at here, and set up long before it is needed
    unsigned long long count_was = p.epoch << 16;
    if (!(starts && ends) && threadIdx.x == 0) count_was = *reinterpret_cast<volatile unsigned long long*>(count);

    // ---- query rows, 16 bytes per thread and turn: loads first
    constexpr int PER_ROW = D / 8, Q_TURNS = (C::ROWS * PER_ROW + THREADS - 1) / THREADS;
    uint4 q[Q_TURNS];
#pragma unroll
    for (int i = 0; i < Q_TURNS; ++i) {
      const int at = i * THREADS + threadIdx.x, row = at / PER_ROW, ch = at % PER_ROW;
      q[i] = make_uint4(0, 0, 0, 0);
      if (row < nrows) {
        const int t = a.token_of(row0 + row), g = row0 + row - t * a.group;
        q[i] = *reinterpret_cast<const uint4*>(a.q + (sh.first + t) * a.q_stride_t +
                                               (static_cast<long long>(head) * a.group + g) * a.q_stride_h + ch * 8);
      }
    }

    // ---- copies of this warp's first steps
    int page_ids = 0, ids_at = -32;  // page of step k_begin + warp + WARPS * (ids_at + lane)
    const int my_steps = k_end - k_begin - warp > 0 ? (k_end - k_begin - warp + WARPS - 1) / WARPS : 0;
    uint32_t good = 0;  // bit: that stage holds or awaits a step whose page is in the cache
    int issued = 0;
    auto issue = [&]() {
      if (issued < my_steps && !late) {
        if (issued >= ids_at + 32) {
          ids_at = issued;
          const int k = k_begin + warp + WARPS * (ids_at + lane);
          page_ids = k < k_end ? table[k >> 1] : -1;
        }
        const int page = __shfl_sync(0xffffffffu, page_ids, issued - ids_at);
        const int k = k_begin + warp + WARPS * issued;
        const int stage = issued % C::STAGES;
        const bool ok = page >= 0 && page < a.pages;
        good = (good & ~(1u << stage)) | (static_cast<uint32_t>(ok) << stage);
        if (ok) {
          const uint8_t* src = a.cache + (static_cast<long long>(page) * a.kv_heads + head) * L::PAGE_BYTES +
                               (k & 1) * C::STEP_BYTES;
          const uint32_t dst = ring + stage * C::STEP_BYTES;
          if (lane == 0) {
            fa::mbar_arrive_expect_tx(copied + 8 * stage, C::STEP_BYTES);
            copy_bulk(dst, src, C::STEP_BYTES, copied + 8 * stage);
          }
        }
        ++issued;
      }
    };
#pragma unroll
    for (int i = 0; i < C::STAGES - 1; ++i) issue();

    // ---- query rows into the order of the B fragments
#pragma unroll
    for (int i = 0; i < Q_TURNS; ++i) {
      const int at = i * THREADS + threadIdx.x;
      if (C::ROWS * PER_ROW % THREADS == 0 || at < C::ROWS * PER_ROW) {
        const int row = at / PER_ROW, ch = at % PER_ROW;
        uint4 x = q[i];
        float f = 1.f;
        if (BF16) {
          // into fp16 (row_exponent): numbers below 2^-14 of the row's largest are
          // rounded by up to 2^-25 of it
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          float y[8], mx = 0.f;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 v = bf162_to_float2(w[e]);
            y[2 * e] = v.x;
            y[2 * e + 1] = v.y;
            mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
#pragma unroll
          for (int d = PER_ROW / 2; d > 0; d /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
          const uint32_t ex = row_exponent(mx);
          f = __uint_as_float(ex << 23);
          const float inv = __uint_as_float((254u - ex) << 23);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] *= inv;
          x = make_uint4(fa::pack_half2(y[0], y[1]), fa::pack_half2(y[2], y[3]), fa::pack_half2(y[4], y[5]),
                         fa::pack_half2(y[6], y[7]));
        }
        if (ch == 0) rowf[row] = f;
        // chunk ch of the row: lane c = ch / (D/32), pair of k-steps ch % (D/32)
        const int lane_to = (row % 8) * 4 + ch / (D / 32);
        *reinterpret_cast<uint4*>(smem + C::Q_OFF + (((row / 8) * (D / 32) + ch % (D / 32)) * 32 + lane_to) * 16) = x;
      }
    }
    if ((count_was >> 16) != p.epoch) atomicCAS(count, count_was, p.epoch << 16);
    __syncthreads();

    Acc<D, NT> acc;
    float factor[NT][2];
    int limit[NT][2];
    int least = INT_MAX;  // first token that some row of the unit does not see
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = nt * 8 + 2 * c + i;
        factor[nt][i] = kf * rowf[row];
        limit[nt][i] = a.causal && row < nrows ? len - tokens + 1 + a.token_of(row0 + row) : len;
        acc.m[nt][i] = -INFINITY;
        acc.l[nt][i] = 0.f;
      }
    acc.large = false;
    least = a.causal ? min(len, len - tokens + 1 + a.token_of(row0)) : len;
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc.o[t][nt][e] = 0.f;

    // ---- this warp's steps
    for (int i = 0; i < my_steps && !late; ++i) {
      issue();
      __syncwarp();
      const int stage = i % C::STAGES;
      if ((good >> stage) & 1u) {
        if (!wait_copy(copied + 8 * stage, (phases >> stage) & 1u, p.timeout_ns)) {
          late = true;
          break;
        }
        phases ^= 1u << stage;
        good &= ~(1u << stage);
        const int key0 = (k_begin + warp + WARPS * i) * STEP;
        if (key0 + STEP > least)
          step<D, NT, true>(acc, ring_at + stage * C::STEP_BYTES, smem + C::Q_OFF, lane, factor, key0, len, limit);
        else
          step<D, NT, false>(acc, ring_at + stage * C::STEP_BYTES, smem + C::Q_OFF, lane, factor, key0, len, limit);
      }
      __syncwarp();  // the stage is free for the next copy
    }
    // a copy that did not come in time: the status word is set, this warp takes no
    // further steps, and waits until none is in flight (at least DRAIN_NS for each,
    // however short the limit: what lands after the block's end lands in another's memory)
    if (late) {
      for (int stage = 0; stage < C::STAGES; ++stage)
        if ((good >> stage) & 1u)
          wait_copy(copied + 8 * stage, (phases >> stage) & 1u, p.timeout_ns > DRAIN_NS ? p.timeout_ns : DRAIN_NS);
    }

    // ---- the four warps' sums become one
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float l = acc.l[nt][i];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        acc.l[nt][i] = l;
        // a row of NaN scores has no maximum, but its sums are NaN and stay
        if (acc.m[nt][i] == -INFINITY && l != l) acc.m[nt][i] = 0.f;
        if (n == 0) ml[warp * C::ROWS + nt * 8 + 2 * c + i] = make_float2(acc.m[nt][i], l);
      }
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem + warp * C::RING);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = nt * 8 + 2 * c + i;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) m = fmaxf(m, ml[w * C::ROWS + row].x);
        const float f = acc.m[nt][i] == -INFINITY ? 0.f : fa::ex2_approx(acc.m[nt][i] - m);
#pragma unroll
        for (int t = 0; t < D / 16; ++t)
          *reinterpret_cast<float2*>(mine + row * C::LD + n * (D / 8) + 2 * t) =
              make_float2(acc.o[t][nt][i] * f, acc.o[t][nt][2 + i] * f);
      }
    __syncthreads();
    const long long slot = static_cast<long long>(blockIdx.x) * 2 + (starts ? 1 : 0);
    for (int at = threadIdx.x; at < nrows * (D / 4); at += THREADS) {
      const int row = at / (D / 4), d = at % (D / 4) * 4;
      float m = -INFINITY, l = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, ml[w * C::ROWS + row].x);
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float2 u = ml[w * C::ROWS + row];
        l += u.x == -INFINITY ? 0.f : u.y * fa::ex2_approx(u.x - m);
        const float4 y = *reinterpret_cast<const float4*>(smem + w * C::RING + (row * C::LD + d) * 4);
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
      }
      if (starts && ends) {
        const float inv = m == -INFINITY ? 0.f : vf / l;
        const int t = a.token_of(row0 + row), g = row0 + row - t * a.group;
        store4<BF16>(a.o + (sh.first + t) * a.o_stride_t +
                         (static_cast<long long>(head) * a.group + g) * a.o_stride_h + d,
                     make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
      } else {
        *reinterpret_cast<float4*>(p.part_o + (slot * C::ROWS + row) * D + d) = x;
        if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * C::ROWS + row) * 2) = make_float2(m, l);
      }
    }
    if (!(starts && ends)) {
      // The block that finishes the unit's last piece joins them, in their
      // order whoever it is. The barrier orders the block's stores before
      // thread 0's fence, and that before its count.
      __syncthreads();
      if (threadIdx.x == 0) {
        const int pieces = split.owner(pos - off + sh.grains - 1) - first_block + 1;
        __threadfence();
        const int before = static_cast<int>(atomicAdd(count, 1ull) & 0xffffull);
        joins = before + 1 == pieces;
        if (joins) {
          __threadfence();
          atomicExch(count, p.epoch << 16);
        }
      }
      __syncthreads();
      if (joins)
        join<D, NT, BF16>(p, reinterpret_cast<float*>(smem), first_block,
                          split.owner(pos - off + sh.grains - 1) - first_block + 1, sh.first, row0, nrows, head, vf);
    }
    pos += stop - off;
    fa::fence_proxy_async_smem();  // what was stored in the rings comes before the next copies
    __syncthreads();               // the merge buffers, Q and row factors are free
  }
  if (a.zero_rest) {
    const int from = min(max(a.query_start[a.requests], 0), a.tokens);
    const long long per = static_cast<long long>(a.kv_heads) * a.group * (D / 4);
    for (long long i = static_cast<long long>(blockIdx.x) * THREADS + threadIdx.x; i < (a.tokens - from) * per;
         i += static_cast<long long>(gridDim.x) * THREADS) {
      const long long t = from + i / per, h = i % per / (D / 4);
      store4<BF16>(a.o + t * a.o_stride_t + h * a.o_stride_h + i % (D / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    }
  }
}

// -------------------------------------------------------------------- host
static bool args_ok(const gfx906_b200_cache4_attn_args& g) {
  return g.dtype >= 0 && g.dtype <= 1 && g.tokens >= 0 && g.heads > 0 && g.kv_heads > 0 && g.heads % g.kv_heads == 0 &&
         g.pages >= 0 && g.requests >= 0 && g.requests <= MAX_REQUESTS && g.width >= 0 &&
         g.width <= INT_MAX / PAGE && g.max_tokens >= 0 && isfinite(g.scale) &&
         static_cast<long long>(g.tokens) * (g.heads / g.kv_heads) <= INT_MAX;
}

struct Plan {
  int nt;      // row tiles of 8 NT rows
  int blocks;
  int shift;   // grains of the line
  size_t ml_off, done_off, many_off, bytes;
  bool fits;
  ManyPlan many;  // max_units 0: no request has that many rows
};
static Plan plan_of(const gfx906_b200_cache4_attn_args& g, int sms) {
  Plan pl{};
  const long long rows = static_cast<long long>(g.max_tokens) * (g.heads / g.kv_heads);
  pl.nt = rows <= 8 ? 1 : 2;
  pl.blocks = sms * (pl.nt == 1 ? Few<128, 1>::PER_SM : Few<128, 2>::PER_SM);
  // the line is counted in 31 bits: in single steps, unless the tables could hold
  // more of them (the lengths are not known here)
  const long long tiles = rows > FEW_ROWS ? static_cast<long long>(g.requests) * (FEW_ROWS / (8 * pl.nt))
                                          : static_cast<long long>(g.tokens) * (g.heads / g.kv_heads) / (8 * pl.nt) + g.requests;
  const long long units = tiles * g.kv_heads, steps = 2ll * g.width + 1;
  pl.fits = units <= INT_MAX;
  while (pl.fits && units * (((steps - 1) >> pl.shift) + 1) > INT_MAX) ++pl.shift;
  // no more blocks than the tables can hold steps for
  const long long most = pl.fits ? units * max(1ll, steps / Few<128, 1>::MIN_STEPS) : 1;
  pl.blocks = static_cast<int>(min(static_cast<long long>(pl.blocks), max(1ll, most)));
  const size_t slots = static_cast<size_t>(pl.blocks) * 2 * 8 * pl.nt;
  pl.ml_off = slots * g.D * sizeof(float);
  pl.done_off = pl.ml_off + slots * 2 * sizeof(float);
  pl.many_off = (pl.done_off + pl.blocks * sizeof(unsigned long long) + 255) & ~static_cast<size_t>(255);
  // of all requests, so many can have more than FEW_ROWS rows
  const long long large = static_cast<long long>(g.tokens) * (g.heads / g.kv_heads) / (FEW_ROWS + 1);
  if (rows > FEW_ROWS && g.requests > 0) {
    pl.many = many_plan(g.tokens, static_cast<int>(min(large, static_cast<long long>(g.requests))), g.heads / g.kv_heads,
                        g.kv_heads, g.D, sms);
    pl.fits = pl.fits && pl.many.fits;
  }
  pl.bytes = pl.many_off + ((pl.many.bytes + 255) & ~static_cast<size_t>(255));
  return pl;
}

template <int D, int NT, bool BF16>
static int launch_few(const FewParams& p, int blocks, cudaStream_t stream) {
  static SmemAttribute smem;
  if (!smem.set(cache4_few_kernel<D, NT, BF16>, Few<D, NT>::SMEM)) return GFX906_B200_ECUDA;
  return launch(cache4_few_kernel<D, NT, BF16>, dim3(blocks), dim3(Few<D, NT>::THREADS), Few<D, NT>::SMEM, stream, p);
}
template <int D, int NT>
static int launch_few_t(const FewParams& p, int dtype, int blocks, cudaStream_t stream) {
  return dtype ? launch_few<D, NT, true>(p, blocks, stream) : launch_few<D, NT, false>(p, blocks, stream);
}

static int attn(const gfx906_b200_cache4_attn_args& g, void* ws, size_t ws_bytes, cudaStream_t stream) {
  if (!head_dim_ok(g.D)) return GFX906_B200_EHEADDIM;
  if (!args_ok(g)) return GFX906_B200_EINVAL;
  if (g.tokens == 0) return GFX906_B200_OK;
  if (!g.q || !g.o || !g.query_start || (g.requests && !g.lengths) || (g.pages && !g.cache) ||
      (static_cast<long long>(g.requests) * g.width && !g.tables))
    return GFX906_B200_EINVAL;
  if (!aligned16(g.q) || !aligned16(g.o) || !aligned16(g.cache) ||
      ((g.q_stride_t | g.q_stride_h | g.o_stride_t | g.o_stride_h) & 7))
    return GFX906_B200_EALIGN;
  int sms = 0;
  const int rc = gfx906_b200_internal_device(&sms);
  if (rc != GFX906_B200_OK) return rc;
  const Plan pl = plan_of(g, sms);
  if (!pl.fits) return GFX906_B200_EINVAL;
  if (!ws || ws_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(ws) & 255u)) return GFX906_B200_EINVAL;
  FewParams p{};
  p.a = {static_cast<const uint16_t*>(g.q), static_cast<uint16_t*>(g.o), static_cast<const uint8_t*>(g.cache), g.tables,
         g.lengths, g.query_start, g.k_scale, g.v_scale, g.q_stride_t, g.q_stride_h, g.o_stride_t, g.o_stride_h,
         g.tokens, g.kv_heads, g.heads / g.kv_heads, g.pages, g.requests, g.width, g.causal != 0, g.zero_rest != 0,
         g.scale * 1.4426950408889634f,
         group_magic(static_cast<long long>(g.tokens) * (g.heads / g.kv_heads), g.heads / g.kv_heads)};
  p.max_rows = INT_MAX;
  p.shift = pl.shift;
  uint8_t* base = static_cast<uint8_t*>(ws);
  if (pl.many.max_units > 0) {
    ManyParams m{};
    m.a = p.a;
    m.min_rows = p.max_rows = FEW_ROWS;
    m.max_units = pl.many.max_units;
    m.sms = sms;
    m.part_o = reinterpret_cast<float*>(base + pl.many_off);
    m.part_ml = reinterpret_cast<float*>(base + pl.many_off + pl.many.ml_off);
    m.done = reinterpret_cast<unsigned long long*>(base + pl.many_off + pl.many.done_off);
    m.epoch = gfx906_b200_internal_next_epoch() & 0xffffffffffffull;
    m.timeout_ns = gfx906_b200_internal_timeout_ns();
    const int st = launch_many(m, g.D, g.dtype, stream);
    if (st != GFX906_B200_OK) return st;
  }
  p.part_o = reinterpret_cast<float*>(base);
  p.part_ml = reinterpret_cast<float*>(base + pl.ml_off);
  p.done = reinterpret_cast<unsigned long long*>(base + pl.done_off);
  p.epoch = gfx906_b200_internal_next_epoch() & 0xffffffffffffull;
  p.timeout_ns = gfx906_b200_internal_timeout_ns();
  if (g.D == 128)
    return pl.nt == 1 ? launch_few_t<128, 1>(p, g.dtype, pl.blocks, stream)
                      : launch_few_t<128, 2>(p, g.dtype, pl.blocks, stream);
  return pl.nt == 1 ? launch_few_t<64, 1>(p, g.dtype, pl.blocks, stream)
                    : launch_few_t<64, 2>(p, g.dtype, pl.blocks, stream);
}

}  // namespace c4

extern "C" {

// 1 when a wait of these kernels ran out; < 0 on a CUDA error.
int gfx906_b200_internal_cache4_few_status(int reset) {
  unsigned int st = 0;
  const unsigned int zero = 0;
  if (cudaMemcpyFromSymbol(&st, c4::g_cache4_few_status, sizeof(st)) != cudaSuccess) return -1;
  if (reset && cudaMemcpyToSymbol(c4::g_cache4_few_status, &zero, sizeof(zero)) != cudaSuccess) return -1;
  return st ? 1 : 0;
}

size_t gfx906_b200_cache4_attn_workspace_size(const gfx906_b200_cache4_attn_args* args) {
  int sms = 0;
  if (!args || !c4::head_dim_ok(args->D) || !c4::args_ok(*args) || args->tokens == 0 ||
      gfx906_b200_internal_device(&sms) != GFX906_B200_OK)
    return 0;
  return c4::plan_of(*args, sms).bytes;
}

int gfx906_b200_cache4_attn(const gfx906_b200_cache4_attn_args* args, void* workspace, size_t workspace_bytes,
                            cudaStream_t stream) {
  if (!args) return c4::done(GFX906_B200_EINVAL);
  return c4::done(c4::attn(*args, workspace, workspace_bytes, stream));
}

}  // extern "C"
