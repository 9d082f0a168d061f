// Attention of many new tokens per request against the paged 4-bit cache
// (cache4.cuh): prompts, and whole blocks of positions.
//
// A unit is 256 query rows (two tiles of 128 rows, a row being one (token, head
// of the group)) of one request and kv head, one per CTA. Its products run on
// the tensor core in fp16 (tcgen05, accumulators in tensor memory):
// S_i = Q_i K^T, O_i += P_i V for the two tiles i and every 128 keys. K and V
// go from 4 bits to fp16 on the way into shared memory: a warpgroup loads the
// codes of the next 128 keys into registers, converts them (exactly) and stores
// the swizzled tiles that the tensor core reads, while it works on the tiles
// before. Both query tiles share each conversion.
//
// Warps: 0-3 and 4-7 the softmax of query tile 0 and 1, one thread per row (the
// row's maximum, sum, exponentials and output scaling); 8-11 the conversion; 12
// issues the products.
//
// Units are dealt to the SMs as these become free, those of the longest requests
// first. The units of the last, partial wave (all of them, if they are fewer
// than the SMs) are cut into pieces of their key range, whose partial sums
// (32 bits, in the workspace) the CTA that finishes the last piece joins.
//
// Every wait is bounded (time limit from the host), as in the dense kernels: one
// that runs out sets the device status word and the CTA ends.
//
// Measured (B200, D = 128): 4096 rows x 24 heads against 16384 keys 760 us, 1085
// TFLOP/s, 0.66 of a library bf16 product's rate; four prompts of 511 to 1021
// tokens behind up to 8192, 32 heads on 8, causal, 249 us (803 TFLOP/s: its units
// differ in length, and the last wave is cut by their number). Called back to back
// for seconds, under the power cap, the former takes 820. Per 128 keys the
// products are 2050 cycles of the tensor core (8192 operations a cycle) out of the
// 4500 that pass at 1.84 to 1.97 GHz; the rest is the chain S -> softmax -> P ->
// next S of each tile, which two tiles hide in part only. Tensor memory (S0, S1,
// O0, O1) leaves no room for a third.
#include <limits.h>
#include <math.h>

#include "attn_row.cuh"
#include "cache4.cuh"
#include "cache4_attn.cuh"
#include "cache4_host.cuh"
#include "cache4_many.cuh"
#include "sm100_ptx.cuh"

namespace c4 {

using namespace fa;  // the PTX wrappers and row helpers

constexpr int M_ROWS = 128;          // query rows of a tile
constexpr int M_THREADS = 512;
constexpr int CONVERT_WARP = 8;      // four of them
constexpr int ISSUE_WARP = 12;
constexpr int BOX = 16384;           // 128 rows x 64 fp16 columns, 128-byte swizzle
// Registers: 512 threads at 128 each are launched; 256 * 184 + 128 * 64 + 128 * 80
// = 65536. The issue loop is on the critical path of every tile: with 32
// registers instead of 80 the compiler spilled in it, and 4096 rows x 24 heads
// against 16384 keys took 1086 us instead of 809 (48: 959, 72: 913).
constexpr uint32_t M_REGS_SOFTMAX = 184;
constexpr uint32_t M_REGS_CONVERT = 64;
constexpr uint32_t M_REGS_ISSUE = 80;
// All exponentials on MUFU here, none by polynomial: the conversions already
// keep the FMA pipe busy (4096 rows x 24 heads against 16384 keys: 775 us; with
// one pair in four on the FMA pipe, as the dense kernels have it, 793; two, 899).
constexpr int M_EMU_PAIRS = 0;
constexpr float M_RESCALE = 8.0f;    // log2 units, see the dense kernels
// A row's reference m is set this far below its largest score, so that P, which
// stays below 2^(M_HEAD + M_RESCALE), uses all of fp16's range: weights down to
// 2^-21 of the largest are rounded to 2^-11 of themselves, smaller ones by 2^-32
// of the largest at most (without it by 2^-25: small weights beside a large one
// would count in l and be lost in O).
constexpr float M_HEAD = 7.0f;
constexpr float M_LARGE = 4194304.f;  // 2^22: half a 32-bit step is 1/4 log2 unit, which fits above 2^15

__device__ unsigned int g_cache4_status = 0;  // 1: a wait ran out

template <int D>
struct Many {
  using L = Layout<D>;
  static constexpr int TILE = D / 64 * BOX;
  static constexpr int SLOTS = D == 128 ? 2 : 4;  // tiles of K, and as many of V
  static constexpr int B_Q = 0;
  static constexpr int B_K_FULL = 1, B_K_EMPTY = B_K_FULL + SLOTS;
  static constexpr int B_V_FULL = B_K_EMPTY + SLOTS, B_V_EMPTY = B_V_FULL + SLOTS;
  static constexpr int B_S = B_V_EMPTY + SLOTS, B_P_HALF = B_S + 2, B_P = B_P_HALF + 2, B_O = B_P + 2;
  static constexpr int B_WG = B_O + 2;  // [2] rendezvous of a softmax warpgroup
  static constexpr int B_DRAIN = B_WG + 2;
  static constexpr int BARS = B_DRAIN + 1;
  static constexpr int K_OFF = 2 * TILE, V_OFF = K_OFF + SLOTS * TILE, BAR_OFF = V_OFF + SLOTS * TILE;
  static constexpr int ROWF_OFF = BAR_OFF + BARS * 8 + 16;  // [2][128] exponents of Q's rows, a byte each
  static constexpr int STAGE_OFF = (ROWF_OFF + 2 * M_ROWS + 127) & ~127;  // 4 KiB per softmax warp
  static constexpr int SMEM = 1024 + STAGE_OFF + 8 * 4096;
  static_assert(SMEM <= 232448, "");
};

// Bounded waits for the barriers at `bars`; the word at `abort_at` stops all of them.
struct Waiter {
  uint32_t bars, abort_at;
  const ManyParams& p;
  __device__ __forceinline__ int aborted() const {
    int v;
    asm volatile("ld.volatile.shared.s32 %0, [%1];" : "=r"(v) : "r"(abort_at) : "memory");
    return v;
  }
  __device__ __forceinline__ bool slow(uint32_t bar, uint32_t parity, bool heed_abort) const {
    const uint64_t t0 = globaltimer_ns();
    uint32_t n = 0;
    while (true) {
      if (mbar_try_wait(bar, parity)) return true;
      if (heed_abort && aborted()) return false;
      if ((++n & 31u) == 0u && (globaltimer_ns() - t0 > (heed_abort ? p.timeout_ns : 100000000ull) || n > (1u << 24))) {
        asm volatile("st.volatile.shared.s32 [%0], %1;" ::"r"(abort_at), "r"(1) : "memory");
        atomicOr(&g_cache4_status, 1u);
        return false;
      }
    }
  }
  // Every lane of the warp gets the same answer.
  __device__ __forceinline__ bool operator()(int idx, uint32_t parity) const {
    const uint32_t bar = bars + 8u * idx;
    bool ok = mbar_try_wait(bar, parity);
    if (!ok) ok = slow(bar, parity, true);
    return __all_sync(0xffffffffu, ok);
  }
};

// Codes of one lane's share of a 16-token block of K or V (see Layout).
template <int D>
struct Codes {
  uint32_t a[D / 32], b[D / 32];  // K: tokens n, n + 8; V: tokens 2c, 2c + 1 and 2c + 8, 2c + 9
  uint32_t scales;
};
template <int D>
__device__ __forceinline__ void load_codes(Codes<D>& r, const uint8_t* block, int which, int lane) {
  using L = Layout<D>;
  if (!block) {  // no such page: its keys take no part, its values are zero
#pragma unroll
    for (int i = 0; i < D / 32; ++i) r.a[i] = r.b[i] = 0;
    r.scales = 0;
    return;
  }
  // the read-only path: the compiler may then move these loads past the barriers
  // of the tile before (plain loads: 3% slower)
  const uint8_t* codes = block + (which ? L::VC : L::KC) + lane * (D / 8);
  if (D == 128) {
    *reinterpret_cast<uint4*>(r.a) = __ldg(reinterpret_cast<const uint4*>(codes));
    *reinterpret_cast<uint4*>(r.b) = __ldg(reinterpret_cast<const uint4*>(codes + 4 * D));
  } else {
    *reinterpret_cast<uint2*>(r.a) = __ldg(reinterpret_cast<const uint2*>(codes));
    *reinterpret_cast<uint2*>(r.b) = __ldg(reinterpret_cast<const uint2*>(codes + 4 * D));
  }
  if (which)
    r.scales = __ldg(reinterpret_cast<const uint32_t*>(block + L::VS + (D == 128 ? lane : (lane >> 3) * 4 + (lane & 3)) * 4));
  else if (D == 128)
    r.scales = __ldg(reinterpret_cast<const uint32_t*>(block + L::KS + lane * 4));
  else
    r.scales = __ldg(reinterpret_cast<const uint16_t*>(block + L::KS + lane * 2));
}

// Eight channels (one word of codes) as fp16 into chunk `ch` of a row of a tile.
__device__ __forceinline__ void put_chunk(uint32_t row_addr, int ch, int row7, uint32_t word, uint32_t scale2) {
  uint32_t x[4];
  codes_to_half2(word, x);
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = mul_half2(x[e], scale2);
  st_shared_v4(row_addr + ((ch ^ row7) << 4), x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void swap_if(bool yes, uint32_t& a, uint32_t& b) {
  const uint32_t x = yes ? b : a, y = yes ? a : b;
  a = x;
  b = y;
}

// A lane's share of 16 tokens of K into rows row0 .. row0 + 15 of the tile at
// `tile`. Lanes whose chunks would meet in one bank group go through theirs in
// another order, so that eight lanes always write eight different ones.
template <int D>
__device__ __forceinline__ void put_k(Codes<D>& r, uint32_t tile, int row0, int lane) {
  const int n = lane >> 2, c = lane & 3;
  if (D == 128) {
    const bool flip = c >= 2;
    uint32_t w = scales_to_half2(r.scales), y = scales_to_half2(r.scales >> 16);
    uint32_t f0 = __byte_perm(w, w, 0x1010), f1 = __byte_perm(w, w, 0x3232);
    uint32_t g0 = __byte_perm(y, y, 0x1010), g1 = __byte_perm(y, y, 0x3232);
    swap_if(flip, r.a[0], r.a[D / 32 - 2]);
    swap_if(flip, r.a[1], r.a[D / 32 - 1]);
    swap_if(flip, r.b[0], r.b[D / 32 - 2]);
    swap_if(flip, r.b[1], r.b[D / 32 - 1]);
    swap_if(flip, f0, f1);
    swap_if(flip, g0, g1);
    const uint32_t at = tile + (c >> 1) * BOX + (row0 + n) * 128;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      const int ch = (c & 1) * 4 + (i ^ (flip ? 2 : 0));
      put_chunk(at, ch, n, r.a[i], i < 2 ? f0 : f1);
      put_chunk(at + 8 * 128, ch, n, r.b[i], i < 2 ? g0 : g1);
    }
  } else {
    const uint32_t w = scales_to_half2(r.scales);
    const uint32_t f = __byte_perm(w, w, 0x1010), g = __byte_perm(w, w, 0x3232);
    const uint32_t at = tile + (row0 + n) * 128;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      put_chunk(at, 2 * c + i, n, r.a[i], f);
      put_chunk(at + 8 * 128, 2 * c + i, n, r.b[i], g);
    }
  }
}
// 16 tokens of V; left: how many of them the request has (the others become zero).
template <int D>
__device__ __forceinline__ void put_v(Codes<D>& r, uint32_t tile, int row0, int left, int lane) {
  const int n = lane >> 2, c = lane & 3;
  uint32_t w = r.scales;
  if (left < BLOCK) {
    if (2 * c >= left) w &= 0xffffff00u;
    if (2 * c + 1 >= left) w &= 0xffff00ffu;
    if (2 * c + 8 >= left) w &= 0xff00ffffu;
    if (2 * c + 9 >= left) w &= 0x00ffffffu;
  }
  const uint32_t x = scales_to_half2(w), y = scales_to_half2(w >> 16);
  const uint32_t f[4] = {__byte_perm(x, x, 0x1010), __byte_perm(x, x, 0x3232), __byte_perm(y, y, 0x1010),
                         __byte_perm(y, y, 0x3232)};
  constexpr int W = D / 64;  // words of a token
  const bool flip = W == 2 && (n & 1);
  if (W == 2) {
    swap_if(flip, r.a[0], r.a[1]);
    swap_if(flip, r.a[D / 32 - 2], r.a[D / 32 - 1]);
    swap_if(flip, r.b[0], r.b[1]);
    swap_if(flip, r.b[D / 32 - 2], r.b[D / 32 - 1]);
  }
  const uint32_t at = tile + (W == 2 ? (n >> 2) * BOX : 0) + row0 * 128;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = 2 * c + (t & 1) + (t >> 1) * 8;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int ch = W == 2 ? 2 * (n & 3) + (i ^ (flip ? 1 : 0)) : n;
      put_chunk(at + row * 128, ch, row & 7, t < 2 ? r.a[(t & 1) * W + i] : r.b[(t & 1) * W + i], f[t]);
    }
  }
}

// What a CTA does: a unit (a block of 256 rows of a request, and a kv head), and
// which of the pieces of its key range.
struct Work {
  int r, block, head;   // r < 0: nothing
  int piece, most;      // piece of at most `most`
  int tail;             // number of the unit among those that are cut
  int slot0;            // its first piece's slot in the workspace
};
// The same with what follows from it, in shared memory.
struct Seg {
  int r, head, row0;     // request, kv head, first of its query rows
  int first, n, len;     // of the request
  int t0, t1;            // tiles of 128 keys
  int tail, slot0, piece, pieces;
};
__device__ __forceinline__ int many_blocks(const ManyParams& p, int r) {
  const Rows t = rows_of(p.a, r);
  const int rows = t.n * p.a.group;
  return rows > p.min_rows ? (rows + 2 * M_ROWS - 1) / (2 * M_ROWS) : 0;
}
// Measured at D = 128, us for four prompts of up to 1021 tokens behind up to 8192
// (8 x 4 heads) / 130 rows x 8 heads against 32768 keys / 100 requests of 70 to 300
// tokens, up to 1000 keys (2 x 4 heads) / 4096 rows x 24 heads, causal, against
// 16384: 275 / 68 / 124 / 482 with the numbers below.
constexpr int MAX_PIECES = 16;  // 8: 275 / 73 / 124 / 482; 32: 275 / 68 / 124 / 482
// Times the SMs: pieces of all units that are cut, at most. 2: 275 / 68 / 124 /
// 460; 6: 276 / 68 / 138 / 484.
constexpr int CUT_CTAS = 3;
constexpr int MIN_TILES = 4;  // of 128 keys, in a piece; 2: 289 / 68 / 123 / 482; 8: 279 / 68 / 124 / 482
constexpr int LOST = 0x8000;  // in a unit's count: a piece did not come

// All threads of the CTA. Units are numbered from the longest request down (up
// to SORTED requests; their loads differ most where they are few), of one request
// from the last block down, which sees the most keys, the kv heads of a block one
// after the other: what is dealt last is short. In the order of the requests the
// cases above take 295 / 68 / 139 / 481 us.
constexpr int SORTED = 128;
__device__ __forceinline__ Work find_work(const ManyParams& p) {
  __shared__ int part[M_THREADS / 32];
  __shared__ int found[2];
  __shared__ int2 loads[SORTED];  // blocks and length of each request
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool sorted = p.a.requests <= SORTED;
  int mine_blocks = 0, mine_len = 0;
  long long blocks = 0;
  for (int base = 0; base < p.a.requests; base += M_THREADS) {
    const int r = base + threadIdx.x;
    mine_blocks = r < p.a.requests ? many_blocks(p, r) : 0;
    if (sorted && r < p.a.requests) {
      mine_len = length_of(p.a, r);
      loads[r] = make_int2(mine_blocks, mine_len);
    }
    const int w = __reduce_add_sync(0xffffffffu, mine_blocks);
    if (lane == 0) part[warp] = w;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < M_THREADS / 32; ++i) blocks += part[i];
    __syncthreads();
  }
  Work out{-1, 0, 0, 0, 1, 0, 0};
  if (blocks > p.max_units / p.a.kv_heads) return out;  // query_start decreases somewhere
  const int units = static_cast<int>(blocks) * p.a.kv_heads;
  const int tail = units % p.sms, whole = units - tail;
  // the number of pieces that ends the last wave soonest (a lane tries each),
  // with a hundredth of a unit as the price of a piece (a thousandth: 275 / 60 /
  // 124 / 482, three: 275 / 85 / 124 / 482)
  const int pieces = lane % MAX_PIECES + 1;
  const int cost = pieces == 1 || tail * pieces <= CUT_CTAS * p.sms
                       ? (tail * pieces + p.sms - 1) / p.sms * 1000 / pieces + 10 * pieces
                       : 1 << 20;
  out.most = static_cast<int>(__reduce_min_sync(0xffffffffu, static_cast<unsigned>(cost) * MAX_PIECES + pieces - 1) %
                              MAX_PIECES) + 1;
  int unit = blockIdx.x;
  if (unit >= whole) {
    const int i = unit - whole;
    out.tail = i / out.most;
    out.piece = i % out.most;
    out.slot0 = i - out.piece;
    unit = whole + out.tail;
  } else {
    out.most = 1;
  }
  if (unit >= units) return out;
  out.head = unit % p.a.kv_heads;
  if (sorted) {
    const int at = unit / p.a.kv_heads;
    if (mine_blocks > 0) {
      int ahead = 0;  // blocks of longer requests
      for (int r = 0; r < p.a.requests; ++r) {
        const int2 other = loads[r];
        if (other.y > mine_len || (other.y == mine_len && r < static_cast<int>(threadIdx.x))) ahead += other.x;
      }
      if (ahead <= at && at < ahead + mine_blocks) {
        found[0] = threadIdx.x;
        found[1] = mine_blocks - 1 - (at - ahead);
      }
    }
    __syncthreads();
    out.r = found[0];
    out.block = found[1];
    return out;
  }
  const int want = static_cast<int>(blocks) - 1 - unit / p.a.kv_heads;
  int before = 0;
  for (int base = 0; base < p.a.requests && before <= want; base += M_THREADS) {
    const int r = base + threadIdx.x;
    const int w = r < p.a.requests ? many_blocks(p, r) : 0;
    int inc = w;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) part[warp] = inc;
    __syncthreads();
    int mine = before + inc - w;
#pragma unroll
    for (int i = 0; i < M_THREADS / 32; ++i) {
      if (i < warp) mine += part[i];
      before += part[i];
    }
    if (mine <= want && want < mine + w) {
      found[0] = r;
      found[1] = want - mine;
    }
    __syncthreads();
  }
  out.r = found[0];
  out.block = found[1];
  return out;
}

// One row of the pieces of a unit, added in their order.
template <int D, bool BF16>
__device__ __forceinline__ void join_row(const ManyParams& p, long long slot0, int pieces, int row, int head,
                                         uint16_t* out) {
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) + slot0 * 2 * M_ROWS + row;
  float m = -INFINITY, l = 0.f;
  for (int k = 0; k < pieces; ++k) m = fmaxf(m, __ldcg(ml + k * 2 * M_ROWS).x);
  for (int k = 0; k < pieces; ++k) {
    const float2 u = __ldcg(ml + k * 2 * M_ROWS);
    l += u.x == -INFINITY ? 0.f : u.y * ex2_approx(u.x - m);
  }
  const float inv = m == -INFINITY ? 0.f : (p.a.v_scale ? p.a.v_scale[head] : 1.f) / l;
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    float x[32];
#pragma unroll
    for (int e = 0; e < 32; ++e) x[e] = 0.f;
#pragma unroll 2
    for (int k = 0; k < pieces; ++k) {
      const float mk = __ldcg(ml + k * 2 * M_ROWS).x;
      const float f = mk == -INFINITY ? 0.f : ex2_approx(mk - m);
      const float4* src = reinterpret_cast<const float4*>(p.part_o + (slot0 + k) * 2 * M_ROWS * D) + row;
      float4 y[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) y[q] = __ldcg(src + (c / 4 + q) * 2 * M_ROWS);
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        x[4 * q] += y[q].x * f;
        x[4 * q + 1] += y[q].y * f;
        x[4 * q + 2] += y[q].z * f;
        x[4 * q + 3] += y[q].w * f;
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t h[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) h[e] = float2_to_pair<BF16>(x[8 * q + 2 * e] * inv, x[8 * q + 2 * e + 1] * inv);
      *reinterpret_cast<uint4*>(out + c + 8 * q) = make_uint4(h[0], h[1], h[2], h[3]);
    }
  }
}

// A warp's 32 rows of a query tile, from row0 on, into the swizzled layout of the
// tensor core's A operand, whole rows per D / 8 lanes; rows behind the request's
// last are zero. Rows of bf16 go into fp16 (row_exponent; numbers below 2^-14 of
// the row's largest are rounded by up to 2^-25 of it); rowf[row] keeps the exponent.
template <int D, bool BF16>
__device__ __forceinline__ void put_q(const AttnParams& a, const Seg& sg, int tile0, int row0, int lane, uint32_t tile,
                                      uint8_t* rowf) {
  constexpr int LANES = D / 8, ROWS = 32 / LANES;  // lanes of a row, rows of an access
  const int total = sg.n * a.group, ch = lane % LANES;
  const uint16_t* q = a.q + sg.first * a.q_stride_t + static_cast<long long>(sg.head) * a.group * a.q_stride_h + ch * 8;
  auto place = [&](int row) { return tile + (ch / 8) * BOX + row * 128 + (((ch % 8) ^ (row & 7)) << 4); };
#pragma unroll 8
  for (int row = row0 + lane / LANES; row < row0 + 32; row += ROWS) {
    const int at = tile0 + row, t = a.token_of(at);
    const bool there = at < total;
    const uint16_t* src = there ? q + t * a.q_stride_t + (at - t * a.group) * a.q_stride_h : a.q;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place(row)), "l"(src), "r"(there ? 16 : 0)
                 : "memory");
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  if (BF16) {  // each lane finds what it fetched itself
#pragma unroll 4
    for (int row = row0 + lane / LANES; row < row0 + 32; row += ROWS) {
      const uint4 x = ld_shared_v4(place(row));
      uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = bf162_to_float2(w[e]);
        mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
      }
#pragma unroll
      for (int d = LANES / 2; d > 0; d /= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
      const uint32_t ex = row_exponent(mx);
      const float inv = __uint_as_float((254u - ex) << 23);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = bf162_to_float2(w[e]);
        w[e] = pack_half2(f.x * inv, f.y * inv);
      }
      if (ch == 0) rowf[row] = static_cast<uint8_t>(ex);
      st_shared_v4(place(row), w[0], w[1], w[2], w[3]);
    }
  }
}

// The thread's number, read anew: nothing that follows from it is kept meanwhile.
__device__ __forceinline__ int fresh_tid() {
  int t;
  asm volatile("mov.u32 %0, %%tid.x;" : "=r"(t));
  return t;
}
__device__ __forceinline__ int tile_of() { return fresh_tid() / M_ROWS; }
// Where a softmax thread is in a unit.
struct Place {
  int tile, row, total, tile0, my_row;  // query tile, row in it; rows of the request, the tile's first, this one
  bool live;
  __device__ __forceinline__ Place(const Seg& s, const AttnParams& a) {
    const int t = fresh_tid();
    tile = t / M_ROWS;
    row = t % M_ROWS;
    total = s.n * a.group;
    tile0 = s.row0 + tile * M_ROWS;
    my_row = tile0 + row;
    live = my_row < total;
  }
};
// Is page i of the unit's request, as far as it holds tokens, outside the cache?
__device__ __forceinline__ bool page_missing(const AttnParams& a, const Seg& s, int i) {
  return i * PAGE < s.len &&
         static_cast<unsigned>(a.tables[static_cast<long long>(s.r) * a.width + i]) >= static_cast<unsigned>(a.pages);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(M_THREADS, 1) cache4_many_kernel(const ManyParams p) {
  using C = Many<D>;
  using L = Layout<D>;
  extern __shared__ uint8_t many_smem[];
  const AttnParams& a = p.a;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();

  __shared__ Seg sg;
  {
    const Work u = find_work(p);
    if (u.r < 0) return;
    const Rows rows = rows_of(a, u.r);
    const int len = length_of(a, u.r), row0 = u.block * 2 * M_ROWS;
    const int last_token = a.token_of(min(rows.n * a.group, row0 + 2 * M_ROWS) - 1);
    const int seen = a.causal ? max(0, min(len, len - rows.n + 1 + last_token)) : len;
    const int tiles = static_cast<int>((static_cast<unsigned>(seen) + BN - 1) / BN);
    const int pieces = max(1, min(u.most, tiles / MIN_TILES));
    if (u.piece >= pieces) return;
    if (threadIdx.x == 0) {
      sg = {u.r, u.head, row0, rows.first, rows.n, len, tiles * u.piece / pieces, tiles * (u.piece + 1) / pieces,
            u.tail, u.slot0, u.piece, pieces};
      for (int i = 0; i < 2 && pieces > 1; ++i) {  // set up the unit's counts, long before they are needed
        unsigned long long* count = p.done + u.tail * 2 + i;
        const unsigned long long was = *reinterpret_cast<volatile unsigned long long*>(count);
        if ((was >> 16) != p.epoch) atomicCAS(count, was, p.epoch << 16);
      }
    }
  }

  const uint32_t raw = smem_u32(many_smem);
  const uint32_t s0 = (raw + 1023u) & ~1023u;
  uint8_t* smem = many_smem + (s0 - raw);
  const uint32_t bars = s0 + C::BAR_OFF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* last_flag = reinterpret_cast<volatile int*>(tmem_slot + 2);  // [2], per tile
  if (threadIdx.x == 0) {
    mbar_init(bars + 8 * C::B_Q, sg.row0 + M_ROWS < sg.n * a.group ? 2 * M_ROWS : M_ROWS);
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(bars + 8 * (C::B_K_FULL + s), 4);
      mbar_init(bars + 8 * (C::B_K_EMPTY + s), 1);
      mbar_init(bars + 8 * (C::B_V_FULL + s), 4);
      mbar_init(bars + 8 * (C::B_V_EMPTY + s), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars + 8 * (C::B_S + i), 1);
      mbar_init(bars + 8 * (C::B_P_HALF + i), M_ROWS);
      mbar_init(bars + 8 * (C::B_P + i), M_ROWS);
      mbar_init(bars + 8 * (C::B_O + i), 1);
      mbar_init(bars + 8 * (C::B_WG + i), M_ROWS);
      last_flag[i] = 0;
    }
    mbar_init(bars + 8 * C::B_DRAIN, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_smem();
  }
  if (warp == ISSUE_WARP) {
    tmem_alloc(smem_u32(tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const Waiter wait{bars, smem_u32(tmem_slot + 1), p};

  if (warp >= ISSUE_WARP) {
    // ------------------------------------------------------ issue of products
    setmaxnreg_dec<M_REGS_ISSUE>();
    const int t0 = sg.t0, t1 = sg.t1;
    const bool has1 = sg.row0 + M_ROWS < sg.n * a.group;
    if (warp == ISSUE_WARP && t0 < t1) {
      constexpr uint32_t IDESC_QK = idesc_f16_f32(M_ROWS, BN, 0, 0);
      constexpr uint32_t IDESC_PV = idesc_f16_f32(M_ROWS, D, 0, 1);
      const uint64_t dQ = sdesc_sw128(s0, 16, 1024);
      const uint64_t dK = sdesc_sw128(s0 + C::K_OFF, 16, 1024);
      const uint64_t dV = sdesc_sw128(s0 + C::V_OFF, BOX, 1024);
      auto issue_qk = [&](int i, int slot) {
        const uint64_t q = dQ + (static_cast<uint32_t>(i * C::TILE) >> 4);
        const uint64_t k = dK + (static_cast<uint32_t>(slot * C::TILE) >> 4);
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const uint32_t o = static_cast<uint32_t>(c * BOX) >> 4;
          mma4_ss_warp(tmem + i * 128, q + o, q + o + 2, q + o + 4, q + o + 6, k + o, k + o + 2, k + o + 4, k + o + 6,
                       IDESC_QK, c > 0 ? 1u : 0u);
        }
        tc_commit_warp(bars + 8 * (C::B_S + i));
      };
      // keys 0-63 once the first half of P is stored, then the rest
      auto issue_pv = [&](int i, int slot, bool acc, uint32_t parity) -> bool {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (!wait((h ? C::B_P : C::B_P_HALF) + i, parity)) return false;
          tc_fence_after();
          const uint64_t v = dV + (static_cast<uint32_t>(slot * C::TILE + 4 * h * 2048) >> 4);
          mma4_ts_warp(tmem + 256 + i * D, tmem + i * 128 + 32 * h, v, v + 128, v + 256, v + 384, IDESC_PV,
                       (acc || h > 0) ? 1u : 0u);
        }
        return true;
      };
      bool ok = wait(C::B_Q, 0);
      tc_fence_after();
      for (int j = t0; ok && j < t1; ++j) {
        const int it = j - t0, slot = it % C::SLOTS;
        const uint32_t ph = (it / C::SLOTS) & 1;
        const int before = (it + C::SLOTS - 1) % C::SLOTS;  // slot of the tile before
        if (!wait(C::B_K_FULL + slot, ph)) { ok = false; break; }
        tc_fence_after();
        issue_qk(0, slot);
        if (has1) {
          if (it > 0) {
            if (!issue_pv(1, before, it > 1, (it - 1) & 1)) { ok = false; break; }
            tc_commit_warp(bars + 8 * (C::B_V_EMPTY + before));
          }
          issue_qk(1, slot);
        }
        tc_commit_warp(bars + 8 * (C::B_K_EMPTY + slot));
        if (!wait(C::B_V_FULL + slot, ph)) { ok = false; break; }
        tc_fence_after();
        if (!issue_pv(0, slot, it > 0, it & 1)) { ok = false; break; }
        if (j + 1 == t1) tc_commit_warp(bars + 8 * (C::B_O + 0));
        if (!has1) tc_commit_warp(bars + 8 * (C::B_V_EMPTY + slot));
      }
      if (ok && has1) {
        const int it = t1 - t0 - 1;
        if (issue_pv(1, it % C::SLOTS, it > 0, it & 1))
          tc_commit_warp(bars + 8 * (C::B_O + 1));
        else
          ok = false;
      }
      if (!ok) {  // let every product end before its memory goes away
        tc_commit_warp(bars + 8 * C::B_DRAIN);
        if (!mbar_try_wait(bars + 8 * C::B_DRAIN, 0)) wait.slow(bars + 8 * C::B_DRAIN, 0, false);
      }
    }
    __syncwarp();
  } else if (warp >= CONVERT_WARP) {
    // ------------------------------------------------------------- conversion
    setmaxnreg_dec<M_REGS_CONVERT>();
    const int w = warp - CONVERT_WARP;  // blocks w and w + 4 of a tile: one in each of its pages
    const int len = sg.len, t0 = sg.t0, t1 = sg.t1;
    const int* table = a.tables + static_cast<long long>(sg.r) * a.width;
    const uint8_t* cache = a.cache + static_cast<long long>(sg.head) * L::PAGE_BYTES + w * L::BLOCK_BYTES;
    const long long page_stride = static_cast<long long>(a.kv_heads) * L::PAGE_BYTES;
    const int pages_held = (len + PAGE - 1) / PAGE;
    // where this warp's block of page 2 j + i is, or null
    auto block_of = [&](int j, int i) -> const uint8_t* {
      const int at = 2 * j + i;
      const int page = j < t1 && at < pages_held ? table[at] : -1;
      return page >= 0 && page < a.pages ? cache + page * page_stride : nullptr;
    };
    Codes<D> k[2], v[2];
    const uint8_t* block[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      block[i] = block_of(t0, i);
      load_codes(k[i], block[i], 0, lane);
      load_codes(v[i], block[i], 1, lane);
      block[i] = block_of(t0 + 1, i);
    }
    for (int j = t0; j < t1; ++j) {
      const int it = j - t0, slot = it % C::SLOTS;
      const uint32_t ph = (it / C::SLOTS) & 1;
      if (!wait(C::B_K_EMPTY + slot, ph ^ 1u)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i) put_k<D>(k[i], s0 + C::K_OFF + slot * C::TILE, (4 * i + w) * BLOCK, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 8 * (C::B_K_FULL + slot));
#pragma unroll
      for (int i = 0; i < 2; ++i) load_codes(k[i], block[i], 0, lane);
      if (!wait(C::B_V_EMPTY + slot, ph ^ 1u)) break;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        put_v<D>(v[i], s0 + C::V_OFF + slot * C::TILE, (4 * i + w) * BLOCK, len - j * BN - (4 * i + w) * BLOCK, lane);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(bars + 8 * (C::B_V_FULL + slot));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        load_codes(v[i], block[i], 1, lane);
        block[i] = block_of(j + 2, i);
      }
    }
  } else {
    // ---------------------------------------------------------------- softmax
    // A score row fills 128 registers, and what else lives through the loop over
    // the tiles decides whether the compiler has to spill it (measured: 1.5
    // times the time). So that is kept to what each tile needs -- the flags
    // are bits of one word -- and everything else is
    // looked up again behind the loop, from the thread's number and the unit.
    setmaxnreg_inc<M_REGS_SOFTMAX>();
    enum : uint32_t { S_PARITY = 1, LARGE = 2, HOLES = 4, FIRST = 8, OK = 16 };
    const uint32_t bar = bars + 8 * (warp >> 2);  // of this query tile: index + tile
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + (warp >> 2) * 128;
    uint32_t st = OK;
    auto tile_wait = [&](int idx, uint32_t parity) -> bool {
      bool ok = mbar_try_wait(bar + 8u * idx, parity);
      if (!ok) ok = wait.slow(bar + 8u * idx, parity, true);
      return __all_sync(0xffffffffu, ok);
    };
    if (sg.row0 + (warp >> 2) * M_ROWS < sg.n * a.group) {
      float sl2 = a.scale_log2 * (a.k_scale ? a.k_scale[sg.head] : 1.f);
      int left = sg.t1 - sg.t0;  // tiles
      int until;                 // keys that this row sees from the next tile's first on
      {
        const Place at(sg, a);
        put_q<D, BF16>(a, sg, at.tile0, at.row - lane, lane, s0 + at.tile * C::TILE, smem + C::ROWF_OFF + at.tile * M_ROWS);
        fence_proxy_async_smem();
        mbar_arrive(bars + 8 * C::B_Q);
        __syncwarp();
        if (BF16) sl2 *= __uint_as_float(static_cast<uint32_t>(smem[C::ROWF_OFF + threadIdx.x]) << 23);
        until = (a.causal && at.live ? min(sg.len, sg.len - sg.n + 1 + a.token_of(at.my_row)) : sg.len) - sg.t0 * BN;
        bool holes = false;
        for (int i = 2 * sg.t0 + lane; i < 2 * sg.t1; i += 32) holes |= page_missing(a, sg, i);
        if (__any_sync(0xffffffffu, holes)) st |= HOLES;
      }
      float m = -INFINITY, l = 0.f;
      st |= FIRST;
#pragma unroll 1
      for (; left > 0; --left, until -= BN) {
        if (!tile_wait(C::B_S, st & S_PARITY)) { st &= ~OK; break; }
        st ^= S_PARITY;
        tc_fence_after();
        uint32_t s[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld32(tS + 32 * c, s + 32 * c);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) reg_fence32(s + 32 * c);
        int lo = 0, hi = min(BN, until);
        if (st & HOLES) {  // pages outside the cache, whose keys take no part
          const int j = sg.t1 - left;
          if (page_missing(a, sg, 2 * j)) lo = PAGE;
          if (page_missing(a, sg, 2 * j + 1)) hi = min(hi, PAGE);
        }
        const bool full = __all_sync(0xffffffffu, lo == 0 && hi == BN);
        const float mx = row_extreme(s, hi, full, sl2 >= 0.f, lo);
        const float m_new = lo < hi ? fmaxf(m, __fsub_rn(__fmul_rn(mx, sl2), M_HEAD)) : m;
        const bool need = m_new > m + M_RESCALE;
        if (__any_sync(0xffffffffu, need)) {
          float f = 1.f;
          if (need) {
            f = ex2_approx(m - m_new);
            m = m_new;
          }
          rescale_rows<D>(tS + 256 - (D == 128 ? 0 : (tile_of() * (128 - D))), !(st & FIRST), f);
          l *= f;
          if (__any_sync(0xffffffffu, fabsf(m) > M_LARGE && m > -INFINITY)) st |= LARGE;
        }
        st &= ~FIRST;
        const float neg_m = m == -INFINITY ? 0.f : -m;
        float sum0, sum1;
        // Where scores are so large that m is a rounded product, each score is
        // rounded as m was, or the largest would lie half a step of m off it.
        if (full && !(st & LARGE))
          row_exp_store<M_EMU_PAIRS, false>(s, sl2, neg_m, hi, tS, sum0, sum1, bar + 8 * C::B_P_HALF, [] {}, [] {});
        else
          row_exp_store<M_EMU_PAIRS, true, true>(s, sl2, neg_m, hi, tS, sum0, sum1, bar + 8 * C::B_P_HALF, [] {}, [] {}, lo);
        l += sum0 + sum1;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar + 8 * C::B_P);
      }
      if (m == -INFINITY && l != l) m = 0.f;  // a row of NaN scores has no maximum, its sums are NaN
      const bool some = sg.t0 < sg.t1;
      if ((st & OK) && some) {
        if (!tile_wait(C::B_O, 0)) st &= ~OK;
        tc_fence_after();
      }
      const Place at(sg, a);
      const uint32_t tO = tS + 256 - at.tile * (128 - D);
      if (sg.pieces == 1 && (st & OK)) {
        // through this warp's staging tile, so that 8 lanes store 128 contiguous bytes of a row
        const float inv = m == -INFINITY ? 0.f : (a.v_scale ? a.v_scale[sg.head] : 1.f) / l;
        uint16_t* const o_head = a.o + sg.first * a.o_stride_t + static_cast<long long>(sg.head) * a.group * a.o_stride_h;
        const uint32_t stg = s0 + C::STAGE_OFF + warp * 4096;
#pragma unroll 1
        for (int hf = 0; hf < D / 64; ++hf) {
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            uint32_t o[32];
            if (some) {
              tmem_ld32(tO + 64 * hf + 32 * cc, o);
              tmem_wait_ld();
              reg_fence32(o);
            }
            // a row that sees no key is zero, whatever the accumulator holds
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = m == -INFINITY ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              uint32_t h[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                h[i] = float2_to_pair<BF16>(__uint_as_float(o[8 * e + 2 * i]), __uint_as_float(o[8 * e + 2 * i + 1]));
              st_shared_v4(stg + lane * 128 + (((cc * 4 + e) ^ (lane & 7)) << 4), h[0], h[1], h[2], h[3]);
            }
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3), ch = lane & 7;
            const uint4 x = ld_shared_v4(stg + r * 128 + ((ch ^ (r & 7)) << 4));
            const int to = at.my_row - lane + r;
            if (to < at.total)
              *reinterpret_cast<uint4*>(o_head + a.token_of(to) * a.o_stride_t +
                                        (to - a.token_of(to) * a.group) * a.o_stride_h + hf * 64 + ch * 8) = x;
          }
          __syncwarp();
        }
      }
      if (sg.pieces > 1) {
        // a piece: unnormalised O, m and l to the workspace, chunk-major (4 columns
        // of one row are 16 bytes, the 256 rows of a chunk are contiguous)
        bool met = st & OK;
        if (met) {
          const long long slot = sg.slot0 + sg.piece;
          *reinterpret_cast<float2*>(p.part_ml + (slot * 2 * M_ROWS + at.tile * M_ROWS + at.row) * 2) = make_float2(m, l);
          if (some) {
            float* dst = p.part_o + slot * 2 * M_ROWS * D + (at.tile * M_ROWS + at.row) * 4;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(tO + 32 * c, o);
              tmem_wait_ld();
              reg_fence32(o);
#pragma unroll
              for (int e = 0; e < 8; ++e)
                *reinterpret_cast<float4*>(dst + (c * 8 + e) * 2 * M_ROWS * 4) =
                    make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]), __uint_as_float(o[4 * e + 2]),
                                __uint_as_float(o[4 * e + 3]));
            }
          }
          // The rendezvous orders the warpgroup's stores before one thread's
          // fence, and that before its count.
          mbar_arrive(bar + 8 * C::B_WG);
          met = tile_wait(C::B_WG, 0);
        }
        if (at.row == 0) {
          unsigned long long* count = p.done + sg.tail * 2 + at.tile;
          if (!met) atomicOr(count, static_cast<unsigned long long>(LOST));
          __threadfence();
          const int before = static_cast<int>(atomicAdd(count, 1ull) & 0xffffull);
          const bool last = (before & ~LOST) + 1 == sg.pieces;
          if (last) {
            __threadfence();
            atomicExch(count, p.epoch << 16);
          }
          last_flag[at.tile] = last && !(before & LOST);
        }
        if (met) {
          mbar_arrive(bar + 8 * C::B_WG);
          met = tile_wait(C::B_WG, 1);
        }
        if (met && last_flag[at.tile] && at.live) {
          const int t = a.token_of(at.my_row);
          join_row<D, BF16>(p, sg.slot0, sg.pieces, at.tile * M_ROWS + at.row, sg.head,
                            a.o + (sg.first + t) * a.o_stride_t +
                                (static_cast<long long>(sg.head + 1) * a.group + at.my_row - (t + 1) * a.group) * a.o_stride_h);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == ISSUE_WARP) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// -------------------------------------------------------------------- host
// requests: those that can have rows for this kernel.
ManyPlan many_plan(int tokens, int requests, int group, int kv_heads, int D, int sms) {
  ManyPlan pl{};
  const long long blocks = static_cast<long long>(tokens) * group / (2 * M_ROWS) + requests;
  if (blocks * kv_heads > INT_MAX - CUT_CTAS * sms) return pl;  // CTAs of a launch
  pl.fits = true;
  pl.max_units = static_cast<int>(blocks * kv_heads);
  // pieces of the units that are cut, fewer than SMs (find_work): 58 MB at D = 128
  const int cut = pl.max_units < sms ? pl.max_units : sms;
  const size_t rows = static_cast<size_t>(cut * MAX_PIECES < CUT_CTAS * sms ? cut * MAX_PIECES : CUT_CTAS * sms) * 2 * M_ROWS;
  pl.ml_off = rows * D * sizeof(float);
  pl.done_off = pl.ml_off + rows * 2 * sizeof(float);
  pl.bytes = pl.done_off + static_cast<size_t>(sms) * 2 * sizeof(unsigned long long);
  return pl;
}

template <int D, bool BF16>
static int launch_many_t(const ManyParams& p, cudaStream_t stream) {
  static SmemAttribute smem;
  if (!smem.set(cache4_many_kernel<D, BF16>, Many<D>::SMEM)) return GFX906_B200_ECUDA;
  // the units, and the pieces of those of the last wave
  const long long cut = static_cast<long long>(p.max_units < p.sms ? p.max_units : p.sms - 1) * (MAX_PIECES - 1);
  const long long ctas = p.max_units + (cut < CUT_CTAS * p.sms ? cut : CUT_CTAS * p.sms);
  return launch(cache4_many_kernel<D, BF16>, dim3(static_cast<unsigned>(ctas)), dim3(M_THREADS), Many<D>::SMEM, stream, p);
}

int launch_many(const ManyParams& p, int D, int dtype, cudaStream_t stream) {
  if (D == 128) return dtype ? launch_many_t<128, true>(p, stream) : launch_many_t<128, false>(p, stream);
  return dtype ? launch_many_t<64, true>(p, stream) : launch_many_t<64, false>(p, stream);
}

}  // namespace c4

// 1 when a wait of these kernels ran out; < 0 on a CUDA error.
extern "C" int gfx906_b200_internal_cache4_status(int reset) {
  unsigned int st = 0;
  const unsigned int zero = 0;
  if (cudaMemcpyFromSymbol(&st, c4::g_cache4_status, sizeof(st)) != cudaSuccess) return -1;
  if (reset && cudaMemcpyToSymbol(c4::g_cache4_status, &zero, sizeof(zero)) != cudaSuccess) return -1;
  return st ? 1 : 0;
}
