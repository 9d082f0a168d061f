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
// When a call has fewer units than half the SMs, each unit's keys are cut into
// `pieces` runs with a CTA each; their partial sums (32 bits, in the workspace)
// are joined by cache4_many_join_kernel.
//
// Every wait is bounded (time limit from the host), as in the dense kernels: one
// that runs out sets the device status word and the CTA ends.
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
// Registers: 512 threads at 128 each are launched; 256 * 192 + 128 * 96 + 128 * 32 = 65536.
constexpr uint32_t M_REGS_SOFTMAX = 192;
constexpr uint32_t M_REGS_CONVERT = 96;
constexpr uint32_t M_REGS_ISSUE = 32;
constexpr float M_RESCALE = 8.0f;    // log2 units, see the dense kernels
constexpr float M_LARGE = 67108864.f;  // 2^26: half a 32-bit step is 2 log2 units

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
  static constexpr int B_DRAIN = B_O + 2;
  static constexpr int BARS = B_DRAIN + 1;
  static constexpr int K_OFF = 2 * TILE, V_OFF = K_OFF + SLOTS * TILE, BAR_OFF = V_OFF + SLOTS * TILE;
  static constexpr int STAGE_OFF = (BAR_OFF + BARS * 8 + 16 + 127) & ~127;  // 4 KiB per softmax warp
  static constexpr int SMEM = 1024 + STAGE_OFF + 8 * 4096;
  static_assert(SMEM <= 232448, "");
};

struct Waiter {
  uint32_t bars;
  volatile int* abort_flag;
  unsigned long long timeout_ns;
  __device__ __forceinline__ bool slow(uint32_t bar, uint32_t parity, bool heed_abort) const {
    const uint64_t t0 = globaltimer_ns();
    uint32_t n = 0;
    while (true) {
      if (mbar_try_wait(bar, parity)) return true;
      if (heed_abort && *abort_flag) return false;
      if ((++n & 31u) == 0u && (globaltimer_ns() - t0 > (heed_abort ? timeout_ns : 100000000ull) || n > (1u << 24))) {
        *abort_flag = 1;
        atomicOr(&g_cache4_status, 1u);
        return false;
      }
    }
  }
  // Every lane of the warp gets the same answer.
  __device__ __forceinline__ bool operator()(int idx, uint32_t parity) const {
    const uint32_t bar = bars + 8u * idx;
    const bool ok = mbar_try_wait(bar, parity) || slow(bar, parity, true);
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

// The unit of CTA `index` of the launch: request, its first block's index among
// all blocks, and the block wanted; false: no such unit.
struct Unit {
  int r, block;  // request, block of 256 rows within it
};
__device__ __forceinline__ int many_blocks(const ManyParams& p, int r) {
  const long long rows = static_cast<long long>(rows_of(p.a, r).n) * p.a.group;
  return rows > p.min_rows ? static_cast<int>((rows + 2 * M_ROWS - 1) / (2 * M_ROWS)) : 0;
}
// Whole block of THREADS threads.
template <int THREADS>
__device__ __forceinline__ bool find_unit(const ManyParams& p, int want, Unit* out) {
  __shared__ int part[THREADS / 32];
  __shared__ int found[2];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  int total = 0;
  if (threadIdx.x == 0) found[0] = -1;
  for (int base = 0; base < p.a.requests && total <= want; base += THREADS) {
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
    int before = total + inc - w;
#pragma unroll
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += part[i];
      total += part[i];
    }
    if (before <= want && want < before + w) {
      found[0] = r;
      found[1] = want - before;
    }
    __syncthreads();
  }
  __syncthreads();
  out->r = found[0];
  out->block = found[1];
  return found[0] >= 0;
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

  // the last blocks of a request see the most keys: they come first
  const int per_block = a.kv_heads * p.pieces;
  const int head = static_cast<int>(blockIdx.x) % per_block / p.pieces;
  const int piece = static_cast<int>(blockIdx.x) % p.pieces;
  const int want = p.max_blocks - 1 - static_cast<int>(blockIdx.x) / per_block;
  Unit u;
  if (!find_unit<M_THREADS>(p, want, &u)) return;
  const Rows rows = rows_of(a, u.r);
  const int len = length_of(a, u.r);
  const int row0 = u.block * 2 * M_ROWS;
  const int total_rows = rows.n * a.group;
  const bool has1 = row0 + M_ROWS < total_rows;
  const int last_token = (min(total_rows, row0 + 2 * M_ROWS) - 1) / a.group;
  const int seen = a.causal ? max(0, min(len, len - rows.n + 1 + last_token)) : len;
  const int all_tiles = (seen + BN - 1) / BN;
  const int t0 = static_cast<int>(static_cast<long long>(all_tiles) * piece / p.pieces);
  const int t1 = static_cast<int>(static_cast<long long>(all_tiles) * (piece + 1) / p.pieces);
  const int* table = a.tables + static_cast<long long>(u.r) * a.width;

  const uint32_t raw = smem_u32(many_smem);
  const uint32_t s0 = (raw + 1023u) & ~1023u;
  uint8_t* smem = many_smem + (s0 - raw);
  const uint32_t bars = s0 + C::BAR_OFF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + C::BARS * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  if (threadIdx.x == 0) {
    mbar_init(bars + 8 * C::B_Q, 2 * M_ROWS);
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
  const Waiter wait{bars, abort_flag, p.timeout_ns};

  if (warp >= ISSUE_WARP) {
    // ------------------------------------------------------ issue of products
    setmaxnreg_dec<M_REGS_ISSUE>();
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
    const uint8_t* cache = a.cache + static_cast<long long>(head) * L::PAGE_BYTES + w * L::BLOCK_BYTES;
    const long long page_stride = static_cast<long long>(a.kv_heads) * L::PAGE_BYTES;
    const int pages_held = (len + PAGE - 1) / PAGE;
    // where this warp's block of page 2 j + i is, or null
    auto block_of = [&](int j, int i) -> const uint8_t* {
      const int at = 2 * j + i;
      const int page = j < t1 && at < pages_held ? __ldg(table + at) : -1;
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
    setmaxnreg_inc<M_REGS_SOFTMAX>();
    const int ti = warp >> 2, quad = warp & 3;
    const int row = quad * 32 + lane;
    const int my_row = row0 + ti * M_ROWS + row;  // of the request
    const bool live = my_row < total_rows;
    float factor = 1.f;
    if (ti == 0 || has1) {
      // this thread's row of q, in the swizzled layout of the tensor core's A operand
      const int t = my_row / a.group, g = my_row % a.group;
      const uint4* src = reinterpret_cast<const uint4*>(
          a.q + (rows.first + t) * a.q_stride_t + (static_cast<long long>(head) * a.group + g) * a.q_stride_h);
      uint4 x[D / 8];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) x[c] = live ? __ldg(src + c) : make_uint4(0, 0, 0, 0);
      if (BF16) {
        // rows of bf16 are brought to [1, 2) by a power of two and then fit fp16
        // (what falls below 2^-24 of a row's largest is lost)
        float mx = 0.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = bf162_to_float2(w[e]);
            mx = fmax3(mx, fabsf(f.x), fabsf(f.y));
          }
        }
        const uint32_t ex = (__float_as_uint(mx) >> 23) & 255u;
        const bool scaled = ex > 0 && ex < 254;
        if (scaled) factor = __uint_as_float(ex << 23);
        const float inv = scaled ? __uint_as_float((254u - ex) << 23) : 1.f;
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = bf162_to_float2(w[e]);
            w[e] = pack_half2(f.x * inv, f.y * inv);
          }
          x[c] = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        st_shared_v4(s0 + ti * C::TILE + (c / 8) * BOX + row * 128 + (((c % 8) ^ (row & 7)) << 4), x[c].x, x[c].y,
                     x[c].z, x[c].w);
    }
    fence_proxy_async_smem();
    mbar_arrive(bars + 8 * C::B_Q);

    if (ti == 0 || has1) {
      const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
      const uint32_t tS = tmem + lane_off + ti * 128;
      const uint32_t tO = tmem + lane_off + 256 + ti * D;
      const float sl2 = a.scale_log2 * (a.k_scale ? a.k_scale[head] : 1.f) * factor;
      const bool pos = sl2 >= 0.f;
      // keys this row sees: [0, limit)
      const int limit = a.causal && live ? min(len, len - rows.n + 1 + my_row / a.group) : len;
      bool holes = false;  // pages outside the cache, whose keys take no part
      for (int i = 2 * t0 + lane; i < 2 * t1 && i * PAGE < len; i += 32)
        holes |= static_cast<unsigned>(__ldg(table + i)) >= static_cast<unsigned>(a.pages);
      holes = __any_sync(0xffffffffu, holes);
      float m = -INFINITY, l = 0.f;
      bool ok = true, large = false;
      for (int j = t0; j < t1; ++j) {
        const uint32_t parity = (j - t0) & 1;
        if (!wait(C::B_S + ti, parity)) { ok = false; break; }
        tc_fence_after();
        uint32_t s[BN];
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) tmem_ld32(tS + 32 * c, s + 32 * c);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < BN / 32; ++c) reg_fence32(s + 32 * c);
        int lo = 0, hi = min(BN, limit - j * BN);
        if (holes) {
          const bool h0 = static_cast<unsigned>(__ldg(table + 2 * j)) >= static_cast<unsigned>(a.pages);
          const bool h1 = (2 * j + 1) * PAGE < len &&
                          static_cast<unsigned>(__ldg(table + 2 * j + 1)) >= static_cast<unsigned>(a.pages);
          if (h0) lo = PAGE;
          if (h1) hi = min(hi, PAGE);
        }
        const bool full = __all_sync(0xffffffffu, lo == 0 && hi == BN);
        const float mx = row_extreme(s, hi, full, pos, lo);
        const float m_cand = lo < hi ? mx * sl2 : -INFINITY;
        const float m_new = fmaxf(m, m_cand);
        const bool need = m_new > m + M_RESCALE;
        float f = 1.f;
        if (need) {
          f = ex2_approx(m - m_new);
          m = m_new;
        }
        if (__any_sync(0xffffffffu, need)) {
          rescale_rows<D>(tO, j > t0, f);
          l *= f;
          large = __any_sync(0xffffffffu, fabsf(m) > M_LARGE && m > -INFINITY);
        }
        float neg_m = m == -INFINITY ? 0.f : -m, mul = sl2;
        if (large) {
          // Scores so large that m is a rounded product: round each score as m
          // was, or the largest would lie half a step of m above or below it.
#pragma unroll
          for (int c = 0; c < BN; ++c)
            s[c] = __float_as_uint(__fadd_rn(__fmul_rn(__uint_as_float(s[c]), sl2), neg_m));
          mul = 1.f;
          neg_m = 0.f;
        }
        const uint32_t half_bar = bars + 8 * (C::B_P_HALF + ti);
        float sum0, sum1;
        if (full)
          row_exp_store<false>(s, mul, neg_m, hi, tS, sum0, sum1, half_bar, [] {}, [] {});
        else
          row_exp_store<true>(s, mul, neg_m, hi, tS, sum0, sum1, half_bar, [] {}, [] {}, lo);
        l += sum0 + sum1;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bars + 8 * (C::B_P + ti));
      }
      if (m == -INFINITY && l != l) m = 0.f;  // a row of NaN scores has no maximum, its sums are NaN
      if (ok && t0 < t1) {
        ok = wait(C::B_O + ti, 0);
        tc_fence_after();
      }
      if (ok) {
        if (p.pieces > 1) {
          // chunk-major: 4 columns of one row are 16 bytes, the 256 rows of a chunk are contiguous
          const long long slot = (static_cast<long long>(want) * a.kv_heads + head) * p.pieces + piece;
          float* dst = p.part_o + slot * 2 * M_ROWS * D + (ti * M_ROWS + row) * 4;
          *reinterpret_cast<float2*>(p.part_ml + (slot * 2 * M_ROWS + ti * M_ROWS + row) * 2) = make_float2(m, l);
          if (t0 < t1) {
#pragma unroll
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
        } else {
          // through this warp's staging tile, so that 8 lanes store 128 contiguous bytes of a row
          const float inv = m == -INFINITY ? 0.f : (a.v_scale ? a.v_scale[head] : 1.f) / l;
          const uint32_t stg = s0 + C::STAGE_OFF + warp * 4096;
#pragma unroll
          for (int hf = 0; hf < D / 64; ++hf) {
#pragma unroll
            for (int cc = 0; cc < 2; ++cc) {
              uint32_t o[32];
              if (t0 < t1) {
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
              const int at = row0 + ti * M_ROWS + quad * 32 + r;
              if (at < total_rows)
                *reinterpret_cast<uint4*>(a.o + (rows.first + at / a.group) * a.o_stride_t +
                                          (static_cast<long long>(head) * a.group + at % a.group) * a.o_stride_h +
                                          hf * 64 + ch * 8) = x;
            }
            __syncwarp();
          }
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

// Joins the pieces of a unit: blockIdx.x is (block, kv head), blockIdx.y 16
// columns; one thread per row. Pieces are added in their order.
template <int D, bool BF16>
__global__ void __launch_bounds__(2 * M_ROWS) cache4_many_join_kernel(const ManyParams p) {
  const AttnParams& a = p.a;
  griddep_wait();
  if (threadIdx.x == 0) griddep_launch_dependents();
  const int head = static_cast<int>(blockIdx.x) % a.kv_heads, want = static_cast<int>(blockIdx.x) / a.kv_heads;
  Unit u;
  if (!find_unit<2 * M_ROWS>(p, want, &u)) return;
  const Rows rows = rows_of(a, u.r);
  const int row = threadIdx.x, at = u.block * 2 * M_ROWS + row;
  if (at >= rows.n * a.group) return;
  const long long slot0 = (static_cast<long long>(want) * a.kv_heads + head) * p.pieces;
  float m = -INFINITY, l = 0.f, x[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) x[e] = 0.f;
  for (int k = 0; k < p.pieces; ++k) m = fmaxf(m, p.part_ml[((slot0 + k) * 2 * M_ROWS + row) * 2]);
  for (int k = 0; k < p.pieces; ++k) {
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + ((slot0 + k) * 2 * M_ROWS + row) * 2);
    if (ml.x == -INFINITY) continue;  // the piece saw no key of this row
    const float f = ex2_approx(ml.x - m);
    l += ml.y * f;
    const float* src = p.part_o + (slot0 + k) * 2 * M_ROWS * D + row * 4;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 y = *reinterpret_cast<const float4*>(src + (blockIdx.y * 4 + q) * 2 * M_ROWS * 4);
      x[4 * q] += y.x * f;
      x[4 * q + 1] += y.y * f;
      x[4 * q + 2] += y.z * f;
      x[4 * q + 3] += y.w * f;
    }
  }
  const float inv = m == -INFINITY ? 0.f : (a.v_scale ? a.v_scale[head] : 1.f) / l;
  uint32_t h[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = float2_to_pair<BF16>(x[2 * e] * inv, x[2 * e + 1] * inv);
  uint4* dst = reinterpret_cast<uint4*>(a.o + (rows.first + at / a.group) * a.o_stride_t +
                                        (static_cast<long long>(head) * a.group + at % a.group) * a.o_stride_h +
                                        blockIdx.y * 16);
  dst[0] = make_uint4(h[0], h[1], h[2], h[3]);
  dst[1] = make_uint4(h[4], h[5], h[6], h[7]);
}

// -------------------------------------------------------------------- host
ManyPlan many_plan(int tokens, int requests, int group, int kv_heads, int D, int sms) {
  ManyPlan pl{};
  const long long blocks = static_cast<long long>(tokens) * group / (2 * M_ROWS) + requests;
  if (blocks * kv_heads > INT_MAX / 8) return pl;
  pl.max_blocks = static_cast<int>(blocks);
  const long long units = blocks * kv_heads;
  pl.pieces = units * 2 <= sms ? static_cast<int>(sms / units < 8 ? sms / units : 8) : 1;
  if (pl.pieces > 1) {
    const size_t rows = static_cast<size_t>(units) * pl.pieces * 2 * M_ROWS;
    pl.ml_off = rows * D * sizeof(float);
    pl.bytes = pl.ml_off + rows * 2 * sizeof(float);
  }
  return pl;
}

template <int D, bool BF16>
static int launch_many_t(const ManyParams& p, cudaStream_t stream) {
  static SmemAttribute smem;
  if (!smem.set(cache4_many_kernel<D, BF16>, Many<D>::SMEM)) return GFX906_B200_ECUDA;
  const int units = p.max_blocks * p.a.kv_heads;
  const int rc = launch(cache4_many_kernel<D, BF16>, dim3(units * p.pieces), dim3(M_THREADS), Many<D>::SMEM, stream, p);
  if (rc != GFX906_B200_OK || p.pieces == 1) return rc;
  return launch(cache4_many_join_kernel<D, BF16>, dim3(units, D / 16), dim3(2 * M_ROWS), 0, stream, p);
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
