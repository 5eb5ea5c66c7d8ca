// The shared prefix of a group on the 5th-generation tensor cores (tcgen05): every (request,
// head) of a kv head is a row of one product against the prefix's keys and values.
//
// A CTA owns up to 256 rows of a group, a kv head and a split of the prefix's 128-token tiles.
// Two softmax streams of 128 rows keep the tensor core busy by turns: with more than 128 rows
// each stream has 128 of them and every tile; else both have the same rows and every other tile,
// and join their sums at the end. For each of its tiles a stream runs
//   S = Q K^T      128 x 128 x D, Q and K from shared memory, S in TMEM
//   P = 2^(S - m)  four warps, a row per thread: no shuffles; P over S in TMEM, in two halves of
//                  the tile's tokens, so that the first half's product runs under the second's
//                  exponentials. P is rounded to the cache's type (half a step of 2^-8 or 2^-11
//                  relative, as the operand type of the product wants); its sum is of fp32 values
//   O += P V       128 x D x 128, P from TMEM, V from shared memory, O in TMEM
// m is the running maximum, raised only when a tile exceeds it by more than 8 in the exponent (O
// and the sum are then rescaled): P stays at most 2^8 and the common factor cancels. (A softmax in one pass
// with a running maximum and sum: Milakov and Gimelshein, Online normalizer calculation for softmax, 2018.)
//
// Warps: 0 loads K and V tiles by TMA (5-D tensor maps over the paged cache, 128-byte swizzle,
// no multicast), 1 and 2 issue a stream's MMAs each, 4-7 and 8-11 are
// the streams' softmax. Shared memory (224 KB at D = 128) and the 512 TMEM columns (two S, two O) are all of
// an SM's, so one CTA runs there. K is the K-major B operand; V, whose rows run along d, the
// MN-major one: no transposition is needed. All waits are bounded; on a timeout the CTA reports
// NIB_DEV_TIMEOUT, lets its copies land, frees its TMEM and returns.
#include "decode_mma.cuh"
#include "tcgen05.cuh"

namespace nib {

constexpr int kPtThreads = 384;
constexpr int kPtTile = 128;   // tokens per tile
constexpr int kPtRows = 128;   // rows per stream
// Shared memory holds seven tiles' worth: Q of each stream that has rows of its own, and a ring of K
// and V tiles in what is left (five or six). A ring's waits tell one use of a slot from the next by
// parity alone, so each stream waits for every load in order and gives every slot back, those of the
// other stream's tiles unused.
constexpr int kPtSlots = 6;
constexpr float kPtRaise = 8.f;

struct PrefixTcParams {
  MmaDecodeParams d;
  int box;  // tokens per TMA copy: the largest power of two that divides block size and tile
};

template <int D>
struct PtSmem {
  static constexpr uint32_t kQ = kPtRows * D * 2;      // one stream's rows
  static constexpr uint32_t kSlot = kPtTile * D * 2;   // a K or V tile
  static_assert(kQ == kSlot, "Q and tiles change places");
  static constexpr uint32_t kBytes = 7 * kSlot + 1024;
};

struct PtBars {
  uint64_t full[kPtSlots], empty[kPtSlots];
  uint64_t s_full[2], p_half[2], p_full[2], o_done[2];
  uint64_t turn[2][4];  // whose exponentials are next, per pair of warps that share a scheduler
  uint64_t landed;  // copies of a tile that is mended before it counts as full
  uint32_t tmem;
  int abort;
};

// a bounded wait that also ends when another warp has given up
__device__ __forceinline__ bool pt_wait(PtBars& s, uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  for (uint32_t it = 0; it < (1u << 30); ++it) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((it & 63u) == 63u) {
      if (*reinterpret_cast<volatile int*>(&s.abort)) return false;
      if (global_ns() - t0 > kWaitLimitNs) break;
    }
  }
  *reinterpret_cast<volatile int*>(&s.abort) = 1;
  return false;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPtThreads, 1)
shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                        const PrefixTcParams pp) {
  using L = PtSmem<D>;
  constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
  __shared__ __align__(8) PtBars bars;
  extern __shared__ unsigned char dsm_raw[];
  const MmaDecodeParams& p = pp.d;
  const uint32_t raw = smem_addr(dsm_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* dsm = dsm_raw + (base - raw);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;

  pdl_enter();

  const int kvh = static_cast<int>(blockIdx.x) % p.num_kv_heads;
  const int split = blockIdx.y;
  const RowTile rt = find_row_tile(p, static_cast<int>(blockIdx.x) / p.num_kv_heads, 2 * kPtRows, lane);
  if (rt.prefix == 0) return;
  const int group_rows = static_cast<int>(rt.end - rt.first) * p.group, row0 = static_cast<int>(rt.row0);
  const int prefix = static_cast<int>(rt.prefix);  // a table covers less than 2^31 tokens
  const int rows = group_rows - row0 < 2 * kPtRows ? group_rows - row0 : 2 * kPtRows;
  const bool both = rows > kPtRows;  // each stream has rows of its own
  const int tiles = static_cast<int>((rt.prefix + kPtTile - 1) / kPtTile);
  const int each = tiles / p.splits, more = tiles - each * p.splits;
  const int tile0 = split * each + (split < more ? split : more), n = each + (split < more ? 1 : 0);
  const int32_t* table = p.tables + rt.leader * p.table_stride;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPtSlots; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 2);  // both streams
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.s_full[i], 1);
      mbar_init(&bars.p_half[i], 128);
      mbar_init(&bars.p_full[i], 128);
      mbar_init(&bars.o_done[i], 1);
      for (int k = 0; k < 4; ++k) mbar_init(&bars.turn[i][k], 1);
    }
    mbar_init(&bars.landed, 1);
    bars.abort = 0;
    fence_mbar_init();
  }
  // stream s: its number of tiles and its i-th one; the ring's load number of tile t's K and V, in
  // the order in which the MMAs want them (a number without a tile is left out)
  auto steps = [&](int s) { return both ? n : (n + 1 - s) / 2; };
  auto tile_of = [&](int s, int i) { return both ? i : 2 * i + s; };
  auto k_load = [&](int t) { return both ? 2 * t : t == 0 ? 0 : 2 * t - 1; };
  auto v_load = [&](int t) { return both ? 2 * t + 1 : 2 * t + 2; };
  const int loads = n > 0 ? (both ? 2 * n : 2 * n + 1) : 0, left_out = both ? -1 : 2 * n - 1;
  const int slots = both ? 5 : 6;

  const uint32_t ring = base + (both ? 2 : 1) * L::kQ;
  unsigned char* const ring_ptr = dsm + (both ? 2 : 1) * L::kQ;
  __syncthreads();

  if (w == 0) {
    // ---------------------------------------------------------------- loads
    const int boxes = kPtTile / pp.box;
    const uint32_t box_bytes = static_cast<uint32_t>(pp.box) * D * 2;
    uint32_t landed_phase = 0, phase = 1;  // the parity of a slot's release, one use behind
    int slot = 0;
    for (int num = 0; num < loads; ++num, phase ^= slot + 1 == slots, slot = slot + 1 == slots ? 0 : slot + 1) {
      if (num == left_out) continue;
      const bool is_v = both || num < 2 ? (both && (num & 1)) : (num & 1) == 0;
      const int t = both ? num >> 1 : num < 2 ? num : is_v ? (num - 2) >> 1 : (num + 1) >> 1;
      const int tok = (tile0 + t) * kPtTile, at = tok + lane * pp.box;
      int page = -1;
      if (lane < boxes && at < prefix) {
        page = __ldg(table + at / p.block_size);
        if (page < 0 || page >= p.num_blocks) {
          page = -1;
          flag(p.status, NIB_DEV_BAD_BLOCK);
        }
      }
      const unsigned have = __ballot_sync(0xffffffffu, page >= 0);
      const bool whole = __popc(have) == boxes && tok + kPtTile <= prefix;
      bool ok = true;
      if (num >= slots) ok = pt_wait(bars, &bars.empty[slot], phase);
      if (!__all_sync(0xffffffffu, ok)) break;
      const bool mend = is_v && !whole;  // rows behind the prefix or without a page become zeros: 0 x NaN is NaN
      uint64_t* bar = mend ? &bars.landed : &bars.full[slot];
      if (lane == 0) mbar_arrive_expect_tx(bar, __popc(have) * box_bytes);
      __syncwarp();
      if (page >= 0) {
        const uint32_t dst = ring + slot * L::kSlot + lane * pp.box * 128;
        const int off = at % p.block_size;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_5d(dst + c * (kPtTile * 128), is_v ? &vmap : &kmap, 0, c, kvh, off, page, bar);
      }
      if (mend) {
        ok = pt_wait(bars, &bars.landed, landed_phase);
        landed_phase ^= 1;
        if (!__all_sync(0xffffffffu, ok)) break;
        for (int e = lane; e < kPtTile * (D / 8); e += 32) {
          const int row = e % kPtTile, c = e / kPtTile;
          if (tok + row >= prefix || !((have >> (row / pp.box)) & 1u))
            *reinterpret_cast<uint4*>(ring_ptr + slot * L::kSlot + (c / 8) * (kPtTile * 128) + row * 128 + (c % 8) * 16) = zero_vec();
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars.full[slot]);
      }
    }
  } else {
    // ---- Q rows into shared memory (swizzled 128-byte rows, one 16 KB region per 64 channels),
    // while warp 0's first tiles are under way
    if (w == 1) tmem_alloc(&bars.tmem, 512);
    {
      constexpr int kTakers = kPtThreads - 32, kVecs = D / 8;
      constexpr int kTake = (2 * kPtRows * kVecs + kTakers - 1) / kTakers;  // vectors per thread
      const uint32_t flip = p.qscale < 0.f ? 0x80008000u : 0u;  // the maximum is taken before the scale
      const int have = (both ? 2 * kPtRows : kPtRows) * kVecs;
      uint4 v[kTake];  // all of a thread's loads in flight
#pragma unroll
      for (int k = 0; k < kTake; ++k) {
        const int e = threadIdx.x - 32 + k * kTakers, r = e / kVecs, row = row0 + r;
        v[k] = zero_vec();
        if (e < have && r < rows) {
          const int request = row / p.group;
          v[k] = ld_vec(static_cast<const T*>(p.q) + (rt.first + request) * p.q_bs +
                        (kvh * p.group + row - request * p.group) * p.q_hs + e % kVecs * 8);
        }
      }
#pragma unroll
      for (int k = 0; k < kTake; ++k) {
        const int e = threadIdx.x - 32 + k * kTakers, r = e / kVecs, c = e % kVecs, in = r % kPtRows;
        const uint32_t at = (r / kPtRows) * L::kQ + (c / 8) * (kPtRows * 128) + in * 128 + (((c % 8) ^ (in & 7)) << 4);
        if (e < have) *reinterpret_cast<uint4*>(dsm + at) = make_uint4(v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip);
      }
      fence_proxy_async();
    }
    tc_fence_before();
    asm volatile("bar.sync 2, %0;" ::"n"(kPtThreads - 32) : "memory");
    tc_fence_after();
  }
  const uint32_t tmem = bars.tmem;
  if (w == 1 || w == 2) {
    // ---------------------------------------------------------------- MMAs, a warp per stream
    // The whole warp runs the loop and waits; one lane issues. Operand addresses change in the
    // descriptors' low words only.
    constexpr uint32_t kIdS = mma_idesc(kBf16, kPtRows, kPtTile, false);
    constexpr uint32_t kIdO = mma_idesc(kBf16, kPtRows, D, true);
    const int s = w - 1, mine = steps(s);
    const uint32_t ts = tmem + s * 128, to = tmem + 256 + s * 128;
    const uint64_t q_desc = smem_desc(base + (both ? s * L::kQ : 0u), 16, 1024);
    const uint64_t k_desc = smem_desc(ring, 16, 1024), v_desc = smem_desc(ring, kPtTile * 128, 1024);
    const bool leader = elect_one();
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, pt_wait(bars, bar, parity)) != 0; };
    // waits for the loads up to `num` in order; the slot of that one
    int seen = 0, at = -1;
    uint32_t phase = 1;
    auto reach = [&](int num) -> bool {
      for (; seen <= num; ++seen) {
        at = at + 1 == slots ? 0 : at + 1;
        phase ^= at == 0;
        if (seen == left_out) continue;
        if (!wait_all(&bars.full[at], phase)) return false;
        if (seen < num && leader) mbar_arrive(&bars.empty[at]);  // the other stream's
      }
      tc_fence_after();
      return true;
    };
    auto scores = [&]() {  // S = Q K^T, K by the load reached
      const uint64_t k = k_desc + at * (L::kSlot >> 4);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          constexpr uint32_t kHalf = kPtRows * 128;
          const uint32_t in = ((kk / 4) * kHalf + (kk % 4) * 32) >> 4;
          tc_mma_ss(ts, q_desc + in, k + in, kIdS, kk > 0);
        }
        tc_commit(&bars.s_full[s]);
        tc_commit(&bars.empty[at]);
      }
    };
    bool ok = true;
    if (mine > 0) {
      ok = reach(k_load(tile_of(s, 0)));
      if (ok) scores();
    }
    for (int i = 0; ok && i < mine; ++i) {
      // P comes in two halves of the tile's tokens: the first half's product runs while the second
      // half's exponentials are computed
      const uint32_t parity = static_cast<uint32_t>(i & 1);
      ok = reach(v_load(tile_of(s, i))) && wait_all(&bars.p_half[s], parity);
      if (!ok) break;
      tc_fence_after();
      const uint64_t v = v_desc + at * (L::kSlot >> 4);
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < kPtTile / 32; ++kk) tc_mma_ts(to, ts + kk * 8, v + kk * (2048 >> 4), kIdO, i > 0 || kk > 0);
      }
      ok = wait_all(&bars.p_full[s], parity);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int kk = kPtTile / 32; kk < kPtTile / 16; ++kk) tc_mma_ts(to, ts + kk * 8, v + kk * (2048 >> 4), kIdO, true);
        tc_commit(&bars.o_done[s]);
        tc_commit(&bars.empty[at]);
      }
      if (i + 1 < mine) {
        // the next scores overwrite P: only after the product that reads it
        ok = reach(k_load(tile_of(s, i + 1))) && wait_all(&bars.o_done[s], parity);
        if (ok) scores();
      }
    }
  } else if (w >= 4) {
    // ---------------------------------------------------------------- softmax
    const int s = (w - 4) >> 2;
    const uint32_t lanes = static_cast<uint32_t>((w & 3) * 32) << 16;
    const uint32_t ts = tmem + s * 128 + lanes, to = tmem + 256 + s * 128 + lanes;
    const float qs = fmaxf(fabsf(p.qscale), 1e-30f);  // masked scores stay -inf with a scale of 0
    const int mine = steps(s);
    const int boxes = kPtTile / pp.box;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int i = 0; i < mine; ++i) {
      const int tok = (tile0 + tile_of(s, i)) * kPtTile, at = tok + lane * pp.box;
      bool here = false;
      if (lane < boxes && at < prefix) {
        const int page = __ldg(table + at / p.block_size);
        here = page >= 0 && page < p.num_blocks;
      }
      const unsigned have = __ballot_sync(0xffffffffu, here);
      ok = __all_sync(0xffffffffu, pt_wait(bars, &bars.s_full[s], static_cast<uint32_t>(i & 1)));
      if (!ok) break;
      tc_fence_after();
      // scores behind the prefix or without a page: -inf (warp-uniform, rare)
      const bool whole = __popc(have) == boxes && tok + kPtTile <= prefix;
      auto mask = [&](uint32_t* x, int c) {
        const int left = prefix - tok - c * 32;
        uint32_t bits = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;  // tokens before the prefix's end
        if (!((have >> (c * 32 / pp.box)) & 1u)) bits &= 0xffff0000u;
        if (!((have >> ((c * 32 + 16) / pp.box)) & 1u)) bits &= 0x0000ffffu;
#pragma unroll
        for (int e = 0; e < 32; ++e)
          if (!((bits >> e) & 1u)) x[e] = 0xff800000u;
      };
      // S is read twice, for the maximum and for P: a row of it does not stay in registers without
      // spills (102 us instead of 100)
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < kPtTile / 32; c += 2) {
        uint32_t x[64];
        tmem_ld32(ts + c * 32, x);
        tmem_ld32(ts + c * 32 + 32, x + 32);
        tmem_wait_ld();
        if (!whole) {
          mask(x, c);
          mask(x + 32, c + 1);
        }
#pragma unroll
        for (int e = 0; e < 64; e += 8) {
#pragma unroll
          for (int k = 0; k < 4; ++k) top[k] = max3(top[k], __uint_as_float(x[e + k]), __uint_as_float(x[e + 4 + k]));
        }
      }
      const float mx = fmaxf(max3(top[0], top[1], top[2]), top[3]) * qs;
      if (i == 0) {
        m = mx;
      } else if (__any_sync(0xffffffffu, mx > m + kPtRaise)) {
        // raise the maximum of the rows that exceed it; the product before must have ended
        ok = __all_sync(0xffffffffu, pt_wait(bars, &bars.o_done[s], static_cast<uint32_t>((i - 1) & 1)));
        if (!ok) break;
        tc_fence_after();
        const bool up = mx > m + kPtRaise;
        const float f = up ? (m == -INFINITY ? 0.f : ex2_fast(m - mx)) : 1.f;
        m = up ? mx : m;
        l *= f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld16(to + c * 16, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st16(to + c * 16, o);
        }
      }
      const float sub = m == -INFINITY ? 0.f : m;  // a row of nothing but masked tokens: all P are 0
      // Streams with rows of their own take turns with the exponentials (stream 0's step i, stream
      // 1's step i, stream 0's step i + 1, ...): one computes while the other's products run. Left
      // to themselves they fall into step (104 us instead of 100). Streams of the same rows, which
      // wait for memory, are left alone.
      if (both && (s == 1 || i > 0)) {
        ok = __all_sync(0xffffffffu, pt_wait(bars, &bars.turn[s][w & 3], static_cast<uint32_t>((s == 1 ? i : i - 1) & 1)));
        if (!ok) break;
      }
      const uint64_t qs2 = pair2(qs, qs), sub2 = pair2(-sub, -sub);
      uint64_t part[2] = {0ull, 0ull};
#pragma unroll
      for (int c = 0; c < kPtTile / 64; ++c) {
        uint32_t pk[32], x[64];
        tmem_ld32(ts + c * 64, x);
        tmem_ld32(ts + c * 64 + 32, x + 32);
        tmem_wait_ld();
        if (!whole) {
          mask(x, 2 * c);
          mask(x + 32, 2 * c + 1);
        }
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const int k = 2 * e;
          const float2 y = unpair2(fma2(pair2(x[k], x[k + 1]), qs2, sub2));
          const float a = ex2_fast(y.x), b = ex2_fast(y.y);
          part[e & 1] = add2(part[e & 1], pair2(a, b));
          pk[e] = pack2<T>(a, b);
        }
        tmem_st32(ts + c * 32, pk);
        if (c == 0) {
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&bars.p_half[s]);
        }
      }
      __syncwarp();
      if (both && lane == 0) mbar_arrive(&bars.turn[1 - s][w & 3]);
      const float2 sum = unpair2(add2(part[0], part[1]));
      l += sum.x + sum.y;
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars.p_full[s]);
    }
    if (ok && mine > 0) ok = __all_sync(0xffffffffu, pt_wait(bars, &bars.o_done[s], static_cast<uint32_t>((mine - 1) & 1)));
    tc_fence_after();
    // ---- partials: rows of their own go straight to the workspace; streams of the same rows
    // meet in shared memory (the ring is free: every tile in it has been used)
    float* meet = reinterpret_cast<float*>(ring_ptr);
    const int r = (w & 3) * 32 + lane;
    if (!both) {
      asm volatile("bar.sync 1, 256;" ::: "memory");  // both streams' last products have ended
      if (s == 1) {
        meet[r] = m;
        meet[kPtRows + r] = l;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(to + c * 32, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) meet[(2 + c * 32 + e) * kPtRows + r] = mine > 0 ? __uint_as_float(o[e]) : 0.f;
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");
    }
    const int row = row0 + (both ? s * kPtRows : 0) + r;
    const bool writes = ok && (both || s == 0) && row < group_rows;
    float fa = 1.f, fb = 0.f;
    if (!both && s == 0) {
      const float m1 = meet[r], top = fmaxf(m, m1);
      fa = m == -INFINITY ? 0.f : ex2_fast(m - top);
      fb = m1 == -INFINITY ? 0.f : ex2_fast(m1 - top);
      l = l * fa + meet[kPtRows + r] * fb;
      m = top;
    }
    if (both || s == 0) {
      // 32 columns of the warp's rows at a time, through the stream's Q (its products have
      // ended), so that eight lanes write 128 bytes of a row
      const int64_t request = rt.first + (row < group_rows ? row / p.group : 0);
      const int64_t place = writes ? (request * p.num_heads + kvh * p.group + row % p.group) * p.slots + p.slot0 + split : -1;
      float4* turn = reinterpret_cast<float4*>(dsm + s * L::kQ) + (w & 3) * 256;
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(to + c * 32, o);
        tmem_wait_ld();
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            v[k] = mine > 0 ? __uint_as_float(o[e + k]) : 0.f;
            if (!both) v[k] = v[k] * fa + meet[(2 + c * 32 + e + k) * kPtRows + r] * fb;
          }
          turn[lane * 8 + ((e / 4) ^ (lane & 7))] = make_float4(v[0], v[1], v[2], v[3]);
        }
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const int from = k * 4 + lane / 8;
          const int64_t at = __shfl_sync(0xffffffffu, place, from);
          if (at >= 0) *reinterpret_cast<float4*>(p.ws + at * D + c * 32 + lane % 8 * 4) = turn[from * 8 + ((lane % 8) ^ (from & 7))];
        }
      }
      if (writes) p.ml[place] = make_float2(m, l);
    }
    tc_fence_before();
  }
  if (__syncthreads_or(bars.abort) && w == 0) {
    if (lane == 0) flag(p.status, kDevTimeout);
    // copies that may still be in flight land before the shared memory goes
    const unsigned long long t0 = global_ns();
    while (global_ns() - t0 < 1000000ull) {
    }
  }
  if (w == 1) {
    tc_fence_after();
    tmem_free(tmem, 512);
  }
}

static int tile_box(int64_t block_size) {
  int box = kPtTile;
  while (block_size % box != 0) box /= 2;  // at least 16: block sizes are multiples of it
  return box;
}

template <typename T, int D>
static int launch_tc(const nib_decode_attention_args& a, const MmaDecodeParams& d, int64_t units, cudaStream_t st) {
  PrefixTcParams p{};
  p.d = d;
  p.box = tile_box(a.block_size);
  CUtensorMap kmap, vmap;
  int rc = make_cache_map(&kmap, a, a.key_cache, p.box);
  if (rc != NIB_OK) return rc;
  rc = make_cache_map(&vmap, a, a.value_cache, p.box);
  if (rc != NIB_OK) return rc;
  constexpr int smem = static_cast<int>(PtSmem<D>::kBytes);
  auto kernel = shared_prefix_tc_kernel<T, D>;
  static int configured[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && configured[dev] < smem) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      set_error("shared_prefix_decode_attention: cannot reserve shared memory: %s", cudaGetErrorString(e));
      return NIB_ERR_CUDA;
    }
    configured[dev] = smem;
  }
  const dim3 grid(static_cast<unsigned>(units * a.num_kv_heads), static_cast<unsigned>(d.splits));
  launch_k(kernel, grid, kPtThreads, smem, st, kmap, vmap, p);
  return launch_status("shared_prefix_decode_attention (prefix)");
}

int64_t prefix_tc_rows() { return 2 * kPtRows; }
int64_t prefix_tc_tile() { return kPtTile; }

int launch_prefix_tc(const nib_decode_attention_args& a, const MmaDecodeParams& p, int64_t units, cudaStream_t st) {
  return NIB_MMA_CASE(a, T, D, launch_tc<T, D>(a, p, units, st));
}

}  // namespace nib
