// Decode attention over the chunks of a context that a cheap score selects, and the per-chunk
// key bounds behind that score.
//
// A chunk is `chunk` consecutive tokens inside a cache block; bounds[block, kv head, chunk, 0/1, :]
// hold the smallest and largest value of each key channel over the chunk's tokens. For a query q
// and any key k between the bounds, q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo
// (q+ = max(q, 0), q- = min(q, 0)), so over the heads h of a kv head
//   score(chunk) = a . hi + b . lo,   a = sum_h q_h+,   b = sum_h q_h-
// bounds the sum of the heads' scores from above with one dot product of 2 D terms, whatever
// the number of heads. Chunks are ranked by their scores in 64 bits (in 32, the order of the
// summation would decide between near neighbours), yet hardly any is computed so: scores are
// summed in 32 bits with a bound of their error, and only the chunks that the bound leaves within
// reach of the last place - mostly none - are scored again in 64 bits.
#include "decode_mma.cuh"

namespace nib {

// ------------------------------------------------------------------ key bounds

struct BoundsParams {
  const void* kc;
  int64_t c_bs, c_ss, c_hs;
  int64_t num_blocks;
  int block_size, chunk, nkv;
  int64_t max_new;
  const int32_t* tables;
  int64_t table_stride, cap;
  const int32_t* starts;
  const int32_t* lens;
  void* bounds;
  int64_t b_bs, b_hs;  // block and head strides (elements)
  unsigned int* status;
};

// packed minimum and maximum; a NaN stays a NaN
__device__ __forceinline__ __nv_bfloat162 min2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 max2(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmax2_nan(a, b); }
__device__ __forceinline__ __half2 min2(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __half2 max2(__half2 a, __half2 b) { return __hmax2_nan(a, b); }

constexpr int kBoundsThreads = 256;
constexpr int kBoundsUnroll = 8;

// One CTA per (window of a request, request): the window's chunk over all kv heads. A thread
// owns one 16-byte vector of the token row (8 channels of a head) and every slices-th token, eight
// loads in flight. Bound by HBM for long prefills; three CTAs per SM (16 x 16,384 tokens of 8 x 128
// 87.5 us, 256 single steps 6.3 us; 80 registers and 16 bytes spilled) against four (64 registers, 28 bytes
// spilled: 85.0 and 7.4), and four with four loads in flight (113.6 and 10.0).
template <typename T, int D>
__global__ void __launch_bounds__(kBoundsThreads, 3)
key_bounds_kernel(const BoundsParams p) {
  pdl_enter();
  using V2 = typename Vec2<T>::type;
  union Vec {
    uint4 u;
    V2 h[4];
  };
  __shared__ Vec part[2][kBoundsThreads];
  const int64_t b = blockIdx.y;
  int64_t len = __ldg(p.lens + b), start = __ldg(p.starts + b);
  if (len < 0 || len > p.cap || start < 0) {
    if (threadIdx.x == 0 && blockIdx.x == 0) flag(p.status, NIB_DEV_BAD_INDEX);
    len = len < 0 ? 0 : len > p.cap ? p.cap : len;
    start = start < 0 ? 0 : start;
  }
  if (start >= len) return;
  const int64_t c = start / p.chunk + blockIdx.x;
  if (blockIdx.x == 0 && threadIdx.x == 0 && len - start > p.max_new)
    flag(p.status, NIB_DEV_BAD_INDEX);  // more new tokens than the caller said
  const int64_t t0 = c * p.chunk;
  if (t0 >= len) return;
  const int count = len - t0 < p.chunk ? static_cast<int>(len - t0) : p.chunk;
  const int blk = __ldg(p.tables + b * p.table_stride + t0 / p.block_size);
  if (blk < 0 || blk >= p.num_blocks) {
    if (threadIdx.x == 0) flag(p.status, NIB_DEV_BAD_BLOCK);
    return;
  }
  const int slot = static_cast<int>(t0 % p.block_size);
  const T* rows = static_cast<const T*>(p.kc) + blk * p.c_bs + slot * p.c_ss;
  T* out = static_cast<T*>(p.bounds) + blk * p.b_bs + (slot / p.chunk) * 2 * D;
  const int units = p.nkv * (D / 8);  // vectors of a token row
  const int slices = units >= kBoundsThreads ? 1 : kBoundsThreads / units;
  const int slice = units >= kBoundsThreads ? 0 : threadIdx.x / units;
  for (int u0 = 0; u0 < units; u0 += kBoundsThreads) {
    const int u = u0 + (units >= kBoundsThreads ? threadIdx.x : threadIdx.x % units);
    const bool active = u < units && slice < slices;
    Vec lo, hi;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      lo.h[i] = Vec2<T>::make(INFINITY, INFINITY);
      hi.h[i] = Vec2<T>::make(-INFINITY, -INFINITY);
    }
    if (active) {
      const T* at = rows + static_cast<int64_t>(u / (D / 8)) * p.c_hs + (u % (D / 8)) * 8;
      for (int t = slice; t < count; t += slices * kBoundsUnroll) {
        Vec x[kBoundsUnroll];
#pragma unroll
        for (int j = 0; j < kBoundsUnroll; ++j)
          if (t + j * slices < count) x[j].u = ld_stream(at + static_cast<int64_t>(t + j * slices) * p.c_ss);
#pragma unroll
        for (int j = 0; j < kBoundsUnroll; ++j)
          if (t + j * slices < count) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              lo.h[i] = min2(lo.h[i], x[j].h[i]);
              hi.h[i] = max2(hi.h[i], x[j].h[i]);
            }
          }
      }
    }
    if (slices > 1) {
      part[0][threadIdx.x].u = lo.u;
      part[1][threadIdx.x].u = hi.u;
      __syncthreads();
      if (active && slice == 0) {
        for (int s = 1; s < slices; ++s) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo.h[i] = min2(lo.h[i], part[0][s * units + u].h[i]);
            hi.h[i] = max2(hi.h[i], part[1][s * units + u].h[i]);
          }
        }
      }
    }
    if (active && slice == 0) {
      T* o = out + static_cast<int64_t>(u / (D / 8)) * p.b_hs + (u % (D / 8)) * 8;
      st_vec(o, lo.u);
      st_vec(o + D, hi.u);
    }
  }
}

// ------------------------------------------------------------------ scores and selection

struct SelectParams {
  MmaDecodeParams d;  // q, tables, lens, heads
  const void* bounds;
  int64_t b_bs, b_hs;
  float* scores;       // [batch * kv heads, max_chunks] in 32 bits
  float* errors;       // [batch * kv heads, error_slots]: bounds of what they are off, by warp
  uint64_t* keys;      // as many as scores: the chunks that are scored in 64 bits
  int64_t max_chunks;
  int error_slots;
  int per, per_shift;  // chunks per block; its log2 where it is a power of two, else -1
  int32_t* selected;   // [batch * kv heads, top]
};

// A lane's share of a chunk's dot product: 8 channels of lo or of hi. The lanes of a chunk are
// 2 D / 8, the first half of them lo's.
template <int D>
struct ScoreLanes {
  static constexpr int kLanes = 2 * D / 8;      // per chunk
  static constexpr int kChunks = 32 / kLanes;   // per warp step
};

// The lane's eight weights: over the kv head's q heads, the positive parts for hi, the negative
// ones for lo, summed in 64 bits.
template <typename T, int D>
__device__ __forceinline__ void score_weights(const SelectParams& p, int64_t b, int kvh, int lane, double (&wt)[8]) {
  constexpr int half = ScoreLanes<D>::kLanes / 2;
  const int part = lane % ScoreLanes<D>::kLanes;
  const bool is_hi = part >= half;
#pragma unroll
  for (int i = 0; i < 8; ++i) wt[i] = 0.0;
  for (int h = 0; h < p.d.group; ++h) {
    float f[8];
    unpack<T>(ld_vec(static_cast<const T*>(p.d.q) + b * p.d.q_bs + (kvh * p.d.group + h) * p.d.q_hs + (part % half) * 8), f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((is_hi ? f[i] > 0.f : f[i] < 0.f) || f[i] != f[i]) wt[i] += static_cast<double>(f[i]);
  }
}

// chunk c's block in its table and its place there
__device__ __forceinline__ int2 chunk_place(const SelectParams& p, int c) {
  if (p.per_shift >= 0) return make_int2(c >> p.per_shift, c & (p.per - 1));
  return make_int2(c / p.per, c % p.per);
}

// the lane's 16 bytes of chunk c, zeros where its block does not exist
template <typename T, int D>
__device__ __forceinline__ uint4 load_bounds(const SelectParams& p, const int32_t* table, int kvh, int c, int lane, bool& ok) {
  constexpr int half = ScoreLanes<D>::kLanes / 2;
  const int part = lane % ScoreLanes<D>::kLanes;
  const int2 at = chunk_place(p, c);
  const int blk = __ldg(table + at.x);
  ok = blk >= 0 && blk < p.d.num_blocks;
  if (!ok) return zero_vec();
  return ld_stream(static_cast<const T*>(p.bounds) + blk * p.b_bs + kvh * p.b_hs + (at.y * 2 + (part >= half ? 1 : 0)) * D +
                   (part % half) * 8);
}

constexpr int kScoreWarps = 8;
constexpr int kScoreUnroll = 8;
constexpr int kScoreResident = 4;  // CTAs per SM that the registers are sized for (64; up to 40 bytes spill)

// Scores of a row's chunks in 32 bits, by one of `parts` CTAs. Error: a weight is a sum of at most
// 16 terms of one sign, a lane adds 8 products with fused operations, five shuffles add the lanes:
// at most 15 + 8 + 5 roundings of 2^-24 relative to the sum of the terms' absolute values. A warp
// bounds that sum for all of its chunks at once, by the largest |value| of each channel; the
// bound's own sum is 2^-19 off at most, so 1.25 * 2^-19 of it covers the error, and 2^-126 terms
// too small for relative errors.
//
// A warp takes groups of kScoreUnroll steps (4 KB of bounds), all loads of a group in flight. The
// lanes' sums of eight steps are added by halving: each exchange halves the steps that a lane is
// left with (9 shuffles for 8 chunks of 32 lanes, not 40).
template <typename T, int D>
__device__ __forceinline__ void score_chunks(const SelectParams& p, int64_t row, int64_t b, int kvh, int chunks, int part_of,
                                             int parts) {
  constexpr int LPC = ScoreLanes<D>::kLanes, CPS = ScoreLanes<D>::kChunks, G = kScoreUnroll * CPS;
  constexpr int half = LPC / 2;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int step = parts * kScoreWarps * G;
  int c0 = (part_of * kScoreWarps + w) * G;
  const int part = lane % LPC;
  const int32_t* table = p.d.tables + b * p.d.table_stride;
  const T* base = static_cast<const T*>(p.bounds) + kvh * p.b_hs + (part >= half ? D : 0) + (part % half) * 8;
  // lane j looks chunk c + j of a group up: where its bounds begin, -1: it has none
  auto look_up = [&](int c) -> int64_t {
    if (lane >= G || c + lane >= chunks) return -1;
    const int2 at = chunk_place(p, c + lane);
    const int blk = __ldg(table + at.x);
    if (blk >= 0 && blk < p.d.num_blocks) return blk * p.b_bs + at.y * 2 * D;
    flag(p.d.status, NIB_DEV_BAD_BLOCK);
    return -1;
  };
  int64_t place = look_up(c0);
  // the weights, with both signs as positive parts; a query that is not finite makes them NaN
  float wt[8], most[8], odd = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) wt[i] = most[i] = 0.f;
  {
    const float sign = part >= half ? 1.f : -1.f;
    const T* q = static_cast<const T*>(p.d.q) + b * p.d.q_bs + kvh * p.d.group * p.d.q_hs + (part % half) * 8;
#pragma unroll 4
    for (int h = 0; h < p.d.group; ++h) {
      float f[8];
      unpack<T>(ld_vec(q + h * p.d.q_hs), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        wt[i] += fmaxf(f[i] * sign, 0.f);
        odd = fmaf(f[i], 0.f, odd);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) wt[i] = fmaf(wt[i], sign, odd);
  }
  float* out = p.scores + row * p.max_chunks;
  for (; c0 < chunks; c0 += step) {
    uint4 v[kScoreUnroll];
    const unsigned have = __ballot_sync(0xffffffffu, place >= 0);
#pragma unroll
    for (int j = 0; j < kScoreUnroll; ++j) {
      const int64_t at = __shfl_sync(0xffffffffu, place, j * CPS + lane / LPC);
      v[j] = zero_vec();
      if (at >= 0) v[j] = ld_stream(base + at);
    }
    place = look_up(c0 + step);
    float s[kScoreUnroll];
#pragma unroll
    for (int j = 0; j < kScoreUnroll; ++j) {
      float f[8];
      unpack<T>(v[j], f);
      s[j] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        s[j] = fmaf(wt[i], f[i], s[j]);
        most[i] = fmaxf(most[i], fabsf(f[i]));
      }
    }
    int mine = 0;  // the step that this lane is left with
#pragma unroll
    for (int n = kScoreUnroll / 2, off = LPC / 2; n >= 1; n /= 2, off /= 2) {
      const bool upper = (lane & off) != 0;
      mine += upper ? n : 0;
#pragma unroll
      for (int j = 0; j < n; ++j) {
        const float keep = upper ? s[j + n] : s[j], give = upper ? s[j] : s[j + n];
        s[j] = keep + __shfl_xor_sync(0xffffffffu, give, off);
      }
    }
#pragma unroll
    for (int off = LPC / 16; off >= 1; off /= 2) s[0] += __shfl_xor_sync(0xffffffffu, s[0], off);
    const int c = mine * CPS + lane / LPC;
    // a chunk without a block ranks below every other (two of them by their index)
    if ((lane & (LPC / 8 - 1)) == 0 && c0 + c < chunks) out[c0 + c] = (have >> c) & 1u ? s[0] : -INFINITY;
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum = fmaf(fabsf(wt[i]), most[i], sum);
#pragma unroll
  for (int off = LPC / 2; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (CPS == 2) sum = fmaxf(sum, __shfl_xor_sync(0xffffffffu, sum, 16)) + (sum - sum);  // a NaN stays one
  if (lane == 0)
    p.errors[row * p.error_slots + part_of * kScoreWarps + w] = fmaf(sum, 1.25f * 1.9073486328125e-6f, 1.1754943508222875e-38f);
}

// A 32-bit score as a whole number of the same order (-0 as 0).
__device__ __forceinline__ uint32_t key_of(float s) {
  const uint32_t bits = __float_as_uint(s + 0.f);
  return bits >> 31 ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float score_of(uint32_t key) {
  return __uint_as_float(key >> 31 ? key & 0x7fffffffu : ~key);
}

// A 64-bit score likewise; NaN and infinity count as the largest finite number.
__device__ __forceinline__ uint64_t key_of(double s) {
  s = s <= 1.7976931348623157e308 ? s + 0.0 : 1.7976931348623157e308;
  const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(s));
  return bits >> 63 ? ~bits : bits | (1ull << 63);
}

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;
constexpr int kSelectShared = 8192;  // chunks whose 32-bit keys are kept in shared memory
constexpr int kSelectBand = 256;     // competing chunks that are ranked by comparing each with each

struct SelectShared {
  uint32_t keys[kSelectShared];
  unsigned int hist[256];
  uint64_t member[kSelectBand], found;
  int digit, need, members;
  int at[kSelectBand];
  uint64_t key[kSelectBand];
  bool in[kSelectBand];
  uint4 range[kSelectWarps];
  unsigned long long counts[kSelectWarps];
  int sums[kSelectWarps];
  int band;
};

// The need-th largest of the keys that key(i, k) yields for i < n (false: i takes no part), from
// bit `top_bit` down (above it all keys are those of `prefix`); need becomes how many of those
// equal to it are among the first need. By the whole CTA: eight bits at a time by counting, until
// the keys that share the bits so far are few enough to compare each with each.
template <typename F>
__device__ __forceinline__ uint64_t nth_largest(SelectShared& s, int n, int& need, int top_bit, uint64_t prefix, F key) {
  static_assert(kSelectThreads == 256 && kSelectBand == 256, "a thread per bin and per member");
  const int tid = threadIdx.x, lane = tid & 31;
  int done = top_bit + 1;  // bits still open
  while (done > 0) {
    const int bits = done < 8 ? done : 8, shift = done - bits;
    s.hist[tid] = 0;
    if (tid == 0) s.members = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelectThreads) {
      uint64_t k;
      if (key(i, k) && (k >> (shift + bits - 1)) >> 1 == prefix)
        atomicAdd(&s.hist[static_cast<int>(k >> shift) & ((1 << bits) - 1)], 1u);
    }
    __syncthreads();
    if (tid < 32) {  // lane l: bins 255 - 8 l down to 248 - 8 l
      int count[8], mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        count[j] = static_cast<int>(s.hist[255 - 8 * lane - j]);
        mine += count[j];
      }
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += v;
      }
      int above = upto - mine;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (above < need && above + count[j] >= need) {  // true for one bin of all
          s.digit = 255 - 8 * lane - j;
          s.need = need - above;
          s.band = count[j];
        }
        above += count[j];
      }
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint64_t>(s.digit);
    need = s.need;
    done = shift;
    if (s.band <= kSelectBand) {
      for (int i = tid; i < n; i += kSelectThreads) {
        uint64_t k;
        if (key(i, k) && k >> shift == prefix) s.member[atomicAdd(&s.members, 1)] = k;
      }
      __syncthreads();
      const int m = s.members;
      if (tid < m) {
        const uint64_t k = s.member[tid];
        int greater = 0, same = 0;
        for (int j = 0; j < m; ++j) {
          greater += s.member[j] > k ? 1 : 0;
          same += s.member[j] == k ? 1 : 0;
        }
        if (greater < need && need <= greater + same) {  // the same for all that hold this key
          s.found = k;
          s.need = need - greater;
        }
      }
      __syncthreads();
      prefix = s.found;
      need = s.need;
      break;
    }
  }
  return prefix;
}

// exclusive prefix sum over the CTA's threads
__device__ __forceinline__ int scan_threads(SelectShared& s, int v) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += x;
  }
  __syncthreads();
  if (lane == 31) s.sums[w] = upto;
  __syncthreads();
  int before = upto - v;
#pragma unroll
  for (int j = 0; j < kSelectWarps; ++j) before += j < w ? s.sums[j] : 0;
  return before;
}

// The `top` best chunks of a row, in ascending order of index: the CTAs of a cluster score the
// row's chunks by turns, then the first of them selects (the others end, and with them their
// SMs are free for other rows). The first and the last chunk are
// in; `rest` others are wanted. With T the rest-th largest 32-bit score and E the row's largest
// error bound, a chunk above T + 2 E is in for certain, one below T - 2 E out, and those between
// compete in 64 bits for the places that are left (unless the places suffice for all of them).
// A score or bound that is not finite makes E infinite: then every chunk competes.
template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, kScoreResident)
chunk_select_kernel(const SelectParams p) {
  static_assert(kSelectThreads == kScoreWarps * 32, "the same CTA scores and selects");
  pdl_enter();
  __shared__ SelectShared s;
  const int64_t row = blockIdx.y;
  const int64_t b = row / p.d.num_kv_heads;
  const int kvh = static_cast<int>(row % p.d.num_kv_heads);
  const int64_t len = clamped_len(p.d, b, threadIdx.x == 0 && blockIdx.x == 0 && kvh == 0);
  const int n = static_cast<int>((len + p.d.chunk - 1) / p.d.chunk);
  const int top = p.d.top;
  int32_t* out = p.selected + row * top;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (n <= top) {  // the whole cluster
    if (blockIdx.x == 0)
      for (int i = tid; i < top; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  score_chunks<T, D>(p, row, b, kvh, n, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  if (blockIdx.x > 0) return;
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  const float* scores = p.scores + row * p.max_chunks;
  const bool shared = n <= kSelectShared;
  auto inner = [&](int i) { return i > 0 && i < n - 1; };
  // the row's error bound (infinite if a score or a bound is not to be trusted: NaN, overflow) and
  // the range of its inner keys
  bool fine = true;
  float worst = 0.f;
  for (int i = tid; i < p.error_slots; i += kSelectThreads) {
    const float e = p.errors[row * p.error_slots + i];
    fine = fine && e <= 3.0e38f;
    worst = fmaxf(worst, e);
  }
  uint32_t least = ~0u, largest = 0u;
  for (int i = tid; i < n; i += kSelectThreads) {
    const float x = scores[i];
    const uint32_t k = key_of(x);
    fine = fine && x <= 3.0e38f;  // -inf next to finite bounds: a chunk without a block
    if (shared) s.keys[i] = k;
    if (inner(i)) {
      least = min(least, k);
      largest = max(largest, k);
    }
  }
  const uint32_t off_by = __reduce_max_sync(0xffffffffu, __float_as_uint(fine ? worst : INFINITY));
  least = __reduce_min_sync(0xffffffffu, least);
  largest = __reduce_max_sync(0xffffffffu, largest);
  if (lane == 0) s.range[w] = make_uint4(off_by, least, largest, 0u);
  __syncthreads();
  worst = 0.f;
#pragma unroll
  for (int j = 0; j < kSelectWarps; ++j) {
    worst = fmaxf(worst, __uint_as_float(s.range[j].x));
    least = min(least, s.range[j].y);
    largest = max(largest, s.range[j].z);
  }
  auto key32 = [&](int i) { return shared ? s.keys[i] : key_of(scores[i]); };
  int rest = top - 2;
  float high = INFINITY, low = INFINITY;  // rest = 0: none of the inner chunks
  if (rest > 0) {
    if (worst < INFINITY) {
      int need = rest;
      const int top_bit = 31 - __clz(least ^ largest);  // -1: all alike
      const uint32_t common = top_bit < 31 ? largest >> (top_bit + 1) : 0u;
      const float t = score_of(static_cast<uint32_t>(nth_largest(s, n, need, top_bit, common, [&](int i, uint64_t& k) {
        k = key32(i);
        return inner(i);
      })));
      // rounded outwards
      high = t + 2.f * worst;
      low = t - 2.f * worst;
      high += fabsf(high) * 2.4e-7f;
      low -= fabsf(low) * 2.4e-7f;
    } else {
      low = -INFINITY;
    }
  }
  auto competes = [&](int i) {
    const float x = score_of(key32(i));
    return rest > 0 && inner(i) && !(x > high) && !(x < low);
  };
  // those certainly in, and those that compete
  __syncthreads();
  if (tid == 0) s.band = 0;
  __syncthreads();
  unsigned long long counts = 0;
  if (rest > 0)
    for (int i = tid; i < n; i += kSelectThreads)
      if (inner(i)) {
        const float x = score_of(key32(i));
        if (x > high) {
          counts += 1ull << 32;
        } else if (!(x < low)) {
          counts += 1ull;
          const int at = atomicAdd(&s.band, 1);
          if (at < kSelectBand) s.at[at] = i;
        }
      }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) counts += __shfl_xor_sync(0xffffffffu, counts, off);
  if (lane == 0) s.counts[w] = counts;
  __syncthreads();
  counts = 0;
#pragma unroll
  for (int j = 0; j < kSelectWarps; ++j) counts += s.counts[j];
  const int sure = static_cast<int>(counts >> 32), band = static_cast<int>(counts & 0xffffffffu);
  const int places = rest - sure;
  const bool ranked = band > places;
  const bool few = band <= kSelectBand;
  uint64_t* keys = p.keys + row * p.max_chunks;
  uint64_t bar = 0;  // many: the 64-bit key that a competing chunk has to exceed,
  int equal = 0;     // and how many of those that reach it are in
  if (ranked) {
    constexpr int LPC = ScoreLanes<D>::kLanes, CPS = ScoreLanes<D>::kChunks;
    const int32_t* table = p.d.tables + b * p.d.table_stride;
    const int candidates = few ? band : n;
    // only in the warps that score one: a row of 8 heads takes eight warps 10 us on the 64-bit pipe
    double wt[8];
    if (w * CPS < candidates) score_weights<T, D>(p, b, kvh, lane, wt);
    for (int j0 = w * CPS; j0 < candidates; j0 += kSelectWarps * CPS) {
      const int j = j0 + lane / LPC;
      const int i = j >= candidates ? -1 : few ? s.at[j] : competes(j) ? j : -1;
      if (!__any_sync(0xffffffffu, i >= 0)) continue;
      bool ok = false;
      const uint4 v = i >= 0 ? load_bounds<T, D>(p, table, kvh, i, lane, ok) : zero_vec();
      float f[8];
      unpack<T>(v, f);
      double x = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) x = fma(wt[e], static_cast<double>(f[e]), x);
#pragma unroll
      for (int off = LPC / 2; off >= 1; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
      if (i >= 0 && lane % LPC == 0) (few ? s.key[j] : keys[i]) = ok ? key_of(x) : 0ull;
    }
    __syncthreads();
    if (few) {
      if (tid < band) {
        const uint64_t k = s.key[tid];
        const int i = s.at[tid];
        int better = 0;
        for (int j = 0; j < band; ++j) better += s.key[j] > k || (s.key[j] == k && s.at[j] < i) ? 1 : 0;
        s.in[tid] = better < places;
      }
      __syncthreads();
    } else if (places > 0) {
      int need = places;
      bar = nth_largest(s, n, need, 63, 0ull, [&](int i, uint64_t& k) {
        if (!competes(i)) return false;
        k = keys[i];
        return true;
      });
      equal = need;
    } else {
      bar = ~0ull;
    }
  }
  // each thread's share of consecutive chunks, in order: `left` of the equal ones are still to take
  const int share = (n + kSelectThreads - 1) / kSelectThreads;
  const int from = tid * share, to = from + share < n ? from + share : n;
  int left = 0;
  if (ranked && !few) {
    int same = 0;
    for (int i = from; i < to; ++i) same += competes(i) && keys[i] == bar ? 1 : 0;
    left = equal - scan_threads(s, same);
  }
  auto selected = [&](int i, int& left) {
    if (!inner(i)) return true;
    const float x = score_of(key32(i));
    if (rest <= 0 || x < low) return false;
    if (x > high || !ranked) return true;
    if (few) {
      bool in = false;
      for (int j = 0; j < band; ++j) in |= s.at[j] == i && s.in[j];
      return in;
    }
    return keys[i] > bar || (keys[i] == bar && left-- > 0);
  };
  int mine = 0, still = left;
  for (int i = from; i < to; ++i) mine += selected(i, still) ? 1 : 0;
  int at = scan_threads(s, mine);
  for (int i = from; i < to; ++i)
    if (selected(i, left)) out[at++] = i;
}

// ------------------------------------------------------------------ host side

struct SparsePlan {
  int splits;
  int64_t max_len, max_chunks;
  int64_t score_ctas;  // per row
  int64_t score_bytes, partial_bytes;  // 64-bit keys, scores and errors; partials
};

static SparsePlan sparse_plan(const nib_sparse_decode_args& s) {
  const nib_decode_attention_args& a = s.attn;
  SparsePlan pl{};
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  pl.max_len = a.max_context_len > 0 && a.max_context_len < cap ? a.max_context_len : cap;
  pl.max_chunks = (pl.max_len + s.chunk - 1) / s.chunk;
  const int64_t rows = a.batch * a.num_kv_heads;
  // every row has as much to read: as many equal splits as fit the SMs' three CTAs each at once.
  // 48 contexts x 8 kv heads, 64 chunks of 32 tokens: 114 us with 1 split, 118 with 2, 129 with 5.
  const int64_t want = 3LL * sm_count();
  int64_t n = rows < 1 || rows >= want ? 1 : want / rows;
  const int64_t tokens = (pl.max_chunks < s.top_chunks ? pl.max_chunks : s.top_chunks) * s.chunk;
  const int64_t by_len = (tokens + 63) / 64;
  if (n > by_len) n = by_len;
  if (n > 256) n = 256;
  pl.splits = static_cast<int>(n < 1 ? 1 : n);
  // score CTAs per row (a cluster): the fewest steps of a warp over all waves, the start and the
  // selection counted as four
  const int64_t per_cta = kScoreWarps * kScoreUnroll * (a.head_dim == 64 ? 2 : 1);
  const int64_t most = (pl.max_chunks + per_cta - 1) / per_cta, resident = static_cast<int64_t>(kScoreResident) * sm_count();
  int64_t best = 0;
  pl.score_ctas = 1;
  for (int64_t c = 1; c <= 8 && c < 2 * most; c *= 2) {
    const int64_t cost = (rows * c + resident - 1) / resident * ((most + c - 1) / c + 4);
    if (best == 0 || cost < best) {
      best = cost;
      pl.score_ctas = c;
    }
  }
  pl.score_bytes = pl.max_chunks > s.top_chunks ? (rows * (pl.max_chunks * 12 + pl.score_ctas * kScoreWarps * 4) + 15) / 16 * 16 : 0;
  pl.partial_bytes = pl.splits > 1 ? nib::partial_bytes(a, pl.splits) : 0;
  return pl;
}

template <typename T, int D>
static int launch_sparse(const nib_sparse_decode_args& s, const SparsePlan& pl, cudaStream_t st) {
  const nib_decode_attention_args& a = s.attn;
  SelectParams sp{};
  sp.d = mma_params(a, pl.splits);
  sp.d.cap = pl.max_len;
  sp.d.chunk = s.chunk;
  sp.d.top = s.top_chunks;
  sp.d.selected = s.selected;
  if (pl.splits > 1) place_partials(sp.d, a, static_cast<char*>(a.workspace) + pl.score_bytes);
  sp.bounds = s.bounds;
  sp.b_bs = s.bounds_block_stride;
  sp.b_hs = s.bounds_head_stride;
  const int64_t rows = a.batch * a.num_kv_heads;
  sp.keys = static_cast<uint64_t*>(a.workspace);
  sp.scores = reinterpret_cast<float*>(sp.keys + rows * pl.max_chunks);
  sp.errors = sp.scores + rows * pl.max_chunks;
  sp.error_slots = static_cast<int>(pl.score_ctas) * kScoreWarps;
  sp.per = static_cast<int>(a.block_size / s.chunk);
  sp.per_shift = -1;
  for (int k = 0; k < 31; ++k)
    if ((1 << k) == sp.per) sp.per_shift = k;
  sp.max_chunks = pl.max_chunks;
  sp.selected = s.selected;
  launch_k_cluster(chunk_select_kernel<T, D>, dim3(static_cast<unsigned>(pl.score_ctas), static_cast<unsigned>(rows)),
                   kSelectThreads, static_cast<unsigned>(pl.score_ctas), 0, st, sp);
  const int rc = launch_mma_mode<T, D, kDecodeSparse>(a, sp.d, rows, st, true);
  if (rc != NIB_OK || pl.splits == 1) return rc;
  return launch_combine_partials<T, D, kDecodeSparse>(a, sp.d, st);
}

static const char* sparse_check(const nib_sparse_decode_args* s) {
  if (s == nullptr || s->struct_size != static_cast<int32_t>(sizeof(nib_sparse_decode_args)))
    return "sparse_decode_attention: args struct size mismatch";
  const char* bad = decode_check(&s->attn);
  if (bad != nullptr) return bad;
  if (s->chunk < 16 || s->chunk % 16 != 0 || s->attn.block_size % s->chunk != 0)
    return "sparse_decode_attention: chunk must be a multiple of 16 that divides the block size";
  if (s->top_chunks < 2) return "sparse_decode_attention: at least two chunks are selected";
  return nullptr;
}

}  // namespace nib

using namespace nib;

extern "C" int nib_paged_key_bounds(int dtype, const void* key_cache, int64_t cache_block_stride,
                                    int64_t cache_slot_stride, int64_t cache_head_stride, int64_t num_blocks,
                                    int64_t block_size, int64_t num_kv_heads, int64_t head_dim, int64_t chunk,
                                    const int32_t* block_tables, int64_t table_stride, int64_t max_blocks_per_seq,
                                    const int32_t* start_lens, const int32_t* context_lens, int64_t batch,
                                    int64_t max_new_tokens, void* bounds, int64_t bounds_block_stride,
                                    int64_t bounds_head_stride, unsigned int* status, void* stream) {
  NIB_REQUIRE(batch >= 0 && num_blocks >= 0 && block_size >= 1 && num_kv_heads >= 1 && max_blocks_per_seq >= 0 &&
                  max_new_tokens >= 0, "paged_key_bounds: bad sizes");
  NIB_REQUIRE(chunk >= 1 && block_size % chunk == 0, "paged_key_bounds: chunk must divide the block size");
  NIB_SUPPORT(dtype == NIB_BF16 || dtype == NIB_F16, "paged_key_bounds: dtype must be bf16 or f16");
  NIB_SUPPORT(head_dim == 64 || head_dim == 128, "paged_key_bounds: head_dim must be 64 or 128");
  if (batch == 0 || max_blocks_per_seq == 0) return NIB_OK;
  NIB_REQUIRE(key_cache && block_tables && start_lens && context_lens && bounds, "paged_key_bounds: null pointer");
  NIB_REQUIRE(block_size < (int64_t{1} << 31) && max_blocks_per_seq * block_size < (int64_t{1} << 31),
              "paged_key_bounds: block table covers too many tokens (2^31 - 4096)");
  NIB_SUPPORT(batch <= 65535 && num_kv_heads <= 4096, "paged_key_bounds: at most 65535 sequences and 4096 kv heads");
  NIB_SUPPORT(aligned16(key_cache) && aligned16(bounds) && cache_block_stride % 8 == 0 && cache_slot_stride % 8 == 0 &&
                  cache_head_stride % 8 == 0 && bounds_block_stride % 8 == 0 && bounds_head_stride % 8 == 0,
              "paged_key_bounds: caches and bounds must be 16-byte aligned with strides of multiples of 8 elements");
  BoundsParams p{};
  p.kc = key_cache;
  p.c_bs = cache_block_stride;
  p.c_ss = cache_slot_stride;
  p.c_hs = cache_head_stride;
  p.num_blocks = num_blocks;
  p.block_size = static_cast<int>(block_size);
  p.chunk = static_cast<int>(chunk);
  p.nkv = static_cast<int>(num_kv_heads);
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.cap = max_blocks_per_seq * block_size;
  p.starts = start_lens;
  p.lens = context_lens;
  p.bounds = bounds;
  p.b_bs = bounds_block_stride;
  p.b_hs = bounds_head_stride;
  p.status = status;
  p.max_new = max_new_tokens;
  // the chunks that max_new_tokens can lie in, the first of them anywhere in its chunk; one for none, to
  // see that there are none
  const int64_t most = max_new_tokens < p.cap ? max_new_tokens : p.cap, all = p.cap / chunk;
  const int64_t windows = most == 0 ? 1 : (most - 1) / chunk + 2;
  const dim3 grid(static_cast<unsigned>(windows < all ? windows : all), static_cast<unsigned>(batch));
  const cudaStream_t st = as_stream(stream);
  if (dtype == NIB_BF16) {
    if (head_dim == 64) launch_k(key_bounds_kernel<__nv_bfloat16, 64>, grid, kBoundsThreads, 0, st, p);
    else launch_k(key_bounds_kernel<__nv_bfloat16, 128>, grid, kBoundsThreads, 0, st, p);
  } else {
    if (head_dim == 64) launch_k(key_bounds_kernel<__half, 64>, grid, kBoundsThreads, 0, st, p);
    else launch_k(key_bounds_kernel<__half, 128>, grid, kBoundsThreads, 0, st, p);
  }
  return launch_status("paged_key_bounds");
}

extern "C" int64_t nib_sparse_decode_workspace_bytes(const nib_sparse_decode_args* s) {
  if (sparse_check(s) != nullptr) return -1;
  const SparsePlan pl = sparse_plan(*s);
  return pl.score_bytes + pl.partial_bytes;
}

extern "C" int nib_sparse_decode_attention(const nib_sparse_decode_args* s, void* stream) {
  const char* bad = sparse_check(s);
  if (bad != nullptr) {
    set_error("%s", bad);
    return NIB_ERR_INVALID;
  }
  const nib_decode_attention_args& a = s->attn;
  if (a.batch == 0) return NIB_OK;
  NIB_REQUIRE(a.q && a.key_cache && a.value_cache && a.block_tables && a.context_lens && a.out && s->bounds && s->selected,
              "sparse_decode_attention: null pointer");
  NIB_SUPPORT(a.batch * a.num_kv_heads <= 65535, "sparse_decode_attention: at most 65535 (request, kv head) pairs");
  NIB_REQUIRE(a.max_blocks_per_seq * a.block_size < kMaxTokens,
              "sparse_decode_attention: block table covers too many tokens (2^31 - 4096)");
  NIB_SUPPORT(aligned16(a.q) && a.q_batch_stride % 8 == 0 && a.q_head_stride % 8 == 0 && aligned16(s->bounds) &&
                  s->bounds_block_stride % 8 == 0 && s->bounds_head_stride % 8 == 0,
              "sparse_decode_attention: q and bounds must be 16-byte aligned with strides of multiples of 8 elements");
  NIB_SUPPORT(decode_mma_eligible(a), "sparse_decode_attention: needs bf16/f16, head_dim 64 or 128, at most 16 q "
              "heads per kv head, a block size that is a multiple of 16 and 16-byte aligned strides");
  const SparsePlan pl = sparse_plan(*s);
  const int64_t need = pl.score_bytes + pl.partial_bytes;
  NIB_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need && aligned16(a.workspace)),
              "sparse_decode_attention: workspace of %lld bytes needed", static_cast<long long>(need));
  const cudaStream_t st = as_stream(stream);
  return NIB_MMA_CASE(a, T, D, launch_sparse<T, D>(*s, pl, st));
}
