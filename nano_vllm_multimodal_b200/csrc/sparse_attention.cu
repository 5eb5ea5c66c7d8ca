// Decode attention over the chunks of a context that a cheap score selects, and the per-chunk
// key bounds behind that score.
//
// A chunk is `chunk` consecutive tokens inside a cache block; bounds[block, kv head, chunk, 0/1, :]
// hold the smallest and largest value of each key channel over the chunk's tokens. For a query q
// and any key k between the bounds, q . k <= sum_d max(q_d lo_d, q_d hi_d) = q+ . hi + q- . lo
// (q+ = max(q, 0), q- = min(q, 0)), so over the heads h of a kv head
//   score(chunk) = a . hi + b . lo,   a = sum_h q_h+,   b = sum_h q_h-
// bounds the sum of the heads' scores from above with one dot product of 2 D terms, whatever
// the number of heads. Scores are summed in 64 bits: chunks are ranked by them, and in 32 bits
// the order of the summation would decide between near neighbours.
#include "decode_mma.cuh"

namespace nib {

// ------------------------------------------------------------------ key bounds

struct BoundsParams {
  const void* kc;
  int64_t c_bs, c_ss, c_hs;
  int64_t num_blocks;
  int block_size, chunk, nkv, max_windows;
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
// owns one 16-byte vector of the token row (8 channels of a head) and every slices-th token.
template <typename T, int D>
__global__ void __launch_bounds__(kBoundsThreads)
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
  if (blockIdx.x == 0 && threadIdx.x == 0 && (len - 1) / p.chunk - start / p.chunk >= p.max_windows)
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
  uint64_t* keys;      // [batch * kv heads, max_chunks]
  int64_t max_chunks;
  int32_t* selected;   // [batch * kv heads, top]
};

// A score as a whole number of the same order. -0 counts as 0; NaN and infinity as the largest
// finite number, so that the first and the last chunk (all ones) rank before every other.
__device__ __forceinline__ uint64_t score_key(double s) {
  s = s <= 1.7976931348623157e308 ? s + 0.0 : 1.7976931348623157e308;
  const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(s));
  return bits >> 63 ? ~bits : bits | (1ull << 63);
}

constexpr int kScoreWarps = 8;
constexpr int kScoreUnroll = 4;

// A warp takes 32 / (2 D / 8) chunks a step: the lanes of a chunk own 8 channels each, the first
// half of them of lo, the others of hi.
template <typename T, int D>
__global__ void __launch_bounds__(kScoreWarps * 32)
chunk_score_kernel(const SelectParams p) {
  pdl_enter();
  constexpr int LPC = 2 * D / 8;   // lanes per chunk
  constexpr int CPS = 32 / LPC;    // chunks per warp step
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t row = blockIdx.y;
  const int64_t b = row / p.d.num_kv_heads;
  const int kvh = static_cast<int>(row % p.d.num_kv_heads);
  const int64_t len = clamped_len(p.d, b, threadIdx.x == 0 && blockIdx.x == 0 && kvh == 0);
  const int chunk = p.d.chunk;
  const int64_t chunks = (len + chunk - 1) / chunk;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kScoreWarps * kScoreUnroll * CPS);
  if (chunks <= p.d.top || first >= chunks) return;  // all of them are selected, or none is here
  const int part = lane % LPC;
  const bool is_hi = part >= LPC / 2;
  const int d0 = (part % (LPC / 2)) * 8;
  double wt[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wt[i] = 0.0;
  for (int h = 0; h < p.d.group; ++h) {
    float f[8];
    unpack<T>(ld_vec(static_cast<const T*>(p.d.q) + b * p.d.q_bs + (kvh * p.d.group + h) * p.d.q_hs + d0), f);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (is_hi ? f[i] > 0.f : f[i] < 0.f) wt[i] += static_cast<double>(f[i]);
      else if (f[i] != f[i]) wt[i] += static_cast<double>(f[i]);
  }
  const int per = p.d.block_size / chunk;
  const int32_t* table = p.d.tables + b * p.d.table_stride;
  const T* base = static_cast<const T*>(p.bounds) + kvh * p.b_hs + (is_hi ? D : 0) + d0;
  uint4 v[kScoreUnroll];
  bool ok[kScoreUnroll];
  const int64_t c0 = first + w * (kScoreUnroll * CPS) + lane / LPC;
#pragma unroll
  for (int j = 0; j < kScoreUnroll; ++j) {
    const int64_t c = c0 + j * CPS;
    ok[j] = false;
    v[j] = zero_vec();
    if (c < chunks) {
      const int blk = __ldg(table + c / per);
      ok[j] = blk >= 0 && blk < p.d.num_blocks;
      if (ok[j]) v[j] = ld_stream(base + blk * p.b_bs + (c % per) * 2 * D);
      else flag(p.d.status, NIB_DEV_BAD_BLOCK);
    }
  }
#pragma unroll
  for (int j = 0; j < kScoreUnroll; ++j) {
    const int64_t c = c0 + j * CPS;
    float f[8];
    unpack<T>(v[j], f);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma(wt[i], static_cast<double>(f[i]), s);
#pragma unroll
    for (int off = LPC / 2; off >= 1; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if (part == 0 && c < chunks)
      p.keys[row * p.max_chunks + c] = c == 0 || c == chunks - 1 ? ~0ull : ok[j] ? score_key(s) : 0ull;
  }
}

constexpr int kSelectThreads = 256;

// The `top` largest keys of a row, the lower index first among equals, in ascending order of index.
__global__ void __launch_bounds__(kSelectThreads)
chunk_select_kernel(const SelectParams p) {
  pdl_enter();
  __shared__ unsigned int hist[256];
  __shared__ uint64_t s_prefix;
  __shared__ int s_need;
  __shared__ int warp_sel[kSelectThreads / 32], warp_eq[kSelectThreads / 32];
  const int64_t row = blockIdx.x;
  const int64_t len = clamped_len(p.d, row / p.d.num_kv_heads, false);
  const int64_t n = (len + p.d.chunk - 1) / p.d.chunk;
  const int top = p.d.top;
  int32_t* out = p.selected + row * top;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  if (n <= top) {
    for (int i = tid; i < top; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* keys = p.keys + row * p.max_chunks;
  if (tid == 0) {
    s_prefix = 0;
    s_need = top;
  }
  // the top-th largest key, eight bits at a time
  for (int shift = 56; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
    __syncthreads();
    const uint64_t prefix = s_prefix;
    const int need = s_need;
    for (int64_t i = tid; i < n; i += kSelectThreads) {
      const uint64_t k = keys[i];
      if (shift == 56 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (w == 0) {  // lane l: bins 255 - 8 l down to 248 - 8 l
      int mine = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) mine += static_cast<int>(hist[255 - 8 * lane - j]);
      int upto = mine;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= off) upto += v;
      }
      const unsigned reach = __ballot_sync(0xffffffffu, upto >= need);
      if (lane == __ffs(reach) - 1) {
        int above = upto - mine;
        for (int j = 0; j < 8; ++j) {
          const int bin = 255 - 8 * lane - j;
          if (above + static_cast<int>(hist[bin]) >= need) {
            s_prefix = (prefix << 8) | static_cast<uint64_t>(bin);
            s_need = need - above;  // still to take among the keys with this prefix
            break;
          }
          above += static_cast<int>(hist[bin]);
        }
      }
    }
    __syncthreads();
  }
  const uint64_t bar = s_prefix;
  const int equal = s_need;
  int done = 0, done_eq = 0;
  for (int64_t i0 = 0; i0 < n; i0 += kSelectThreads) {
    const int64_t i = i0 + tid;
    const uint64_t k = i < n ? keys[i] : 0;
    const bool eq = i < n && k == bar;
    const unsigned eqs = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) warp_eq[w] = __popc(eqs);
    __syncthreads();
    int before_eq = done_eq + __popc(eqs & ((1u << lane) - 1));
    int all_eq = 0;
    for (int j = 0; j < kSelectThreads / 32; ++j) {
      if (j < w) before_eq += warp_eq[j];
      all_eq += warp_eq[j];
    }
    const bool sel = (i < n && k > bar) || (eq && before_eq < equal);
    const unsigned sels = __ballot_sync(0xffffffffu, sel);
    if (lane == 0) warp_sel[w] = __popc(sels);
    __syncthreads();
    int before = done + __popc(sels & ((1u << lane) - 1));
    int all = 0;
    for (int j = 0; j < kSelectThreads / 32; ++j) {
      if (j < w) before += warp_sel[j];
      all += warp_sel[j];
    }
    if (sel) out[before] = static_cast<int32_t>(i);
    done += all;
    done_eq += all_eq;
  }
}

// ------------------------------------------------------------------ host side

struct SparsePlan {
  int splits;
  int64_t max_len, max_chunks;
  int64_t keys_bytes, partial_bytes;
};

static SparsePlan sparse_plan(const nib_sparse_decode_args& s) {
  const nib_decode_attention_args& a = s.attn;
  SparsePlan pl{};
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  pl.max_len = a.max_context_len > 0 && a.max_context_len < cap ? a.max_context_len : cap;
  pl.max_chunks = (pl.max_len + s.chunk - 1) / s.chunk;
  const int64_t rows = a.batch * a.num_kv_heads;
  const int64_t want = 12LL * sm_count();
  int64_t n = rows < 1 || rows >= want ? 1 : (want + rows - 1) / rows;
  const int64_t tokens = (pl.max_chunks < s.top_chunks ? pl.max_chunks : s.top_chunks) * s.chunk;
  const int64_t by_len = (tokens + 63) / 64;
  if (n > by_len) n = by_len;
  if (n > 256) n = 256;
  pl.splits = static_cast<int>(n < 1 ? 1 : n);
  pl.keys_bytes = pl.max_chunks > s.top_chunks ? (rows * pl.max_chunks * 8 + 15) / 16 * 16 : 0;
  pl.partial_bytes = pl.splits > 1 ? a.batch * a.num_heads * static_cast<int64_t>(pl.splits) * (a.head_dim + 2) *
                                         static_cast<int64_t>(sizeof(float)) : 0;
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
  sp.d.ws = pl.splits > 1 ? reinterpret_cast<float*>(static_cast<char*>(a.workspace) + pl.keys_bytes) : nullptr;
  sp.bounds = s.bounds;
  sp.b_bs = s.bounds_block_stride;
  sp.b_hs = s.bounds_head_stride;
  sp.keys = static_cast<uint64_t*>(a.workspace);
  sp.max_chunks = pl.max_chunks;
  sp.selected = s.selected;
  const int64_t rows = a.batch * a.num_kv_heads;
  if (pl.keys_bytes > 0) {
    constexpr int kChunks = kScoreWarps * kScoreUnroll * (32 / (2 * D / 8));
    const dim3 grid(static_cast<unsigned>((pl.max_chunks + kChunks - 1) / kChunks), static_cast<unsigned>(rows));
    launch_k(chunk_score_kernel<T, D>, grid, kScoreWarps * 32, 0, st, sp);
  }
  launch_k(chunk_select_kernel, static_cast<unsigned>(rows), kSelectThreads, 0, st, sp);
  const int rc = launch_mma_mode<T, D, kDecodeSparse>(a, sp.d, rows, st);
  if (rc != NIB_OK || pl.splits == 1) return rc;
  launch_k_after(combine_partials_kernel<T, D, kDecodeSparse>, static_cast<unsigned>(a.batch * a.num_heads), D, 0, st, sp.d);
  return launch_status("sparse_decode_attention");
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
  if (batch == 0 || max_new_tokens == 0 || max_blocks_per_seq == 0) return NIB_OK;
  NIB_REQUIRE(key_cache && block_tables && start_lens && context_lens && bounds, "paged_key_bounds: null pointer");
  NIB_REQUIRE(block_size < (int64_t{1} << 31) && max_blocks_per_seq * block_size < (int64_t{1} << 31),
              "paged_key_bounds: block table covers 2^31 tokens or more");
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
  const int64_t most = max_new_tokens < p.cap ? max_new_tokens : p.cap;
  p.max_windows = static_cast<int>((most - 1) / chunk + 2);  // the first new token may sit anywhere in its chunk
  const dim3 grid(static_cast<unsigned>(p.max_windows), static_cast<unsigned>(batch));
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
  return pl.keys_bytes + pl.partial_bytes;
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
  NIB_REQUIRE(a.max_blocks_per_seq * a.block_size < (int64_t{1} << 31),
              "sparse_decode_attention: block table covers 2^31 tokens or more");
  NIB_SUPPORT(aligned16(a.q) && a.q_batch_stride % 8 == 0 && a.q_head_stride % 8 == 0 && aligned16(s->bounds) &&
                  s->bounds_block_stride % 8 == 0 && s->bounds_head_stride % 8 == 0,
              "sparse_decode_attention: q and bounds must be 16-byte aligned with strides of multiples of 8 elements");
  NIB_SUPPORT(decode_mma_eligible(a), "sparse_decode_attention: needs bf16/f16, head_dim 64 or 128, at most 16 q "
              "heads per kv head, a block size that is a multiple of 16 and 16-byte aligned strides");
  const SparsePlan pl = sparse_plan(*s);
  const int64_t need = pl.keys_bytes + pl.partial_bytes;
  NIB_REQUIRE(need == 0 || (a.workspace && a.workspace_bytes >= need && aligned16(a.workspace)),
              "sparse_decode_attention: workspace of %lld bytes needed", static_cast<long long>(need));
  const cudaStream_t st = as_stream(stream);
  return NIB_MMA_CASE(a, T, D, launch_sparse<T, D>(*s, pl, st));
}
