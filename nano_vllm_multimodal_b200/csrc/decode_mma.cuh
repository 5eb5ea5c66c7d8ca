// Paged attention of single query tokens on the tensor cores: the device code that
// decode_attention_mma.cu (every token of a context), shared_prefix.cu (a group's shared
// first tokens, and each request's own tokens behind them) and sparse_attention.cu (the
// chunks that a selection keeps) launch with a token source each.
//
// Paged decode attention on the tensor cores (the default kernel of
// nib_decode_attention for bf16/f16, head_dim 64/128, up to 16 q heads per kv
// head, block sizes that are multiples of 16).
//
// Same contract as decode_attention.cu (flash_attn_with_kvcache's decode call,
// nanovllm/layers/attention.py:122-130; the reference's SDPA decode branch,
// attention.py:286-300): out[b, h] = softmax(q[b, h] . K^T * scale) V over the
// request's first context_lens[b] cached tokens, kv head h / group.
//
// A CTA owns (request, kv head, split of the context). The kv head's q heads
// (at most 16) are the M rows of mma.sync m16n8k16 tiles, the context's
// tokens the N columns: S = Q K^T per 16-token tile (D/16 k-steps x 2 n-tiles),
// then O += P V (one k-step of 16 tokens x D/8 n-tiles). q heads beyond the
// group are zero rows. With at most 16 q heads per kv head this spends the
// same tensor-core issue on grouped-query (GQA 8) as on GQA 2, so the kernel
// stays HBM-bound where the CUDA-core kernel's fp32 FMAs per cached byte grow
// with the group.
//
// Each warp owns every kMmaWarps-th tile of the CTA's range and a private ring
// of kMmaStages (2) shared-memory stages, so 3 CTAs (12 warps) fit on an SM:
// with 3 stages and 2 CTAs per SM the GQA-8 C2 decode took 0.210 ms instead of
// 0.203 ms. Lane 0 loads a tile with two TMA tensor copies per 64-element
// half of the head, one from each cache (cp.async.bulk.tensor, 5-D maps over
// [blocks, block_size, kv_heads, D/64, 64], 128-byte swizzle, no multicast),
// completing on the stage's mbarrier; the waits are bounded in wall time like every wait of this
// library (on timeout: NIB_DEV_TIMEOUT, wait for the warp's other copies,
// return). Fragments come from shared memory with ldmatrix (.trans for V);
// the swizzle keeps those reads free of bank conflicts. Scores are kept in
// the log2 domain with an online max and sum per q head; warps and splits are
// merged with max-rescaled sums (the split partials use the CUDA-core
// kernel's workspace format and its combine kernel).
#pragma once

#include <cuda.h>

#include <mutex>
#include <type_traits>

#include "bulk_copy.cuh"
#include "dispatch.cuh"

namespace nib {

constexpr int kMmaWarps = 4;
constexpr int kMmaStages = 2;  // ring stages per warp: 3 CTAs (12 warps) per SM fit
constexpr int kMmaTile = 16;   // tokens per tile

// Contexts stay below this, so that token arithmetic a tile beyond them fits 32 bits.
constexpr int64_t kMaxTokens = (int64_t{1} << 31) - 4096;

// Which rows and tokens a CTA takes.
enum DecodeMode : int {
  kDecodeFull = 0,    // a request's heads against all of its tokens
  kDecodeSuffix = 1,  // a request's heads against its tokens behind the prefix that its group shares
  kDecodeShared = 2,  // one launch: 16 rows (request, head) of a group against the prefix that they
                      // share (the first prefix_ctas CTAs), and kDecodeSuffix's work
  kDecodeSparse = 3   // a request's heads against the chunks selected for them
};

struct MmaDecodeParams {
  const void* q;
  int64_t q_bs, q_hs;
  const int32_t* tables;
  int64_t table_stride, num_blocks;
  int64_t cap;  // tokens that a request may have
  int block_size;
  const int32_t* lens;
  float qscale;  // softmax scale * log2(e)
  void* out;
  int64_t o_bs, o_hs;
  float* ws;   // partials; null: one split writes `out`. kDecodeFull: [batch, num_heads, splits, D + 2]
               // (output, maximum, sum), else [batch, num_heads, slots, D] with
  float2* ml;  // [batch, num_heads, slots] (maximum, sum)
  int num_heads, num_kv_heads, group, splits;
  int slots, slot0;  // partials per (request, head), and this launch's first
  bool early;  // kDecodeSuffix: launched behind the prefix kernel, of whose results it reads none
  unsigned int* status;
  // kDecodeSuffix, kDecodeShared
  int prefix_ctas, prefix_splits;
  int64_t batch;
  const int32_t* group_offsets;  // [num_groups + 1]
  const int32_t* prefix_lens;    // [num_groups]
  int num_groups;
  // kDecodeSparse
  const int32_t* selected;  // [batch, num_kv_heads, top] ascending
  int chunk, top;
};

// A request's length, clamped to what it may have (what its table can hold, or less).
__device__ __forceinline__ int64_t clamped_len(const MmaDecodeParams& p, int64_t b, bool report) {
  const int64_t len = __ldg(p.lens + b);
  if (len >= 0 && len <= p.cap) return len;
  if (report) flag(p.status, NIB_DEV_BAD_INDEX);
  return len < 0 ? 0 : p.cap;
}

// The tokens of request b that its group shares (0: none), by a whole warp. A request that
// is shorter than its group's prefix takes no part in the sharing.
__device__ __forceinline__ int64_t shared_prefix_of(const MmaDecodeParams& p, int64_t b, int64_t len, int lane) {
  for (int g0 = 0; g0 < p.num_groups; g0 += 32) {
    const int g = g0 + lane;
    const bool in = g < p.num_groups && b >= __ldg(p.group_offsets + g) && b < __ldg(p.group_offsets + g + 1);
    const unsigned found = __ballot_sync(0xffffffffu, in);
    if (found) {
      const int64_t pre = __ldg(p.prefix_lens + g0 + __ffs(found) - 1);
      return pre > 0 && pre <= len ? pre : 0;
    }
  }
  return 0;
}

// How many of the launch's splits share a request's `own` tokens behind the prefix: 256 tokens each at
// least. The others write nothing and the merge passes them over.
constexpr int kOwnTokens = 256;
__device__ __forceinline__ int own_splits(int64_t own, int splits) {
  const int64_t n = (own + kOwnTokens - 1) / kOwnTokens;
  return n < 1 ? 1 : n < splits ? static_cast<int>(n) : splits;
}

// Row tile `tile` (tile_rows rows each, a group's last one ragged) of the groups in order:
// its group's requests and its place among the group's tiles. By a whole warp. Tile 0 looks every group
// over and reports what is wrong, whether or not it has rows.
struct RowTile {
  int64_t first, end;  // the group's requests
  int64_t row0;        // the tile's first row: row = (request - first) * heads per kv head + head
  int64_t prefix;      // tokens that the group shares; 0: nothing to do
  int64_t leader;      // the request whose table names the prefix's pages
};

__device__ __forceinline__ RowTile find_row_tile(const MmaDecodeParams& p, int64_t tile, int tile_rows, int lane) {
  RowTile r{0, 0, 0, 0, -1};
  int64_t base = 0;
  int found_g = -1;
  for (int g0 = 0; g0 < p.num_groups; g0 += 32) {
    const int g = g0 + lane;
    int64_t lo = 0, hi = 0;
    if (g < p.num_groups) {
      lo = __ldg(p.group_offsets + g);
      hi = __ldg(p.group_offsets + g + 1);
      const int shared = tile == 0 ? __ldg(p.prefix_lens + g) : 0;
      if (tile == 0 && (lo < 0 || hi < lo || hi > p.batch || shared < 0)) flag(p.status, NIB_DEV_BAD_INDEX);
      lo = lo < 0 ? 0 : lo;
      hi = hi > p.batch ? p.batch : hi;
      if (hi < lo) hi = lo;
    }
    const int64_t mine = ((hi - lo) * p.group + tile_rows - 1) / tile_rows;
    int64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= off) upto += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, tile < base + upto);
    if (hit && found_g < 0) {
      const int src = __ffs(hit) - 1;
      r.first = __shfl_sync(0xffffffffu, lo, src);
      r.end = __shfl_sync(0xffffffffu, hi, src);
      r.row0 = (tile - base - __shfl_sync(0xffffffffu, upto - mine, src)) * tile_rows;
      found_g = g0 + src;
      if (tile > 0) break;
    }
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (found_g < 0) return r;
  const int64_t pre = __ldg(p.prefix_lens + found_g);
  if (pre <= 0) return r;
  for (int64_t b0 = r.first; b0 < r.end; b0 += 32) {
    const bool holds = b0 + lane < r.end && clamped_len(p, b0 + lane, false) >= pre;
    const unsigned any = __ballot_sync(0xffffffffu, holds);
    if (any) {
      r.leader = b0 + __ffs(any) - 1;
      r.prefix = pre;
      break;
    }
  }
  return r;
}

// byte offset of (token t, element d) inside a stage's K or V tile. The tile is
// D/64 regions (one per 64-element half of the head, one tensor copy each) of
// kMmaTile 128-byte rows, row = token, whose 16-byte chunks are XOR-swizzled by
// row % 8 - how a SWIZZLE_128B tensor copy lays its box out. An ldmatrix phase
// reads the same chunk of 8 consecutive tokens: 8 different rows, 8 different
// swizzled chunks, no bank conflict. (With both halves of a token in one box,
// consecutive tokens sit 2 rows apart and every phase conflicts 2-way: 48% of
// the shared-memory wavefronts in the first version of this kernel.)
template <int D>
__device__ __forceinline__ uint32_t swz(int t, int d) {
  return static_cast<uint32_t>((d >> 6) * (kMmaTile * 128) + t * 128 + ((((d & 63) >> 3) ^ (t & 7)) << 4) +
                               (d & 7) * 2);
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2,
                                            int c3, int c4, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_addr(bar))
      : "memory");
}

__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// c += a (16x16, row) * b (16x8, col), fp32 accumulate
template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
        " {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9},"
        " {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  typename Vec2<T>::type v = Vec2<T>::make(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

__device__ __forceinline__ float ex2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Zero the K and V rows of the tokens outside [lo, hi) (tile-relative) of one
// stage, whatever the cache holds there: their scores are masked, but 0 x NaN
// would still reach the sums. The fence orders these generic writes before
// the stage's next tensor copy.
template <int D>
__device__ __forceinline__ void zero_rows(unsigned char* kg, int lo, int hi, int lane) {
  constexpr uint32_t kTileBytes = kMmaTile * D * 2;
  for (int e = lane; e < kMmaTile * (D / 8); e += 32) {  // 16-byte units of one tile
    const int t = e % kMmaTile;  // a token's row in each region (the chunk order within does not matter)
    if (t < lo || t >= hi) {
      const int u = e / kMmaTile;  // (region, chunk)
      const uint32_t at = (u >> 3) * (kMmaTile * 128) + t * 128 + (u & 7) * 16;
      *reinterpret_cast<uint4*>(kg + at) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(kg + kTileBytes + at) = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async();
  __syncwarp();
}

// Q fragments: the A operand. q0 and q1 are this lane's rows r0 and r0 + 8 (null: a zero row).
template <typename T, int D>
__device__ __forceinline__ void load_q_rows(uint32_t (&qa)[D / 16][4], const T* q0, const T* q1, int lane) {
  const int cq = (lane & 3) * 2;
  const bool ok0 = q0 != nullptr, ok1 = q1 != nullptr;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const int k = ks * 16 + cq;
    qa[ks][0] = ok0 ? __ldg(reinterpret_cast<const uint32_t*>(q0 + k)) : 0u;
    qa[ks][1] = ok1 ? __ldg(reinterpret_cast<const uint32_t*>(q1 + k)) : 0u;
    qa[ks][2] = ok0 ? __ldg(reinterpret_cast<const uint32_t*>(q0 + k + 8)) : 0u;
    qa[ks][3] = ok1 ? __ldg(reinterpret_cast<const uint32_t*>(q1 + k + 8)) : 0u;
  }
}

// Q fragments of one (request, kv head): rows = the kv head's q heads, zero past the group.
template <typename T, int D>
__device__ __forceinline__ void load_q_frags(uint32_t (&qa)[D / 16][4], const T* qb, int64_t q_hs, int first_head,
                                             int group, int lane) {
  const int r0 = lane >> 2;
  load_q_rows<T, D>(qa, r0 < group ? qb + static_cast<int64_t>(first_head + r0) * q_hs : nullptr,
                    r0 + 8 < group ? qb + static_cast<int64_t>(first_head + r0 + 8) * q_hs : nullptr, lane);
}

// One 16-token tile of a stage (K at kt, V at kt + tile bytes) into the online
// softmax state of rows r0 (a) and r0 + 8 (b): S = Q K^T, scores of tokens
// outside [lo, hi) (tile-relative) masked, then O += P V. A row whose scores are all NaN so far keeps
// a NaN in its sum (and, below, in the result): only a row of masked scores counts as empty.
template <typename T, int D>
__device__ __forceinline__ void mma_tile(const uint32_t (&qa)[D / 16][4], uint32_t kt, int lo, int hi, float qscale,
                                         float (&o)[D / 8][4], float& m_a, float& m_b, float& l_a, float& l_b,
                                         int lane) {
  constexpr int KS = D / 16;
  constexpr int ND = D / 8;
  const uint32_t vt = kt + kMmaTile * D * 2;
  const int cq = (lane & 3) * 2;
  // ---- S = Q K^T (2 n-tiles of 8 tokens)
  float s[2][4];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
    s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ks += 2) {
      uint32_t kb[4];
      // matrices (tokens 8nt..8nt+7) x (d chunks 2ks .. 2ks+3): lane L gives row L%8 of matrix L/8
      ldsm_x4(kt + swz<D>(nt * 8 + (lane & 7), (ks * 2 + (lane >> 3)) * 8), kb);
      mma16816<T>(s[nt], qa[ks], kb[0], kb[1]);
      mma16816<T>(s[nt], qa[ks + 1], kb[2], kb[3]);
    }
  }
  // ---- online softmax (log2 domain); mask tokens outside the range
  float mx_a = -INFINITY, mx_b = -INFINITY;
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int t = nt * 8 + cq + c;
      const bool in = t >= lo && t < hi;
      s[nt][c] = in ? s[nt][c] * qscale : -INFINITY;
      s[nt][c + 2] = in ? s[nt][c + 2] * qscale : -INFINITY;
      mx_a = fmaxf(mx_a, s[nt][c]);
      mx_b = fmaxf(mx_b, s[nt][c + 2]);
    }
  }
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    mx_a = fmaxf(mx_a, __shfl_xor_sync(0xffffffffu, mx_a, off));
    mx_b = fmaxf(mx_b, __shfl_xor_sync(0xffffffffu, mx_b, off));
  }
  const float na = fmaxf(m_a, mx_a), nb = fmaxf(m_b, mx_b);
  // nothing but masked (-inf) and NaN scores so far: less 0, so that these become 0 and NaN
  const float sa = na == -INFINITY ? 0.f : na, sb = nb == -INFINITY ? 0.f : nb;
  const float ra = ex2_fast(m_a - sa), rb = ex2_fast(m_b - sb);
  m_a = na;
  m_b = nb;
  float pa[2][2], pb[2][2];
#pragma unroll
  for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      pa[nt][c] = ex2_fast(s[nt][c] - sa);
      pb[nt][c] = ex2_fast(s[nt][c + 2] - sb);
    }
  }
  l_a = l_a * ra + (pa[0][0] + pa[0][1]) + (pa[1][0] + pa[1][1]);
  l_b = l_b * rb + (pb[0][0] + pb[0][1]) + (pb[1][0] + pb[1][1]);
#pragma unroll
  for (int n = 0; n < ND; ++n) {
    o[n][0] *= ra;
    o[n][1] *= ra;
    o[n][2] *= rb;
    o[n][3] *= rb;
  }
  // P as the A fragment of one 16-token k-step (the C layout of two n-tiles)
  uint32_t pf[4];
  pf[0] = pack2<T>(pa[0][0], pa[0][1]);
  pf[1] = pack2<T>(pb[0][0], pb[0][1]);
  pf[2] = pack2<T>(pa[1][0], pa[1][1]);
  pf[3] = pack2<T>(pb[1][0], pb[1][1]);
  // ---- O += P V (V^T fragments by ldmatrix.trans: rows = tokens, 8 d values each)
#pragma unroll
  for (int n2 = 0; n2 < ND; n2 += 2) {
    uint32_t vb[4];
    // matrices: (tokens 0-7, d chunk n2), (tokens 8-15, n2), (0-7, n2+1), (8-15, n2+1)
    ldsm_x4_t(vt + swz<D>((lane & 7) + ((lane >> 3) & 1) * 8, (n2 + (lane >> 4)) * 8), vb);
    mma16816<T>(o[n2], pf, vb[0], vb[1]);
    mma16816<T>(o[n2 + 1], pf, vb[2], vb[3]);
  }
}

template <typename T, int D, int MODE>
__global__ void __launch_bounds__(kMmaWarps * 32, 3)
decode_attention_mma_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                            const MmaDecodeParams p) {
  constexpr int KS = D / 16;          // k-steps of Q K^T
  constexpr int ND = D / 8;           // n-tiles of P V
  constexpr uint32_t kTileBytes = kMmaTile * D * 2;  // one of K or V
  constexpr uint32_t kStageBytes = 2 * kTileBytes;
  __shared__ __align__(8) uint64_t bars[kMmaWarps][kMmaStages];
  extern __shared__ unsigned char dsm_raw[];
  // the 128-byte swizzle repeats every 1,024 bytes: stages start on that boundary
  const uint32_t raw = smem_addr(dsm_raw);
  const uint32_t base_all = (raw + 1023u) & ~1023u;
  unsigned char* dsm = dsm_raw + (base_all - raw);

  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  if (lane == 0) {
    for (int s = 0; s < kMmaStages; ++s) mbar_init(&bars[w][s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  // the barrier set-up above overlaps the previous kernel's tail
  if (MODE == kDecodeSuffix && p.early) pdl_launch_dependents();  // runs next to it; waits for it at the end
  else pdl_enter();

  // kDecodeShared: a 1-D grid; else (rows x kv heads, splits)
  const bool is_prefix = MODE == kDecodeShared && static_cast<int>(blockIdx.x) < p.prefix_ctas;
  int splits = is_prefix ? p.prefix_splits : p.splits;
  int unit = blockIdx.x, split = blockIdx.y;
  if constexpr (MODE == kDecodeShared) {
    if (is_prefix) {
      split = unit % splits;
      unit /= splits;
    } else {  // every request's first split before the others, which may have nothing to do
      const int rows = static_cast<int>(p.batch) * p.num_kv_heads;
      unit -= p.prefix_ctas;
      split = unit / rows;
      unit -= split * rows;
    }
  }
  const int kvh = unit % p.num_kv_heads;
  int64_t b;          // the request whose table is read
  int64_t skip = 0;   // tokens before the range that the splits share
  int64_t len;        // length of that range (kDecodeSparse: of the selected chunks, end to end)
  int64_t ctx = 0;    // kDecodeSparse: the request's length
  RowTile rt{};
  if (is_prefix) {
    rt = find_row_tile(p, unit / p.num_kv_heads, 16, lane);
    if (rt.prefix == 0) return;  // no such tile, or nothing shared
    b = rt.leader;
    len = rt.prefix;
  } else {
    b = unit / p.num_kv_heads;
    len = clamped_len(p, b, threadIdx.x == 0 && split == 0);
    if constexpr (MODE == kDecodeSuffix || MODE == kDecodeShared) {
      skip = shared_prefix_of(p, b, len, lane);
      len -= skip;
      splits = own_splits(len, splits);
      if (split >= splits) {
        if (MODE == kDecodeSuffix && p.early) pdl_wait();
        return;
      }
    }
    if constexpr (MODE == kDecodeSparse) {
      ctx = len;
      const int chunks = static_cast<int>(len / p.chunk) + (len % p.chunk != 0);
      len = static_cast<int64_t>(chunks < p.top ? chunks : p.top) * p.chunk;
    }
  }
  int64_t t_begin, t_end, tile0, n_tiles;
  if constexpr (MODE == kDecodeFull) {
    // Split boundaries: the splits of a context shrink linearly toward the last one
    // (split y gets a share s - y of s + (s-1) + ... + 1), and the grid's rows are
    // dispatched in split order, so its final wave holds the smallest CTAs.
    auto split_start = [&](int y) -> int64_t {
      const int64_t sp = p.splits;
      const int64_t before = y * sp - static_cast<int64_t>(y) * (y - 1) / 2;
      return len * before / (sp * (sp + 1) / 2);
    };
    t_begin = split_start(split);
    t_end = split_start(split + 1);
    tile0 = t_begin / kMmaTile;
    n_tiles = t_end > t_begin ? (t_end + kMmaTile - 1) / kMmaTile - tile0 : 0;
  } else {
    // equal shares of whole tiles: one wave of CTAs is what these launches ask for
    const int first = static_cast<int>(skip) / kMmaTile;
    const int total = len > 0 ? static_cast<int>(skip + len + kMmaTile - 1) / kMmaTile - first : 0;
    const int each = total / splits, more = total - each * splits;
    tile0 = first + split * each + (split < more ? split : more);
    n_tiles = each + (split < more ? 1 : 0);
    t_begin = tile0 * kMmaTile > skip ? tile0 * kMmaTile : skip;
    t_end = (tile0 + n_tiles) * kMmaTile < skip + len ? (tile0 + n_tiles) * kMmaTile : skip + len;
  }
  const int64_t n_mine = n_tiles > w ? (n_tiles - w + kMmaWarps - 1) / kMmaWarps : 0;  // warp-uniform

  const int r0 = lane >> 2, cq = (lane & 3) * 2;
  uint32_t qa[KS][4];
  if (is_prefix) {
    auto q_row = [&](int r) -> const T* {
      if (r >= (rt.end - rt.first) * p.group) return nullptr;
      return static_cast<const T*>(p.q) + (rt.first + r / p.group) * p.q_bs + (kvh * p.group + r % p.group) * p.q_hs;
    };
    load_q_rows<T, D>(qa, q_row(static_cast<int>(rt.row0) + r0), q_row(static_cast<int>(rt.row0) + r0 + 8), lane);
  } else {
    load_q_frags<T, D>(qa, static_cast<const T*>(p.q) + b * p.q_bs, p.q_hs, kvh * p.group, p.group, lane);
  }

  float o[ND][4];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m_a = -INFINITY, m_b = -INFINITY, l_a = 0.f, l_b = 0.f;  // rows r0 and r0 + 8

  const int32_t* table = p.tables + b * p.table_stride;
  const uint32_t ring = base_all + static_cast<uint32_t>(w) * kMmaStages * kStageBytes;
  uint32_t ok_bits = 0;  // per stage: its tile was loaded
  bool timed_out = false;

  // kDecodeFull: a tile's place is looked up when it is issued. Else by 32 tiles of the warp at
  // once, a tile per lane: the chain list -> table -> copy is too long to walk for each tile.
  const int32_t* list = MODE == kDecodeSparse ? p.selected + (b * p.num_kv_heads + kvh) * p.top : nullptr;
  int batch_t0 = 0, batch_blk = -1;          // this lane's tile of the batch: first token, block (-1: none)
  int stage_t0[kMmaStages], stage_ok[kMmaStages];

  auto issue = [&](int64_t i) {
    if (i >= n_mine) return;
    const int st = static_cast<int>(i % kMmaStages);
    if constexpr (MODE != kDecodeFull) {
      if ((i & 31) == 0) {
        batch_blk = -1;
        if (i + lane < n_mine) {
          int t0 = static_cast<int>(tile0 + w + (i + lane) * kMmaWarps) * kMmaTile;  // tokens stay below 2^31
          if constexpr (MODE == kDecodeSparse) {
            const int nth = t0 / p.chunk, c = __ldg(list + nth);
            t0 = c < 0 ? static_cast<int>(ctx) : c * p.chunk + (t0 - nth * p.chunk);
          }
          batch_t0 = t0;
          if (MODE != kDecodeSparse || t0 < ctx) {  // a last chunk's empty tiles are left out
            batch_blk = __ldg(table + t0 / p.block_size);
            if (batch_blk < 0 || batch_blk >= p.num_blocks) {
              flag(p.status, NIB_DEV_BAD_BLOCK);
              batch_blk = -1;
            }
          }
        }
      }
      const int t0 = __shfl_sync(0xffffffffu, batch_t0, static_cast<int>(i & 31));
      const int blk = __shfl_sync(0xffffffffu, batch_blk, static_cast<int>(i & 31));
#pragma unroll
      for (int s = 0; s < kMmaStages; ++s)
        if (s == st) {
          stage_t0[s] = t0;
          stage_ok[s] = blk >= 0;
        }
      if (lane == 0) {
        fence_proxy_async();  // this stage's generic zero-fill (if any) before the copies
        mbar_arrive_expect_tx(&bars[w][st], blk >= 0 ? kStageBytes : 0u);
        if (blk >= 0) {
          const int off = t0 % p.block_size;
          const uint32_t dst = ring + st * kStageBytes;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            tma_load_5d(dst + c * kMmaTile * 128, &kmap, 0, c, kvh, off, blk, &bars[w][st]);
            tma_load_5d(dst + kTileBytes + c * kMmaTile * 128, &vmap, 0, c, kvh, off, blk, &bars[w][st]);
          }
        }
      }
      return;
    }
    if (lane == 0) {
      const int64_t t0 = (tile0 + w + i * kMmaWarps) * kMmaTile;
      const int64_t bi = t0 / p.block_size;
      const int blk = __ldg(table + bi);
      const bool ok = blk >= 0 && blk < p.num_blocks;
      if (!ok) flag(p.status, NIB_DEV_BAD_BLOCK);
      fence_proxy_async();  // this stage's generic zero-fill (if any) before the copies
      mbar_arrive_expect_tx(&bars[w][st], ok ? kStageBytes : 0u);
      if (ok) {
        const int off = static_cast<int>(t0 - bi * p.block_size);
        const uint32_t dst = ring + st * kStageBytes;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {  // one region per 64-element half
          tma_load_5d(dst + c * kMmaTile * 128, &kmap, 0, c, kvh, off, blk, &bars[w][st]);
          tma_load_5d(dst + kTileBytes + c * kMmaTile * 128, &vmap, 0, c, kvh, off, blk, &bars[w][st]);
        }
      }
      ok_bits = (ok_bits & ~(1u << st)) | (static_cast<uint32_t>(ok) << st);
    }
  };

#pragma unroll
  for (int i = 0; i < kMmaStages - 1; ++i) issue(i);
  for (int64_t i = 0; i < n_mine; ++i) {
    issue(i + kMmaStages - 1);
    const int st = static_cast<int>(i % kMmaStages);
    const bool done = mbar_wait(&bars[w][st], static_cast<uint32_t>((i / kMmaStages) & 1));
    if (!__all_sync(0xffffffffu, done)) {
      if (lane == 0) flag(p.status, kDevTimeout);
      // let the warp's other copies land (bounded) before leaving
      for (int64_t j = i + 1; j < i + kMmaStages && j < n_mine; ++j)
        (void)mbar_wait(&bars[w][j % kMmaStages], static_cast<uint32_t>((j / kMmaStages) & 1));
      timed_out = true;
      break;
    }
    bool ok;
    int64_t t0;
    if constexpr (MODE == kDecodeFull) {
      ok = (__shfl_sync(0xffffffffu, ok_bits, 0) >> st) & 1u;
      t0 = (tile0 + w + i * kMmaWarps) * kMmaTile;
    } else {
      ok = st == 0 ? stage_ok[0] : stage_ok[1];
      t0 = st == 0 ? stage_t0[0] : stage_t0[1];
      static_assert(kMmaStages == 2, "two stages");
    }
    const uint32_t kt = ring + st * kStageBytes;
    if (!ok) continue;  // bad block id: its tokens take no part
    // the tile's tokens in [t_begin, t_end), tile-relative (only the first and last tile are partial)
    const int64_t from = MODE == kDecodeSparse ? 0 : t_begin, to = MODE == kDecodeSparse ? ctx : t_end;
    const int lo = from > t0 ? static_cast<int>(from - t0) : 0;
    const int hi = to - t0 < kMmaTile ? static_cast<int>(to - t0) : kMmaTile;
    if (lo > 0 || hi < kMmaTile) zero_rows<D>(dsm + (kt - base_all), lo, hi, lane);
    mma_tile<T, D>(qa, kt, lo, hi, p.qscale, o, m_a, m_b, l_a, l_b, lane);
    __syncwarp();  // every lane has read the stage before it is refilled
  }

  // ---- per-row sums over the quad; merge the warps through shared memory
#pragma unroll
  for (int off = 1; off < 4; off <<= 1) {
    l_a += __shfl_xor_sync(0xffffffffu, l_a, off);
    l_b += __shfl_xor_sync(0xffffffffu, l_b, off);
  }
  if (__syncthreads_or(timed_out)) {  // the rows are incomplete; the status bit says so
    if (MODE == kDecodeSuffix && p.early) pdl_wait();
    return;
  }
  constexpr int SW = D + 2;
  float* red = reinterpret_cast<float*>(dsm);  // [warps][16 rows][D + 2], over the rings
#pragma unroll
  for (int n = 0; n < ND; ++n) {
    const int d = n * 8 + cq;
    red[(w * 16 + r0) * SW + d] = o[n][0];
    red[(w * 16 + r0) * SW + d + 1] = o[n][1];
    red[(w * 16 + r0 + 8) * SW + d] = o[n][2];
    red[(w * 16 + r0 + 8) * SW + d + 1] = o[n][3];
  }
  if ((lane & 3) == 0) {
    red[(w * 16 + r0) * SW + D] = m_a;
    red[(w * 16 + r0) * SW + D + 1] = l_a;
    red[(w * 16 + r0 + 8) * SW + D] = m_b;
    red[(w * 16 + r0 + 8) * SW + D + 1] = l_b;
  }
  __syncthreads();
  const int rows = is_prefix ? 16 : p.group;
  for (int idx = threadIdx.x; idx < rows * D; idx += blockDim.x) {
    const int r = idx / D, d = idx % D;
    int64_t rb = b;
    int h = kvh * p.group + r;
    if (is_prefix) {
      const int row = static_cast<int>(rt.row0) + r;
      if (row >= (rt.end - rt.first) * p.group) continue;
      rb = rt.first + row / p.group;
      h = kvh * p.group + row % p.group;
    }
    float M = -INFINITY;
#pragma unroll
    for (int ww = 0; ww < kMmaWarps; ++ww) M = fmaxf(M, red[(ww * 16 + r) * SW + D]);
    float L = 0.f, A = 0.f;
    if (M != -INFINITY) {
#pragma unroll
      for (int ww = 0; ww < kMmaWarps; ++ww) {
        const float* rr = red + (ww * 16 + r) * SW;
        const float f = rr[D] == -INFINITY ? 0.f : ex2_fast(rr[D] - M);
        L += rr[D + 1] * f;
        A += rr[d] * f;
      }
    } else {
#pragma unroll
      for (int ww = 0; ww < kMmaWarps; ++ww) L += red[(ww * 16 + r) * SW + D + 1];  // 0, or the NaN of NaN scores
    }
    if (p.ws == nullptr) {
      static_cast<T*>(p.out)[rb * p.o_bs + h * p.o_hs + d] = Elem<T>::from_f(attention_row(A, L));
    } else if constexpr (MODE == kDecodeFull) {
      float* ws = p.ws + ((rb * p.num_heads + h) * p.splits + split) * SW;
      ws[d] = A;
      if (d == 0) {
        ws[D] = M;
        ws[D + 1] = L;
      }
    } else {
      const int64_t at = (rb * p.num_heads + h) * p.slots + (is_prefix ? 0 : p.slot0) + split;
      p.ws[at * D + d] = A;
      if (d == 0) p.ml[at] = make_float2(M, L);
    }
  }
  if (MODE == kDecodeSuffix && p.early) pdl_wait();  // so that the next kernel follows both
}


// out[b, h] from the partials of (b, h). MODE kDecodeSuffix: the first slot0 partials are the
// prefix's, which only a request that shares one has; behind them as many as its own tokens fill. WPR warps take a row's partials by turns; a
// warp's first eight outputs are requested together with the maxima and sums, before it is known
// which of them count: one round trip to memory is most of this kernel's time. (Four warps a row
// where rows are few, one where they fill the SMs: 4,096 rows of ten partials, 13.2 us with four.)
constexpr int kCombineWarps = 4, kCombineBatch = 8;

template <typename T, int D, int MODE, int WPR>
__global__ void __launch_bounds__(kCombineWarps * 32)
combine_partials_kernel(const MmaDecodeParams p) {
  pdl_enter();
  constexpr int E = D / 32;  // channels per lane
  using Vec = typename std::conditional<E == 4, float4, float2>::type;
  __shared__ float red[WPR > 1 ? kCombineWarps : 1][D];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int row = static_cast<int>(blockIdx.x) * (kCombineWarps / WPR) + w / WPR, part = w % WPR;
  if (row >= static_cast<int>(p.batch) * p.num_heads) return;  // WPR = 1 alone
  const int b = row / p.num_heads, h = row - b * p.num_heads;
  const float2* ml = p.ml + static_cast<int64_t>(row) * p.slots;
  const Vec* ws = reinterpret_cast<const Vec*>(p.ws + static_cast<int64_t>(row) * p.slots * D) + lane;
  Vec v[kCombineBatch];
#pragma unroll
  for (int k = 0; k < kCombineBatch; ++k)
    if (part + k * WPR < p.slots) v[k] = ws[static_cast<int64_t>(part + k * WPR) * 32];
  const float2 first = lane < p.slots ? ml[lane] : make_float2(-INFINITY, 0.f);
  int s0 = 0, s1 = p.slots;
  if constexpr (MODE == kDecodeSuffix) {  // and after kDecodeShared
    const int64_t len = clamped_len(p, b, false), shared = shared_prefix_of(p, b, len, lane);
    if (shared == 0) s0 = p.slot0;
    s1 = p.slot0 + own_splits(len - shared, p.splits);
  }
  auto counts = [&](int s) { return s >= s0 && s < s1; };
  float M = counts(lane) ? first.x : -INFINITY;
  for (int s = 32 + lane; s < s1; s += 32)
    if (s >= s0) M = fmaxf(M, ml[s].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, off));
  // a NaN sum (of NaN scores) makes the row NaN
  bool odd = counts(lane) && first.y != first.y;
  for (int s = 32 + lane; s < s1; s += 32) odd |= s >= s0 && ml[s].y != ml[s].y;
  odd = __any_sync(0xffffffffu, odd);
  float L = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
  if (M != -INFINITY && !odd) {
    // a split without tokens has no output and the weight 0
    auto weight = [&](float2 x, int s) { return counts(s) && x.x != -INFINITY ? ex2_fast(x.x - M) : 0.f; };
    const float f = weight(first, lane);
    L = f > 0.f ? first.y * f : 0.f;
    for (int s = 32 + lane; s < s1; s += 32) {
      const float2 x = ml[s];
      const float g = weight(x, s);
      if (g > 0.f) L += x.y * g;
    }
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) L += __shfl_xor_sync(0xffffffffu, L, off);
    auto add = [&](const Vec& x, float g) {
      const float* xs = reinterpret_cast<const float*>(&x);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += xs[e] * g;
    };
#pragma unroll
    for (int k = 0; k < kCombineBatch; ++k) {
      const int s = part + k * WPR;  // below 32
      const float g = __shfl_sync(0xffffffffu, f, s);
      if (s < s1 && g > 0.f) add(v[k], g);
    }
    for (int s = part + kCombineBatch * WPR; s < s1; s += WPR) {
      const float g = weight(ml[s], s);
      if (g > 0.f) add(ws[static_cast<int64_t>(s) * 32], g);
    }
  }
  T* out = static_cast<T*>(p.out) + b * p.o_bs + h * p.o_hs;
  const float none = odd ? __int_as_float(0x7fffffff) : 0.f;
  if constexpr (WPR == 1) {
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<typename Vec2<T>::type*>(out + lane * E + e) =
          Vec2<T>::make(L > 0.f ? acc[e] / L : none, L > 0.f ? acc[e + 1] / L : none);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) red[w][lane * E + e] = acc[e];
    __syncthreads();
    static_assert(WPR == kCombineWarps, "a CTA per row");
    for (int d = threadIdx.x; d < D; d += kCombineWarps * 32) {
      float A = 0.f;
#pragma unroll
      for (int ww = 0; ww < kCombineWarps; ++ww) A += red[ww][d];
      out[d] = Elem<T>::from_f(L > 0.f ? A / L : none);
    }
  }
}

// Device bytes of the partials of a launch sequence (any mode but kDecodeFull).
inline int64_t partial_bytes(const nib_decode_attention_args& a, int64_t slots) {
  return a.batch * a.num_heads * slots * (a.head_dim + 2) * static_cast<int64_t>(sizeof(float));
}
// their places in `at` (16-byte aligned)
inline void place_partials(MmaDecodeParams& p, const nib_decode_attention_args& a, void* at) {
  p.ws = static_cast<float*>(at);
  p.ml = reinterpret_cast<float2*>(p.ws + a.batch * a.num_heads * static_cast<int64_t>(p.slots) * a.head_dim);
}

template <typename T, int D, int MODE>
int launch_combine_partials(const nib_decode_attention_args& a, const MmaDecodeParams& p, cudaStream_t st) {
  static_assert(kCombineBatch * kCombineWarps <= 32, "a batch's weights lie in one warp");
  const int64_t rows = a.batch * a.num_heads;
  // one warp a row once that gives every SM 16 warps; it stores pairs, for which `out` has to be 4-byte
  // aligned with even strides (the other form stores single elements)
  const bool pairs = reinterpret_cast<uintptr_t>(a.out) % 4 == 0 && a.out_batch_stride % 2 == 0 && a.out_head_stride % 2 == 0;
  if (pairs && rows >= 16LL * sm_count()) {
    const unsigned grid = static_cast<unsigned>((rows + kCombineWarps - 1) / kCombineWarps);
    launch_k_after(combine_partials_kernel<T, D, MODE, 1>, grid, kCombineWarps * 32, 0, st, p);
  } else {
    launch_k_after(combine_partials_kernel<T, D, MODE, kCombineWarps>, static_cast<unsigned>(rows), kCombineWarps * 32, 0, st, p);
  }
  return launch_status("decode_attention (combine)");
}

// ------------------------------------------------------------------ host side

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_tiled() {
  static std::once_flag once;
  static EncodeTiledFn fn = nullptr;
  std::call_once(once, [] {
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault) == cudaSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(f);
  });
  return fn;
}

// whether the tensor-core kernels take this call
bool decode_mma_eligible(const nib_decode_attention_args& a);
// the checks of decode attention's arguments: null, or what is wrong
const char* decode_check(const nib_decode_attention_args* a);
size_t decode_mma_smem(int head_dim);

// boxes of `tokens` consecutive slots of a block x one 64-element half of a head
inline int make_cache_map(CUtensorMap* map, const nib_decode_attention_args& a, const void* cache,
                          int tokens = kMmaTile) {
  const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(a.head_dim / 64), static_cast<cuuint64_t>(a.num_kv_heads),
                              static_cast<cuuint64_t>(a.block_size), static_cast<cuuint64_t>(a.num_blocks)};
  const cuuint64_t strides[4] = {128, static_cast<cuuint64_t>(a.cache_head_stride * 2),
                                 static_cast<cuuint64_t>(a.cache_slot_stride * 2),
                                 static_cast<cuuint64_t>(a.cache_block_stride * 2)};
  const cuuint32_t box[5] = {64, 1, 1, static_cast<cuuint32_t>(tokens), 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUtensorMapDataType dt =
      a.dtype == NIB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = encode_tiled()(map, dt, 5, const_cast<void*>(cache), dims, strides, box, estr,
                                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("decode_attention: cuTensorMapEncodeTiled failed (%d)", static_cast<int>(r));
    return NIB_ERR_CUDA;
  }
  return NIB_OK;
}

// The parameters that every token source shares.
inline MmaDecodeParams mma_params(const nib_decode_attention_args& a, int splits) {
  MmaDecodeParams p{};
  p.q = a.q;
  p.q_bs = a.q_batch_stride;
  p.q_hs = a.q_head_stride;
  p.tables = a.block_tables;
  p.table_stride = a.block_table_stride;
  p.cap = a.max_blocks_per_seq * a.block_size;
  p.num_blocks = a.num_blocks;
  p.block_size = static_cast<int>(a.block_size);
  p.lens = a.context_lens;
  p.qscale = a.scale * 1.4426950408889634f;
  p.out = a.out;
  p.o_bs = a.out_batch_stride;
  p.o_hs = a.out_head_stride;
  p.num_heads = a.num_heads;
  p.num_kv_heads = a.num_kv_heads;
  p.group = a.num_heads / a.num_kv_heads;
  p.splits = splits;
  p.slots = splits;
  p.batch = a.batch;
  p.status = a.status;
  return p;
}

// The kernel over `row_blocks` (request, kv head) pairs and p.splits splits; kDecodeShared: over
// `row_blocks` CTAs.
// `after`: behind the kernel before it as a programmatic dependent.
template <typename T, int D, int MODE>
int launch_mma_mode(const nib_decode_attention_args& a, const MmaDecodeParams& p, int64_t row_blocks, cudaStream_t st,
                    bool after = false) {
  CUtensorMap kmap, vmap;
  int rc = make_cache_map(&kmap, a, a.key_cache);
  if (rc != NIB_OK) return rc;
  rc = make_cache_map(&vmap, a, a.value_cache);
  if (rc != NIB_OK) return rc;
  const size_t smem = decode_mma_smem(D);
  auto kernel = decode_attention_mma_kernel<T, D, MODE>;
  static int configured[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && configured[dev] < static_cast<int>(smem)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) {
      set_error("decode_attention: cannot reserve shared memory: %s", cudaGetErrorString(e));
      return NIB_ERR_CUDA;
    }
    configured[dev] = static_cast<int>(smem);
  }
  const dim3 grid(static_cast<unsigned>(row_blocks), MODE == kDecodeShared ? 1u : static_cast<unsigned>(p.splits));
  launch_k_pdl(after || pdl_enabled(), kernel, grid, kMmaWarps * 32, smem, st, kmap, vmap, p);
  return launch_status("decode_attention (tensor cores)");
}

// Calls f(type tag, integral_constant<int, D>) for the call's dtype and head size.
#define NIB_MMA_CASE(a, T_, D_, ...)                                                   \
  [&]() -> int {                                                                       \
    if ((a).dtype == NIB_BF16) {                                                       \
      using T_ = __nv_bfloat16;                                                        \
      if ((a).head_dim == 64) { constexpr int D_ = 64; return __VA_ARGS__; }           \
      constexpr int D_ = 128;                                                          \
      return __VA_ARGS__;                                                              \
    }                                                                                  \
    using T_ = __half;                                                                 \
    if ((a).head_dim == 64) { constexpr int D_ = 64; return __VA_ARGS__; }             \
    constexpr int D_ = 128;                                                            \
    return __VA_ARGS__;                                                                \
  }()

}  // namespace nib
