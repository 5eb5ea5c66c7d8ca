// Moving the pages (blocks) of a paged cache: copying given pages, forking sequences, releasing
// them, compacting the live pages to the front.
//
// A cache is `planes` arrays of num_blocks pages (K and V of each layer: the runner allocates
// [2, layers, blocks, block_size, kv_heads, head_dim]); block b of plane p lies at
// p * plane_stride + b * block_bytes. A block table row names a sequence's pages in order, -1
// behind its last; ref_counts[b] says how many rows name page b, 0: free.
//
// Index work is a few kilobytes and one CTA (plan_*); the bytes are moved by a grid of a
// fixed size in units of (page, plane, 32 KB piece) with 16-byte vectors, eight in flight per thread.
// Both run behind one another on the stream without a look from the host: how many pages move
// stays on the device.
#include "copy_rows.cuh"

namespace nib {

constexpr int kMoveThreads = 256;
constexpr int kMoveVecs = 8;  // vectors of a thread and unit
constexpr int kPlanThreads = 1024;

struct PageMove {
  char* cache;
  int64_t planes, plane_stride, num_blocks, block_bytes, slot_bytes;
  const int32_t* src;    // pairs: page src[i] to page dst[i]
  const int32_t* dst;
  const int32_t* slots;  // how many slots of the page (null: all)
  const int32_t* count;  // how many pairs (null: max_pairs)
  int64_t max_pairs;
  unsigned int* status;
};

// Whether pair i of a caller's list may be copied, by the whole CTA: both pages exist, and its
// destination is no other pair's source or destination - else the result would depend on
// which copy runs first.
__device__ __forceinline__ bool pair_allowed(const PageMove& m, int64_t i) {
  const int s = __ldg(m.src + i), d = __ldg(m.dst + i);
  if (s < 0 || d < 0 || s >= m.num_blocks || d >= m.num_blocks || s == d) {
    const bool padding = s == -1 || d == -1 || (s == d && s >= 0 && s < m.num_blocks);
    if (!padding && threadIdx.x == 0) flag(m.status, NIB_DEV_BAD_BLOCK);
    return false;  // the same for the whole CTA
  }
  bool clash = false;
  for (int64_t j = threadIdx.x; j < m.max_pairs; j += kMoveThreads)
    if (j != i && (__ldg(m.dst + j) == d ? __ldg(m.src + j) != -1 : __ldg(m.src + j) == d && __ldg(m.dst + j) != -1)) clash = true;
  if (!__syncthreads_or(clash)) return true;
  if (threadIdx.x == 0) flag(m.status, NIB_DEV_BAD_INDEX);
  return false;
}

// bytes [at, at + kMoveThreads * kMoveVecs * VW) of a page, as far as `bytes`
template <int VW>
__device__ __forceinline__ void move_piece(char* dst, const char* src, int64_t at, int64_t bytes) {
  using V = typename VecOf<VW>::type;
  V buf[kMoveVecs];
#pragma unroll
  for (int k = 0; k < kMoveVecs; ++k) {
    const int64_t o = at + (k * kMoveThreads + threadIdx.x) * static_cast<int64_t>(VW);
    if (o < bytes) buf[k] = *reinterpret_cast<const V*>(src + o);
  }
#pragma unroll
  for (int k = 0; k < kMoveVecs; ++k) {
    const int64_t o = at + (k * kMoveThreads + threadIdx.x) * static_cast<int64_t>(VW);
    if (o < bytes) *reinterpret_cast<V*>(dst + o) = buf[k];
  }
}

template <int VW>
__device__ __forceinline__ void move_unit(const PageMove& m, int64_t i, int64_t plane, int64_t piece) {
  const int s = __ldg(m.src + i), d = __ldg(m.dst + i);
  if (s < 0 || d < 0) return;
  const int64_t bytes = m.slots ? __ldg(m.slots + i) * m.slot_bytes : m.block_bytes;
  char* base = m.cache + plane * m.plane_stride;
  move_piece<VW>(base + d * m.block_bytes, base + s * m.block_bytes, piece * (kMoveThreads * kMoveVecs * VW), bytes);
}

// A caller's pairs: each CTA takes consecutive units, so that it looks at few pairs.
template <int VW>
__global__ void __launch_bounds__(kMoveThreads)
copy_pages_kernel(const PageMove m) {
  pdl_enter();
  constexpr int64_t kPiece = kMoveThreads * kMoveVecs * VW;
  const int64_t pieces = (m.block_bytes + kPiece - 1) / kPiece;
  const int64_t per_pair = m.planes * pieces, units = m.max_pairs * per_pair;
  const int64_t from = units * blockIdx.x / gridDim.x, to = units * (blockIdx.x + 1) / gridDim.x;
  int64_t u = from;
  while (u < to) {
    const int64_t i = u / per_pair;
    const int64_t stop = (i + 1) * per_pair < to ? (i + 1) * per_pair : to;
    if (pair_allowed(m, i))
      for (; u < stop; ++u) move_unit<VW>(m, i, u % per_pair / pieces, u % pieces);
    u = stop;
  }
}

template <int VW>
__device__ __forceinline__ void move_all(const PageMove& m) {
  constexpr int64_t kPiece = kMoveThreads * kMoveVecs * VW;
  const int64_t pieces = (m.block_bytes + kPiece - 1) / kPiece;
  const int64_t per_pair = m.planes * pieces;
  const int64_t units = (m.count ? static_cast<int64_t>(__ldg(m.count)) : m.max_pairs) * per_pair;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) move_unit<VW>(m, u / per_pair, u % per_pair / pieces, u % pieces);
}

// ------------------------------------------------------------------ block-wide sums

// exclusive prefix sum over the CTA's kPlanThreads values; `total` is the sum of all
__device__ __forceinline__ int scan_exclusive(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int upto = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= off) upto += x;
  }
  __syncthreads();  // the sums of the call before have been read
  if (lane == 31) warp_sums[w] = upto;
  __syncthreads();
  if (w == 0) {
    int s = warp_sums[lane];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, off);
      if (lane >= off) s += x;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  total = warp_sums[kPlanThreads / 32 - 1];
  return (w > 0 ? warp_sums[w - 1] : 0) + upto - v;
}

// ------------------------------------------------------------------ fork

struct ForkParams {
  const int32_t* tables;
  int64_t table_stride, rows, width, block_size;
  const int32_t* lens;
  const int32_t* refs;
  int64_t num_blocks;
  const int32_t* parents;
  const int32_t* children;
  int64_t n;
  int32_t* tables_out;  // [rows, width]
  int32_t* lens_out;
  int32_t* refs_out;
  int32_t* copies;   // [3, n]: source page, fresh page, slots; -1, -1, 0: nothing is copied
  int32_t* granted;  // [n] 1: the fork takes place
  int32_t* winner;   // [rows] scratch: the first fork of a child row
  int32_t* fresh;    // [n] scratch: the free pages in ascending order
  unsigned int* status;
};

// CTA 0 decides which forks take place and which pages they get; the others copy the tables,
// lengths and counts, which the next kernel then amends.
__global__ void __launch_bounds__(kPlanThreads)
fork_plan_kernel(const ForkParams p) {
  pdl_enter();
  const int tid = threadIdx.x;
  if (blockIdx.x > 0) {
    const int64_t step = static_cast<int64_t>(gridDim.x - 1) * kPlanThreads;
    const int64_t i0 = (blockIdx.x - 1) * static_cast<int64_t>(kPlanThreads) + tid;
    for (int64_t i = i0; i < p.rows * p.width; i += step) p.tables_out[i] = __ldg(p.tables + i / p.width * p.table_stride + i % p.width);
    for (int64_t i = i0; i < p.rows; i += step) p.lens_out[i] = __ldg(p.lens + i);
    for (int64_t i = i0; i < p.num_blocks; i += step) p.refs_out[i] = __ldg(p.refs + i);
    return;
  }
  __shared__ int sums[32];
  for (int64_t i = tid; i < p.rows; i += kPlanThreads) p.winner[i] = 0x7fffffff;
  __syncthreads();
  for (int64_t i = tid; i < p.n; i += kPlanThreads) {
    const int c = __ldg(p.children + i);
    if (c >= 0 && c < p.rows && __ldg(p.parents + i) != -1) atomicMin(p.winner + c, static_cast<int>(i));
  }
  __syncthreads();
  int needed = 0;  // forks of earlier passes that need a page
  for (int64_t i0 = 0; i0 < p.n; i0 += kPlanThreads) {
    const int64_t i = i0 + tid;
    bool ok = false, part = false;
    if (i < p.n) {
      const int a = __ldg(p.parents + i), c = __ldg(p.children + i);
      const bool padding = a == -1 || c == -1;
      ok = a >= 0 && a < p.rows && c >= 0 && c < p.rows;
      if (ok) {
        const int len = __ldg(p.lens + a);
        ok = len >= 0 && len <= p.width * p.block_size && __ldg(p.lens + c) == 0 && __ldcg(p.winner + c) == i;
        part = ok && len % p.block_size != 0;
        if (part) {
          const int last = __ldg(p.tables + a * p.table_stride + len / p.block_size);
          if (last < 0 || last >= p.num_blocks) {
            flag(p.status, NIB_DEV_BAD_BLOCK);
            ok = part = false;
          } else {
            p.copies[i] = last;
            p.copies[2 * p.n + i] = static_cast<int>(len % p.block_size);
          }
        } else if (!ok) {
          flag(p.status, NIB_DEV_BAD_INDEX);
        }
      } else if (!padding) {
        flag(p.status, NIB_DEV_BAD_INDEX);
      }
      if (!part) {
        p.copies[i] = -1;
        p.copies[2 * p.n + i] = 0;
      }
    }
    int total;
    const int before = scan_exclusive(part ? 1 : 0, sums, total);
    if (i < p.n) {
      p.granted[i] = ok ? 1 : 0;
      p.copies[p.n + i] = part ? needed + before : -1;  // the rank of its page, for now
    }
    needed += total;
  }
  // the first `needed` free pages: each thread counts its share of them, then writes them down
  const int64_t share = (p.num_blocks + kPlanThreads - 1) / kPlanThreads;
  const int64_t b0 = tid * share, b1 = b0 + share < p.num_blocks ? b0 + share : p.num_blocks;
  int mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += __ldg(p.refs + b) == 0 ? 1 : 0;
  int free_pages;
  int at = scan_exclusive(mine, sums, free_pages);
  for (int64_t b = b0; b < b1 && at < needed; ++b)
    if (__ldg(p.refs + b) == 0) p.fresh[at++] = static_cast<int>(b);
  __syncthreads();
  for (int64_t i = tid; i < p.n; i += kPlanThreads) {
    const int rank = p.copies[p.n + i];
    if (rank < 0) continue;
    if (rank < free_pages) {
      p.copies[p.n + i] = __ldcg(p.fresh + rank);
    } else {
      flag(p.status, NIB_DEV_NO_PAGE);
      p.copies[i] = p.copies[p.n + i] = -1;
      p.copies[2 * p.n + i] = 0;
      p.granted[i] = 0;
    }
  }
}

template <int VW>
__global__ void __launch_bounds__(kMoveThreads)
fork_apply_kernel(const ForkParams p, const PageMove m) {
  pdl_enter();
  for (int64_t i = blockIdx.x; i < p.n; i += gridDim.x) {
    if (!__ldg(p.granted + i)) continue;
    const int a = __ldg(p.parents + i), c = __ldg(p.children + i);
    const int len = __ldg(p.lens + a);
    const int64_t full = len / p.block_size;
    for (int64_t j = threadIdx.x; j < p.width; j += kMoveThreads) {
      int page = -1;
      if (j < full) {
        page = __ldg(p.tables + a * p.table_stride + j);
        if (page >= 0 && page < p.num_blocks) atomicAdd(p.refs_out + page, 1);
        else flag(p.status, NIB_DEV_BAD_BLOCK);
      } else if (j == full) {
        page = __ldg(p.copies + p.n + i);
        if (page >= 0) atomicAdd(p.refs_out + page, 1);
      }
      p.tables_out[c * p.width + j] = page;
    }
    if (threadIdx.x == 0) p.lens_out[c] = len;
  }
  move_all<VW>(m);
}

// ------------------------------------------------------------------ release

struct FreeParams {
  const int32_t* tables;
  int64_t table_stride, rows, width, block_size;
  const int32_t* lens;
  const int32_t* refs;
  int64_t num_blocks;
  const int32_t* list;
  int64_t n;
  int32_t* tables_out;
  int32_t* lens_out;
  int32_t* refs_out;
  unsigned int* status;
};

// whether row r is in the list, by the whole CTA
__device__ __forceinline__ bool listed(const FreeParams& p, int64_t r) {
  bool in = false;
  for (int64_t i = threadIdx.x; i < p.n; i += blockDim.x) in |= __ldg(p.list + i) == r;
  return __syncthreads_or(in) != 0;
}

__global__ void __launch_bounds__(kMoveThreads)
free_rows_kernel(const FreeParams p) {
  pdl_enter();
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const bool gone = listed(p, r);
    for (int64_t j = threadIdx.x; j < p.width; j += kMoveThreads)
      p.tables_out[r * p.width + j] = gone ? -1 : __ldg(p.tables + r * p.table_stride + j);
    if (threadIdx.x == 0) p.lens_out[r] = gone ? 0 : __ldg(p.lens + r);
  }
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x, step = static_cast<int64_t>(gridDim.x) * kMoveThreads;
  for (int64_t i = i0; i < p.num_blocks; i += step) p.refs_out[i] = __ldg(p.refs + i);
  for (int64_t i = i0; i < p.n; i += step) {
    const int r = __ldg(p.list + i);
    if (r != -1 && (r < 0 || r >= p.rows)) flag(p.status, NIB_DEV_BAD_INDEX);
  }
}

// Each released row gives its pages back; a row that the list names twice does so once. A count
// stays at 0: a decrement that finds nothing left is undone and reported.
__global__ void __launch_bounds__(kMoveThreads)
free_pages_kernel(const FreeParams p) {
  pdl_enter();
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    if (!listed(p, r)) continue;
    int64_t len = __ldg(p.lens + r);
    if (len < 0 || len > p.width * p.block_size) {
      if (threadIdx.x == 0) flag(p.status, NIB_DEV_BAD_INDEX);
      len = len < 0 ? 0 : p.width * p.block_size;
    }
    const int64_t held = (len + p.block_size - 1) / p.block_size;
    for (int64_t j = threadIdx.x; j < held; j += kMoveThreads) {
      const int page = __ldg(p.tables + r * p.table_stride + j);
      if (page < 0 || page >= p.num_blocks) {
        flag(p.status, NIB_DEV_BAD_BLOCK);
      } else if (atomicSub(p.refs_out + page, 1) <= 0) {
        atomicAdd(p.refs_out + page, 1);
        flag(p.status, NIB_DEV_BAD_INDEX);
      }
    }
  }
}

// ------------------------------------------------------------------ compact

struct CompactParams {
  const int32_t* tables;
  int64_t table_stride, rows, width;
  const int32_t* refs;
  int64_t num_blocks;
  int32_t* tables_out;
  int32_t* refs_out;
  int32_t* live;   // [1]
  int32_t* moves;  // [2, max_moves]: source, destination; -1 behind the last
  int64_t max_moves;
  int32_t* count;  // [1] how many
  int32_t* remap;  // [num_blocks] where a page's contents are now
  unsigned int* status;
};

// One CTA: L = live pages; the i-th live page behind place L goes to the i-th free place before it.
__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(const CompactParams p) {
  pdl_enter();
  __shared__ int sums[32];
  const int tid = threadIdx.x;
  const int64_t share = (p.num_blocks + kPlanThreads - 1) / kPlanThreads;
  const int64_t b0 = tid * share, b1 = b0 + share < p.num_blocks ? b0 + share : p.num_blocks;
  int mine = 0;
  for (int64_t b = b0; b < b1; ++b) mine += __ldg(p.refs + b) > 0 ? 1 : 0;
  int live;
  scan_exclusive(mine, sums, live);
  int holes = 0, far = 0;
  for (int64_t b = b0; b < b1; ++b) {
    const bool used = __ldg(p.refs + b) > 0;
    holes += !used && b < live ? 1 : 0;
    far += used && b >= live ? 1 : 0;
  }
  int moves, same;
  int at_hole = scan_exclusive(holes, sums, same);
  int at_far = scan_exclusive(far, sums, moves);  // as many as holes
  for (int64_t b = b0; b < b1; ++b) {
    const int r = __ldg(p.refs + b);
    if (r <= 0 && b < live) p.moves[p.max_moves + at_hole++] = static_cast<int>(b);
    else if (r > 0 && b >= live) p.moves[at_far++] = static_cast<int>(b);
    p.remap[b] = static_cast<int>(b);
    p.refs_out[b] = r;
  }
  for (int64_t i = moves + tid; i < p.max_moves; i += kPlanThreads) p.moves[i] = p.moves[p.max_moves + i] = -1;
  if (tid == 0) {
    p.live[0] = live;
    p.count[0] = moves;
  }
  __syncthreads();
  for (int64_t i = tid; i < moves; i += kPlanThreads) {
    const int s = __ldcg(p.moves + i), d = __ldcg(p.moves + p.max_moves + i);
    p.remap[s] = d;
    p.refs_out[d] = __ldg(p.refs + s);
    p.refs_out[s] = 0;
  }
}

template <int VW>
__global__ void __launch_bounds__(kMoveThreads)
compact_apply_kernel(const CompactParams p, const PageMove m) {
  pdl_enter();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMoveThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kMoveThreads + threadIdx.x; i < p.rows * p.width; i += step) {
    int page = __ldg(p.tables + i / p.width * p.table_stride + i % p.width);
    if (page >= 0 && page < p.num_blocks) page = __ldg(p.remap + page);
    else if (page != -1) flag(p.status, NIB_DEV_BAD_BLOCK);
    p.tables_out[i] = page;
  }
  move_all<VW>(m);
}

// ------------------------------------------------------------------ host side

static int page_move(PageMove& m, int& vw, void* cache, int64_t planes, int64_t plane_stride, int64_t num_blocks,
                     int64_t block_bytes, int64_t slot_bytes, unsigned int* status) {
  NIB_REQUIRE(planes >= 0 && num_blocks >= 0 && block_bytes >= 2 && plane_stride >= 0, "paged pages: bad cache sizes");
  NIB_REQUIRE(num_blocks < (int64_t{1} << 31), "paged pages: 2^31 blocks or more");
  NIB_REQUIRE(planes <= 1 || plane_stride >= num_blocks * block_bytes, "paged pages: planes overlap");
  NIB_SUPPORT(block_bytes % 2 == 0 && slot_bytes % 2 == 0 && plane_stride % 2 == 0 && (reinterpret_cast<uintptr_t>(cache) & 1) == 0,
              "paged pages: sizes and addresses must be even");
  m.cache = static_cast<char*>(cache);
  m.planes = planes;
  m.plane_stride = plane_stride;
  m.num_blocks = num_blocks;
  m.block_bytes = block_bytes;
  m.slot_bytes = slot_bytes;
  m.status = status;
  vw = pick_vec_width({reinterpret_cast<uint64_t>(cache), static_cast<uint64_t>(plane_stride),
                       static_cast<uint64_t>(block_bytes), static_cast<uint64_t>(slot_bytes)});
  return NIB_OK;
}

// Eight CTAs per SM at most: the movers' 64 to 80 registers (16-byte vectors) let three or four of them run
// at once, the others follow as SMs become free.
static unsigned move_grid(const PageMove& m, int vw, int64_t pairs, int64_t at_least) {
  const int64_t piece = static_cast<int64_t>(kMoveThreads) * kMoveVecs * vw;
  int64_t units = pairs * m.planes * ((m.block_bytes + piece - 1) / piece);
  if (units < at_least) units = at_least;
  const int64_t most = 8LL * sm_count();
  return static_cast<unsigned>(units < 1 ? 1 : units > most ? most : units);
}

}  // namespace nib

using namespace nib;

extern "C" int nib_paged_copy_blocks(void* cache, int64_t planes, int64_t plane_stride_bytes, int64_t num_blocks,
                                     int64_t block_bytes, const int32_t* src_blocks, const int32_t* dst_blocks,
                                     int64_t n, unsigned int* status, void* stream) {
  PageMove m{};
  int vw = 16;
  NIB_REQUIRE(n >= 0, "paged_copy_blocks: negative pair count");
  const int rc = page_move(m, vw, cache, planes, plane_stride_bytes, num_blocks, block_bytes, 16, status);
  if (rc != NIB_OK) return rc;
  if (n == 0 || planes == 0) return NIB_OK;
  NIB_REQUIRE(cache && src_blocks && dst_blocks, "paged_copy_blocks: null pointer");
  NIB_SUPPORT(n <= 65536, "paged_copy_blocks: at most 65536 pairs per call");
  m.src = src_blocks;
  m.dst = dst_blocks;
  m.max_pairs = n;
  const unsigned grid = move_grid(m, vw, n, 1);
  NIB_VW_SWITCH(vw, VW, launch_k(copy_pages_kernel<VW>, grid, kMoveThreads, 0, as_stream(stream), m));
  return launch_status("paged_copy_blocks");
}

extern "C" int64_t nib_paged_fork_workspace_bytes(int64_t rows, int64_t n) { return rows < 0 || n < 0 ? -1 : 4 * (rows + 2 * n); }

extern "C" int nib_paged_fork(void* cache, int64_t planes, int64_t plane_stride_bytes, int64_t num_blocks,
                              int64_t block_bytes, int64_t block_size, const int32_t* block_tables,
                              int64_t table_stride, int64_t rows, int64_t max_blocks_per_seq,
                              const int32_t* context_lens, const int32_t* ref_counts, const int32_t* parents,
                              const int32_t* children, int64_t n, int32_t* tables_out, int32_t* lens_out,
                              int32_t* refs_out, int32_t* copies, void* workspace, int64_t workspace_bytes,
                              unsigned int* status, void* stream) {
  PageMove m{};
  int vw = 16;
  NIB_REQUIRE(n >= 0 && rows >= 0 && max_blocks_per_seq >= 0 && block_size >= 1, "paged_fork: bad sizes");
  NIB_REQUIRE(block_bytes % block_size == 0, "paged_fork: a block is not whole slots");
  const int rc = page_move(m, vw, cache, planes, plane_stride_bytes, num_blocks, block_bytes, block_bytes / block_size, status);
  if (rc != NIB_OK) return rc;
  NIB_REQUIRE(rows == 0 || (context_lens && lens_out), "paged_fork: null pointer");
  NIB_REQUIRE(rows * max_blocks_per_seq == 0 || (block_tables && tables_out), "paged_fork: null pointer");
  NIB_REQUIRE(num_blocks == 0 || (cache && ref_counts && refs_out), "paged_fork: null pointer");
  NIB_REQUIRE(n == 0 || (parents && children && copies), "paged_fork: null pointer");
  NIB_REQUIRE(max_blocks_per_seq * block_size < (int64_t{1} << 31) && rows < (int64_t{1} << 31) && n < (int64_t{1} << 31),
              "paged_fork: sizes of 2^31 or more");
  const int64_t need = nib_paged_fork_workspace_bytes(rows, n);
  NIB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "paged_fork: workspace of %lld bytes needed",
              static_cast<long long>(need));
  ForkParams p{};
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.rows = rows;
  p.width = max_blocks_per_seq;
  p.block_size = block_size;
  p.lens = context_lens;
  p.refs = ref_counts;
  p.num_blocks = num_blocks;
  p.parents = parents;
  p.children = children;
  p.n = n;
  p.tables_out = tables_out;
  p.lens_out = lens_out;
  p.refs_out = refs_out;
  p.copies = copies;
  p.granted = static_cast<int32_t*>(workspace);
  p.fresh = p.granted + n;
  p.winner = p.fresh + n;
  p.status = status;
  int64_t most = rows * max_blocks_per_seq;
  if (most < num_blocks) most = num_blocks;
  if (most < rows) most = rows;
  const int64_t copiers = (most + kPlanThreads - 1) / kPlanThreads, sms = sm_count();
  const cudaStream_t st = as_stream(stream);
  launch_k(fork_plan_kernel, static_cast<unsigned>(1 + (copiers < 1 ? 1 : copiers > 2 * sms ? 2 * sms : copiers)), kPlanThreads, 0, st, p);
  if (n > 0) {
    m.src = copies;
    m.dst = copies + n;
    m.slots = copies + 2 * n;
    m.max_pairs = n;
    const unsigned grid = move_grid(m, vw, n, n);
    NIB_VW_SWITCH(vw, VW, launch_k_after(fork_apply_kernel<VW>, grid, kMoveThreads, 0, st, p, m));
  }
  return launch_status("paged_fork");
}

extern "C" int nib_paged_free(const int32_t* block_tables, int64_t table_stride, int64_t rows,
                              int64_t max_blocks_per_seq, int64_t block_size, const int32_t* context_lens,
                              const int32_t* ref_counts, int64_t num_blocks, const int32_t* free_rows, int64_t n,
                              int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, unsigned int* status,
                              void* stream) {
  NIB_REQUIRE(n >= 0 && rows >= 0 && max_blocks_per_seq >= 0 && block_size >= 1 && num_blocks >= 0, "paged_free: bad sizes");
  NIB_REQUIRE(rows == 0 || (context_lens && lens_out), "paged_free: null pointer");
  NIB_REQUIRE(rows * max_blocks_per_seq == 0 || (block_tables && tables_out), "paged_free: null pointer");
  NIB_REQUIRE(num_blocks == 0 || (ref_counts && refs_out), "paged_free: null pointer");
  NIB_REQUIRE(n == 0 || free_rows, "paged_free: null pointer");
  NIB_REQUIRE(max_blocks_per_seq * block_size < (int64_t{1} << 31) && num_blocks < (int64_t{1} << 31),
              "paged_free: sizes of 2^31 or more");
  FreeParams p{};
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.rows = rows;
  p.width = max_blocks_per_seq;
  p.block_size = block_size;
  p.lens = context_lens;
  p.refs = ref_counts;
  p.num_blocks = num_blocks;
  p.list = free_rows;
  p.n = n;
  p.tables_out = tables_out;
  p.lens_out = lens_out;
  p.refs_out = refs_out;
  p.status = status;
  const int64_t by_pages = (num_blocks + kMoveThreads - 1) / kMoveThreads, sms = sm_count();
  int64_t ctas = rows > by_pages ? rows : by_pages;
  ctas = ctas < 1 ? 1 : ctas > 8 * sms ? 8 * sms : ctas;
  const cudaStream_t st = as_stream(stream);
  launch_k(free_rows_kernel, static_cast<unsigned>(ctas), kMoveThreads, 0, st, p);
  if (n > 0 && rows > 0) {
    const int64_t row_ctas = rows > 8 * sms ? 8 * sms : rows;
    launch_k_after(free_pages_kernel, static_cast<unsigned>(row_ctas), kMoveThreads, 0, st, p);
  }
  return launch_status("paged_free");
}

extern "C" int64_t nib_paged_compact_workspace_bytes(int64_t num_blocks) { return num_blocks < 0 ? -1 : 4 * (num_blocks + 1); }

extern "C" int nib_paged_compact(void* cache, int64_t planes, int64_t plane_stride_bytes, int64_t num_blocks,
                                 int64_t block_bytes, const int32_t* block_tables, int64_t table_stride, int64_t rows,
                                 int64_t max_blocks_per_seq, const int32_t* ref_counts, int32_t* tables_out,
                                 int32_t* refs_out, int32_t* live, int32_t* moves, void* workspace,
                                 int64_t workspace_bytes, unsigned int* status, void* stream) {
  PageMove m{};
  int vw = 16;
  NIB_REQUIRE(rows >= 0 && max_blocks_per_seq >= 0, "paged_compact: bad sizes");
  const int rc = page_move(m, vw, cache, planes, plane_stride_bytes, num_blocks, block_bytes, 16, status);
  if (rc != NIB_OK) return rc;
  NIB_REQUIRE(rows * max_blocks_per_seq == 0 || (block_tables && tables_out), "paged_compact: null pointer");
  NIB_REQUIRE(live && (num_blocks == 0 || (cache && ref_counts && refs_out)) && (num_blocks < 2 || moves),
              "paged_compact: null pointer");
  const int64_t need = nib_paged_compact_workspace_bytes(num_blocks);
  NIB_REQUIRE(workspace && workspace_bytes >= need, "paged_compact: workspace of %lld bytes needed", static_cast<long long>(need));
  CompactParams p{};
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.rows = rows;
  p.width = max_blocks_per_seq;
  p.refs = ref_counts;
  p.num_blocks = num_blocks;
  p.tables_out = tables_out;
  p.refs_out = refs_out;
  p.live = live;
  p.moves = moves;
  p.max_moves = num_blocks / 2;
  p.count = static_cast<int32_t*>(workspace);
  p.remap = p.count + 1;
  p.status = status;
  m.src = moves;
  m.dst = moves + p.max_moves;
  m.count = p.count;
  const cudaStream_t st = as_stream(stream);
  launch_k(compact_plan_kernel, 1, kPlanThreads, 0, st, p);
  const int64_t table_ctas = (rows * max_blocks_per_seq + kMoveThreads - 1) / kMoveThreads;
  const unsigned grid = move_grid(m, vw, p.max_moves, table_ctas);
  NIB_VW_SWITCH(vw, VW, launch_k_after(compact_apply_kernel<VW>, grid, kMoveThreads, 0, st, p, m));
  return launch_status("paged_compact");
}
