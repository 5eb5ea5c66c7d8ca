// Decode attention of a batch whose groups share their first tokens: the shared part is read
// and computed once for a group, not once for each of its requests.
//
// For a group of n requests whose first P tokens are the same, softmax(q K^T) V splits over
// the token axis: over [0, P) every (request, head) of a kv head is a row of one product
// against the same K and V; over [P, len) each request has tokens of its own. Both halves
// leave partials (max, sum, unnormalised output) that the combine kernel joins.
//
// With few rows: one launch over the prefixes' row tiles (x kv heads x splits) and the suffixes
// (requests x kv heads x splits), and the combine. With many: the prefixes by shared_prefix_tc.cu, the
// suffixes, the combine. There the suffix kernel reads nothing of the prefix kernel's: it starts as
// soon as every CTA of that one has, on SMs that are free and as SMs become free, and waits for it
// only before its own end, so that the combine follows both.
#include "decode_mma.cuh"

namespace nib {

// the prefix kernel of shared_prefix_tc.cu: rows per CTA, tokens per tile, launch
int64_t prefix_tc_rows();
int64_t prefix_tc_tile();
int launch_prefix_tc(const nib_decode_attention_args& a, const MmaDecodeParams& p, int64_t units, cudaStream_t st);

struct SharedPrefixPlan {
  bool tc;  // the tcgen05 kernel computes the prefixes
  int prefix_splits, suffix_splits;
  int64_t row_tiles;  // an upper bound: every group's last tile may be ragged
};

static SharedPrefixPlan shared_prefix_plan(const nib_shared_prefix_args& s) {
  const nib_decode_attention_args& a = s.attn;
  SharedPrefixPlan pl{};
  const int group = a.num_heads / a.num_kv_heads;
  const int64_t cap = a.max_blocks_per_seq * a.block_size;
  const int64_t max_len = a.max_context_len > 0 && a.max_context_len < cap ? a.max_context_len : cap;
  const int64_t max_prefix = s.max_prefix_len > 0 && s.max_prefix_len < max_len ? s.max_prefix_len : max_len;
  // sum over the groups of ceil(rows / tile) <= (all rows + (tile - 1) groups) / tile
  const int64_t rows = a.batch * group;
  auto row_tiles = [&](int64_t tile) { return (rows + (tile - 1) * s.num_groups) / tile; };
  // The tcgen05 kernel reads a tile for up to 256 rows, the 16-row kernel for 16, but a CTA of the
  // first has an SM to itself and takes microseconds to start and end: it runs with more than 32
  // rows a group and at least 6,144 tokens x row tiles for each (group, kv head), and as many
  // again for two. Measured, us a call, 16-row / tcgen05 kernel (16/2 heads of 128, 40 tokens
  // behind the prefix): one group of 160 rows behind 1,024 tokens 15.0 / 16.1, 320 rows 20.5 / 17.3;
  // 40 rows behind 4,096 tokens 19.0 / 15.7; five groups of 64 rows behind 1,024 tokens 18.3 / 23.9, of
  // 128 rows 23.1 / 21.8; 16/8 heads: one group of 20 rows behind 16,384 tokens 26.4 / 29.1, of 40 rows
  // 34.5 / 30.1.
  pl.tc = a.variant == 2 || (a.variant == 0 && rows > 32 * s.num_groups &&
                             row_tiles(16) * a.num_kv_heads * max_prefix >= 6144 * (s.num_groups * a.num_kv_heads + 2));
  pl.row_tiles = row_tiles(pl.tc ? prefix_tc_rows() : 16);
  // as many splits as fit the SMs' three CTAs each at once, of at least `least` tokens: 64 requests
  // of up to 1,024 tokens behind 8,192 shared ones 57.4 us with 3 CTAs per SM wanted, 63.2 with 12;
  // 93 of up to 333 (fp16, D = 64) 24.7 us with 256 tokens at least, 28.4 with 64
  const int64_t want = 3LL * sm_count();
  auto splits = [&](int64_t ctas, int64_t tokens, int64_t least) -> int {
    int64_t n = ctas < 1 || ctas >= want ? 1 : want / ctas;
    const int64_t by_len = (tokens + least - 1) / least;
    if (n > by_len) n = by_len;
    return static_cast<int>(n < 1 ? 1 : n > 256 ? 256 : n);
  };
  if (pl.tc) {
    // one CTA runs on an SM: the split count with the fewest tile steps over all waves, each
    // CTA's start and end counted as two more
    const int64_t ctas = pl.row_tiles * a.num_kv_heads, tiles = (max_prefix + prefix_tc_tile() - 1) / prefix_tc_tile();
    int64_t best = 0;
    for (int64_t n = 1; n <= tiles && n <= 64; ++n) {
      const int64_t cost = (ctas * n + sm_count() - 1) / sm_count() * ((tiles + n - 1) / n + 2);
      if (best == 0 || cost < best) {
        best = cost;
        pl.prefix_splits = static_cast<int>(n);
      }
    }
    if (pl.prefix_splits < 1) pl.prefix_splits = 1;
  } else {
    pl.prefix_splits = splits(pl.row_tiles * a.num_kv_heads, max_prefix, 64);
  }
  // What a request has to itself is max_len - max_prefix tokens where its group shares the longest prefix,
  // but all of them where it is in no group, shorter than its group's prefix, or its group's is short: a
  // split for each 1,024 of those. How many it uses goes by what it has. us a call, 16/8 heads, with
  // max_len - max_prefix alone -> so: 32,768 tokens in no group 519 -> 32; four requests of 100 + 16,000
  // tokens next to four of 20,000 + 50, 274 -> 71; two of 30,000 + 20, whose added splits are empty, 34.0 ->
  // 33.7. Requests that fill the SMs get one split each, a long one among them too: 32,768 tokens in no
  // group next to 32 requests of 8,192 + 512, 495 us.
  const int64_t own = s.num_groups == 0 ? max_len : max_len - max_prefix, by_own = (own + kOwnTokens - 1) / kOwnTokens;
  const int64_t by_all = (max_len + 1023) / 1024;
  pl.suffix_splits = splits(a.batch * a.num_kv_heads, (by_own > by_all ? by_own : by_all) * kOwnTokens, kOwnTokens);
  return pl;
}

static int64_t shared_prefix_workspace(const nib_shared_prefix_args& s, const SharedPrefixPlan& pl) {
  return partial_bytes(s.attn, pl.prefix_splits + pl.suffix_splits);
}

template <typename T, int D>
static int launch_shared_prefix(const nib_shared_prefix_args& s, const SharedPrefixPlan& pl, cudaStream_t st) {
  const nib_decode_attention_args& a = s.attn;
  MmaDecodeParams p = mma_params(a, pl.prefix_splits);
  p.slots = pl.prefix_splits + pl.suffix_splits;
  place_partials(p, a, a.workspace);
  p.group_offsets = s.group_offsets;
  p.prefix_lens = s.prefix_lens;
  p.num_groups = static_cast<int>(s.num_groups);
  if (s.num_groups > 0 && pl.tc) {
    const int rc = launch_prefix_tc(a, p, pl.row_tiles, st);
    if (rc != NIB_OK) return rc;
  }
  p.prefix_splits = pl.prefix_splits;
  p.splits = pl.suffix_splits;
  p.slot0 = pl.prefix_splits;
  int rc;
  if (s.num_groups > 0 && !pl.tc) {
    p.prefix_ctas = static_cast<int>(pl.row_tiles * a.num_kv_heads * pl.prefix_splits);
    rc = launch_mma_mode<T, D, kDecodeShared>(a, p, p.prefix_ctas + a.batch * a.num_kv_heads * pl.suffix_splits, st);
  } else {
    p.early = s.num_groups > 0;
    rc = launch_mma_mode<T, D, kDecodeSuffix>(a, p, a.batch * a.num_kv_heads, st, p.early);
  }
  if (rc != NIB_OK) return rc;
  return launch_combine_partials<T, D, kDecodeSuffix>(a, p, st);
}

static const char* shared_prefix_check(const nib_shared_prefix_args* s) {
  if (s == nullptr || s->struct_size != static_cast<int32_t>(sizeof(nib_shared_prefix_args)))
    return "shared_prefix_decode_attention: args struct size mismatch";
  const char* bad = decode_check(&s->attn);
  if (bad != nullptr) return bad;
  if (s->attn.variant < 0 || s->attn.variant > 2) return "shared_prefix_decode_attention: bad variant";
  if (s->num_groups < 0 || s->num_groups > (1 << 20)) return "shared_prefix_decode_attention: bad group count";
  return nullptr;
}

}  // namespace nib

using namespace nib;

extern "C" int64_t nib_shared_prefix_workspace_bytes(const nib_shared_prefix_args* s) {
  if (shared_prefix_check(s) != nullptr) return -1;
  return shared_prefix_workspace(*s, shared_prefix_plan(*s));
}

extern "C" int nib_shared_prefix_decode_attention(const nib_shared_prefix_args* s, void* stream) {
  const char* bad = shared_prefix_check(s);
  if (bad != nullptr) {
    set_error("%s", bad);
    return NIB_ERR_INVALID;
  }
  const nib_decode_attention_args& a = s->attn;
  if (a.batch == 0) return NIB_OK;
  NIB_REQUIRE(a.q && a.key_cache && a.value_cache && a.block_tables && a.context_lens && a.out &&
                  (s->num_groups == 0 || (s->group_offsets && s->prefix_lens)),
              "shared_prefix_decode_attention: null pointer");
  const int64_t group = a.num_heads / a.num_kv_heads;
  NIB_REQUIRE((a.batch * group + s->num_groups) * a.num_kv_heads <= (1LL << 24) && a.batch * a.num_heads <= (1LL << 24),
              "shared_prefix_decode_attention: batch too large");
  NIB_REQUIRE(a.max_blocks_per_seq * a.block_size < kMaxTokens,
              "shared_prefix_decode_attention: block table covers too many tokens (2^31 - 4096)");
  NIB_SUPPORT(aligned16(a.q) && a.q_batch_stride % 8 == 0 && a.q_head_stride % 8 == 0,
              "shared_prefix_decode_attention: q must be 16-byte aligned with strides of multiples of 8 elements");
  NIB_SUPPORT(decode_mma_eligible(a), "shared_prefix_decode_attention: needs bf16/f16, head_dim 64 or 128, at most 16 q "
              "heads per kv head, a block size that is a multiple of 16 and 16-byte aligned strides");
  const SharedPrefixPlan pl = shared_prefix_plan(*s);
  const int64_t need = shared_prefix_workspace(*s, pl);
  NIB_REQUIRE(a.workspace && a.workspace_bytes >= need && aligned16(a.workspace),
              "shared_prefix_decode_attention: workspace of %lld bytes needed", static_cast<long long>(need));
  const cudaStream_t st = as_stream(stream);
  return NIB_MMA_CASE(a, T, D, launch_shared_prefix<T, D>(*s, pl, st));
}
