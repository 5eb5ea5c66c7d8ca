// The default kernel of nib_decode_attention: decode_mma.cuh's over every token of a context.
#include "decode_mma.cuh"

namespace nib {

// whether the tensor-core kernel takes this call
bool decode_mma_eligible(const nib_decode_attention_args& a) {
  if (a.dtype != NIB_BF16 && a.dtype != NIB_F16) return false;
  if (a.head_dim != 64 && a.head_dim != 128) return false;
  if (a.num_heads / a.num_kv_heads > 16) return false;
  if (a.block_size % kMmaTile != 0 || a.block_size > 256 * 16) return false;
  const int64_t es = 2;
  // tensor-map rules: 16-byte aligned base and strides, extents below 2^32
  if (!aligned16(a.key_cache) || !aligned16(a.value_cache)) return false;
  for (int64_t s : {a.cache_block_stride, a.cache_slot_stride, a.cache_head_stride})
    if ((s * es) % 16 != 0 || s * es >= (int64_t{1} << 40)) return false;
  if (a.num_blocks >= (int64_t{1} << 31) || a.num_blocks < 1) return false;
  return encode_tiled() != nullptr;
}

size_t decode_mma_smem(int head_dim) {
  return static_cast<size_t>(kMmaWarps) * kMmaStages * 2 * kMmaTile * head_dim * 2 + 1024;
}

int launch_decode_mma(const nib_decode_attention_args& a, int splits, cudaStream_t st) {
  MmaDecodeParams p = mma_params(a, splits);
  p.ws = splits > 1 ? static_cast<float*>(a.workspace) : nullptr;
  return NIB_MMA_CASE(a, T, D, launch_mma_mode<T, D, kDecodeFull>(a, p, a.batch * a.num_kv_heads, st));
}

}  // namespace nib
