// The paged Q4_0 key/value cache: where a token's blocks lie, and the conversions of the activation
// types that go with it.
//
// A page holds `groups` groups of 16 tokens for each kv head, page-major, then head, then group; a
// group of one head is 18 * D bytes (D = 32 * nb, so 9/16 byte a value, as in a row of block_q4_0):
//   [0, 8D)    key quants     32-bit word (half, g, t, b): bytes 4t..4t+3 of block b of token g + 8 * half
//   [8D, 16D)  value quants   32-bit word (half, g, t, b): bytes 2g, 2g+1 of block b of token 2t + 8 * half
//                             in the low half, the same bytes of the token after it in the high half
//   [16D, 17D) key scales     fp16 (token, b)
//   [17D, 18D) value scales   fp16 (token, b)
// with half < 2, g < 8, t < 4, b < nb, the last index fastest.  A block's 16 quant bytes are those of
// block_q4_0: byte j holds element j low and element j + 16 high, each plus 8.  The order is that of
// the tensor cores' 16 x 16 operand: lane 4g + t reads its nb words of each half as one aligned run,
// lanes side by side, and one AND with 0x000f000f leaves two neighbours of a k step in a register.
#pragma once

#include <cuda_bf16.h>

#include "tcrv_common.cuh"

namespace tcrv {

constexpr int kGroupTokens = 16;

__host__ __device__ constexpr uint32_t kv_group_bytes(uint32_t dim) { return 18 * dim; }

// Byte offsets inside a group of `dim` = 32 * nb.
__device__ __forceinline__ uint32_t kv_key_word(uint32_t nb, uint32_t token, uint32_t t, uint32_t b) {
  return 4 * ((token * 4 + t) * nb + b);
}
__device__ __forceinline__ uint32_t kv_value_half(uint32_t nb, uint32_t token, uint32_t g, uint32_t b) {
  return 256 * nb + 4 * ((((token >> 3) * 8 + g) * 4 + ((token & 7) >> 1)) * nb + b) + 2 * (token & 1);
}
__device__ __forceinline__ uint32_t kv_key_scale(uint32_t nb, uint32_t token, uint32_t b) {
  return 512 * nb + 2 * (token * nb + b);
}
__device__ __forceinline__ uint32_t kv_value_scale(uint32_t nb, uint32_t token, uint32_t b) {
  return 544 * nb + 2 * (token * nb + b);
}

// ---- activation types (TCRV_CUDA_TYPE_*)
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of an array whose type is known at run time.
__device__ __forceinline__ float load_typed(const void *p, size_t i, int type) {
  if (type == TCRV_CUDA_TYPE_F32)
    return static_cast<const float *>(p)[i];
  if (type == TCRV_CUDA_TYPE_F16)
    return __half2float(static_cast<const __half *>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}
__device__ __forceinline__ void store_typed(void *p, size_t i, int type, float v) {
  if (type == TCRV_CUDA_TYPE_F32)
    static_cast<float *>(p)[i] = v;
  else if (type == TCRV_CUDA_TYPE_F16)
    static_cast<__half *>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

inline size_t type_bytes(int type) { return type == TCRV_CUDA_TYPE_F32 ? 4 : 2; }

}  // namespace tcrv
