// The paged key / value cache as the kernels see it (mcpuKvCache of
// include/mcpu_ops.h), and the argument checks its entry points share.
#pragma once

#include <cuda_fp8.h>

#include "common.cuh"

namespace mcpu {
namespace kv {

// Address of a page: block ids come from device memory, so an id outside the
// cache is replaced by block 0 and reported instead of being followed.
__device__ __forceinline__ long long checked_block(int id, long long num_blocks, int* error) {
  if (id < 0 || id >= num_blocks) {
    atomicOr(error, 1);
    return 0;
  }
  return id;
}


// What every entry point asks of a cache: its sizes, and 16-byte-aligned rows.
inline orError_t check_cache(const mcpuKvCache* c, int dtype, const char* op) {
  MCPU_ARG_CHECK(c != nullptr, "%s: cache is NULL", op);
  MCPU_ARG_CHECK(dtype == MCPU_BFLOAT16 || dtype == MCPU_FLOAT16, "%s: bfloat16 or float16 tensors expected", op);
  MCPU_ARG_CHECK(c->dtype == dtype || c->dtype == MCPU_FLOAT8_E4M3 || c->dtype == MCPU_INT8,
                 "%s: the cache holds the tensors' type, float8_e4m3fn or int8", op);
  const bool small = c->dtype != dtype;
  MCPU_ARG_CHECK(c->num_blocks >= 0 && c->num_blocks < (1LL << 31) && c->block_size > 0 && c->kv_heads > 0 &&
                     c->head_size > 0,
                 "%s: bad cache sizes", op);
  MCPU_ARG_CHECK(c->head_size % 16 == 0 && c->head_size <= 512, "%s: head_size %d must be a multiple of 16, at most 512",
                 op, c->head_size);
  MCPU_ARG_CHECK(c->scale_mode == (small ? c->scale_mode : MCPU_KV_SCALE_NONE) &&
                     c->scale_mode >= MCPU_KV_SCALE_NONE && c->scale_mode <= MCPU_KV_SCALE_TOKEN &&
                     (!small || c->scale_mode != MCPU_KV_SCALE_NONE),
                 "%s: an 8-bit cache has scales, a 16-bit cache has none", op);
  const int align = small ? 16 : 8;  // elements per 16 bytes
  for (int i = 0; i < 3; ++i)
    MCPU_ARG_CHECK(c->key_stride[i] >= 0 && c->value_stride[i] >= 0 && c->key_stride[i] % align == 0 &&
                       c->value_stride[i] % align == 0,
                   "%s: cache strides must be multiples of 16 bytes", op);
  if (c->num_blocks > 0) {
    MCPU_ARG_CHECK(c->key && c->value && (!small || (c->k_scale && c->v_scale)), "%s: NULL cache pointer", op);
    MCPU_ARG_CHECK(((reinterpret_cast<uintptr_t>(c->key) | reinterpret_cast<uintptr_t>(c->value)) & 15) == 0,
                   "%s: the cache must be 16-byte aligned", op);
  }
  return orSuccess;
}

}  // namespace kv
}  // namespace mcpu
