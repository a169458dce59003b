// paged.cuh -- address arithmetic of the paged key / value cache (turt_paged_kv), shared by the
// kernels that write and read it.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/turt_cuda.h"
#include "common.cuh"

namespace turt {

// The descriptor as kernels see it: strides resolved, sizes checked by paged_layout().
struct PagedLayout {
  const uint32_t* table;
  const uint32_t* lens;
  size_t page_stride, head_stride, slot_stride;
  uint32_t n_pages, page_size, max_pages;
  int kv_heads, dim, batch;
};

// Checks a descriptor and resolves its strides (0 = packed [page][head][slot][dim]).
int paged_layout(const turt_paged_kv* kv, PagedLayout* out);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline size_t cache_type_size(int dtype) { return dtype == TURT_CACHE_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace turt
