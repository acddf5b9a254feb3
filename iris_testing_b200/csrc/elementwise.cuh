// Typed 16-byte (or single-element) accesses and row reductions of the kernels that work on rows of activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

// Element types as the host names them.
enum ElemType : int { ELEM_F32 = 0, ELEM_BF16 = 1, ELEM_F16 = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

template <typename T, int VEC>
struct __align__(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// VEC consecutive elements as fp32; `p` is aligned to the whole pack.
template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[VEC]) {
  const Pack<T, VEC> k = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int j = 0; j < VEC; ++j) out[j] = to_f32(k.v[j]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[VEC]) {
  Pack<T, VEC> k;
#pragma unroll
  for (int j = 0; j < VEC; ++j) k.v[j] = from_f32<T>(in[j]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = k;
}
// A parameter vector that is kept in T or in fp32; its address is aligned to VEC elements of either.
template <typename T, int VEC>
__device__ __forceinline__ void load_param(const void* base, int f32, size_t i, float (&out)[VEC]) {
  if (f32) {
    constexpr int Q = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int q = 0; q < VEC; q += Q) {
      float part[Q];
      load_pack<float, Q>(static_cast<const float*>(base) + i + q, part);
#pragma unroll
      for (int j = 0; j < Q; ++j) out[q + j] = part[j];
    }
  } else {
    load_pack<T, VEC>(static_cast<const T*>(base) + i, out);
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the threads that share a row: one warp, or the whole block through `slot` (32 floats that no other
// reduction of the same row uses, so that one barrier is enough).  Every thread gets the same bits.
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  v = warp_sum(v);
  if constexpr (WARP_ROW) {
    return v;
  } else {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    if (lane == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(lane < warps ? slot[lane] : 0.f);
  }
}

}  // namespace b200
