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

// Two 16-bit values of a word as fp32, and back (rounded to nearest).
template <typename T> __device__ __forceinline__ void split_word(uint32_t w, float& lo, float& hi);
template <> __device__ __forceinline__ void split_word<__nv_bfloat16>(uint32_t w, float& lo, float& hi) {
  lo = __uint_as_float(w << 16);           // bf16 is the upper half of an fp32
  hi = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void split_word<__half>(uint32_t w, float& lo, float& hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = f.x;
  hi = f.y;
}
template <typename T> __device__ __forceinline__ uint32_t join_word(float lo, float hi);
template <> __device__ __forceinline__ uint32_t join_word<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t join_word<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// The values of a pack as fp32.
template <typename T, int VEC>
__device__ __forceinline__ void unpack(const Pack<T, VEC>& k, float (&out)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    const uint4 w = *reinterpret_cast<const uint4*>(&k);
    split_word<T>(w.x, out[0], out[1]);
    split_word<T>(w.y, out[2], out[3]);
    split_word<T>(w.z, out[4], out[5]);
    split_word<T>(w.w, out[6], out[7]);
  } else {
#pragma unroll
    for (int j = 0; j < VEC; ++j) out[j] = to_f32(k.v[j]);
  }
}
// VEC consecutive elements as fp32; `p` is aligned to the whole pack.
template <typename T, int VEC>
__device__ __forceinline__ void load_pack(const T* p, float (&out)[VEC]) {
  const Pack<T, VEC> k = *reinterpret_cast<const Pack<T, VEC>*>(p);
  unpack<T, VEC>(k, out);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const float (&in)[VEC]) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(join_word<T>(in[0], in[1]), join_word<T>(in[2], in[3]), join_word<T>(in[4], in[5]),
                                              join_word<T>(in[6], in[7]));
  } else {
    Pack<T, VEC> k;
#pragma unroll
    for (int j = 0; j < VEC; ++j) k.v[j] = from_f32<T>(in[j]);
    *reinterpret_cast<Pack<T, VEC>*>(p) = k;
  }
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

// Asynchronous 16-byte copies into slots of shared memory that only the copying thread reads: rows in flight without
// registers to hold them and without a barrier.
__device__ __forceinline__ void async_copy_16(void* smem, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(smem))), "l"(global)
               : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Hardware approximations: 2^x (two units in the last place) and 1 / x (one).
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The larger one, NaN where either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
constexpr float LOG2_E = 1.4426950408889634f;

// Arithmetic on the values of a pack, two at a time: d = a b + c and the like, each an fp32 operation of its own.
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
  unsigned long long v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpair(unsigned long long v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ void fma_2(float& d0, float& d1, float a0, float a1, float b0, float b1, float c0, float c1) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair_of(a0, a1)), "l"(pair_of(b0, b1)), "l"(pair_of(c0, c1)));
  unpair(d, d0, d1);
}
__device__ __forceinline__ void mul_2(float& d0, float& d1, float a0, float a1, float b0, float b1) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair_of(a0, a1)), "l"(pair_of(b0, b1)));
  unpair(d, d0, d1);
}
template <int N>
__device__ __forceinline__ void v_fma(float (&d)[N], const float (&a)[N], const float (&b)[N], const float (&c)[N]) {
  if constexpr (N == 1) d[0] = fmaf(a[0], b[0], c[0]);
  else {
#pragma unroll
    for (int j = 0; j < N; j += 2) fma_2(d[j], d[j + 1], a[j], a[j + 1], b[j], b[j + 1], c[j], c[j + 1]);
  }
}
template <int N>
__device__ __forceinline__ void v_fma(float (&d)[N], const float (&a)[N], float s, const float (&c)[N]) {
  if constexpr (N == 1) d[0] = fmaf(a[0], s, c[0]);
  else {
#pragma unroll
    for (int j = 0; j < N; j += 2) fma_2(d[j], d[j + 1], a[j], a[j + 1], s, s, c[j], c[j + 1]);
  }
}
template <int N>
__device__ __forceinline__ void v_mul(float (&d)[N], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N == 1) d[0] = a[0] * b[0];
  else {
#pragma unroll
    for (int j = 0; j < N; j += 2) mul_2(d[j], d[j + 1], a[j], a[j + 1], b[j], b[j + 1]);
  }
}
template <int N>
__device__ __forceinline__ void v_mul(float (&d)[N], const float (&a)[N], float s) {
  if constexpr (N == 1) d[0] = a[0] * s;
  else {
#pragma unroll
    for (int j = 0; j < N; j += 2) mul_2(d[j], d[j + 1], a[j], a[j + 1], s, s);
  }
}
// sum[0] + sum[1] += a . b
template <int N>
__device__ __forceinline__ void v_dot(float (&sum)[2], const float (&a)[N], const float (&b)[N]) {
  if constexpr (N == 1) sum[0] = fmaf(a[0], b[0], sum[0]);
  else {
#pragma unroll
    for (int j = 0; j < N; j += 2) fma_2(sum[0], sum[1], a[j], a[j + 1], b[j], b[j + 1], sum[0], sum[1]);
  }
}

// Sum over the threads that share a row: one warp, or the whole block through `slot` (32 floats, zero behind the block's
// warps, that no other sum of the same row uses, so that one barrier is enough).  Every thread gets the same bits.
template <bool WARP_ROW>
__device__ __forceinline__ float row_sum(float v, float* slot) {
  v = warp_sum(v);
  if constexpr (WARP_ROW) {
    return v;
  } else {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x >> 5] = v;
    __syncthreads();
    const float4* s = reinterpret_cast<const float4*>(slot);
    float4 t = s[0];
    for (int i = 4; i < warps; i += 4) {
      const float4 o = s[i >> 2];
      t.x += o.x; t.y += o.y; t.z += o.z; t.w += o.w;
    }
    return (t.x + t.y) + (t.z + t.w);
  }
}

}  // namespace b200
