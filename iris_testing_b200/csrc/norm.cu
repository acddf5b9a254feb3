// RMS norm in front of a block, and the junction behind it: norm of the block's output, gate, residual with its
// scale, and the norm in front of the next block, forward and backward.
//
//   r1 = rsqrt(mean(y^2) + eps)   u = y r1 w   (or u = y)        h = s res + gate u
//   r2 = rsqrt(mean(h^2) + eps)   n = h r2 w2
//
//   t = dn w2          gh = dh + r2 (t - hh mean(t hh))   hh = h r2       dw2 = sum_rows dn hh
//   dres = s gh        dgate = sum over what the gate was spread over of gh u
//   q = gate gh w      dy = r1 (q - yh mean(q yh))        yh = y r1       dw  = sum_rows gate gh yh
//
// A row stays in the registers of the threads that share it (a warp up to 32 packs of a row, a block above that),
// so every tensor is read and written once.  The backward pass computes h again from y and res, which are
// kept for it anyway, instead of reading the rounded h.  Sums over rows (dw, dw2, dgate of one value per column) are
// kept per thread over the rows of a block, written once per block and added up in a fixed order by a second kernel.
#include <cuda_runtime.h>

#include "elementwise.cuh"
#include "launch.h"
#include "moe_args.h"
#include "sm100_ptx.cuh"

extern "C" {
typedef struct b200_norm_args {
  const void* y;          // [T, H], row stride ld_y
  const void* res;        // [T, H], row stride ld_res, or null: h = u
  const void* w;          // [H] or null
  const void* gate;       // by gate_kind
  const void* w2;         // [H]: the next norm's weight (null: no second output)
  void* h;                // [T, H]
  void* n;                // [T, H] (with w2)
  float* r1;              // [T] (null: not kept)
  float* r2;              // [T]
  const void* dh;         // backward: gradient of h, or null
  const void* dn;         // gradient of n, or null
  void* dy;               // [T, H]
  void* dres;             // [T, H] or null
  void* dgate;            // gate_kind 2: [T], 3: [T, H]; 1: [H], written by the finishing kernel
  void* dw;               // [H] or null
  void* dw2;              // [H] or null
  float* partial;         // [3][parts][H]: dw, dw2, dgate of each block
  long long ld_y, ld_res, ld_gate, ld_dh, ld_dn;
  int T, H;
  int elem;               // ElemType of y, res, h, n
  int w_f32, w2_f32, gate_f32;
  int norm;               // 0: u = y
  int gate_kind;          // 0 none, 1 [H], 2 one per row, 3 [T, H]
  int aligned;            // every row starts on 16 bytes and H is a whole number of packs
  int parts;              // rows of `partial`
  float scale, eps;
} b200_norm_args;
}

namespace b200 {

constexpr int NORM_MAX_H = 16384;
constexpr int NORM_WARP_ROWS = 4;     // rows of a block where a warp has a row

template <typename T, int VEC, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? NORM_WARP_ROWS * 32 : 1024) norm_forward_kernel(const b200_norm_args a) {
  __shared__ float slot[2][32];
  const int row = WARP_ROW ? blockIdx.x * NORM_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
  const int stride = (WARP_ROW ? 32 : blockDim.x) * VEC;
  if (row >= a.T) return;
  const T* y = static_cast<const T*>(a.y) + row * a.ld_y;
  const T* res = static_cast<const T*>(a.res) + (a.res != nullptr ? row * a.ld_res : 0);
  const size_t out = static_cast<size_t>(row) * a.H;
  const float inv_h = 1.f / static_cast<float>(a.H);

  float u[VPT][VEC], v[VPT][VEC];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[i][j] = v[i][j] = 0.f;
    if (c < a.H) {
      load_pack<T, VEC>(y + c, u[i]);
      if (a.res != nullptr) load_pack<T, VEC>(res + c, v[i]);
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) ss += u[i][j] * u[i][j];
  }
  float r1 = 1.f;
  if (a.norm) {
    r1 = rsqrtf(row_sum<WARP_ROW>(ss, slot[0]) * inv_h + a.eps);
    if (a.r1 != nullptr && t == 0) a.r1[row] = r1;
  }
  float gate_row = 1.f;
  if (a.gate_kind == 2) load_param<T, 1>(a.gate, a.gate_f32, static_cast<size_t>(row) * a.ld_gate, reinterpret_cast<float(&)[1]>(gate_row));
  float ss2 = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
    if (c >= a.H) continue;
    float w[VEC], g[VEC];
#pragma unroll
    for (int j = 0; j < VEC; ++j) { w[j] = 1.f; g[j] = gate_row; }
    if (a.w != nullptr) load_param<T, VEC>(a.w, a.w_f32, c, w);
    if (a.gate_kind == 1) load_param<T, VEC>(a.gate, a.gate_f32, c, g);
    if (a.gate_kind == 3) load_pack<T, VEC>(static_cast<const T*>(a.gate) + row * a.ld_gate + c, g);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      const float uu = u[i][j] * r1 * w[j];
      u[i][j] = a.res != nullptr ? fmaf(g[j], uu, a.scale * v[i][j]) : uu;
      ss2 += u[i][j] * u[i][j];
    }
    store_pack<T, VEC>(static_cast<T*>(a.h) + out + c, u[i]);
  }
  if (a.w2 == nullptr) return;
  const float r2 = rsqrtf(row_sum<WARP_ROW>(ss2, slot[1]) * inv_h + a.eps);
  if (a.r2 != nullptr && t == 0) a.r2[row] = r2;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
    if (c >= a.H) continue;
    float w[VEC];
    load_param<T, VEC>(a.w2, a.w2_f32, c, w);
#pragma unroll
    for (int j = 0; j < VEC; ++j) u[i][j] *= r2 * w[j];
    store_pack<T, VEC>(static_cast<T*>(a.n) + out + c, u[i]);
  }
}

template <typename T, int VEC, int VPT, bool WARP_ROW>
__global__ void __launch_bounds__(WARP_ROW ? NORM_WARP_ROWS * 32 : 1024) norm_backward_kernel(const b200_norm_args a) {
  __shared__ float slot[2][3][32];       // two sets: a row's sums while a slow warp still reads the row before's
  const int part = WARP_ROW ? blockIdx.x * NORM_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
  const int stride = (WARP_ROW ? 32 : blockDim.x) * VEC;
  const float inv_h = 1.f / static_cast<float>(a.H);
  const bool junction = a.res != nullptr;

  float acc_w[VPT][VEC], acc_w2[VPT][VEC], acc_g[VPT][VEC];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc_w[i][j] = acc_w2[i][j] = acc_g[i][j] = 0.f;

  int set = 0;
  for (int row = part; row < a.T; row += a.parts, set ^= 1) {
    const float r1 = a.norm ? a.r1[row] : 1.f;
    const float r2 = a.dn != nullptr ? a.r2[row] : 0.f;
    float gate_row = 1.f;
    if (a.gate_kind == 2) load_param<T, 1>(a.gate, a.gate_f32, static_cast<size_t>(row) * a.ld_gate, reinterpret_cast<float(&)[1]>(gate_row));
    float yh[VPT][VEC], hh[VPT][VEC], gh[VPT][VEC];
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
#pragma unroll
      for (int j = 0; j < VEC; ++j) yh[i][j] = hh[i][j] = gh[i][j] = 0.f;
      if (c >= a.H) continue;
      load_pack<T, VEC>(static_cast<const T*>(a.y) + row * a.ld_y + c, yh[i]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) yh[i][j] *= r1;
      if (a.dn != nullptr) {
        float res[VEC], w[VEC], g[VEC], dn[VEC], w2[VEC];
        load_pack<T, VEC>(static_cast<const T*>(a.res) + row * a.ld_res + c, res);
        load_pack<T, VEC>(static_cast<const T*>(a.dn) + row * a.ld_dn + c, dn);
        load_param<T, VEC>(a.w2, a.w2_f32, c, w2);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { w[j] = 1.f; g[j] = gate_row; }
        if (a.w != nullptr) load_param<T, VEC>(a.w, a.w_f32, c, w);
        if (a.gate_kind == 1) load_param<T, VEC>(a.gate, a.gate_f32, c, g);
        if (a.gate_kind == 3) load_pack<T, VEC>(static_cast<const T*>(a.gate) + row * a.ld_gate + c, g);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          hh[i][j] = fmaf(g[j], yh[i][j] * w[j], a.scale * res[j]) * r2;
          acc_w2[i][j] += dn[j] * hh[i][j];
          gh[i][j] = dn[j] * w2[j];
          m += gh[i][j] * hh[i][j];
        }
      }
    }
    if (a.dn != nullptr) m = row_sum<WARP_ROW>(m, slot[set][0]) * inv_h;
    float mq = 0.f, mg = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      float w[VEC], g[VEC], d[VEC], p[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) { w[j] = 1.f; g[j] = gate_row; d[j] = 0.f; }
      if (a.dh != nullptr) load_pack<T, VEC>(static_cast<const T*>(a.dh) + row * a.ld_dh + c, d);
      if (a.w != nullptr) load_param<T, VEC>(a.w, a.w_f32, c, w);
      if (a.gate_kind == 1) load_param<T, VEC>(a.gate, a.gate_f32, c, g);
      if (a.gate_kind == 3) load_pack<T, VEC>(static_cast<const T*>(a.gate) + row * a.ld_gate + c, g);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (a.dn != nullptr) d[j] += r2 * (gh[i][j] - hh[i][j] * m);
        p[j] = d[j] * yh[i][j] * w[j];          // d(gate)
        mg += p[j];
        acc_g[i][j] += p[j];
        const float du = g[j] * d[j];
        acc_w[i][j] += du * yh[i][j];
        gh[i][j] = du * w[j];                   // q
        mq += gh[i][j] * yh[i][j];
        d[j] *= a.scale;
      }
      if (a.dres != nullptr) store_pack<T, VEC>(static_cast<T*>(a.dres) + static_cast<size_t>(row) * a.H + c, d);
      if (junction && a.gate_kind == 3 && a.dgate != nullptr)
        store_pack<T, VEC>(static_cast<T*>(a.dgate) + static_cast<size_t>(row) * a.H + c, p);
    }
    if (a.gate_kind == 2 && a.dgate != nullptr) {
      mg = row_sum<WARP_ROW>(mg, slot[set][1]);
      if (t == 0) {
        if (a.gate_f32) static_cast<float*>(a.dgate)[row] = mg;
        else static_cast<T*>(a.dgate)[row] = from_f32<T>(mg);
      }
    }
    if (a.norm) mq = row_sum<WARP_ROW>(mq, slot[set][2]) * inv_h;
    if (a.dy != nullptr) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = t * VEC + i * stride;
        if (c >= a.H) continue;
        float d[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) d[j] = a.norm ? r1 * (gh[i][j] - yh[i][j] * mq) : gh[i][j];
        store_pack<T, VEC>(static_cast<T*>(a.dy) + static_cast<size_t>(row) * a.H + c, d);
      }
    }
  }
  const size_t plane = static_cast<size_t>(a.parts) * a.H, at = static_cast<size_t>(part) * a.H;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
    if (c >= a.H) continue;
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if (a.dw != nullptr) a.partial[at + c + j] = acc_w[i][j];
      if (a.dw2 != nullptr) a.partial[plane + at + c + j] = acc_w2[i][j];
      if (a.gate_kind == 1 && a.dgate != nullptr) a.partial[2 * plane + at + c + j] = acc_g[i][j];
    }
  }
}

// out[c] = sum over the parts of partial[.][c], in their order within each of eight interleaved shares.
template <typename T>
__global__ void __launch_bounds__(256) norm_columns_kernel(const b200_norm_args a) {
  __shared__ float share[8][33];
  chain_wait();
  const int which = blockIdx.y;
  void* out = which == 0 ? a.dw : which == 1 ? a.dw2 : (a.gate_kind == 1 ? a.dgate : nullptr);
  if (out == nullptr) return;
  const int f32 = which == 0 ? a.w_f32 : which == 1 ? a.w2_f32 : a.gate_f32;
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), s = threadIdx.x >> 5;
  const float* p = a.partial + static_cast<size_t>(which) * a.parts * a.H;
  float v = 0.f;
  if (c < a.H)
    for (int k = s; k < a.parts; k += 8) v += p[static_cast<size_t>(k) * a.H + c];
  share[s][threadIdx.x & 31] = v;
  __syncthreads();
  if (s == 0 && c < a.H) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += share[k][threadIdx.x];
    if (f32) static_cast<float*>(out)[c] = v;
    else static_cast<T*>(out)[c] = from_f32<T>(v);
  }
}

// How a row is shared: packs of VEC elements, VPT of them per thread, `threads` threads (32: a warp per row).
struct NormShape {
  int threads, vpt;
};
static NormShape norm_shape(int H, int vec) {
  const int packs = (H + vec - 1) / vec;
  const int vpt = vec > 1 ? (packs <= 32 ? 1 : packs <= 1024 ? 2 : 4) : (packs <= 1024 ? 4 : 16);
  int threads = ((packs + vpt - 1) / vpt + 31) / 32 * 32;
  return {threads, vpt};
}

static int norm_vec(const b200_norm_args& a) { return a.aligned ? (a.elem == ELEM_F32 ? 4 : 8) : 1; }

template <bool BACK, typename T, int VEC, int VPT>
static cudaError_t norm_launch(const b200_norm_args& a, int threads, cudaStream_t st) {
  const bool warp_row = threads <= 32;
  b200_count_launches(1);
  if constexpr (!BACK) {
    if (warp_row) norm_forward_kernel<T, VEC, VPT, true><<<(a.T + NORM_WARP_ROWS - 1) / NORM_WARP_ROWS, NORM_WARP_ROWS * 32, 0, st>>>(a);
    else norm_forward_kernel<T, VEC, VPT, false><<<a.T, threads, 0, st>>>(a);
    return cudaGetLastError();
  } else {
    if (warp_row) norm_backward_kernel<T, VEC, VPT, true><<<a.parts / NORM_WARP_ROWS, NORM_WARP_ROWS * 32, 0, st>>>(a);
    else norm_backward_kernel<T, VEC, VPT, false><<<a.parts, threads, 0, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || (a.dw == nullptr && a.dw2 == nullptr && !(a.gate_kind == 1 && a.dgate != nullptr))) return e;
    b200_count_launches(1);
    return launch_chained(norm_columns_kernel<T>, dim3((a.H + 31) / 32, 3), dim3(256), 0, st, a);
  }
}

template <bool BACK, typename T>
static cudaError_t norm_dispatch(const b200_norm_args& a, cudaStream_t st) {
  constexpr int VEC = 16 / sizeof(T);
  const NormShape s = norm_shape(a.H, a.aligned ? VEC : 1);
  if (a.aligned) {
    if (s.vpt == 1) return norm_launch<BACK, T, VEC, 1>(a, s.threads, st);
    if (s.vpt == 2) return norm_launch<BACK, T, VEC, 2>(a, s.threads, st);
    return norm_launch<BACK, T, VEC, 4>(a, s.threads, st);
  }
  if (s.vpt == 4) return norm_launch<BACK, T, 1, 4>(a, s.threads, st);
  return norm_launch<BACK, T, 1, 16>(a, s.threads, st);
}

template <bool BACK>
static int norm_run(const b200_norm_args* a, void* stream) {
  if (a == nullptr || a->T < 1 || a->H < 1 || a->H > NORM_MAX_H || a->y == nullptr || a->gate_kind < 0 || a->gate_kind > 3) return -10;
  if ((a->gate_kind != 0 && (a->gate == nullptr || a->res == nullptr)) || (a->w2 != nullptr && a->res == nullptr)) return -11;
  if (!BACK && (a->h == nullptr || (a->w2 != nullptr && a->n == nullptr))) return -12;
  if (BACK && (a->parts < 1 || (a->norm && a->r1 == nullptr) || (a->dn != nullptr && (a->r2 == nullptr || a->w2 == nullptr)))) return -13;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->elem) {
    case ELEM_F32: return static_cast<int>(norm_dispatch<BACK, float>(*a, st));
    case ELEM_BF16: return static_cast<int>(norm_dispatch<BACK, __nv_bfloat16>(*a, st));
    case ELEM_F16: return static_cast<int>(norm_dispatch<BACK, __half>(*a, st));
  }
  return -14;
}

}  // namespace b200

extern "C" {

int b200_norm_forward(const b200_norm_args* a, void* stream) { return b200::norm_run<false>(a, stream); }
int b200_norm_backward(const b200_norm_args* a, void* stream) { return b200::norm_run<true>(a, stream); }

// Rows of `partial` that a backward call of this shape uses: one per block, or per warp where a warp has a row.
int b200_norm_parts(int T, int H, int elem, int aligned, int sms) {
  using namespace b200;
  const NormShape s = norm_shape(H, aligned ? (elem == ELEM_F32 ? 4 : 8) : 1);
  if (s.threads <= 32) {
    const int blocks = (T + NORM_WARP_ROWS - 1) / NORM_WARP_ROWS;
    return NORM_WARP_ROWS * (blocks < 4 * sms ? blocks : 4 * sms);
  }
  const int per_sm = s.threads <= 128 ? 4 : s.threads <= 256 ? 2 : 1;
  return T < per_sm * sms ? T : per_sm * sms;
}

int b200_abi_size_norm_args() { return static_cast<int>(sizeof(b200_norm_args)); }
int b200_norm_max_columns() { return b200::NORM_MAX_H; }

}  // extern "C"
