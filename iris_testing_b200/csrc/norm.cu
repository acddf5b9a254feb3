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
// A row stays in the registers of the threads that share it, 16 elements each (a warp up to 512 columns, a block above
// that), so every tensor is read and written once; blocks are persistent, and the next rows are on their way
// (cp.async into slots that each thread fills and reads itself) while a row is reduced.  With 8 elements a thread, the
// reductions were a third of 46 instructions per 32 elements and the kernels bound by issue.  The backward
// pass computes h again from y and res, which are kept for it anyway, instead of reading the rounded h.  Sums over rows
// (dw2, and A = sum gh yh, of which dw is gate times and the gradient of a gate per column w times) are kept per thread
// over the rows of a block, written once per block and added up in a fixed order by a second kernel.
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
  float* partial;         // [2][parts][H]: A and dw2 of each block
  long long ld_y, ld_res, ld_gate, ld_dh, ld_dn;
  int T, H;
  int elem;               // ElemType of y, res, h, n
  int w_f32, w2_f32, gate_f32;
  int norm;               // 0: u = y
  int gate_kind;          // 0 none, 1 [H], 2 one per row, 3 [T, H]
  int aligned;            // every row starts on 16 bytes and H is a whole number of packs
  int parts;              // rows in work at once (set by the launcher)
  float scale, eps;
} b200_norm_args;
}

namespace b200 {

constexpr int NORM_MAX_H = 16384;
constexpr int NORM_MAX_ROWS = 1 << 30;  // rows ahead of the last one still have numbers of 32 bits
constexpr int NORM_WARP_ROWS = 4;      // rows of a block where a warp has a row
constexpr int NORM_ELEMS = 16;         // elements of a row per thread (8 where that is enough)

// Threads of a block and blocks of an SM of a variant: MAXT is the most threads that share a row (32: a warp).  512
// threads an SM leave 128 registers each; where 1024 threads share a row (more than 8192 columns) it is 64, and the backward
// kernels spill 260 - 440 bytes a thread (4096 rows of 16384 bf16 columns, without / with a next norm: forward 100 / 152 us,
// backward 185 / 368, for 42 / 83 and 62 / 125 of bytes at the copy rate; nothing is fetched ahead there either).  The forward
// kernel of 16-bit rows above 4096 and up to 6144 columns needs 78 and so has two blocks of 384 threads on an SM instead of
// one: 8192 rows of 5120 columns 52 -> 40 us, with a residual 58 -> 48, with a next norm 75 -> 62; of 6144 columns
// 52 -> 44, 59 -> 56, 77 -> 77.  For fp32 rows the two are even (68 -> 62, 87 -> 93, 122 -> 118), and one block stays.
template <bool BACK, int MAXT>
constexpr int NORM_BLOCKS = MAXT == 32 ? 4 : MAXT == 256 || (MAXT == 384 && !BACK) ? 2 : 1;
template <int MAXT>
constexpr int NORM_THREADS = MAXT == 32 ? NORM_WARP_ROWS * 32 : MAXT;
// Rows on their way ahead of the one in work: up to three, by the slots that fit beside each other on an SM (two tensors
// forward, four and the two column vectors backward); none for the widest rows and for rows that do not lie on 16 bytes,
// which go straight to registers (8192 rows of 4099 columns: forward 207 us, backward 335; of 4096: 32 and 46).  The forms
// without a next norm have room for w2's factors too, and do not use it.
constexpr int NORM_SLOT_BYTES = 200 * 1024;
template <bool BACK, int VEC, int VPT, int MAXT>
constexpr int NORM_VECTOR_BYTES = BACK && VEC > 1 && MAXT != 1024 ? 2 * VPT * VEC * 4 * NORM_THREADS<MAXT> : 0;
template <bool BACK, int VEC, int VPT, int MAXT>
constexpr int NORM_FIT = (NORM_SLOT_BYTES / NORM_BLOCKS<BACK, MAXT> - NORM_VECTOR_BYTES<BACK, VEC, VPT, MAXT>) / ((BACK ? 4 : 2) * VPT * 16 * NORM_THREADS<MAXT>);
template <bool BACK, int VEC, int VPT, int MAXT>
constexpr int NORM_STAGES = VEC == 1 || MAXT == 1024 ? 0 : NORM_FIT<BACK, VEC, VPT, MAXT> < 3 ? NORM_FIT<BACK, VEC, VPT, MAXT> : 3;

// Asks for every pack that this thread takes of a row.
template <typename T, int VEC, int VPT>
__device__ __forceinline__ void fetch_row(const void* base, long long ld, int row, int H, int t, int stride, uint4* slot, int threads) {
  if (base == nullptr) return;
  const T* p = static_cast<const T*>(base) + row * ld;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
    if (c < H) async_copy_16(slot + i * threads, p + c);
  }
}

// One pack of a tensor: from this thread's slot, or straight from memory where rows are not fetched ahead.
template <typename T, int VEC, int S>
__device__ __forceinline__ void read_pack(const uint4* slot, const void* base, long long ld, int row, int c, float (&out)[VEC]) {
  if constexpr (S > 0) load_pack<T, VEC>(reinterpret_cast<const T*>(slot), out);
  else load_pack<T, VEC>(static_cast<const T*>(base) + row * ld + c, out);
}

// What a pack's values of norm(y) are multiplied with in every row: w, times the gate where that has a value per column.
template <typename T, int VEC>
__device__ __forceinline__ void column_factor(const b200_norm_args& a, int c, float (&f)[VEC]) {
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = 1.f;
  if (a.w != nullptr) load_param<T, VEC>(a.w, a.w_f32, c, f);
  if (a.gate_kind == 1) {
    float g[VEC];
    load_param<T, VEC>(a.gate, a.gate_f32, c, g);
    v_mul<VEC>(f, f, g);
  }
}
// What a row is multiplied with: the gate where that has a value per row.
template <typename T>
__device__ __forceinline__ float row_factor(const b200_norm_args& a, int row) {
  float g[1] = {1.f};
  if (a.gate_kind == 2) load_param<T, 1>(a.gate, a.gate_f32, static_cast<size_t>(row) * a.ld_gate, g);
  return g[0];
}

template <typename T, int VEC, int VPT, int MAXT>
__global__ void __launch_bounds__(NORM_THREADS<MAXT>, NORM_BLOCKS<false, MAXT>) norm_forward_kernel(const b200_norm_args a) {
  extern __shared__ uint4 slots[];
  __shared__ __align__(16) float sums[2][2][32];       // two sets: a row's sums while a slow warp still reads the row before's
  constexpr bool WARP_ROW = MAXT == 32;
  constexpr int S = NORM_STAGES<false, VEC, VPT, MAXT>;
  const int part = WARP_ROW ? blockIdx.x * NORM_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
  const int threads = blockDim.x, stride = (WARP_ROW ? 32 : threads) * VEC;
  const float inv_h = 1.f / static_cast<float>(a.H);
  const int tensors = a.res != nullptr ? 2 : 1;
  uint4* mine = slots + threadIdx.x;                       // [stage][tensor][VPT][threads]
  auto at = [&](int stage, int tensor) { return mine + (stage * tensors + tensor) * VPT * threads; };
  auto fetch = [&](int row, int stage) {
    if constexpr (S > 0) {
      if (row < a.T) {
        fetch_row<T, VEC, VPT>(a.y, a.ld_y, row, a.H, t, stride, at(stage, 0), threads);
        fetch_row<T, VEC, VPT>(a.res, a.ld_res, row, a.H, t, stride, at(stage, 1), threads);
      }
      async_commit();
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(part + s * a.parts, s);
  if constexpr (!WARP_ROW) {
    if (threadIdx.x < 128) (&sums[0][0][0])[threadIdx.x] = 0.f;
    for (int i = threadIdx.x + threads; i < 128; i += threads) (&sums[0][0][0])[i] = 0.f;
    __syncthreads();
  }
  // the columns' factors stay in registers (of the widest rows they are read again for every row)
  constexpr bool HELD = MAXT != 1024;
  float f1[HELD ? VPT : 1][VEC], f2[HELD ? VPT : 1][VEC];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      column_factor<T, VEC>(a, c, f1[i]);
      if (a.w2 != nullptr) load_param<T, VEC>(a.w2, a.w2_f32, c, f2[i]);
    }
  }

  int set = 0, stage = 0;
  for (int row = part; row < a.T; row += a.parts, set ^= 1, stage = stage + 1 >= S ? 0 : stage + 1) {
    if constexpr (S > 0) async_wait<S - 1>();
    const size_t out = static_cast<size_t>(row) * a.H;
    float r1 = row_factor<T>(a, row);
    float u[VPT][VEC], v[VPT][VEC];
    float ss[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
#pragma unroll
      for (int j = 0; j < VEC; ++j) u[i][j] = v[i][j] = 0.f;
      if (c < a.H) {
        read_pack<T, VEC, S>(at(stage, 0) + i * threads, a.y, a.ld_y, row, c, u[i]);
        if (a.res != nullptr) read_pack<T, VEC, S>(at(stage, 1) + i * threads, a.res, a.ld_res, row, c, v[i]);
      }
      v_dot<VEC>(ss, u[i], u[i]);
    }
    if (a.norm) {
      const float r = rsqrtf(row_sum<WARP_ROW>(ss[0] + ss[1], sums[set][0]) * inv_h + a.eps);
      if (a.r1 != nullptr && t == 0) a.r1[row] = r;
      r1 *= r;
    }
    fetch(row + S * a.parts, stage);
    ss[0] = ss[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      float x[VEC];
      if constexpr (!HELD) column_factor<T, VEC>(a, c, x);
      float(&f)[VEC] = HELD ? f1[HELD ? i : 0] : x;
      v_mul<VEC>(u[i], u[i], r1);
      if (a.gate_kind == 3) {
        float g[VEC];
        load_pack<T, VEC>(static_cast<const T*>(a.gate) + row * a.ld_gate + c, g);
        v_mul<VEC>(u[i], u[i], g);
      }
      v_mul<VEC>(v[i], v[i], a.scale);              // zeros without a residual
      v_fma<VEC>(u[i], u[i], f, v[i]);
      if (a.w2 != nullptr) v_dot<VEC>(ss, u[i], u[i]);
      store_pack<T, VEC>(static_cast<T*>(a.h) + out + c, u[i]);
    }
    if (a.w2 == nullptr) continue;
    const float r2 = rsqrtf(row_sum<WARP_ROW>(ss[0] + ss[1], sums[set][1]) * inv_h + a.eps);
    if (a.r2 != nullptr && t == 0) a.r2[row] = r2;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      float x[VEC];
      if constexpr (!HELD) load_param<T, VEC>(a.w2, a.w2_f32, c, x);
      float(&f)[VEC] = HELD ? f2[HELD ? i : 0] : x;
      v_mul<VEC>(u[i], u[i], r2);
      v_mul<VEC>(u[i], u[i], f);
      store_pack<T, VEC>(static_cast<T*>(a.n) + out + c, u[i]);
    }
  }
  if constexpr (S > 0) async_wait<0>();
}

// FORM says which of two conditions hold, a next norm and a gate of the rows' own shape, both of which stand around every
// pack: known beforehand they cost neither registers nor branches.  Found out at run time (NORM_ANY) the kernel took 88 us
// for 8192 x 4096 with a next norm, and 79 for 5003 x 6144 without one; as forms of their own 74 and 61.  Rows that do not
// lie on 16 bytes, and those of more than 8192 columns, keep the one kernel for all.
enum NormForm : int { NORM_NEXT = 1, NORM_FULL_GATE = 2, NORM_ANY = 4 };

template <typename T, int VEC, int VPT, int MAXT, int FORM>
__global__ void __launch_bounds__(NORM_THREADS<MAXT>, NORM_BLOCKS<true, MAXT>) norm_backward_kernel(const b200_norm_args a) {
  extern __shared__ uint4 slots[];
  __shared__ __align__(16) float sums[2][2][32];
  constexpr bool WARP_ROW = MAXT == 32;
  constexpr int S = NORM_STAGES<true, VEC, VPT, MAXT>;
  constexpr int VQ = VEC / 4;                              // float4 of a pack's column factors
  const int part = WARP_ROW ? blockIdx.x * NORM_WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x;
  const int t = WARP_ROW ? threadIdx.x & 31 : threadIdx.x;
  const int threads = blockDim.x, stride = (WARP_ROW ? 32 : threads) * VEC;
  const float inv_h = 1.f / static_cast<float>(a.H);
  const bool next = FORM == NORM_ANY ? a.dn != nullptr : (FORM & NORM_NEXT) != 0;
  const bool full_gate = FORM == NORM_ANY ? a.gate_kind == 3 : (FORM & NORM_FULL_GATE) != 0;
  // [w times gate, w2][VPT][VQ][threads], then [stage][y, dh, res, dn][VPT][threads]: a thread's own, all of them
  float4* factors = reinterpret_cast<float4*>(slots) + threadIdx.x;
  uint4* mine = slots + (S > 0 ? 2 * VPT * VQ * threads : 0) + threadIdx.x;
  const int tensors = next ? 4 : 2;
  auto at = [&](int stage, int tensor) { return mine + (stage * tensors + tensor) * VPT * threads; };
  auto fetch = [&](int row, int stage) {
    if constexpr (S > 0) {
      if (row < a.T) {
        fetch_row<T, VEC, VPT>(a.y, a.ld_y, row, a.H, t, stride, at(stage, 0), threads);
        fetch_row<T, VEC, VPT>(a.dh, a.ld_dh, row, a.H, t, stride, at(stage, 1), threads);
        if (next) {
          fetch_row<T, VEC, VPT>(a.res, a.ld_res, row, a.H, t, stride, at(stage, 2), threads);
          fetch_row<T, VEC, VPT>(a.dn, a.ld_dn, row, a.H, t, stride, at(stage, 3), threads);
        }
      }
      async_commit();
    }
  };
#pragma unroll
  for (int s = 0; s < S; ++s) fetch(part + s * a.parts, s);
  if constexpr (!WARP_ROW) {
    for (int i = threadIdx.x; i < 128; i += threads) (&sums[0][0][0])[i] = 0.f;
    __syncthreads();
  }
  auto factor = [&](int which, int i, int c, float (&f)[VEC]) {
    if constexpr (S > 0) {
#pragma unroll
      for (int q = 0; q < VQ; ++q) {
        const float4 x = factors[((which * VPT + i) * VQ + q) * threads];
        f[4 * q] = x.x; f[4 * q + 1] = x.y; f[4 * q + 2] = x.z; f[4 * q + 3] = x.w;
      }
    } else if (which == 0) {
      column_factor<T, VEC>(a, c, f);
    } else {
      load_param<T, VEC>(a.w2, a.w2_f32, c, f);
    }
  };
  if constexpr (S > 0) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      float f[VEC];
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        if (which == 0) column_factor<T, VEC>(a, c, f);
        else if (next) load_param<T, VEC>(a.w2, a.w2_f32, c, f);
#pragma unroll
        for (int q = 0; q < VQ; ++q)
          factors[((which * VPT + i) * VQ + q) * threads] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
      }
    }
  }

  float acc[VPT][VEC], acc2[VPT][VEC];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) acc[i][j] = acc2[i][j] = 0.f;

  // a row's three numbers, read while the row before is in work
  float n1 = 1.f, n2 = 0.f, ng = 1.f;
  auto numbers = [&](int row) {
    if (row >= a.T) return;
    if (a.norm) n1 = a.r1[row];
    if (next) n2 = a.r2[row];
    ng = row_factor<T>(a, row);
  };
  numbers(part);

  int set = 0, stage = 0;
  for (int row = part; row < a.T; row += a.parts, set ^= 1, stage = stage + 1 >= S ? 0 : stage + 1) {
    if constexpr (S > 0) async_wait<S - 1>();
    const float r1 = n1, r2 = n2, gate_row = ng;
    numbers(row + a.parts);
    auto times_full_gate = [&](int c, float (&x)[VEC]) {
      if (!full_gate) return;
      float g[VEC];
      load_pack<T, VEC>(static_cast<const T*>(a.gate) + row * a.ld_gate + c, g);
      v_mul<VEC>(x, x, g);
    };
    float yh[VPT][VEC], hh[VPT][VEC], gh[VPT][VEC];
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
#pragma unroll
      for (int j = 0; j < VEC; ++j) yh[i][j] = hh[i][j] = gh[i][j] = 0.f;
      if (c >= a.H) continue;
      read_pack<T, VEC, S>(at(stage, 0) + i * threads, a.y, a.ld_y, row, c, yh[i]);
      v_mul<VEC>(yh[i], yh[i], r1);
      if (next) {
        float x[VEC], f[VEC];
        read_pack<T, VEC, S>(at(stage, 2) + i * threads, a.res, a.ld_res, row, c, hh[i]);
        v_mul<VEC>(hh[i], hh[i], a.scale);
        v_mul<VEC>(x, yh[i], gate_row);
        times_full_gate(c, x);
        factor(0, i, c, f);
        v_fma<VEC>(hh[i], x, f, hh[i]);
        v_mul<VEC>(hh[i], hh[i], r2);
        read_pack<T, VEC, S>(at(stage, 3) + i * threads, a.dn, a.ld_dn, row, c, gh[i]);
        v_fma<VEC>(acc2[i], gh[i], hh[i], acc2[i]);
        factor(1, i, c, f);
        v_mul<VEC>(gh[i], gh[i], f);
        v_dot<VEC>(m, gh[i], hh[i]);
      }
    }
    const float mean = next ? row_sum<WARP_ROW>(m[0] + m[1], sums[set][0]) * inv_h : 0.f;
    m[0] = m[1] = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = t * VEC + i * stride;
      if (c >= a.H) continue;
      float d[VEC], f[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) d[j] = 0.f;
      if (a.dh != nullptr) read_pack<T, VEC, S>(at(stage, 1) + i * threads, a.dh, a.ld_dh, row, c, d);
      if (next) {
        v_fma<VEC>(gh[i], hh[i], -mean, gh[i]);
        v_fma<VEC>(d, gh[i], r2, d);
      }
      factor(0, i, c, f);
      // A takes in a gate that changes from row to row; gh becomes q but for the row's gate
      float g[VEC];
      v_mul<VEC>(g, d, gate_row);
      if (full_gate) {
        float p[VEC];
        v_mul<VEC>(p, d, f);
        v_mul<VEC>(p, p, yh[i]);
        if (a.dgate != nullptr) store_pack<T, VEC>(static_cast<T*>(a.dgate) + static_cast<size_t>(row) * a.H + c, p);
        times_full_gate(c, g);
        v_mul<VEC>(gh[i], g, f);
      } else {
        v_mul<VEC>(gh[i], d, f);
      }
      v_fma<VEC>(acc[i], g, yh[i], acc[i]);
      v_dot<VEC>(m, gh[i], yh[i]);
      if (a.dres != nullptr) {
        v_mul<VEC>(d, d, a.scale);
        store_pack<T, VEC>(static_cast<T*>(a.dres) + static_cast<size_t>(row) * a.H + c, d);
      }
    }
    fetch(row + S * a.parts, stage);
    const bool row_gate = a.gate_kind == 2 && a.dgate != nullptr;
    float sum = 0.f;                                 // gate per row: its gradient, and the mean of q yh but for the gate
    if (a.norm || row_gate) sum = row_sum<WARP_ROW>(m[0] + m[1], sums[set][1]);
    if (row_gate && t == 0) {
      if (a.gate_f32) static_cast<float*>(a.dgate)[row] = sum;
      else static_cast<T*>(a.dgate)[row] = from_f32<T>(sum);
    }
    if (a.dy != nullptr) {
      const float mean_q = a.norm ? sum * inv_h : 0.f, r = r1 * gate_row;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = t * VEC + i * stride;
        if (c >= a.H) continue;
        v_fma<VEC>(gh[i], yh[i], -mean_q, gh[i]);
        v_mul<VEC>(gh[i], gh[i], r);
        store_pack<T, VEC>(static_cast<T*>(a.dy) + static_cast<size_t>(row) * a.H + c, gh[i]);
      }
    }
  }
  if constexpr (S > 0) async_wait<0>();
  if (a.partial == nullptr) return;
  const size_t plane = static_cast<size_t>(a.parts) * a.H, here = static_cast<size_t>(part) * a.H;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int c = t * VEC + i * stride;
    if (c >= a.H) continue;
    constexpr int Q = VEC < 4 ? VEC : 4;
#pragma unroll
    for (int q = 0; q < VEC; q += Q) {
      store_pack<float, Q>(a.partial + here + c + q, reinterpret_cast<float(&)[Q]>(acc[i][q]));
      if (a.dw2 != nullptr) store_pack<float, Q>(a.partial + plane + here + c + q, reinterpret_cast<float(&)[Q]>(acc2[i][q]));
    }
  }
}

// Column sums over the parts, in their order within each of 32 interleaved shares: dw = gate A, the gate's w A, and dw2.
template <typename T>
__global__ void __launch_bounds__(1024) norm_columns_kernel(const b200_norm_args a) {
  __shared__ float share[32][33];
  chain_wait();
  const int lane = threadIdx.x & 31, s = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  if (blockIdx.y == 1 ? a.dw2 == nullptr : a.dw == nullptr && a.dgate == nullptr) return;
  const float* p = a.partial + static_cast<size_t>(blockIdx.y) * a.parts * a.H;
  float v = 0.f;
  if (c < a.H) {
#pragma unroll 4
    for (int k = s; k < a.parts; k += 32) v += p[static_cast<size_t>(k) * a.H + c];
  }
  share[s][lane] = v;
  __syncthreads();
  if (s != 0 || c >= a.H) return;
#pragma unroll
  for (int k = 1; k < 32; ++k) v += share[k][lane];
  auto put = [&](void* out, int f32, float x) {
    if (f32) static_cast<float*>(out)[c] = x;
    else static_cast<T*>(out)[c] = from_f32<T>(x);
  };
  if (blockIdx.y == 1) {
    put(a.dw2, a.w2_f32, v);
    return;
  }
  float w[1] = {1.f}, g[1] = {1.f};
  if (a.w != nullptr) load_param<T, 1>(a.w, a.w_f32, c, w);
  if (a.gate_kind == 1) load_param<T, 1>(a.gate, a.gate_f32, c, g);
  if (a.dw != nullptr) put(a.dw, a.w_f32, g[0] * v);
  if (a.gate_kind == 1 && a.dgate != nullptr) put(a.dgate, a.gate_f32, w[0] * v);
}

// How a row is shared: a warp while 16 elements a lane are enough, which needs no barrier, otherwise the threads of a block.
template <int MAXT>
static int norm_row_threads(int H, int vec, int vpt) {
  const int packs = (H + vec - 1) / vec;
  return MAXT == 32 ? 32 : ((packs + vpt - 1) / vpt + 31) / 32 * 32;
}

// Rows (of warps, or of blocks) in work at once: the blocks that the registers of the variant and the slots leave room
// for on every SM, and no more rows than there are.
template <bool BACK, int MAXT>
static int norm_parts(int T, int threads, size_t smem, int sms) {
  const int rows = MAXT == 32 ? NORM_WARP_ROWS : 1;
  int per_sm = MAXT == 32 ? NORM_BLOCKS<BACK, 32> : MAXT * NORM_BLOCKS<BACK, MAXT> / threads;
  const int fit = static_cast<int>((224u * 1024u) / (smem + 2048));      // beside 1 KB of the system's and the sums
  if (fit < per_sm) per_sm = fit > 0 ? fit : 1;
  const int blocks = (T + rows - 1) / rows;
  return rows * (blocks < per_sm * sms ? blocks : per_sm * sms);
}

template <bool BACK, typename T, int VEC, int VPT, int MAXT>
static cudaError_t norm_launch(b200_norm_args a, int sms, cudaStream_t st) {
  using Kernel = void (*)(const b200_norm_args);
  const int threads = norm_row_threads<MAXT>(a.H, VEC, VPT);
  const int block = MAXT == 32 ? NORM_WARP_ROWS * 32 : threads;
  const int tensors = BACK ? (a.dn != nullptr ? 4 : 2) : (a.res != nullptr ? 2 : 1);
  constexpr int S = NORM_STAGES<BACK, VEC, VPT, MAXT>;
  const size_t smem = (static_cast<size_t>(S) * tensors * VPT * 16 + (BACK && S > 0 ? 2 * VPT * VEC * 4 : 0)) * block;   // at most 200 KB
  a.parts = norm_parts<BACK, MAXT>(a.T, threads, smem, sms);
  const dim3 grid(MAXT == 32 ? a.parts / NORM_WARP_ROWS : a.parts);
  Kernel kern;
  int form = 0;
  if constexpr (!BACK) {
    kern = norm_forward_kernel<T, VEC, VPT, MAXT>;
  } else if constexpr (S == 0) {
    kern = norm_backward_kernel<T, VEC, VPT, MAXT, NORM_ANY>;
  } else {
    form = (a.dn != nullptr ? NORM_NEXT : 0) | (a.gate_kind == 3 ? NORM_FULL_GATE : 0);
    kern = form == 0 ? norm_backward_kernel<T, VEC, VPT, MAXT, 0>
         : form == NORM_NEXT ? norm_backward_kernel<T, VEC, VPT, MAXT, NORM_NEXT>
         : form == NORM_FULL_GATE ? norm_backward_kernel<T, VEC, VPT, MAXT, NORM_FULL_GATE>
                                  : norm_backward_kernel<T, VEC, VPT, MAXT, NORM_NEXT | NORM_FULL_GATE>;
  }
  static std::atomic<unsigned long long> allowed[4];
  if (S > 0) {
    const cudaError_t e = allow_shared_memory(kern, NORM_SLOT_BYTES, allowed[form]);
    if (e != cudaSuccess) return e;
  }
  b200_count_launches(1);
  kern<<<grid, block, smem, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (!BACK || e != cudaSuccess || a.partial == nullptr) return e;
  b200_count_launches(1);
  return launch_chained(norm_columns_kernel<T>, dim3((a.H + 31) / 32, a.dw2 != nullptr ? 2 : 1), dim3(1024), 0, st, a);
}

// Calls f<VEC, VPT, MAXT> for rows of H elements.
template <typename T, typename F>
static auto norm_variant(int H, bool aligned, F&& f) {
  constexpr int V = 16 / sizeof(T);
  if (!aligned) {
    if (H <= 32 * NORM_ELEMS) return f.template operator()<1, NORM_ELEMS, 32>();
    if (H <= 256 * NORM_ELEMS) return f.template operator()<1, NORM_ELEMS, 256>();
    return f.template operator()<1, NORM_ELEMS, 1024>();
  }
  if (H <= 256) return f.template operator()<V, 8 / V, 32>();
  if (H <= 32 * NORM_ELEMS) return f.template operator()<V, NORM_ELEMS / V, 32>();
  if (H <= 256 * NORM_ELEMS) return f.template operator()<V, NORM_ELEMS / V, 256>();
  if constexpr (V == 8)
    if (H <= 384 * NORM_ELEMS) return f.template operator()<V, NORM_ELEMS / V, 384>();
  if (H <= 512 * NORM_ELEMS) return f.template operator()<V, NORM_ELEMS / V, 512>();
  return f.template operator()<V, NORM_ELEMS / V, 1024>();
}

template <bool BACK, typename T>
struct NormLaunch {
  const b200_norm_args& a;
  int sms;
  cudaStream_t st;
  template <int VEC, int VPT, int MAXT>
  int operator()() const { return static_cast<int>(norm_launch<BACK, T, VEC, VPT, MAXT>(a, sms, st)); }
};
template <typename T>
static int norm_dispatch(bool back, const b200_norm_args& a, int sms, cudaStream_t st) {
  return back ? norm_variant<T>(a.H, a.aligned != 0, NormLaunch<true, T>{a, sms, st})
              : norm_variant<T>(a.H, a.aligned != 0, NormLaunch<false, T>{a, sms, st});
}

// The most rows that a backward pass has in work at once.
struct NormPartsOf {
  int T, H, sms;
  template <int VEC, int VPT, int MAXT>
  int operator()() const { return norm_parts<true, MAXT>(T, norm_row_threads<MAXT>(H, VEC, VPT), 0, sms); }
};

template <bool BACK>
static int norm_run(const b200_norm_args* a, int sms, void* stream) {
  if (a == nullptr || sms < 1 || a->T < 1 || a->T > NORM_MAX_ROWS || a->H < 1 || a->H > NORM_MAX_H || a->y == nullptr || a->gate_kind < 0 || a->gate_kind > 3) return -10;
  if ((a->gate_kind != 0 && (a->gate == nullptr || a->res == nullptr)) || (a->w2 != nullptr && a->res == nullptr)) return -11;
  if (!BACK && (a->h == nullptr || (a->w2 != nullptr && a->n == nullptr))) return -12;
  if (BACK && ((a->norm && a->r1 == nullptr) || (a->dn != nullptr && (a->r2 == nullptr || a->w2 == nullptr)))) return -13;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->elem) {
    case ELEM_F32: return norm_dispatch<float>(BACK, *a, sms, st);
    case ELEM_BF16: return norm_dispatch<__nv_bfloat16>(BACK, *a, sms, st);
    case ELEM_F16: return norm_dispatch<__half>(BACK, *a, sms, st);
  }
  return -14;
}

}  // namespace b200

extern "C" {

int b200_norm_forward(const b200_norm_args* a, int sms, void* stream) { return b200::norm_run<false>(a, sms, stream); }
// `partial` has 2 * b200_norm_parts() * H floats where dw, dw2 or the gradient of a gate per column is asked for.
int b200_norm_backward(const b200_norm_args* a, int sms, void* stream) { return b200::norm_run<true>(a, sms, stream); }

int b200_norm_parts(int T, int H, int elem, int aligned, int sms) {
  using namespace b200;
  const NormPartsOf f{T, H, sms};
  return elem == ELEM_F32 ? norm_variant<float>(H, aligned != 0, f) : norm_variant<__half>(H, aligned != 0, f);
}

int b200_abi_size_norm_args() { return static_cast<int>(sizeof(b200_norm_args)); }
int b200_norm_max_columns() { return b200::NORM_MAX_H; }

}  // extern "C"
