// Matrix products with bias, activation and residual in their epilogue, dense or with one weight per group of packed
// rows, and their backward products, on tcgen05 tensor cores.
//
//   forward   z_g = x_g W_g^T + b_g,  y = act(z) + res          x [M, K], W [G, N, K]
//   dX        dx_g = dz_g W_g                                    dz = dy act'(z), [M, N]
//   dW        dW_g = dz_g^T x_g                                  db_g = column sums of dz_g
//
// Few rows per group: the weights are streamed once for all of them, with tokens on the narrow side of the MMA and the work
// cut into equal shares (see linear_rows_kernel).
//
// Otherwise one persistent kernel for the three products: warp 0 loads (TMA), warp 1 issues the MMAs, warps 2-5 drain the
// accumulators, warps 6-7 mend ragged ends.  An operand whose contracted dimension is contiguous is K-major
// (x and W forward, dz for dX); the others (W for dX, both of dW) are read as they lie in memory, MN-major, in boxes of 64
// columns x 64 contracted rows, so that nothing is ever transposed in memory.
//
// dW contracts over a group's rows, whose end lies anywhere inside a block of 64.  The last block is multiplied as far as it
// has rows, in steps of 16; the rows of the last step that belong to the next group (or to nothing) are set to zero in
// shared memory, in both operands, so that what lies there, infinities and NaN included, has no part in the product.  Such a
// block is loaded first and multiplied third, which hides the mending (64 groups of 1023 rows: 612 us, 631 when it came last;
// 603 for 1024 rows, which need none).
//
// The pre-activations z are kept for the backward pass, of bf16 products as fp16 under a power of two that 32 columns of a row share,
// kept in a byte: off by 2^-11 |z|, and by 2^-30 in absolute terms.  fp16 spans too little for 32 columns that hold both a value of
// 1024 or more and one 2^31 times smaller than it: those are kept as bf16, off by 2^-8 |z| whatever the size (beside
// 1e12, a 1 under a shared power of two would be kept as nothing, and its slope and its products with it).  (Kept as bf16
// throughout, dX and dW of a gated bf16 product are 3.0e-3 off instead of 2.4e-3, relative; 1.7e-3 is what rounding the result
// alone costs.)  Of fp16 products z is the upper 24 bits of the fp32 sum, 16 of them in z and a byte beside it: off by 2^-15 |z|.
// (With 11 bits, dX and dW of a gated fp16 product were 3.7e-4 off instead of 3.0e-4, which is what rounding dz and the result costs;
// the result alone 2.1e-4.)
// dz is rounded to the element type, since the tensor cores multiply 16-bit values: at most half a step of each value, which
// averages out over the contracted dimension.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <atomic>
#include <type_traits>

#include "elementwise.cuh"
#include "launch.h"
#include "moe_args.h"
#include "sm100_ptx.cuh"
#include "tile_order.cuh"

extern "C" {
typedef struct b200_linear_args {
  const void* a;            // forward: x [M, K]; dX: dz [M, N]; dW: dz [M, N]
  const void* b;            // forward, dX: W [G, N, K]; dW: x [M, K]
  void* out;                // y [M, n_out]; dx [M, K]; dW [G, N, K]
  void* z;                  // forward: [M, N] of 16 bits or null; what they are, zexp says
  unsigned char* zexp;      // with z, bf16: [M][ceil(N / 256) * 8], exponents of 32 columns each; fp16: [M][ceil(N / 256) * 256], z's next 8 bits
  const void* bias;         // [G, N] or null
  union {
    const void* res;            // forward: [M, n_out] or null
    const unsigned int* peak;   // dX, dW: what dz is under a power of two by (see dz_shift), or null: it is as it is
  };
  const int* group_rows;    // [G] or null: one group of all M rows
  int* status;
  unsigned long long wait_budget_ns;
  int mode;                 // LinearMode
  int G, M, N, K, n_out;
  int elem;                 // ELEM_BF16 or ELEM_F16
  int act;                  // LinearAct
  int pair;                 // two CTAs per tile (256 rows)
  int group_m;              // M-tiles per chunk (see decode_tile)
  float* record;            // split product: scratch of b200_linear_record_floats(); null: whole tiles
} b200_linear_args;

typedef struct b200_act_grad_args {
  const void* dy;           // [M, n_out]
  const void* z;            // [M, N] as the forward product left it, or null (no activation)
  const unsigned char* zexp;   // as the forward product left it
  void* dz;                 // [M, N] or null (no activation: dz is dy)
  void* dres;               // [M, n_out] or null: dy of the groups' rows, zero behind them
  void* dbias;              // [G, N] or null
  float* record;            // [chunks + G][N] sums over the rows of a group in a chunk
  const int* group_rows;
  unsigned int* peak;       // fp16 with an activation: [1], left for the products of dz
  int G, M, N, n_out, elem, act;
  int chunks, chunk_rows;
} b200_act_grad_args;
}

namespace b200 {

enum LinearMode : int { LIN_FORWARD = 0, LIN_DX = 1, LIN_DW = 2 };
enum LinearAct : int { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_SILU_GATE = 4 };

constexpr int LBM = 128;                 // rows of a tile per CTA
constexpr int LBN = 256;                 // columns of a tile
constexpr int LBK = 64;                  // contracted elements per stage
constexpr int LIN_THREADS = 256;
constexpr int LIN_MENDERS = 2;           // warps 6 and 7
constexpr int LIN_MAX_ROWS = 0x7fffffff - 1023;      // a last tile that is partly empty still has row numbers of 32 bits
constexpr int LIN_A_BYTES = LBM * LBK * 2;
constexpr int LIN_MN_BOX = 64 * LBK * 2; // bytes of one MN-major box
constexpr int LIN_BOX = 32 * 128;        // a warp's staging box: 32 rows x 64 columns, 16-byte chunks XOR-swizzled by row

// Stages and staging boxes per variant.  An epilogue warp's boxes form a ring, so that it fills one while bulk stores still
// read others (with one box, a 256 x 256 tile took 3.2 us to drain).  Forward, a pass fills up to three (z of the
// gate, z of the up half, y).
template <int MODE, int CG>
struct LinGeo {
  static constexpr int B_ROWS = LBN / CG;
  static constexpr int B_BYTES = B_ROWS * LBK * 2;
  static constexpr int STAGE = LIN_A_BYTES + B_BYTES;
  static constexpr int BOXES = MODE == LIN_FORWARD ? 4 : 2;
  static constexpr int STAGES = CG == 2 ? (MODE == LIN_FORWARD ? 5 : 6) : (MODE == LIN_FORWARD ? 3 : 4);
  static constexpr int TM = LBM * CG;
};
constexpr int LIN_MAX_STAGES = 6;

struct __align__(16) LinControl {
  uint64_t full[LIN_MAX_STAGES], empty[LIN_MAX_STAGES];
  uint64_t part_full[LIN_MAX_STAGES];    // dW: this CTA's own bytes of a block that has to be mended
  uint64_t mended[LIN_MAX_STAGES];       // dW: both CTAs have mended theirs
  uint64_t tmem_full[2], tmem_empty[2], drain;
  uint32_t tmem_base;
  int abort_flag;
  int g_rows[B200_MAX_GROUPS];
  int g_row_start[B200_MAX_GROUPS + 1];
  int g_sched_start[B200_MAX_GROUPS + 1];
};
template <int MODE, int CG>
constexpr int lin_smem() {
  using S = LinGeo<MODE, CG>;
  return S::STAGES * S::STAGE + 4 * S::BOXES * LIN_BOX + static_cast<int>(sizeof(LinControl)) + 1024;
}
static_assert(lin_smem<LIN_FORWARD, 1>() <= 232448 && lin_smem<LIN_FORWARD, 2>() <= 232448 && lin_smem<LIN_DW, 1>() <= 232448 &&
                  lin_smem<LIN_DW, 2>() <= 232448, "exceeds 227 KiB of shared memory per CTA");

// q = 1 / (1 + exp(-v)): 1 - q, and q where v is negative, are off by up to 2^-21 + 1.3 |v| 2^-24, relative (the rounding of the
// exponent, log2(e) v, grows with it), which is 2^-17 where fp32 ends.  A 16-bit result is rounded to 2^-11.
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_approx(1.f + exp2_approx(__fmul_rn(-LOG2_E, v))); }
constexpr float GELU_A = 2.f * 0.7978845608028654f, GELU_B = GELU_A * 0.044715f;    // tanh form: v * sigmoid(A v + B v^3)
// The products are rounded before anything is added to them, so that a result does not depend on what else its kernel
// keeps or adds.
__device__ __forceinline__ float act_value(float v, int act) {
  if (act == ACT_RELU) return v < 0.f ? 0.f : v;
  if (act == ACT_SILU) return __fmul_rn(v, sigmoid_f(v));
  if (act == ACT_GELU) return __fmul_rn(v, sigmoid_f(v * fmaf(GELU_B, v * v, GELU_A)));
  return v;
}
__device__ __forceinline__ float gated_value(float gate, float up) { return __fmul_rn(__fmul_rn(gate, sigmoid_f(gate)), up); }
// Slopes, from q and 1 - q: the difference's rounding, 2^-24, is multiplied with v only while q is not yet 1.
__device__ __forceinline__ float silu_slope(float v, float q) { return q * fmaf(v, 1.f - q, 1.f); }
__device__ __forceinline__ float act_slope(float v, int act) {
  if (act == ACT_RELU) return v > 0.f ? 1.f : 0.f;
  if (act == ACT_SILU) return silu_slope(v, sigmoid_f(v));
  v = v > 50.f ? 50.f : v < -50.f ? -50.f : v;         // 1 and 0 from there on, and the powers of v stay finite
  const float vv = v * v, q = sigmoid_f(v * fmaf(GELU_B, vv, GELU_A));
  return q * fmaf(v * fmaf(3.f * GELU_B, vv, GELU_A), 1.f - q, 1.f);
}

// z of bf16 products, in fp16 under a shared power of two: E is the largest finite magnitude's exponent (biased, 15 at least), the
// values are scaled into [0, 2^15], where fp16 has 11 bits down to 2^-14, 8 down to 2^-17 and an absolute error of 2^-25.
// Infinities and NaN stay what they are; so near to fp32's largest value that rounding reaches 2^128, z becomes infinite.
// Scales of 2^-5 and below (E >= 137: a value of 1024) leave an absolute error that ordinary values may feel: there, where the
// smallest that is not zero lies below the 8 bits, the values are bf16, and the byte is Z_BF16.
constexpr int Z_BF16 = 255;
__device__ __forceinline__ int shared_exponent(uint32_t largest_finite_bits) { return max(15, static_cast<int>(largest_finite_bits >> 23)); }
__device__ __forceinline__ float z_scale(int E) { return __uint_as_float(static_cast<uint32_t>(268 - E) << 23); }      // 2^(141 - E)
__device__ __forceinline__ float z_unscale(int E) { return __uint_as_float(static_cast<uint32_t>(E - 14) << 23); }    // 2^(E - 141)
__device__ __forceinline__ bool z_spans_much(int E, float smallest) { return E >= 137 && smallest * z_scale(E) < 0x1p-17f; }
__device__ __forceinline__ long long zexp_pitch(int N) { return (N + 255) / 256 * 8; }
// Of fp16 products: the upper 16 bits of fp32 values beside each other, and the 8 bits below of four values.  (Cut, not
// rounded, so that infinities and NaN stay what they are.)
__device__ __forceinline__ long long zlow_pitch(int N) { return (N + 255) / 256 * 256; }
__device__ __forceinline__ uint32_t upper_halves(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
__device__ __forceinline__ uint32_t lower_bytes(const uint32_t* x) {
  return __byte_perm(__byte_perm(x[0], x[1], 0x0051), __byte_perm(x[2], x[3], 0x0051), 0x5410);
}

// dz of fp16 products: the tensor cores take it in 16 bits like the weights and x that it is multiplied with, off by 2^-11 |dz|
// and 2^-25 in absolute terms.  (Of bf16, by 2^-8 |dz| at any size.)  Where a call's largest finite |dz| (its fp32 bits are `peak`)
// would round to infinity, or is below 2^-10, so that what is lost below 2^-25 would count, dz is multiplied with the power of two that
// takes the largest into [2^14, 2^15), and the products are multiplied back before they are rounded.  Returned is the power's
// negative exponent.  It stays at 10 at most: a single value of 2^26 may not take the bits of all others.
constexpr float DZ_LARGEST = 65520.f;      // rounds to infinity
__device__ __forceinline__ int dz_shift(unsigned int peak) {
  const int E = static_cast<int>(peak >> 23);
  if (__uint_as_float(peak) >= DZ_LARGEST) return min(E - 141, 10);
  return peak != 0u && E < 117 ? max(E - 141, -100) : 0;
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

__device__ __forceinline__ uint32_t pack_16(float lo, float hi, bool bf16) {
  if (bf16) return pack_bf16x2(lo, hi);
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float2 unpack_16(uint32_t v, bool bf16) {
  if (bf16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

struct LinTables {
  int *g_rows, *g_row_start, *g_sched_start;
};
// Rows and first row of every group, and its first scheduling tile (tiles per group: by its rows, or `fixed`).  One warp.
// Returns the rows of all groups.
__device__ __forceinline__ long long lin_scan(const LinTables& c, const int* group_rows, int G, int M, int lane, int tile_rows, int fixed) {
  long long carry = 0;
  int tcarry = 0;
  for (int base = 0; base < G; base += 32) {
    const int g = base + lane;
    const int rows = g < G ? (group_rows != nullptr ? max(0, group_rows[g]) : M) : 0;
    const int tiles = g < G ? (fixed > 0 ? fixed : (rows + tile_rows - 1) / tile_rows) : 0;
    long long rs = rows;
    int ts = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long r2 = __shfl_up_sync(0xffffffffu, rs, o);
      const int t2 = __shfl_up_sync(0xffffffffu, ts, o);
      if (lane >= o) { rs += r2; ts += t2; }
    }
    if (g < G) {
      c.g_rows[g] = rows;
      c.g_row_start[g] = static_cast<int>(min(carry + rs - rows, 0x7fffffffll));
      c.g_sched_start[g] = tcarry + ts - tiles;
    }
    carry += __shfl_sync(0xffffffffu, rs, 31);
    tcarry += __shfl_sync(0xffffffffu, ts, 31);
  }
  if (lane == 0) {
    c.g_row_start[G] = static_cast<int>(min(carry, 0x7fffffffll));
    c.g_sched_start[G] = tcarry;
  }
  return carry;
}

// Writes one staging box: 32 rows x 64 columns at (row, col) of a row-major matrix.  Whole boxes leave as one bulk tensor
// store, others row segment by row segment; either way the box is one bulk group of lane 0.
__device__ __forceinline__ void store_box(const uint8_t* box, const CUtensorMap* tmap, char* base, long long ld_bytes, long long row,
                                          int col, int cols, int rows_here, int lane) {
  if (rows_here >= 32) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0 && col < cols) tma_store_2d(tmap, box, col, static_cast<int>(row));
  } else {
    __syncwarp();
    const int c = col + (lane & 7) * 8;
#pragma unroll
    for (int rr = 0; rr < 8; ++rr) {
      const int r = rr * 4 + (lane >> 3);
      if (r < rows_here && c < cols)
        st_16(base + (row + r) * ld_bytes + c * 2ll, *reinterpret_cast<const uint4*>(box + r * 128 + (((lane & 7) ^ (r & 7)) << 4)));
    }
  }
  if (lane == 0) bulk_commit_group();
}

// Z24: how z is kept, of fp16 products (forward).
template <int MODE, int CG, bool GATED, bool Z24>
__global__ void __launch_bounds__(LIN_THREADS, 1)
linear_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
              const __grid_constant__ CUtensorMap tmap_o, const __grid_constant__ CUtensorMap tmap_z, const b200_linear_args la) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  using S = LinGeo<MODE, CG>;
  constexpr int STAGES = S::STAGES;
  constexpr bool A_MN = MODE == LIN_DW, B_MN = MODE != LIN_FORWARD;
  uint8_t* staging = smem + STAGES * S::STAGE;
  LinControl& c = *reinterpret_cast<LinControl*>(staging + 4 * S::BOXES * LIN_BOX);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = la.G;
  const uint32_t cta_rank = CG == 2 ? cluster_ctarank() : 0u;
  const bool bf16 = la.elem == ELEM_BF16;
  // the product's own sizes: rows of a tile's group (dW: features), columns, contracted length of a group
  const int cols = MODE == LIN_FORWARD ? la.N : la.K;
  const int TN = (cols + LBN - 1) / LBN;

  WaitCtx w;
  w.abort_flag = &c.abort_flag;
  w.status = la.status;
  w.budget_ns = la.wait_budget_ns;

  if (tid == 0) {
    c.abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&c.full[s], 1);
      mbar_init(&c.empty[s], 1);
      mbar_init(&c.part_full[s], 1);
      mbar_init(&c.mended[s], LIN_MENDERS * CG);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&c.tmem_full[a], 1);
      mbar_init(&c.tmem_empty[a], 128 * CG);
    }
    mbar_init(&c.drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    tma_prefetch_desc(&tmap_o);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_pair(&c.tmem_base, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&c.tmem_base, 512);
      tmem_relinquish();
    }
  }
  __syncthreads();                      // abort_flag is set below
  if (warp == 0) {
    const LinTables tables{c.g_rows, c.g_row_start, c.g_sched_start};
    const long long rows = lin_scan(tables, la.group_rows, G, la.M, lane, S::TM, MODE == LIN_DW ? (la.N + S::TM - 1) / S::TM : 0);
    // more rows than the buffers hold: nothing is computed, the host reads the status
    if (lane == 0 && rows > la.M) {
      report_status(w.status, ST_OVERFLOW);
      if (w.status != nullptr) atomicMax(w.status + 1, c.g_row_start[G]);
      c.abort_flag = 1;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();      // the peer's barriers exist before anyone signals them
  tc_fence_after_sync();

  const uint32_t tmem_base = c.tmem_base;
  const bool overflow = c.abort_flag != 0;
  const int total_tiles = overflow ? 0 : c.g_sched_start[G] * TN;
  int tile_first, tile_stride;
  tile_walk(total_tiles, gridDim.x / CG, blockIdx.x / CG, tile_first, tile_stride);
  // every role reads the flag above before any of them may set it
  __syncthreads();

  // blocks of the contracted dimension in a tile of group g
  auto k_blocks = [&](int g) { return ((MODE == LIN_FORWARD ? la.K : MODE == LIN_DX ? la.N : c.g_rows[g]) + LBK - 1) / LBK; };
  // dW: contracted rows in the last block of group g (64: whole); a number that is no multiple of 16 has to be mended
  auto tail_rows = [&](int g) { return MODE == LIN_DW ? ((c.g_rows[g] - 1) & (LBK - 1)) + 1 : LBK; };

  if (warp == 0) {
    // ------------------------------------------------------------ loads
    if (lane == 0) {
      int cursor = 0, stage = 0, issued = 0;
      uint32_t phase = 0, part_phase = 0, part_used = 0;      // a bit per stage
      bool ok = true;
      for (int idx = tile_first; ok && idx < total_tiles; idx += tile_stride) {
        int g, m, n;
        if (!decode_tile(c, G, TN, la.group_m, idx, cursor, g, m, n)) break;
        const int KB = k_blocks(g);
        const bool ragged = MODE == LIN_DW && tail_rows(g) % 16 != 0;
        const int mrow = m * S::TM + static_cast<int>(cta_rank) * LBM;      // first row (dW: feature) of my half
        const int ncol = n * LBN + static_cast<int>(cta_rank) * S::B_ROWS;  // first column of my share of B
        const int row0 = c.g_row_start[g];
        for (int pos = 0; pos < KB; ++pos) {
          const int kb = !ragged ? pos : pos == 0 ? KB - 1 : pos - 1;
          if (!mbar_wait(&c.empty[stage], phase ^ 1u, w, ST_TIMEOUT_PIPE_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * S::STAGE;
          uint8_t* sb = sa + LIN_A_BYTES;
          const bool part = MODE == LIN_DW && ragged && pos == 0;
          if (part) {
            // this CTA's bytes go to its own barrier; the pair's goes on at once, the MMAs wait for `mended`
            if (cta_rank == 0) mbar_arrive(&c.full[stage]);
            mbar_expect_tx(&c.part_full[stage], S::STAGE);
#pragma unroll
            for (int i = 0; i < LBM / 64; ++i)
              tma_load_2d(sa + i * LIN_MN_BOX, &tmap_a, &c.part_full[stage], mrow + i * 64, row0 + kb * LBK);
#pragma unroll
            for (int i = 0; i < S::B_ROWS / 64; ++i)
              tma_load_2d(sb + i * LIN_MN_BOX, &tmap_b, &c.part_full[stage], ncol + i * 64, row0 + kb * LBK);
            part_phase ^= 1u << stage;
            part_used |= 1u << stage;
          } else if constexpr (CG == 2) {
            if (cta_rank == 0) mbar_expect_tx(&c.full[stage], S::STAGE * 2);
            const uint32_t bar = map_to_cta(&c.full[stage], 0);
            if constexpr (A_MN) {
#pragma unroll
              for (int i = 0; i < LBM / 64; ++i) tma_load_2d_pair(sa + i * LIN_MN_BOX, &tmap_a, bar, mrow + i * 64, row0 + kb * LBK);
            } else {
              tma_load_2d_pair(sa, &tmap_a, bar, kb * LBK, row0 + mrow);
            }
            if constexpr (MODE == LIN_FORWARD) {
              tma_load_2d_pair(sb, &tmap_b, bar, kb * LBK, g * la.N + ncol);
            } else {
#pragma unroll
              for (int i = 0; i < S::B_ROWS / 64; ++i) {
                if constexpr (MODE == LIN_DX) tma_load_3d_pair(sb + i * LIN_MN_BOX, &tmap_b, bar, ncol + i * 64, kb * LBK, g);
                else tma_load_2d_pair(sb + i * LIN_MN_BOX, &tmap_b, bar, ncol + i * 64, row0 + kb * LBK);
              }
            }
          } else {
            mbar_expect_tx(&c.full[stage], S::STAGE);
            if constexpr (A_MN) {
#pragma unroll
              for (int i = 0; i < LBM / 64; ++i) tma_load_2d(sa + i * LIN_MN_BOX, &tmap_a, &c.full[stage], mrow + i * 64, row0 + kb * LBK);
            } else {
              tma_load_2d(sa, &tmap_a, &c.full[stage], kb * LBK, row0 + mrow);
            }
            if constexpr (MODE == LIN_FORWARD) {
              tma_load_2d(sb, &tmap_b, &c.full[stage], kb * LBK, g * la.N + ncol);
            } else {
#pragma unroll
              for (int i = 0; i < S::B_ROWS / 64; ++i) {
                if constexpr (MODE == LIN_DX) tma_load_3d(sb + i * LIN_MN_BOX, &tmap_b, &c.full[stage], ncol + i * 64, kb * LBK, g);
                else tma_load_2d(sb + i * LIN_MN_BOX, &tmap_b, &c.full[stage], ncol + i * 64, row0 + kb * LBK);
              }
            }
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
      }
      // Retire the loads still in flight before shared memory is released.  The pair leader's barriers account for both
      // CTAs' loads; blocks to be mended are on each CTA's own.
      int no_abort = 0;
      WaitCtx wd = w;
      wd.abort_flag = &no_abort;
      const int behind = CG == 2 && cta_rank != 0 ? 0 : min(issued, STAGES);
      for (int i = 0; i < behind; ++i) {
        int s = stage - 1 - i;
        uint32_t ph = phase;
        if (s < 0) { s += STAGES; ph ^= 1u; }
        mbar_wait(&c.full[s], ph, wd, ST_TIMEOUT_DRAIN);
      }
      for (int s = 0; s < STAGES; ++s)
        if (part_used >> s & 1u) mbar_wait(&c.part_full[s], (part_phase >> s & 1u) ^ 1u, wd, ST_TIMEOUT_DRAIN);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs
    if (lane == 0 && cta_rank == 0) {
      const uint32_t idesc = make_idesc_16bit(S::TM, LBN, bf16, A_MN, B_MN);
      int cursor = 0, stage = 0, it = 0;
      uint32_t phase = 0, mend_phase = 0;
      bool ok = true;
      for (int idx = tile_first; ok && idx < total_tiles; idx += tile_stride, ++it) {
        int g, m, n;
        if (!decode_tile(c, G, TN, la.group_m, idx, cursor, g, m, n)) break;
        const int KB = k_blocks(g);
        const int tail = tail_rows(g);
        const int acc = it & 1;
        if (!mbar_wait(&c.tmem_empty[acc], ((it >> 1) & 1) ^ 1u, w, ST_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + acc * LBN;
        // a block to be mended lies first and is taken after the next two
        const bool ragged = MODE == LIN_DW && tail % 16 != 0;
        const int third = min(2, KB - 1), stage0 = stage;
        const uint32_t phase0 = phase;
        for (int j = 0; j < KB; ++j) {
          int s = stage;
          uint32_t ph = phase;
          bool last = MODE == LIN_DW && !ragged && j == KB - 1;
          if (ragged && j <= third) {
            last = j == third;
            s = stage0 + (last ? 0 : j + 1);
            ph = phase0;
            if (s >= STAGES) { s -= STAGES; ph ^= 1u; }
          }
          if (!mbar_wait(&c.full[s], ph, w, ST_TIMEOUT_PIPE_FULL)) { ok = false; break; }
          if (ragged && last) {
            if (!mbar_wait_cluster(&c.mended[s], mend_phase >> s & 1u, w, ST_TIMEOUT_PIPE_FULL)) { ok = false; break; }
            mend_phase ^= 1u << s;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + s * S::STAGE), sb = sa + LIN_A_BYTES;
          const uint64_t ad = A_MN ? make_smem_desc_mn_sw128(sa, LIN_MN_BOX) : make_smem_desc_sw128(sa);
          const uint64_t bd = B_MN ? make_smem_desc_mn_sw128(sb, LIN_MN_BOX) : make_smem_desc_sw128(sb);
          // 16 steps of K: 32 bytes along a K-major row, 2048 bytes down an MN-major box
          constexpr int ASTEP = A_MN ? 2048 / 16 : 2, BSTEP = B_MN ? 2048 / 16 : 2;
#pragma unroll
          for (int k = 0; k < LBK / 16; ++k) {
            if (last && k * 16 >= tail) continue;
            if constexpr (CG == 2) umma_bf16_ss_pair(d, ad + ASTEP * k, bd + BSTEP * k, idesc, (j | k) != 0 ? 1u : 0u);
            else umma_bf16_ss(d, ad + ASTEP * k, bd + BSTEP * k, idesc, (j | k) != 0 ? 1u : 0u);
          }
          if constexpr (CG == 2) umma_commit_pair(&c.empty[s], 3);
          else umma_commit(&c.empty[s]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        if constexpr (CG == 2) umma_commit_pair(&c.tmem_full[acc], 3);
        else umma_commit(&c.tmem_full[acc]);
      }
      if constexpr (CG == 2) umma_commit_pair(&c.drain, 1);
      else umma_commit(&c.drain);
      int no_abort = 0;
      WaitCtx wd = w;
      wd.abort_flag = &no_abort;
      mbar_wait(&c.drain, 0, wd, ST_TIMEOUT_DRAIN);
    }
  } else if (warp < 6) {
    // ------------------------------------------------------------ epilogue
    constexpr int OUT_TILE = GATED ? LBN / 2 : LBN;
    const int q = warp & 3;                            // TMEM lane quarter this warp may read
    uint8_t* boxes = staging + q * S::BOXES * LIN_BOX;
    int ring = 0;                                      // the next box
    const bool save_z = MODE == LIN_FORWARD && la.z != nullptr;
    float unshift = 1.f;
    if constexpr (MODE != LIN_FORWARD)
      if (la.peak != nullptr) unshift = power_of_two(dz_shift(*la.peak));
    auto take_box = [&]() {
      uint8_t* box = boxes + ring * LIN_BOX;
      ring = ring + 1 == S::BOXES ? 0 : ring + 1;
      return box;
    };
    int cursor = 0, it = 0;
    const uint32_t empty_addr[2] = {map_to_cta(&c.tmem_empty[0], 0), map_to_cta(&c.tmem_empty[1], 0)};
    for (int idx = tile_first; idx < total_tiles; idx += tile_stride, ++it) {
      int g, m, n;
      if (!decode_tile(c, G, TN, la.group_m, idx, cursor, g, m, n)) break;
      const int acc = it & 1;
      const int half0 = m * S::TM + static_cast<int>(cta_rank) * LBM + q * 32;     // this warp's first row in the group
      const int rows_here = (MODE == LIN_DW ? la.N : c.g_rows[g]) - half0;         // may be <= 0
      const long long row0 = MODE == LIN_DW ? static_cast<long long>(g) * la.N + half0 : c.g_row_start[g] + half0;
      const bool zero = MODE == LIN_DW && c.g_rows[g] == 0;
      const bool got = mbar_wait(&c.tmem_full[acc], (it >> 1) & 1, w, ST_TIMEOUT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after_sync();
      const uint32_t t_acc = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * LBN;
      const bool row_ok = lane < rows_here;
      unsigned long long exponents = 0;                // of this row's eight chunks of 32 columns
#pragma unroll 1
      for (int p = 0; p < OUT_TILE / 64; ++p) {
        const int ycol = n * OUT_TILE + p * 64;        // first output column of the pass
        // of the boxes of this pass, the stores that read them last are done
        if (lane == 0) {
          if (!save_z) bulk_wait_group_read<S::BOXES - 1>();
          else if (GATED) bulk_wait_group_read<(S::BOXES > 2 ? S::BOXES - 3 : 0)>();
          else bulk_wait_group_read<S::BOXES - 2>();
        }
        __syncwarp();
        uint8_t* ybox = take_box();
        uint8_t* zbox = save_z ? take_box() : nullptr;
        uint8_t* ubox = save_z && GATED ? take_box() : nullptr;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int cc = p * 64 + h * 32;
          uint32_t v[32];
          tmem_ld_32x32b_x32(t_acc + cc, v);
          uint32_t u[GATED ? 32 : 1];
          if constexpr (GATED) tmem_ld_32x32b_x32(t_acc + LBN / 2 + cc, u);
          tmem_ld_wait();
          if (zero) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
          }
          if constexpr (MODE != LIN_FORWARD) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * unshift);
          } else {
            const int zcol = n * LBN + cc;             // column of z (of the gate half)
            auto add_bias = [&](uint32_t (&x)[32], int col) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (col + i * 8 >= la.N) continue;
                const uint4 b = *reinterpret_cast<const uint4*>(static_cast<const char*>(la.bias) + (static_cast<size_t>(g) * la.N + col + i * 8) * 2);
                const uint32_t bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float2 f = unpack_16(bb[j], bf16);
                  x[i * 8 + 2 * j] = __float_as_uint(__uint_as_float(x[i * 8 + 2 * j]) + f.x);
                  x[i * 8 + 2 * j + 1] = __float_as_uint(__uint_as_float(x[i * 8 + 2 * j + 1]) + f.y);
                }
              }
            };
            if (la.bias != nullptr) {
              add_bias(v, zcol);
              if constexpr (GATED) add_bias(reinterpret_cast<uint32_t(&)[32]>(u), zcol + LBN / 2);
            }
            if (save_z) {
              auto put = [&](const uint32_t (&x)[32], uint8_t* box, int col, int chunk) {
                if constexpr (Z24) {
                  uint32_t low[8];
#pragma unroll
                  for (int i = 0; i < 8; ++i) low[i] = lower_bytes(x + 4 * i);
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(box + lane * 128 + (((h * 4 + i) ^ (lane & 7)) << 4)) =
                        make_uint4(upper_halves(x[8 * i], x[8 * i + 1]), upper_halves(x[8 * i + 2], x[8 * i + 3]),
                                   upper_halves(x[8 * i + 4], x[8 * i + 5]), upper_halves(x[8 * i + 6], x[8 * i + 7]));
                  if (!row_ok) return;
                  uint4* bytes = reinterpret_cast<uint4*>(la.zexp + (row0 + lane) * zlow_pitch(la.N) + col);
                  bytes[0] = make_uint4(low[0], low[1], low[2], low[3]);
                  bytes[1] = make_uint4(low[4], low[5], low[6], low[7]);
                  return;
                }
                float m = 0.f;
#pragma unroll
                for (int i = 0; i < 32; ++i)
                  if (col + (i & ~7) < la.N) m = fmaxf(m, fabsf(__uint_as_float(x[i])));
                if (m > 3.402823466e38f) {             // an infinity: the largest of the others
                  m = 0.f;
                  for (int i = 0; i < 32; ++i) {
                    const float f = fabsf(__uint_as_float(x[i]));
                    if (col + (i & ~7) < la.N && f <= 3.402823466e38f) m = fmaxf(m, f);
                  }
                }
                int E = shared_exponent(__float_as_uint(m));
                if (E >= 137) {                        // rare
                  float least = m;
                  for (int i = 0; i < 32; ++i) {
                    const float f = fabsf(__uint_as_float(x[i]));
                    if (col + (i & ~7) < la.N && f > 0.f) least = fminf(least, f);
                  }
                  if (z_spans_much(E, least)) E = Z_BF16;
                }
                exponents |= static_cast<unsigned long long>(E) << (8 * chunk);
                auto fill = [&](float s, bool as_bf16) {
#pragma unroll
                  for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<uint4*>(box + lane * 128 + (((h * 4 + i) ^ (lane & 7)) << 4)) =
                        make_uint4(pack_16(__uint_as_float(x[8 * i]) * s, __uint_as_float(x[8 * i + 1]) * s, as_bf16),
                                   pack_16(__uint_as_float(x[8 * i + 2]) * s, __uint_as_float(x[8 * i + 3]) * s, as_bf16),
                                   pack_16(__uint_as_float(x[8 * i + 4]) * s, __uint_as_float(x[8 * i + 5]) * s, as_bf16),
                                   pack_16(__uint_as_float(x[8 * i + 6]) * s, __uint_as_float(x[8 * i + 7]) * s, as_bf16));
                };
                if (E != Z_BF16) fill(z_scale(E), false);
                else fill(1.f, true);
              };
              put(v, zbox, zcol, p * 2 + h);
              if constexpr (GATED) put(reinterpret_cast<uint32_t(&)[32]>(u), ubox, zcol + LBN / 2, 4 + p * 2 + h);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float f = __uint_as_float(v[i]);
              if constexpr (GATED) v[i] = __float_as_uint(gated_value(f, __uint_as_float(u[i])));
              else v[i] = __float_as_uint(act_value(f, la.act));
            }
            if (la.res != nullptr && row_ok) {
              const int col = ycol + h * 32;
              const char* src = static_cast<const char*>(la.res) + ((row0 + lane) * la.n_out + col) * 2;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                if (col + i * 8 >= la.n_out) continue;
                const uint4 b = ld_16(src + i * 16);
                const uint32_t bb[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const float2 f = unpack_16(bb[j], bf16);
                  v[i * 8 + 2 * j] = __float_as_uint(__uint_as_float(v[i * 8 + 2 * j]) + f.x);
                  v[i * 8 + 2 * j + 1] = __float_as_uint(__uint_as_float(v[i * 8 + 2 * j + 1]) + f.y);
                }
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(ybox + lane * 128 + (((h * 4 + i) ^ (lane & 7)) << 4)) =
                make_uint4(pack_16(__uint_as_float(v[8 * i]), __uint_as_float(v[8 * i + 1]), bf16),
                           pack_16(__uint_as_float(v[8 * i + 2]), __uint_as_float(v[8 * i + 3]), bf16),
                           pack_16(__uint_as_float(v[8 * i + 4]), __uint_as_float(v[8 * i + 5]), bf16),
                           pack_16(__uint_as_float(v[8 * i + 6]), __uint_as_float(v[8 * i + 7]), bf16));
        }
        if (p == OUT_TILE / 64 - 1) {
          tc_fence_before_sync();
          if constexpr (CG == 2) mbar_arrive_cluster(empty_addr[acc]);
          else mbar_arrive(&c.tmem_empty[acc]);
        }
        store_box(ybox, &tmap_o, static_cast<char*>(la.out), static_cast<long long>(la.n_out) * 2, row0, ycol, la.n_out, rows_here, lane);
        if (save_z) {
          const long long ldz = static_cast<long long>(la.N) * 2;
          store_box(zbox, &tmap_z, static_cast<char*>(la.z), ldz, row0, n * LBN + p * 64, la.N, rows_here, lane);
          if constexpr (GATED)
            store_box(ubox, &tmap_z, static_cast<char*>(la.z), ldz, row0, n * LBN + LBN / 2 + p * 64, la.N, rows_here, lane);
        }
      }
      if (!Z24 && save_z && row_ok)
        *reinterpret_cast<unsigned long long*>(la.zexp + (row0 + lane) * zexp_pitch(la.N) + n * 8) = exponents;
    }
    if (lane == 0) bulk_wait_group<0>();               // shared memory stays allocated until the stores are done
  } else {
    // ------------------------------------------------------------ ragged ends
    if constexpr (MODE == LIN_DW) {
      int cursor = 0, blocks = 0;
      uint32_t phase = 0;
      for (int idx = tile_first; idx < total_tiles; idx += tile_stride) {
        int g, m, n;
        if (!decode_tile(c, G, TN, la.group_m, idx, cursor, g, m, n)) break;
        const int KB = k_blocks(g), stage = blocks % STAGES, tail = tail_rows(g);
        blocks += KB;
        if (KB == 0 || tail % 16 == 0) continue;
        const bool got = mbar_wait(&c.part_full[stage], phase >> stage & 1u, w, ST_TIMEOUT_PIPE_FULL);
        if (!__all_sync(0xffffffffu, got)) break;
        phase ^= 1u << stage;
        uint8_t* s = smem + stage * S::STAGE;
        constexpr int NBOX = S::STAGE / LIN_MN_BOX;
        // the rows from tail to the end of its step, of every box: whole 128-byte rows, which the swizzle does not leave
        const int chunks = (16 - tail % 16) * 8;
        for (int i = tid - 6 * 32; i < NBOX * chunks; i += LIN_MENDERS * 32) {
          const int box = i / chunks, r = i - box * chunks;
          *reinterpret_cast<uint4*>(s + box * LIN_MN_BOX + tail * 128 + r * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          if constexpr (CG == 2) mbar_arrive_cluster(map_to_cta(&c.mended[stage], 0));
          else mbar_arrive(&c.mended[stage]);
        }
      }
    } else if (!overflow) {
      // rows of the buffer behind the last group
      const long long first = static_cast<long long>(c.g_row_start[G]) * la.n_out / 8, last = static_cast<long long>(la.M) * la.n_out / 8;
      uint4* out = reinterpret_cast<uint4*>(la.out);
      const long long step = static_cast<long long>(gridDim.x) * LIN_MENDERS * 32;
      for (long long i = first + blockIdx.x * (LIN_MENDERS * 32) + tid - 6 * 32; i < last; i += step) out[i] = make_uint4(0, 0, 0, 0);
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    if constexpr (CG == 2) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

// The larger magnitude, of finite ones.
__device__ __forceinline__ float finite_max(float top, float v) {
  v = fabsf(v);
  return v <= 3.402823466e38f ? fmaxf(top, v) : top;
}
// Eight values of z as they were kept, with what belongs to them beside z.
template <typename T>
struct ZBeside;
template <>
struct ZBeside<__nv_bfloat16> {
  int e = 141;
  static __device__ __forceinline__ long long pitch(int N) { return zexp_pitch(N); }
  static __device__ __forceinline__ int column(int c) { return c / 32; }
  __device__ __forceinline__ void load(const unsigned char* p) { e = *p; }
  __device__ __forceinline__ void values(const Pack<__half, 8>& k, float (&v)[8]) const {
    if (e == Z_BF16) {
      unpack<__nv_bfloat16, 8>(*reinterpret_cast<const Pack<__nv_bfloat16, 8>*>(&k), v);
    } else {
      unpack<__half, 8>(k, v);
      v_mul<8>(v, v, z_unscale(e));
    }
  }
};
template <>
struct ZBeside<__half> {
  uint2 low = {0u, 0u};
  static __device__ __forceinline__ long long pitch(int N) { return zlow_pitch(N); }
  static __device__ __forceinline__ int column(int c) { return c; }
  __device__ __forceinline__ void load(const unsigned char* p) { low = *reinterpret_cast<const uint2*>(p); }
  // the byte stands for the last eight bits as well, which leaves 0 and all numbers of 16 bits as they are
  __device__ __forceinline__ void values(const Pack<__half, 8>& k, float (&v)[8]) const {
    const uint4 w = *reinterpret_cast<const uint4*>(&k);
    v[0] = __uint_as_float(__byte_perm(w.x, low.x, 0x1044));
    v[1] = __uint_as_float(__byte_perm(w.x, low.x, 0x3255));
    v[2] = __uint_as_float(__byte_perm(w.y, low.x, 0x1066));
    v[3] = __uint_as_float(__byte_perm(w.y, low.x, 0x3277));
    v[4] = __uint_as_float(__byte_perm(w.z, low.y, 0x1044));
    v[5] = __uint_as_float(__byte_perm(w.z, low.y, 0x3255));
    v[6] = __uint_as_float(__byte_perm(w.w, low.y, 0x1066));
    v[7] = __uint_as_float(__byte_perm(w.w, low.y, 0x3277));
  }
};

// dz = act'(z) dy and the column sums of dz over each group.  A thread takes eight columns of the output down a run of
// rows, the next row under way while it works on one; the sums of a (run, group) go to record run + group (both only ever
// advance), added up in order by the next kernel.  Bound by memory traffic with SUMS off; 64 registers, so that an SM holds
// 1024 threads (the gated form with SUMS spills 36 - 56 bytes for that).  fp16: the largest |dz| is found on the way; AGAIN,
// launched behind it, ends at once as a rule, and otherwise writes dz once more under the power of two that it asks for.
template <typename T, bool GATED, bool SUMS, bool AGAIN>
__global__ void __launch_bounds__(128, 8) act_grad_kernel(const b200_act_grad_args a) {
  using P = Pack<T, 8>;
  using Z = Pack<__half, 8>;
  constexpr bool PEAK = std::is_same<T, __half>::value && !AGAIN;
  float shift = 1.f, top = 0.f;
  if constexpr (AGAIN) {
    chain_wait();
    const int s = dz_shift(*a.peak);
    if (s == 0) return;
    shift = power_of_two(-s);
  }
  // of the gated form, a thread's columns belong to eight columns of the gate and of the up half
  const int oc = (blockIdx.y * 128 + threadIdx.x) * 8;
  if (oc >= a.n_out) return;
  const int zc = GATED ? (oc / 128) * 256 + oc % 128 : oc;
  long long start = 0;
  int g = 0;
  const long long first = static_cast<long long>(blockIdx.x) * a.chunk_rows, r1 = min(static_cast<long long>(a.M), first + a.chunk_rows);
  auto rows_of = [&](int i) { return a.group_rows != nullptr ? max(0, a.group_rows[i]) : a.M; };
  while (g < a.G && start + rows_of(g) <= first) start += rows_of(g++);
  const T* dy = static_cast<const T*>(a.dy) + oc;
  const __half* z = static_cast<const __half*>(a.z) + zc;
  const bool active = a.z != nullptr;
  using Beside = ZBeside<T>;
  const unsigned char* zexp = a.zexp + Beside::column(zc);
  const long long pitch = Beside::pitch(a.N);
  long long pos = first;
  for (; g < a.G && pos < r1; ++g) {
    const long long end = min(r1, start + rows_of(g));
    start += rows_of(g);
    if (end <= pos) continue;
    float sum[8], sum2[8];
    if constexpr (SUMS) {
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] = sum2[j] = 0.f;
    }
    P kd;
    Z kz, ku;
    Beside ez, eu;
    auto load = [&](long long r) {
      kd = *reinterpret_cast<const P*>(dy + r * a.n_out);
      if (active) {
        kz = *reinterpret_cast<const Z*>(z + r * a.N);
        ez.load(zexp + r * pitch);
      }
      if (GATED) {
        ku = *reinterpret_cast<const Z*>(z + r * a.N + 128);
        eu.load(zexp + r * pitch + Beside::column(128));
      }
    };
    load(pos);
    for (long long r = pos; r < end; ++r) {
      const P cd = kd;
      const Z cz = kz, cu = ku;
      const Beside cez = ez, ceu = eu;
      if (r + 1 < end) load(r + 1);
      if (a.dres != nullptr) *reinterpret_cast<P*>(static_cast<T*>(a.dres) + r * a.n_out + oc) = cd;
      float d[8], v[8];
      unpack<T, 8>(cd, d);
      if (active) {
        T* dz = static_cast<T*>(a.dz) + r * a.N + zc;
        cez.values(cz, v);
        if constexpr (GATED) {
          float u[8], du[8];
          ceu.values(cu, u);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float q = sigmoid_f(v[j]);
            du[j] = d[j] * (q * v[j]);
            d[j] *= u[j] * silu_slope(v[j], q);
            if constexpr (SUMS) sum2[j] += du[j];
            if constexpr (PEAK) top = finite_max(top, du[j]);
            if constexpr (AGAIN) du[j] *= shift;
          }
          store_pack<T, 8>(dz + 128, du);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] *= act_slope(v[j], a.act);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if constexpr (PEAK) top = finite_max(top, d[j]);
          if constexpr (AGAIN) d[j] *= shift;
        }
        store_pack<T, 8>(dz, d);
      }
      if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += d[j];
      }
    }
    if constexpr (SUMS) {
      float* rec = a.record + (static_cast<size_t>(blockIdx.x) + g) * a.N + zc;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        rec[j] = sum[j];
        if (GATED) rec[128 + j] = sum2[j];
      }
    }
    pos = end;
  }
  if (a.dres != nullptr) {
    const float none[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (long long r = pos; r < r1; ++r) store_pack<T, 8>(static_cast<T*>(a.dres) + r * a.n_out + oc, none);
  }
  if constexpr (PEAK) {
    if (active) {
      const unsigned int here = __activemask(), most = __reduce_max_sync(here, __float_as_uint(top));
      if ((threadIdx.x & 31) == __ffs(here) - 1 && most != 0u) atomicMax(a.peak, most);
    }
  }
}

// A warp takes 32 columns and an eighth of a group's records; the eight sums are added in order.
template <typename T>
__global__ void __launch_bounds__(256) bias_grad_kernel(const b200_act_grad_args a) {
  __shared__ float share[8][33];
  chain_wait();
  const int g = blockIdx.y, lane = threadIdx.x & 31, s = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  long long start = 0;
  for (int i = 0; i < g; ++i) start += max(0, a.group_rows[i]);
  const long long rows = a.group_rows != nullptr ? max(0, a.group_rows[g]) : a.M;
  const long long end = min(static_cast<long long>(a.M), start + rows);
  float v = 0.f;
  if (c < a.N && end > start) {
    const long long last = (end - 1) / a.chunk_rows;
#pragma unroll 4
    for (long long k = start / a.chunk_rows + s; k <= last; k += 8) v += a.record[(static_cast<size_t>(k) + g) * a.N + c];
  }
  share[s][lane] = v;
  __syncthreads();
  if (s != 0 || c >= a.N) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) v += share[i][lane];
  static_cast<T*>(a.dbias)[static_cast<size_t>(g) * a.N + c] = from_f32<T>(v);
}

// ----------------------------------------------------------------------------
// Fewer tiles than SMs: the contracted dimension is split.  A tile is 128 features (rows of the MMA) x TT tokens (its
// columns); the blocks of 64 contracted elements of all tiles are one list, cut into equal runs, one per CTA, whatever the
// number of tiles.  With few tokens the time is that of reading the weights, and every SM reads as many as any other.  A
// run ends inside a tile as a rule: a CTA leaves its fp32 sums of each tile it touched in record CTA + tile (both only ever
// advance, so no two share one), and linear_join_kernel adds a tile's records in their order and does the epilogue.  The
// same inputs give the same bits.  Gated: a tile is 64 gate rows and their 64 up rows.  dW (dense only: rows behind the
// last come as zeros) takes x's columns for features and dz's for tokens.
// Measured, one token: 28672 x 4096 gated weights 40 us (5.8 TB/s), 4096 x 14336 23 us; 112 and 16 tiles of 256 columns
// took 58 and 115.
// ----------------------------------------------------------------------------
constexpr int ROWS_FEATURES = 128;
constexpr int ROWS_THREADS = 192;
constexpr int ROWS_LEAST = 4;            // blocks of a run at least: a record costs as much as reading one
template <int TT>
struct RowsGeo {
  static constexpr int STAGE = ROWS_FEATURES * LBK * 2 + TT * LBK * 2;
  static constexpr int STAGES = TT <= 32 ? 5 : TT == 64 ? 4 : TT == 128 ? 6 : 4;
  static constexpr int PER_SM = TT <= 64 ? 2 : 1;
  static constexpr int ACC = TT < 64 ? 64 : TT;          // TMEM columns of an accumulator; there are two
};
static int rows_per_sm(int TT) { return TT <= 64 ? 2 : 1; }
struct __align__(16) RowsControl {
  uint64_t full[6], empty[6], tmem_full[2], tmem_empty[2], drain;
  uint32_t tmem_base;
  int abort_flag;
  int g_rows[B200_MAX_GROUPS];
  int g_row_start[B200_MAX_GROUPS + 1];
  int g_sched_start[B200_MAX_GROUPS + 1];      // token tiles
};
template <int TT>
constexpr int rows_smem() { return RowsGeo<TT>::STAGES * RowsGeo<TT>::STAGE + static_cast<int>(sizeof(RowsControl)) + 1024; }
static_assert(rows_smem<64>() <= 113 * 1024 && rows_smem<32>() <= 113 * 1024, "two CTAs per SM");
static_assert(rows_smem<256>() <= 232448 && rows_smem<128>() <= 232448, "exceeds 227 KiB of shared memory per CTA");

// Sizes of a product: features, tokens (of the one group, where there are no group sizes) and blocks of the contraction.
__host__ __device__ __forceinline__ int rows_features(int mode, int N, int K) { return mode == LIN_FORWARD ? N : K; }
__host__ __device__ __forceinline__ int rows_tokens(int mode, int M, int N) { return mode == LIN_DW ? N : M; }
__host__ __device__ __forceinline__ int rows_blocks(int mode, int M, int N, int K) {
  return ((mode == LIN_FORWARD ? K : mode == LIN_DX ? N : M) + LBK - 1) / LBK;
}
// Blocks of a CTA's run.
__host__ __device__ __forceinline__ long long rows_quota(long long units, int ctas) {
  const long long q = (units + ctas - 1) / ctas;
  return q < ROWS_LEAST ? ROWS_LEAST : q;
}

// Tile t: its group, its feature tile and its token tile (token tiles of a feature tile one after another, so that its
// weights are still in L2 for the next).
__device__ __forceinline__ void rows_tile(const int* sched_start, int G, int FT, int t, int& cursor, int& ft, int& tt) {
  while (cursor < G - 1 && t >= FT * sched_start[cursor + 1]) ++cursor;
  const int per = sched_start[cursor + 1] - sched_start[cursor], j = t - FT * sched_start[cursor];
  ft = j / per;
  tt = j - ft * per;
}

template <int MODE, int TT>
__global__ void __launch_bounds__(ROWS_THREADS, RowsGeo<TT>::PER_SM)
linear_rows_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const b200_linear_args la) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  constexpr int STAGES = RowsGeo<TT>::STAGES, STAGE = RowsGeo<TT>::STAGE, ACC = RowsGeo<TT>::ACC;
  RowsControl& c = *reinterpret_cast<RowsControl*>(smem + STAGES * STAGE);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = la.G;
  const int features = rows_features(MODE, la.N, la.K), KB = rows_blocks(MODE, la.M, la.N, la.K);
  const int FT = (features + ROWS_FEATURES - 1) / ROWS_FEATURES;
  const bool gated = MODE == LIN_FORWARD && la.act == ACT_SILU_GATE;
  const bool bf16 = la.elem == ELEM_BF16;
  WaitCtx w;
  w.abort_flag = &c.abort_flag;
  w.status = la.status;
  w.budget_ns = la.wait_budget_ns;
  if (tid == 0) {
    c.abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&c.full[s], 1);
      mbar_init(&c.empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&c.tmem_full[a], 1);
      mbar_init(&c.tmem_empty[a], 128);
    }
    mbar_init(&c.drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmap_w);
    tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc(&c.tmem_base, 2 * ACC);
    tmem_relinquish();
  }
  __syncthreads();
  chain_release();
  if (warp == 0) {
    LinTables tables{c.g_rows, c.g_row_start, c.g_sched_start};
    const long long rows = lin_scan(tables, la.group_rows, G, rows_tokens(MODE, la.M, la.N), lane, TT, 0);
    if (lane == 0 && rows > rows_tokens(MODE, la.M, la.N)) {
      report_status(w.status, ST_OVERFLOW);
      if (w.status != nullptr) atomicMax(w.status + 1, c.g_row_start[G]);
      c.abort_flag = 1;
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = c.tmem_base;
  const bool overflow = c.abort_flag != 0;
  const long long units = overflow ? 0 : static_cast<long long>(c.g_sched_start[G]) * FT * KB;
  const long long quota = rows_quota(units, gridDim.x);
  const long long u0 = min(units, quota * blockIdx.x), u1 = min(units, u0 + quota);
  __syncthreads();

  if (warp == 0) {
    if (lane == 0) {
      int cursor = 0, stage = 0, issued = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long u = u0; ok && u < u1;) {
        const int t = static_cast<int>(u / KB), kb0 = static_cast<int>(u - static_cast<long long>(t) * KB);
        const int kb1 = static_cast<int>(min(static_cast<long long>(KB), kb0 + (u1 - u)));
        int ft, tt;
        rows_tile(c.g_sched_start, G, FT, t, cursor, ft, tt);
        const int f0 = gated ? (ft >> 1) * 256 + (ft & 1) * 64 : ft * ROWS_FEATURES, f1 = gated ? f0 + 128 : f0 + 64;
        const int row = c.g_row_start[cursor] + tt * TT;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&c.empty[stage], phase ^ 1u, w, ST_TIMEOUT_PIPE_EMPTY)) { ok = false; break; }
          uint8_t* sa = smem + stage * STAGE;
          mbar_expect_tx(&c.full[stage], STAGE);
          if constexpr (MODE == LIN_FORWARD) {
            tma_load_2d(sa, &tmap_w, &c.full[stage], kb * LBK, cursor * la.N + f0);
            tma_load_2d(sa + LIN_MN_BOX, &tmap_w, &c.full[stage], kb * LBK, cursor * la.N + f1);
          } else if constexpr (MODE == LIN_DX) {
            tma_load_3d(sa, &tmap_w, &c.full[stage], f0, kb * LBK, cursor);
            tma_load_3d(sa + LIN_MN_BOX, &tmap_w, &c.full[stage], f1, kb * LBK, cursor);
          } else {
            tma_load_2d(sa, &tmap_w, &c.full[stage], f0, kb * LBK);
            tma_load_2d(sa + LIN_MN_BOX, &tmap_w, &c.full[stage], f1, kb * LBK);
          }
          if constexpr (MODE == LIN_DW) {
#pragma unroll
            for (int i = 0; i < TT / 64; ++i) tma_load_2d(sa + (2 + i) * LIN_MN_BOX, &tmap_x, &c.full[stage], row + i * 64, kb * LBK);
          } else {
            tma_load_2d(sa + 2 * LIN_MN_BOX, &tmap_x, &c.full[stage], kb * LBK, row);
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        u += kb1 - kb0;
      }
      int no_abort = 0;
      WaitCtx wd = w;
      wd.abort_flag = &no_abort;
      for (int i = 0; i < min(issued, STAGES); ++i) {
        int s = stage - 1 - i;
        uint32_t ph = phase;
        if (s < 0) { s += STAGES; ph ^= 1u; }
        mbar_wait(&c.full[s], ph, wd, ST_TIMEOUT_DRAIN);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr bool A_MN = MODE != LIN_FORWARD, B_MN = MODE == LIN_DW;
      const uint32_t idesc = make_idesc_16bit(ROWS_FEATURES, TT, bf16, A_MN, B_MN);
      int stage = 0, it = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (long long u = u0; ok && u < u1; ++it) {
        const int kb0 = static_cast<int>(u % KB), n = static_cast<int>(min(static_cast<long long>(KB - kb0), u1 - u));
        const int acc = it & 1;
        if (!mbar_wait(&c.tmem_empty[acc], ((it >> 1) & 1) ^ 1u, w, ST_TIMEOUT_TMEM_EMPTY)) break;
        tc_fence_after_sync();
        for (int i = 0; i < n; ++i) {
          if (!mbar_wait(&c.full[stage], phase, w, ST_TIMEOUT_PIPE_FULL)) { ok = false; break; }
          tc_fence_after_sync();
          const uint32_t sa = smem_u32(smem + stage * STAGE);
          const uint64_t ad = A_MN ? make_smem_desc_mn_sw128(sa, LIN_MN_BOX) : make_smem_desc_sw128(sa);
          const uint64_t bd = B_MN ? make_smem_desc_mn_sw128(sa + 2 * LIN_MN_BOX, LIN_MN_BOX) : make_smem_desc_sw128(sa + 2 * LIN_MN_BOX);
          constexpr int ASTEP = A_MN ? 2048 / 16 : 2, BSTEP = B_MN ? 2048 / 16 : 2;
#pragma unroll
          for (int k = 0; k < LBK / 16; ++k) umma_bf16_ss(tmem_base + acc * ACC, ad + ASTEP * k, bd + BSTEP * k, idesc, (i | k) != 0 ? 1u : 0u);
          umma_commit(&c.empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit(&c.tmem_full[acc]);
        u += n;
      }
      umma_commit(&c.drain);
      int no_abort = 0;
      WaitCtx wd = w;
      wd.abort_flag = &no_abort;
      mbar_wait(&c.drain, 0, wd, ST_TIMEOUT_DRAIN);
    }
  } else {
    const int q = warp & 3;
    int cursor = 0, it = 0;
    for (long long u = u0; u < u1; ++it) {
      const int t = static_cast<int>(u / KB), kb0 = static_cast<int>(u - static_cast<long long>(t) * KB);
      u += min(static_cast<long long>(KB - kb0), u1 - u);
      int ft, tt;
      rows_tile(c.g_sched_start, G, FT, t, cursor, ft, tt);
      const int tokens = min(TT, c.g_rows[cursor] - tt * TT), acc = it & 1;
      const bool got = mbar_wait(&c.tmem_full[acc], (it >> 1) & 1, w, ST_TIMEOUT_TMEM_FULL);
      if (!__all_sync(0xffffffffu, got)) break;
      tc_fence_after_sync();
      float* rec = la.record + (static_cast<size_t>(blockIdx.x) + t) * (ROWS_FEATURES * TT) + q * 32 + lane;
#pragma unroll 1
      for (int h = 0; h < TT; h += 16) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + acc * ACC + h, v);
        tmem_ld_wait();
        if (h + 16 >= TT) {
          tc_fence_before_sync();
          mbar_arrive(&c.tmem_empty[acc]);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (h + i < tokens) rec[(h + i) * ROWS_FEATURES] = __uint_as_float(v[i]);
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 2 * ACC);
  }
}

// Adds a tile's records and does the epilogue: a block takes four of a tile's 4 * `quads` tokens, a thread a feature of each
// (gated: an output of two of them).
constexpr int JOIN_TOKENS = 4;
// z of column c, by a warp that has 32 columns of the row, those that a byte of exponents is for.
template <typename T>
__device__ __forceinline__ void keep_z(const b200_linear_args& la, size_t row, int c, bool in, float z) {
  if constexpr (std::is_same<T, __half>::value) {
    if (!in) return;
    static_cast<unsigned short*>(la.z)[row * la.N + c] = static_cast<unsigned short>(__float_as_uint(z) >> 16);
    la.zexp[row * zlow_pitch(la.N) + c] = static_cast<unsigned char>(__float_as_uint(z) >> 8);
    return;
  }
  const uint32_t bits = __float_as_uint(fabsf(z));
  int E = shared_exponent(__reduce_max_sync(0xffffffffu, in && bits < 0x7f800000u ? bits : 0u));
  if (E >= 137 && z_spans_much(E, __uint_as_float(__reduce_min_sync(0xffffffffu, in && bits != 0u && bits < 0x7f800000u ? bits : 0x7f7fffffu)))) E = Z_BF16;
  if ((threadIdx.x & 31) == 0 && in) la.zexp[row * zexp_pitch(la.N) + c / 32] = static_cast<unsigned char>(E);
  if (!in) return;
  const size_t i = row * la.N + c;
  if (E != Z_BF16) static_cast<__half*>(la.z)[i] = __float2half_rn(z * z_scale(E));
  else static_cast<__nv_bfloat16*>(la.z)[i] = __float2bfloat16_rn(z);
}
template <int MODE, int TT, typename T>
__global__ void __launch_bounds__(ROWS_FEATURES) linear_join_kernel(const b200_linear_args la, int ctas, int quads) {
  __shared__ int g_rows[B200_MAX_GROUPS], g_row_start[B200_MAX_GROUPS + 1], g_sched_start[B200_MAX_GROUPS + 1];
  __shared__ int too_many;
  const int tid = threadIdx.x;
  const int features = rows_features(MODE, la.N, la.K), KB = rows_blocks(MODE, la.M, la.N, la.K);
  const int FT = (features + ROWS_FEATURES - 1) / ROWS_FEATURES;
  chain_wait();
  if (tid < 32) {
    LinTables tables{g_rows, g_row_start, g_sched_start};
    const long long rows = lin_scan(tables, la.group_rows, la.G, rows_tokens(MODE, la.M, la.N), tid, TT, 0);
    if (tid == 0) too_many = rows > rows_tokens(MODE, la.M, la.N);
  }
  __syncthreads();
  if (too_many) return;
  const int tiles = g_sched_start[la.G] * FT;
  const long long units = static_cast<long long>(tiles) * KB, quota = rows_quota(units, ctas);
  const bool gated = MODE == LIN_FORWARD && la.act == ACT_SILU_GATE;
  const float unshift = MODE != LIN_FORWARD && la.peak != nullptr ? power_of_two(dz_shift(*la.peak)) : 1.f;
  const long long jobs = static_cast<long long>(tiles) * quads;
  int cursor = 0;
  for (long long job = blockIdx.x; job < jobs; job += gridDim.x) {
    const int t = static_cast<int>(job / quads), k0 = static_cast<int>(job % quads) * JOIN_TOKENS;
    int ft, tt;
    rows_tile(g_sched_start, la.G, FT, t, cursor, ft, tt);
    const int g = cursor, tokens = min(TT, g_rows[g] - tt * TT) - k0;      // of this block, up to JOIN_TOKENS
    if (tokens <= 0) continue;
    const size_t row0 = static_cast<size_t>(g_row_start[g]) + tt * TT + k0;
    const int first = static_cast<int>(static_cast<long long>(t) * KB / quota), last = static_cast<int>((static_cast<long long>(t + 1) * KB - 1) / quota);
    // this thread's four sums: feature f of tokens k, k + step, ...; gated: gate and up of two tokens
    const int f = gated ? tid & 63 : tid, k = gated ? tid >> 6 : 0, step = gated ? 2 : 1;
    const float* rec = la.record + (static_cast<size_t>(first) + t) * (ROWS_FEATURES * TT) + static_cast<size_t>(k0 + k) * ROWS_FEATURES + f;
    auto at = [&](int j) { return gated ? (j >> 1) * 2 * ROWS_FEATURES + (j & 1) * 64 : j * ROWS_FEATURES; };
    bool have[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) have[j] = k + (gated ? j >> 1 : j) * step < tokens;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int i = first; i <= last; ++i) {
      const float* r = rec + static_cast<size_t>(i - first) * (ROWS_FEATURES * TT);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += r[at(j)];      // tokens that are none read what lies in the record, and end below
    }
    T* y = static_cast<T*>(la.out);
    if (gated) {
      const int zc = (ft >> 1) * 256 + (ft & 1) * 64 + f, yc = ft * 64 + f;
      if (la.bias != nullptr) {
        const T* b = static_cast<const T*>(la.bias) + static_cast<size_t>(g) * la.N + zc;
        const float bg = to_f32(b[0]), bu = to_f32(b[128]);
        v[0] += bg; v[1] += bu; v[2] += bg; v[3] += bu;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (!have[2 * j]) continue;
        const size_t row = row0 + k + 2 * j;
        if (la.z != nullptr) {
          keep_z<T>(la, row, zc, true, v[2 * j]);
          keep_z<T>(la, row, zc + 128, true, v[2 * j + 1]);
        }
        float o = gated_value(v[2 * j], v[2 * j + 1]);
        if (la.res != nullptr) o += to_f32(static_cast<const T*>(la.res)[row * la.n_out + yc]);
        y[row * la.n_out + yc] = from_f32<T>(o);
      }
    } else {
      const int c = ft * ROWS_FEATURES + tid;
      const bool in = c < features;
      const float b = MODE == LIN_FORWARD && la.bias != nullptr && in ? to_f32(static_cast<const T*>(la.bias)[static_cast<size_t>(g) * la.N + c]) : 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!have[j]) continue;
        const size_t row = row0 + j;
        float o = v[j];
        if constexpr (MODE == LIN_FORWARD) {
          o += b;
          if (la.z != nullptr) keep_z<T>(la, row, c, in, o);
          o = act_value(o, la.act);
          if (la.res != nullptr && in) o += to_f32(static_cast<const T*>(la.res)[row * la.n_out + c]);
        } else {
          o *= unshift;
        }
        if (in) y[row * la.n_out + c] = from_f32<T>(o);
      }
    }
  }
  // rows of the buffer behind the last group
  const long long begin = static_cast<long long>(g_row_start[la.G]) * la.n_out / 8, end = static_cast<long long>(rows_tokens(MODE, la.M, la.N)) * la.n_out / 8;
  uint4* out = reinterpret_cast<uint4*>(la.out);
  for (long long i = begin + static_cast<long long>(blockIdx.x) * ROWS_FEATURES + tid; i < end; i += static_cast<long long>(gridDim.x) * ROWS_FEATURES)
    out[i] = make_uint4(0, 0, 0, 0);
}

// ------------------------------------------------------------------ host side
typedef CUresult (*LinEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static LinEncodeFn lin_encode() {
  static std::atomic<void*> fn{nullptr};
  void* p = fn.load(std::memory_order_relaxed);
  if (p == nullptr) {
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &qres) != cudaSuccess || qres != cudaDriverEntryPointSuccess) return nullptr;
    fn.store(p, std::memory_order_relaxed);
  }
  return reinterpret_cast<LinEncodeFn>(p);
}

// Row-major [planes][rows][cols] of 16-bit elements (two dimensions where planes is 0), boxes of 64 columns x box_rows.
static int lin_map(CUtensorMap* tm, const void* base, int elem, long long planes, long long rows, long long cols, int box_rows) {
  LinEncodeFn enc = lin_encode();
  if (enc == nullptr) return -1;
  if ((reinterpret_cast<uintptr_t>(base) & 15u) != 0 || cols % 8 != 0 || rows <= 0) return -2;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(planes)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(cols) * rows * 2};
  const cuuint32_t box[3] = {64u, static_cast<cuuint32_t>(box_rows), 1u};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = enc(tm, elem == ELEM_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, planes > 0 ? 3 : 2,
                         const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -3;
}

template <int MODE, int CG, bool GATED, bool Z24 = false>
static int linear_launch(const b200_linear_args& la, int ctas, cudaStream_t st) {
  static std::atomic<unsigned long long> configured{0};
  using S = LinGeo<MODE, CG>;
  auto kern = linear_kernel<MODE, CG, GATED, Z24>;
  constexpr int smem = lin_smem<MODE, CG>();
  // The device's context becomes current: the thread that runs a backward pass may not have met it yet, and tensor maps
  // are encoded by the CUDA driver, which does not do so itself.
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);
  if (e == cudaSuccess) e = allow_shared_memory(kern, smem, configured);
  if (e != cudaSuccess) return static_cast<int>(e);
  CUtensorMap ta, tb, to, tz;
  const long long out_rows = MODE == LIN_DW ? static_cast<long long>(la.G) * la.N : la.M;
  int r = MODE == LIN_FORWARD ? lin_map(&ta, la.a, la.elem, 0, la.M, la.K, LBM)
          : MODE == LIN_DX    ? lin_map(&ta, la.a, la.elem, 0, la.M, la.N, LBM)
                              : lin_map(&ta, la.a, la.elem, 0, la.M, la.N, LBK);
  if (r == 0)
    r = MODE == LIN_FORWARD ? lin_map(&tb, la.b, la.elem, 0, static_cast<long long>(la.G) * la.N, la.K, S::B_ROWS)
        : MODE == LIN_DX    ? lin_map(&tb, la.b, la.elem, la.G, la.N, la.K, LBK)
                            : lin_map(&tb, la.b, la.elem, 0, la.M, la.K, LBK);
  if (r == 0) r = lin_map(&to, la.out, la.elem, 0, out_rows, la.n_out, 32);
  tz = to;
  if (r == 0 && la.z != nullptr) r = lin_map(&tz, la.z, la.elem, 0, la.M, la.N, 32);
  if (r != 0) return r;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(ctas / CG * CG, 1, 1);
  cfg.blockDim = dim3(LIN_THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  b200_count_launches(1);
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, ta, tb, to, tz, la));
}

template <bool Z24>
static int linear_forward(const b200_linear_args& la, bool gated, int ctas, cudaStream_t st) {
  if (gated) return la.pair ? linear_launch<LIN_FORWARD, 2, true, Z24>(la, ctas, st) : linear_launch<LIN_FORWARD, 1, true, Z24>(la, ctas, st);
  return la.pair ? linear_launch<LIN_FORWARD, 2, false, Z24>(la, ctas, st) : linear_launch<LIN_FORWARD, 1, false, Z24>(la, ctas, st);
}

// Tokens of a tile: as few as hold an average group.
static int rows_tile_tokens(int mode, int M, int N, int G) {
  const long long n = rows_tokens(mode, M, N), g = G;
  if (mode == LIN_DW) return n <= 64 ? 64 : n <= 128 ? 128 : 256;      // whole boxes of 64
  return n <= 16 * g ? 16 : n <= 32 * g ? 32 : n <= 64 * g ? 64 : n <= 128 * g ? 128 : 256;
}
static long long rows_tiles_most(int mode, int M, int N, int K, int G) {
  const int n = rows_tokens(mode, M, N), TT = rows_tile_tokens(mode, M, N, G);
  const long long token_tiles = (static_cast<long long>(n) + TT - 1) / TT + (G > 1 ? (G < n ? G : n) : 0);   // each group may leave one partly filled
  return token_tiles * ((rows_features(mode, N, K) + ROWS_FEATURES - 1) / ROWS_FEATURES);
}

template <int MODE, int TT>
static int linear_rows_launch(const b200_linear_args& la, int sms, cudaStream_t st) {
  static std::atomic<unsigned long long> configured{0};
  auto kern = linear_rows_kernel<MODE, TT>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaSetDevice(dev);       // as in linear_launch
  if (e == cudaSuccess) e = allow_shared_memory(kern, rows_smem<TT>(), configured);
  if (e != cudaSuccess) return static_cast<int>(e);
  CUtensorMap tw, tx;
  int r = MODE == LIN_FORWARD ? lin_map(&tw, la.b, la.elem, 0, static_cast<long long>(la.G) * la.N, la.K, 64)
          : MODE == LIN_DX    ? lin_map(&tw, la.b, la.elem, la.G, la.N, la.K, LBK)
                              : lin_map(&tw, la.b, la.elem, 0, la.M, la.K, LBK);
  if (r == 0) r = lin_map(&tx, la.a, la.elem, 0, la.M, MODE == LIN_FORWARD ? la.K : la.N, MODE == LIN_DW ? LBK : TT);
  if (r != 0) return r;
  const int ctas = RowsGeo<TT>::PER_SM * sms;
  b200_count_launches(2);
  kern<<<ctas, ROWS_THREADS, rows_smem<TT>(), st>>>(tw, tx, la);
  e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  const int tokens = rows_tokens(MODE, la.M, la.N);
  const int quads = ((tokens < TT ? tokens : TT) + JOIN_TOKENS - 1) / JOIN_TOKENS;      // no tile has more tokens than there are
  const long long jobs = rows_tiles_most(MODE, la.M, la.N, la.K, la.G) * quads;
  const dim3 grid(static_cast<unsigned>(jobs < 16ll * sms ? jobs : 16ll * sms));
  e = la.elem == ELEM_BF16 ? launch_chained(linear_join_kernel<MODE, TT, __nv_bfloat16>, grid, dim3(ROWS_FEATURES), 0, st, la, ctas, quads)
                           : launch_chained(linear_join_kernel<MODE, TT, __half>, grid, dim3(ROWS_FEATURES), 0, st, la, ctas, quads);
  return static_cast<int>(e);
}
template <int MODE>
static int linear_rows(const b200_linear_args& la, int sms, cudaStream_t st) {
  const int TT = rows_tile_tokens(MODE, la.M, la.N, la.G);
  if constexpr (MODE != LIN_DW) {
    if (TT == 16) return linear_rows_launch<MODE, 16>(la, sms, st);
    if (TT == 32) return linear_rows_launch<MODE, 32>(la, sms, st);
  }
  if (TT == 64) return linear_rows_launch<MODE, 64>(la, sms, st);
  if (TT == 128) return linear_rows_launch<MODE, 128>(la, sms, st);
  return linear_rows_launch<MODE, 256>(la, sms, st);
}

template <typename T>
static cudaError_t act_grad_launch(const b200_act_grad_args& a, cudaStream_t st) {
  const dim3 grid(a.chunks, (a.n_out / 8 + 127) / 128);
  const bool gated = a.act == ACT_SILU_GATE, sums = a.dbias != nullptr;
  auto kern = gated ? (sums ? act_grad_kernel<T, true, true, false> : act_grad_kernel<T, true, false, false>)
                    : (sums ? act_grad_kernel<T, false, true, false> : act_grad_kernel<T, false, false, false>);
  if (a.peak != nullptr) {
    const cudaError_t e = cudaMemsetAsync(a.peak, 0, sizeof(unsigned int), st);
    if (e != cudaSuccess) return e;
  }
  b200_count_launches(1);
  kern<<<grid, 128, 0, st>>>(a);
  return cudaGetLastError();
}
// dz under its power of two, where it needs one.
static cudaError_t act_grad_again(b200_act_grad_args a, cudaStream_t st) {
  const dim3 grid(a.chunks, (a.n_out / 8 + 127) / 128);
  a.dres = nullptr;
  b200_count_launches(1);
  return a.act == ACT_SILU_GATE ? launch_chained(act_grad_kernel<__half, true, false, true>, grid, dim3(128), 0, st, a)
                                : launch_chained(act_grad_kernel<__half, false, false, true>, grid, dim3(128), 0, st, a);
}

}  // namespace b200

extern "C" {

int b200_linear(const b200_linear_args* args, int ctas, void* stream) {
  using namespace b200;
  if (args == nullptr || args->G < 1 || args->G > B200_MAX_GROUPS || args->M < 1 || args->N < 1 || args->K < 1 || ctas < 2) return -10;
  b200_linear_args la = *args;
  if (la.N % 8 != 0 || la.K % 8 != 0 || (la.elem != ELEM_BF16 && la.elem != ELEM_F16)) return -11;
  if (la.mode < LIN_FORWARD || la.mode > LIN_DW) return -15;
  if ((la.group_rows == nullptr && la.G != 1) || la.M > LIN_MAX_ROWS || static_cast<long long>(la.G) * la.N > LIN_MAX_ROWS) return -12;
  const bool gated = la.mode == LIN_FORWARD && la.act == ACT_SILU_GATE;
  if (gated && la.N % 256 != 0) return -13;
  if ((la.z != nullptr) != (la.zexp != nullptr) || (reinterpret_cast<uintptr_t>(la.zexp) & 15u) != 0) return -17;
  if (la.mode != LIN_FORWARD && la.peak != nullptr && la.elem != ELEM_F16) return -18;
  if (la.n_out != (la.mode != LIN_FORWARD ? la.K : gated ? la.N / 2 : la.N)) return -14;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (la.record != nullptr) {
    if (la.mode == LIN_FORWARD) return linear_rows<LIN_FORWARD>(la, ctas, st);
    if (la.mode == LIN_DX) return linear_rows<LIN_DX>(la, ctas, st);
    return la.mode == LIN_DW && la.group_rows == nullptr ? linear_rows<LIN_DW>(la, ctas, st) : -16;
  }
  // rows of tiles that share a stretch of the weights while it is in L2: about 48 MB of the row operand, at most 16 tiles
  const long long tile_bytes = static_cast<long long>(la.pair ? 2 * LBM : LBM) * (la.mode == LIN_DX ? la.N : la.K) * 2;
  const long long gm = (48ll << 20) / tile_bytes;
  la.group_m = static_cast<int>(gm < 1 ? 1 : gm > 16 ? 16 : gm);
  switch (la.mode) {
    case LIN_FORWARD: return la.elem == ELEM_F16 ? linear_forward<true>(la, gated, ctas, st) : linear_forward<false>(la, gated, ctas, st);
    case LIN_DX: return la.pair ? linear_launch<LIN_DX, 2, false>(la, ctas, st) : linear_launch<LIN_DX, 1, false>(la, ctas, st);
    case LIN_DW: return la.pair ? linear_launch<LIN_DW, 2, false>(la, ctas, st) : linear_launch<LIN_DW, 1, false>(la, ctas, st);
  }
  return -15;
}

// Floats of `record` for a split product: a record per CTA and tile that a CTA's run may end in.
long long b200_linear_record_floats(int mode, int M, int N, int K, int G, int sms) {
  using namespace b200;
  const int TT = rows_tile_tokens(mode, M, N, G);
  return (rows_per_sm(TT) * sms + rows_tiles_most(mode, M, N, K, G)) * ROWS_FEATURES * TT;
}

int b200_act_grad(const b200_act_grad_args* args, void* stream) {
  using namespace b200;
  if (args == nullptr || args->G < 1 || args->M < 1 || args->N < 8 || args->N % 8 != 0 || args->chunk_rows < 1 ||
      static_cast<long long>(args->chunks) * args->chunk_rows < args->M || (args->group_rows == nullptr && args->G != 1))
    return -10;
  if (args->dbias != nullptr && args->record == nullptr) return -11;
  if ((args->act != ACT_NONE) != (args->z != nullptr) || (args->z != nullptr) != (args->dz != nullptr)) return -12;
  if (args->elem != ELEM_BF16 && args->elem != ELEM_F16) return -13;
  if ((args->z != nullptr) != (args->zexp != nullptr)) return -14;
  if ((args->peak != nullptr) != (args->z != nullptr && args->elem == ELEM_F16)) return -15;
  const b200_act_grad_args& a = *args;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = a.elem == ELEM_BF16 ? act_grad_launch<__nv_bfloat16>(a, st) : act_grad_launch<__half>(a, st);
  if (e == cudaSuccess && a.dbias != nullptr) {
    b200_count_launches(1);
    const dim3 fin((a.N + 31) / 32, a.G);
    e = a.elem == ELEM_BF16 ? launch_chained(bias_grad_kernel<__nv_bfloat16>, fin, dim3(256), 0, st, a)
                            : launch_chained(bias_grad_kernel<__half>, fin, dim3(256), 0, st, a);
  }
  if (e == cudaSuccess && a.peak != nullptr) e = act_grad_again(a, st);
  return static_cast<int>(e);
}

void b200_abi_sizes_linear(int* out) {
  out[0] = static_cast<int>(sizeof(b200_linear_args));
  out[1] = static_cast<int>(sizeof(b200_act_grad_args));
}

}  // extern "C"
