// The router's auxiliary losses with per-expert counts, forward and backward.
//
// Over the tokens of sequence s that take part (n_s of them), with p = softmax(logits), lse = log sum exp(logits) and c_se the
// routed copies of expert e among them (k per token):
//
//   loss = (coef / S') sum_s sum_e  E c_se / (k n_s) * (1 / n_s) sum_t p_te   +   (z / n) sum_t lse_t^2
//   dlogits_te = p_te (a_se - sum_j a_sj p_tj) + (2 z / n) lse_t p_te,   a_se = (coef / S') E c_se / (k n_s^2)
//
// S' is the number of sequences that hold such a token and n that of such tokens.  A token takes no part (zero gradient,
// not counted) behind the last sequence, where the mask is false, and where its logits have no usable maximum: a NaN,
// +infinity, or none above the type's lowest value (every expert masked).
//
// A block takes a run of tokens and walks the sequences in it one after another; 2^x lanes share a token, each with whole
// packs of 16 bytes of its logits, and hold the next token's while they work on one.  Column sums stay in registers until the sequence or the run ends; then one record per (run, sequence) is written: sums of p,
// counts, tokens, sum of lse^2.  Runs and sequences only ever advance, so run + sequence numbers the records
// without gaps.  A second kernel adds a sequence's records in their order.  No atomics on floating-point values: the same
// inputs give the same bits.
#include <cuda_runtime.h>
#include <math_constants.h>

#include "elementwise.cuh"
#include "launch.h"
#include "moe_args.h"
#include "sm100_ptx.cuh"

extern "C" {
typedef struct b200_balance_args {
  const void* logits;        // [T, E], row stride ld
  const int* idx;            // [T, k]
  const int* seq_rows;       // [S] or null: one sequence of all T tokens
  const unsigned char* mask; // [T] or null
  float* loss;               // [1]
  int* counts;               // [S, E]
  int* kept;                 // [S, E]: the same again, for the backward pass (the caller may change its own)
  float* record;             // [runs + S][2 E + 2]: sums of p, counts (int), tokens (int), sum of lse^2
  float* seq_loss;           // [S][ceil(E / 32)]: 32 experts' part of a sequence's term
  float* seq_z;              // [S]: its sum of lse^2
  int* seq_tokens;           // [S]
  float* total;              // [2]: 1 / S' (0 without a token), 1 / n
  int* ticket;               // [1]
  const float* grad_loss;    // [1] (backward)
  void* grad;                // [T, E] (backward)
  int* status;
  long long ld;
  int T, E, k, S;
  int elem;
  int runs;                  // blocks
  int run_tokens;            // tokens per block
  float coef, z;
} b200_balance_args;
}

namespace b200 {

constexpr int BAL_THREADS = 256;
constexpr int BAL_MAX_E = 1024;
constexpr int BAL_MOST = 0x7fffffff - 0xfffff;      // tokens, and blocks of 32 experts of all sequences: their numbers have 32 bits
// Blocks of an SM: as many runs as these make no second, half empty round.  (The registers that this leaves, 64 and 80, make the
// fp32 forms of the forward kernel spill 12 - 20 bytes, its forms for rows off 16 bytes up to 104, and the backward one for fp32
// rows of 257 experts and more 12.)
constexpr int BAL_FORWARD_BLOCKS = 4, BAL_BACKWARD_BLOCKS = 3;

template <typename T> __device__ __forceinline__ float lowest();
template <> __device__ __forceinline__ float lowest<float>() { return -3.402823466e38f; }
template <> __device__ __forceinline__ float lowest<__nv_bfloat16>() { return -3.389531390e38f; }
template <> __device__ __forceinline__ float lowest<__half>() { return -65504.f; }

// The sequence that token t0 lies in, and where that sequence starts; S where it lies behind the last.  Every
// thread sums its share of the lengths, the block scans the sums, and the thread whose share holds t0 walks it.
__device__ __forceinline__ void find_sequence(const b200_balance_args& a, long long t0, int& seq, long long& start) {
  __shared__ long long warp_total[BAL_THREADS / 32];
  __shared__ int found_seq;
  __shared__ long long found_start;
  const int tid = threadIdx.x, lane = tid & 31;
  const int per = (a.S + BAL_THREADS - 1) / BAL_THREADS;
  const int s0 = min(a.S, tid * per), s1 = min(a.S, s0 + per);
  long long mine = 0;
  for (int s = s0; s < s1; ++s) mine += max(0, a.seq_rows[s]);
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long other = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += other;
  }
  if (lane == 31) warp_total[tid >> 5] = incl;
  if (tid == 0) { found_seq = a.S; found_start = 0; }
  __syncthreads();
  for (int w = 0; w < (tid >> 5); ++w) incl += warp_total[w];
  if (tid == BAL_THREADS - 1 && blockIdx.x == 0 && incl > a.T) report_status(a.status, ST_OVERFLOW);
  long long at = incl - mine;
  if (at <= t0 && t0 < incl) {
    for (int s = s0; s < s1; ++s) {
      const int n = max(0, a.seq_rows[s]);
      if (t0 < at + n) { found_seq = s; found_start = at; break; }
      at += n;
    }
  }
  __syncthreads();
  seq = found_seq;
  start = found_start;
}

// How a token's experts lie on the LPT lanes that share it: P packs of V logits per lane; value i of a lane is expert
// expert_of(i, sub).  V is 1 where rows do not start on 16 bytes.
template <int LPT, int V>
__device__ __forceinline__ int expert_of(int i, int sub) { return (i / V * LPT + sub) * V + i % V; }

template <typename T, int V, int P>
struct TokenRow {
  Pack<T, V> k[P];
};

template <typename T> __device__ __forceinline__ T minus_infinity();
template <> __device__ __forceinline__ float minus_infinity<float>() { return -CUDART_INF_F; }
template <> __device__ __forceinline__ __nv_bfloat16 minus_infinity<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ __half minus_infinity<__half>() { return __ushort_as_half(0xfc00); }

// Loads one token's logits; minus infinity behind the last expert, and everywhere where `in` is false (a masked token's are
// loaded all the same: waiting for the mask first would put one latency behind another).
template <typename T, int LPT, int V, int P>
__device__ __forceinline__ void load_token(const b200_balance_args& a, long long t, bool in, int sub, TokenRow<T, V, P>& row) {
  const T* p = static_cast<const T*>(a.logits) + t * a.ld;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    const int e = (i * LPT + sub) * V;
    if (in && e < a.E) row.k[i] = *reinterpret_cast<const Pack<T, V>*>(p + e);
    else {
#pragma unroll
      for (int j = 0; j < V; ++j) row.k[i].v[j] = minus_infinity<T>();
    }
  }
}

// One token's exponentials over the lanes that share it and the inverse of their sum.  False: it takes no part.
// exp(l - max) is 2^((l - max) log2 e): the difference comes first, so that logits next to the type's largest do not overflow.
template <typename T, int LPT, int V, int P>
__device__ __forceinline__ bool token_softmax(const TokenRow<T, V, P>& row, bool take, float (&p)[V * P], float& inv, float& lse) {
  constexpr int C = V * P;
  float mx = -CUDART_INF_F;
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float x[V];
    unpack<T, V>(row.k[i], x);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      p[i * V + j] = x[j];
      mx = max_nan(mx, x[j]);
    }
  }
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) mx = max_nan(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const bool ok = take && mx > lowest<T>() && mx < CUDART_INF_F;      // no for a NaN
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    p[i] = exp2_approx((p[i] - mx) * LOG2_E);
    sum += p[i];
  }
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (!ok) {
#pragma unroll
    for (int i = 0; i < C; ++i) p[i] = 0.f;
  }
  inv = ok ? 1.f / sum : 0.f;
  lse = ok ? mx + logf(sum) : 0.f;
  return ok;
}

template <typename T, int LPT, int V, int P>
__global__ void __launch_bounds__(BAL_THREADS, V * P <= 16 ? BAL_FORWARD_BLOCKS : 2) balance_forward_kernel(const b200_balance_args a) {
  extern __shared__ float sm[];              // [warps][E] sums of p, then int [E] counts
  __shared__ float warp_z[BAL_THREADS / 32];
  __shared__ int warp_n[BAL_THREADS / 32];
  constexpr int WARPS = BAL_THREADS / 32, TOK = 32 / LPT, C = V * P;
  int* cnt = reinterpret_cast<int*>(sm + WARPS * a.E);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LPT, slot = lane / LPT;
  const long long t0 = static_cast<long long>(blockIdx.x) * a.run_tokens;
  const long long t1 = min(static_cast<long long>(a.T), t0 + a.run_tokens);
  if (blockIdx.x == 0 && tid == 0) *a.ticket = 0;
  int seq = 0;
  long long start = 0;
  if (a.seq_rows != nullptr) find_sequence(a, t0, seq, start);
  long long pos = t0;
  for (; seq < a.S && pos < t1; ++seq) {
    const long long len = a.seq_rows != nullptr ? max(0, a.seq_rows[seq]) : a.T;
    const long long end = min(t1, start + len);
    if (len == 0) continue;
    for (int e = tid; e < a.E; e += BAL_THREADS) cnt[e] = 0;
    __syncthreads();
    float col[C];
#pragma unroll
    for (int i = 0; i < C; ++i) col[i] = 0.f;
    float zsum = 0.f;
    int tokens = 0;
    long long t = pos + warp * TOK;
    TokenRow<T, V, P> row, next;
    bool take = false, next_take = false;
    int chosen = -1, next_chosen = -1;         // this lane's first copy of the token
    auto load = [&](long long at, TokenRow<T, V, P>& r, bool& take, int& chosen) {
      const bool in = at < end;
      load_token<T, LPT, V, P>(a, at, in, sub, r);
      take = in && (a.mask == nullptr || a.mask[at] != 0);
      chosen = in && sub < a.k ? a.idx[at * a.k + sub] : -1;
    };
    load(t + slot, row, take, chosen);
    for (; t < end; t += WARPS * TOK) {
      const long long mine = t + slot;
      load(mine + WARPS * TOK, next, next_take, next_chosen);
      float p[C], inv, lse;
      const bool ok = token_softmax<T, LPT, V, P>(row, take, p, inv, lse);
#pragma unroll
      for (int i = 0; i < C; ++i) col[i] = fmaf(p[i], inv, col[i]);
      if (ok) {
        if (chosen >= 0 && chosen < a.E) atomicAdd(cnt + chosen, 1);
        for (int j = sub + LPT; j < a.k; j += LPT) {
          const int e = a.idx[mine * a.k + j];
          if (e >= 0 && e < a.E) atomicAdd(cnt + e, 1);
        }
        if (sub == 0) {
          if (a.z != 0.f) zsum += lse * lse;       // may be infinite, and nothing times that is not nothing
          ++tokens;
        }
      }
      row = next;
      take = next_take;
      chosen = next_chosen;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int o = LPT; o < 32; o <<= 1) col[i] += __shfl_xor_sync(0xffffffffu, col[i], o);
      if (slot == 0 && expert_of<LPT, V>(i, sub) < a.E) sm[warp * a.E + expert_of<LPT, V>(i, sub)] = col[i];
    }
    zsum = warp_sum(zsum);
    tokens = __reduce_add_sync(0xffffffffu, tokens);
    if (lane == 0) { warp_z[warp] = zsum; warp_n[warp] = tokens; }
    __syncthreads();
    float* rec = a.record + (static_cast<size_t>(blockIdx.x) + seq) * (2 * a.E + 2);
    for (int e = tid; e < a.E; e += BAL_THREADS) {
      float v = 0.f;
      for (int w = 0; w < WARPS; ++w) v += sm[w * a.E + e];
      rec[e] = v;
      reinterpret_cast<int*>(rec)[a.E + e] = cnt[e];
    }
    if (tid == 0) {
      float z = 0.f;
      int n = 0;
      for (int w = 0; w < WARPS; ++w) { z += warp_z[w]; n += warp_n[w]; }
      reinterpret_cast<int*>(rec)[2 * a.E] = n;
      rec[2 * a.E + 1] = z;
    }
    __syncthreads();
    start += len;
    pos = end;
  }
}

// Block (s, c) adds the records of 32 experts of a sequence, each of 16 warps a share of the runs in their order, and
// writes the counts and the experts' part of sum_e c_e P_e; the last block of all adds the parts.
constexpr int FIN_WARPS = 16;
__global__ void __launch_bounds__(FIN_WARPS * 32) balance_finish_kernel(const b200_balance_args a) {
  __shared__ float sh_p[FIN_WARPS][33], sh_z[FIN_WARPS];
  __shared__ int sh_c[FIN_WARPS][33], sh_n[FIN_WARPS];
  __shared__ long long sh_start[FIN_WARPS];
  __shared__ double sh_d[2][FIN_WARPS];
  __shared__ int last;
  chain_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunks = (a.E + 31) / 32, stride = 2 * a.E + 2;
  for (int job = blockIdx.x; job < a.S * chunks; job += gridDim.x) {
    const int s = job / chunks, e = (job - s * chunks) * 32 + lane;
    long long start = 0;
    if (a.seq_rows != nullptr) {
      for (int q = tid; q < s; q += FIN_WARPS * 32) start += max(0, a.seq_rows[q]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) start += __shfl_xor_sync(0xffffffffu, start, o);
      if (lane == 0) sh_start[warp] = start;
      __syncthreads();
      start = 0;
      for (int w = 0; w < FIN_WARPS; ++w) start += sh_start[w];
    }
    // the runs that hold a token of s (none: nothing was recorded); record numbers are run + s
    const long long len = a.seq_rows != nullptr ? max(0, a.seq_rows[s]) : a.T;
    const long long end = min(static_cast<long long>(a.T), start + len);
    const int r0 = static_cast<int>(min(start, static_cast<long long>(a.T)) / a.run_tokens);
    const int r1 = end > start ? static_cast<int>((end - 1) / a.run_tokens) : r0 - 1;
    float p = 0.f, z = 0.f;
    int c = 0, n = 0;
#pragma unroll 4
    for (int r = r0 + warp; r <= r1; r += FIN_WARPS) {
      const float* rec = a.record + (static_cast<size_t>(r) + s) * stride;
      if (e < a.E) {
        p += rec[e];
        c += reinterpret_cast<const int*>(rec)[a.E + e];
      }
      n += reinterpret_cast<const int*>(rec)[2 * a.E];
      z += rec[2 * a.E + 1];
    }
    sh_p[warp][lane] = p;
    sh_c[warp][lane] = c;
    if (lane == 0) { sh_z[warp] = z; sh_n[warp] = n; }
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < FIN_WARPS; ++w) { p += sh_p[w][lane]; c += sh_c[w][lane]; z += sh_z[w]; n += sh_n[w]; }
      if (e < a.E) {
        a.counts[static_cast<size_t>(s) * a.E + e] = c;
        a.kept[static_cast<size_t>(s) * a.E + e] = c;
      }
      const float dot = warp_sum(p * static_cast<float>(c));
      if (lane == 0) {
        const float nn = static_cast<float>(n);
        a.seq_loss[job] = n > 0 ? static_cast<float>(a.E) * (dot / nn) / (static_cast<float>(a.k) * nn) : 0.f;
        if (job == s * chunks) {
          a.seq_z[s] = z;
          a.seq_tokens[s] = n;
        }
      }
    }
    __syncthreads();
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) last = atomicAdd(a.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0, zs = 0.0;
  int full = 0, tokens = 0;
  for (int j = tid; j < a.S * chunks; j += FIN_WARPS * 32) sum += __ldcg(a.seq_loss + j);
  for (int s = tid; s < a.S; s += FIN_WARPS * 32) {
    zs += __ldcg(a.seq_z + s);
    const int n = __ldcg(a.seq_tokens + s);
    full += n > 0;
    tokens += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    zs += __shfl_xor_sync(0xffffffffu, zs, o);
  }
  full = __reduce_add_sync(0xffffffffu, full);
  tokens = __reduce_add_sync(0xffffffffu, tokens);
  if (lane == 0) { sh_d[0][warp] = sum; sh_d[1][warp] = zs; sh_c[warp][0] = full; sh_n[warp] = tokens; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < FIN_WARPS; ++w) { sum += sh_d[0][w]; zs += sh_d[1][w]; full += sh_c[w][0]; tokens += sh_n[w]; }
    *a.loss = full > 0 ? static_cast<float>(a.coef * sum / full + a.z * zs / tokens) : 0.f;
    a.total[0] = full > 0 ? 1.f / static_cast<float>(full) : 0.f;
    a.total[1] = tokens > 0 ? 1.f / static_cast<float>(tokens) : 0.f;
  }
}

template <typename T, int LPT, int V, int P>
__global__ void __launch_bounds__(BAL_THREADS, V * P <= 16 ? BAL_BACKWARD_BLOCKS : 2) balance_backward_kernel(const b200_balance_args a) {
  constexpr int WARPS = BAL_THREADS / 32, TOK = 32 / LPT, C = V * P;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % LPT, slot = lane / LPT;
  const long long t0 = static_cast<long long>(blockIdx.x) * a.run_tokens;
  const long long t1 = min(static_cast<long long>(a.T), t0 + a.run_tokens);
  int seq = 0;
  long long start = 0;
  if (a.seq_rows != nullptr) find_sequence(a, t0, seq, start);
  const float g = *a.grad_loss;
  const float zc = 2.f * a.z * a.total[1];
  long long pos = t0;
  while (pos < t1) {
    const bool behind = seq >= a.S;
    const long long len = behind ? 0 : a.seq_rows != nullptr ? max(0, a.seq_rows[seq]) : a.T;
    const long long end = behind ? t1 : min(t1, start + len);
    const int n = behind ? 0 : a.seq_tokens[seq];
    const float scale = n > 0 ? a.coef * a.total[0] * static_cast<float>(a.E) / (static_cast<float>(a.k) * static_cast<float>(n)) / static_cast<float>(n) : 0.f;
    float coef[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int e = expert_of<LPT, V>(i, sub);
      coef[i] = n > 0 && e < a.E ? scale * static_cast<float>(a.kept[static_cast<size_t>(seq) * a.E + e]) : 0.f;
    }
    long long t = pos + warp * TOK;
    TokenRow<T, V, P> row, next;
    bool take = false, next_take = false;
    auto load = [&](long long at, TokenRow<T, V, P>& r, bool& take) {
      const bool in = n > 0 && at < end;
      load_token<T, LPT, V, P>(a, at, in, sub, r);
      take = in && (a.mask == nullptr || a.mask[at] != 0);
    };
    load(t + slot, row, take);
    for (; t < end; t += WARPS * TOK) {
      const long long mine = t + slot;
      load(mine + WARPS * TOK, next, next_take);
      float p[C], inv, lse;
      const bool ok = token_softmax<T, LPT, V, P>(row, take, p, inv, lse);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) dot = fmaf(p[i], coef[i], dot);
#pragma unroll
      for (int o = LPT / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (mine < end) {
        T* out = static_cast<T*>(a.grad) + mine * a.E;
        const float shift = zc * lse - dot * inv, scaled = ok ? g * inv : 0.f;      // an infinite g leaves other tokens at 0
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const int e = (q * LPT + sub) * V;
          float d[V];
#pragma unroll
          for (int j = 0; j < V; ++j) d[j] = scaled * p[q * V + j] * (coef[q * V + j] + shift);
          if (e < a.E) store_pack<T, V>(out + e, d);
        }
      }
      row = next;
      take = next_take;
    }
    __syncwarp();
    pos = end;
    start += len;
    ++seq;
  }
}

template <bool BACK, typename T, int LPT, int V, int P>
static cudaError_t balance_launch(const b200_balance_args& a, cudaStream_t st) {
  b200_count_launches(1);
  if constexpr (BACK) {
    balance_backward_kernel<T, LPT, V, P><<<a.runs, BAL_THREADS, 0, st>>>(a);
    return cudaGetLastError();
  } else {
    const size_t smem = (BAL_THREADS / 32 + 1) * static_cast<size_t>(a.E) * 4;      // 36 KB at 1024 experts
    balance_forward_kernel<T, LPT, V, P><<<a.runs, BAL_THREADS, smem, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    b200_count_launches(1);
    const long long jobs = static_cast<long long>(a.S) * ((a.E + 31) / 32);
    return launch_chained(balance_finish_kernel, dim3(static_cast<unsigned>(jobs < 592 ? jobs : 592)), dim3(FIN_WARPS * 32), 0, st, a);
  }
}

// Lanes per token: 16 experts a lane, so that a warp has several tokens in work and what is done once per token (shuffles,
// addresses, counts) is shared; with 8 a lane the kernels took half as many instructions again.
// Rows that do not start on 16 bytes have fewer forms.
template <bool BACK, typename T, int V>
static cudaError_t balance_lanes(const b200_balance_args& a, cudaStream_t st) {
  constexpr int P = 16 / V;
  if constexpr (V > 1) {
    if (a.E <= 8) return balance_launch<BACK, T, 1, V, 8 / V>(a, st);
    if (a.E > 16 && a.E <= 32) return balance_launch<BACK, T, 2, V, P>(a, st);
    if (a.E > 32 && a.E <= 64) return balance_launch<BACK, T, 4, V, P>(a, st);
    if (a.E > 128 && a.E <= 256) return balance_launch<BACK, T, 16, V, P>(a, st);
  }
  if (a.E <= 16) return balance_launch<BACK, T, 1, V, P>(a, st);
  if (a.E <= 128) return balance_launch<BACK, T, 8, V, P>(a, st);
  if (a.E <= 512) return balance_launch<BACK, T, 32, V, P>(a, st);
  return balance_launch<BACK, T, 32, V, 2 * P>(a, st);
}

template <bool BACK, typename T>
static cudaError_t balance_dispatch(const b200_balance_args& a, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const bool aligned = a.E % V == 0 && a.ld % V == 0 && reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
  return aligned ? balance_lanes<BACK, T, V>(a, st) : balance_lanes<BACK, T, 1>(a, st);
}

template <bool BACK>
static int balance_run(const b200_balance_args* a, void* stream) {
  if (a == nullptr || a->T < 1 || a->T > BAL_MOST || a->E < 1 || a->E > BAL_MAX_E || a->k < 1 || a->S < 1 || a->runs < 1 || a->run_tokens < 1 ||
      static_cast<long long>(a->runs) * a->run_tokens < a->T || static_cast<long long>(a->runs - 1) * a->run_tokens >= a->T ||
      static_cast<long long>(a->S) * ((a->E + 31) / 32) > BAL_MOST)
    return -10;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (a->elem) {
    case ELEM_F32: return static_cast<int>(balance_dispatch<BACK, float>(*a, st));
    case ELEM_BF16: return static_cast<int>(balance_dispatch<BACK, __nv_bfloat16>(*a, st));
    case ELEM_F16: return static_cast<int>(balance_dispatch<BACK, __half>(*a, st));
  }
  return -14;
}

}  // namespace b200

extern "C" {

int b200_balance_forward(const b200_balance_args* a, void* stream) { return b200::balance_run<false>(a, stream); }
int b200_balance_backward(const b200_balance_args* a, void* stream) { return b200::balance_run<true>(a, stream); }

// Blocks (runs of tokens) of a call: as many as are in work at once, but no shorter than 32 KB of logits (a record is written
// and read per run).
int b200_balance_runs(int T, int E, int elem, int backward, int sms) {
  const long long bytes = static_cast<long long>(T) * E * (elem == b200::ELEM_F32 ? 4 : 2);
  const long long want = (bytes + 32767) / 32768, most = static_cast<long long>(backward ? b200::BAL_BACKWARD_BLOCKS : b200::BAL_FORWARD_BLOCKS) * sms;
  const long long runs = want < most ? want : most;
  return static_cast<int>(runs < T ? runs : T);
}

int b200_balance_max_experts() { return b200::BAL_MAX_E; }
int b200_abi_size_balance_args() { return static_cast<int>(sizeof(b200_balance_args)); }

}  // extern "C"
