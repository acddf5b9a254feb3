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
// A block takes a run of tokens and walks the sequences in it one after another; 2^x lanes share a token.  Column
// sums stay in registers until the sequence or the run ends; then one record per (run, sequence) is written: sums of p,
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
  float* seq_loss;           // [S][2]: a sequence's balance term, its sum of lse^2
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

// One token's softmax over the lanes that share it: p[i] for expert i * LPT + sub.  False: it takes no part.
template <typename T, int LPT, int C>
__device__ __forceinline__ bool token_softmax(const b200_balance_args& a, long long t, bool in, int sub, float (&p)[C], float& lse) {
  if (in && a.mask != nullptr) in = a.mask[t] != 0;
  const T* row = static_cast<const T*>(a.logits) + t * a.ld;
  float mx = -CUDART_INF_F;
  bool ok = true;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int e = i * LPT + sub;
    p[i] = in && e < a.E ? to_f32(row[e]) : -CUDART_INF_F;
    ok = ok && !(p[i] != p[i]);
    mx = fmaxf(mx, p[i]);
  }
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  ok = ok && mx > lowest<T>() && mx < CUDART_INF_F;
  // every lane of the token has to have seen no NaN
  const unsigned all = __ballot_sync(0xffffffffu, ok);
  const unsigned mine = (LPT == 32 ? 0xffffffffu : ((1u << LPT) - 1u) << ((threadIdx.x & 31) / LPT * LPT));
  ok = (all & mine) == mine;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    p[i] = ok ? expf(p[i] - mx) : 0.f;
    sum += p[i];
  }
#pragma unroll
  for (int o = LPT / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = ok ? 1.f / sum : 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) p[i] *= inv;
  lse = ok ? mx + logf(sum) : 0.f;
  return ok;
}

template <typename T, int LPT, int C>
__global__ void __launch_bounds__(BAL_THREADS) balance_forward_kernel(const b200_balance_args a) {
  extern __shared__ float sm[];              // [warps][E] sums of p, then int [E] counts
  __shared__ float warp_z[BAL_THREADS / 32];
  __shared__ int warp_n[BAL_THREADS / 32];
  constexpr int WARPS = BAL_THREADS / 32, TOK = 32 / LPT;
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
    for (long long t = pos + warp * TOK; t < end; t += WARPS * TOK) {
      float p[C], lse;
      const long long mine = t + slot;
      const bool ok = token_softmax<T, LPT, C>(a, mine, mine < end, sub, p, lse);
      if (!ok) continue;
#pragma unroll
      for (int i = 0; i < C; ++i) col[i] += p[i];
      for (int j = sub; j < a.k; j += LPT) {
        const int e = a.idx[mine * a.k + j];
        if (e >= 0 && e < a.E) atomicAdd(cnt + e, 1);
      }
      if (sub == 0) { zsum += lse * lse; ++tokens; }
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int o = LPT; o < 32; o <<= 1) col[i] += __shfl_xor_sync(0xffffffffu, col[i], o);
      if (slot == 0 && i * LPT + sub < a.E) sm[warp * a.E + i * LPT + sub] = col[i];
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

// One block per sequence: adds its records, writes its counts and its term; the last block adds the terms.
__global__ void __launch_bounds__(BAL_THREADS) balance_finish_kernel(const b200_balance_args a) {
  __shared__ float red[BAL_THREADS / 32];
  __shared__ double dred[2][BAL_THREADS / 32];
  __shared__ int nred[2][BAL_THREADS / 32];
  __shared__ long long ired[BAL_THREADS / 32];
  __shared__ int last;
  chain_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int stride = 2 * a.E + 2;
  for (int s = blockIdx.x; s < a.S; s += gridDim.x) {
    // tokens [start, start + len) lie in runs start / run_tokens ... ; record numbers are run + s
    long long start = 0;
    if (a.seq_rows != nullptr) {
      long long part = 0;
      for (int q = tid; q < s; q += BAL_THREADS) part += max(0, a.seq_rows[q]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
      if (lane == 0) ired[warp] = part;
      __syncthreads();
      for (int w = 0; w < BAL_THREADS / 32; ++w) start += ired[w];
      __syncthreads();
    }
    const long long len = a.seq_rows != nullptr ? max(0, a.seq_rows[s]) : a.T;
    const long long end = min(static_cast<long long>(a.T), start + len);
    // runs that hold a token of s; none: no record is read
    const int r0 = static_cast<int>(min(start, static_cast<long long>(a.T)) / a.run_tokens);
    const int r1 = end > start ? static_cast<int>((end - 1) / a.run_tokens) : r0 - 1;
    int n = 0;
    float z = 0.f;
    for (int r = r0; r <= r1; ++r) {
      const float* rec = a.record + (static_cast<size_t>(r) + s) * stride;
      n += reinterpret_cast<const int*>(rec)[2 * a.E];
      z += rec[2 * a.E + 1];
    }
    float dot = 0.f;
    for (int e = tid; e < a.E; e += BAL_THREADS) {
      float p = 0.f;
      int c = 0;
      for (int r = r0; r <= r1; ++r) {
        const float* rec = a.record + (static_cast<size_t>(r) + s) * stride;
        p += rec[e];
        c += reinterpret_cast<const int*>(rec)[a.E + e];
      }
      a.counts[static_cast<size_t>(s) * a.E + e] = c;
      a.kept[static_cast<size_t>(s) * a.E + e] = c;
      dot += p * static_cast<float>(c);
    }
    dot = warp_sum(dot);
    if (lane == 0) red[warp] = dot;
    __syncthreads();
    if (tid == 0) {
      float v = 0.f;
      for (int w = 0; w < BAL_THREADS / 32; ++w) v += red[w];
      const float nn = static_cast<float>(n);
      a.seq_loss[2 * s] = n > 0 ? static_cast<float>(a.E) * (v / nn) / (static_cast<float>(a.k) * nn) : 0.f;
      a.seq_loss[2 * s + 1] = z;
      a.seq_tokens[s] = n;
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
  int full = 0;
  long long tokens = 0;
  for (int s = tid; s < a.S; s += BAL_THREADS) {
    sum += __ldcg(a.seq_loss + 2 * s);
    zs += __ldcg(a.seq_loss + 2 * s + 1);
    const int n = __ldcg(a.seq_tokens + s);
    full += n > 0;
    tokens += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    zs += __shfl_xor_sync(0xffffffffu, zs, o);
    full += __shfl_xor_sync(0xffffffffu, full, o);
    tokens += __shfl_xor_sync(0xffffffffu, tokens, o);
  }
  if (lane == 0) { dred[0][warp] = sum; dred[1][warp] = zs; nred[0][warp] = full; nred[1][warp] = static_cast<int>(tokens); }
  __syncthreads();
  if (tid == 0) {
    sum = zs = 0.0;
    full = 0;
    int n = 0;
    for (int w = 0; w < BAL_THREADS / 32; ++w) { sum += dred[0][w]; zs += dred[1][w]; full += nred[0][w]; n += nred[1][w]; }
    const float inv_s = full > 0 ? 1.f / static_cast<float>(full) : 0.f, inv_n = n > 0 ? 1.f / static_cast<float>(n) : 0.f;
    *a.loss = full > 0 ? static_cast<float>(a.coef * sum / full + a.z * zs / n) : 0.f;
    a.total[0] = inv_s;
    a.total[1] = inv_n;
  }
}

template <typename T, int LPT, int C>
__global__ void __launch_bounds__(BAL_THREADS) balance_backward_kernel(const b200_balance_args a) {
  constexpr int WARPS = BAL_THREADS / 32, TOK = 32 / LPT;
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
      const int e = i * LPT + sub;
      coef[i] = n > 0 && e < a.E ? scale * static_cast<float>(a.kept[static_cast<size_t>(seq) * a.E + e]) : 0.f;
    }
    for (long long t = pos + warp * TOK; t < end; t += WARPS * TOK) {
      float p[C], lse;
      const long long mine = t + slot;
      const bool in = mine < end;
      const bool ok = token_softmax<T, LPT, C>(a, mine, in && n > 0, sub, p, lse);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < C; ++i) dot += p[i] * coef[i];
#pragma unroll
      for (int o = LPT / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (!in) continue;
      T* out = static_cast<T*>(a.grad) + mine * a.E;
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int e = i * LPT + sub;
        if (e < a.E) out[e] = from_f32<T>(ok ? g * (p[i] * (coef[i] - dot) + zc * lse * p[i]) : 0.f);
      }
    }
    __syncwarp();
    pos = end;
    start += len;
    ++seq;
  }
}

template <bool BACK, typename T, int LPT, int C>
static cudaError_t balance_launch(const b200_balance_args& a, cudaStream_t st) {
  b200_count_launches(1);
  if constexpr (BACK) {
    balance_backward_kernel<T, LPT, C><<<a.runs, BAL_THREADS, 0, st>>>(a);
    return cudaGetLastError();
  } else {
    const size_t smem = (BAL_THREADS / 32 + 1) * static_cast<size_t>(a.E) * 4;      // 36 KB at 1024 experts
    balance_forward_kernel<T, LPT, C><<<a.runs, BAL_THREADS, smem, st>>>(a);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    b200_count_launches(1);
    return launch_chained(balance_finish_kernel, dim3(a.S < 592 ? a.S : 592), dim3(BAL_THREADS), 0, st, a);
  }
}

template <bool BACK, typename T>
static cudaError_t balance_dispatch(const b200_balance_args& a, cudaStream_t st) {
  if (a.E <= 4) return balance_launch<BACK, T, 1, 4>(a, st);
  if (a.E <= 8) return balance_launch<BACK, T, 2, 4>(a, st);
  if (a.E <= 16) return balance_launch<BACK, T, 4, 4>(a, st);
  if (a.E <= 32) return balance_launch<BACK, T, 8, 4>(a, st);
  if (a.E <= 64) return balance_launch<BACK, T, 16, 4>(a, st);
  if (a.E <= 128) return balance_launch<BACK, T, 32, 4>(a, st);
  if (a.E <= 256) return balance_launch<BACK, T, 32, 8>(a, st);
  return balance_launch<BACK, T, 32, 32>(a, st);
}

template <bool BACK>
static int balance_run(const b200_balance_args* a, void* stream) {
  if (a == nullptr || a->T < 1 || a->E < 1 || a->E > BAL_MAX_E || a->k < 1 || a->S < 1 || a->runs < 1 || a->run_tokens < 1 ||
      static_cast<long long>(a->runs) * a->run_tokens < a->T || static_cast<long long>(a->runs - 1) * a->run_tokens >= a->T)
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

// Blocks (runs of tokens) of a call: as many as fill the GPU four times over, but no fewer tokens each than the
// warps of a block take in one turn.
int b200_balance_runs(int T, int E, int sms) {
  int lanes = 1;
  while (lanes < 32 && lanes * 4 < E) lanes *= 2;
  const int turn = b200::BAL_THREADS / lanes;
  const int want = (T + turn - 1) / turn, most = 4 * sms;
  return want < most ? want : most;
}

int b200_abi_size_balance_args() { return static_cast<int>(sizeof(b200_balance_args)); }

}  // extern "C"
