// Order in which persistent GEMM kernels take the tiles of a grouped product.
#pragma once
#include <cuda_runtime.h>

namespace b200 {

// Maps a linear tile index to (group, m-tile, n-tile).  Tiles are ordered per
// group in chunks of `gm` M-tiles; inside a chunk the M index runs fastest so
// that concurrently running CTAs share a few weight tiles and a chunk of A
// that stays resident in L2 while the N index sweeps.
template <typename Tables>
__host__ __device__ __forceinline__ bool decode_tile(const Tables& c, int G, int TN, int gm, int idx, int& cursor,
                                            int& g, int& m, int& n) {
  while (cursor < G && idx >= TN * c.g_sched_start[cursor + 1]) ++cursor;
  if (cursor >= G) return false;
  g = cursor;
  const int tm = c.g_sched_start[g + 1] - c.g_sched_start[g];
  const int j = idx - TN * c.g_sched_start[g];
  // even out the chunks of this group: 16 M-tiles with a target of 12 become 8 + 8, not 12 + 4
  const int nchunks = (tm + gm - 1) / gm;
  gm = (tm + nchunks - 1) / nchunks;
  const int chunk_tiles = gm * TN;
  const int ch = j / chunk_tiles;
  const int r = j - ch * chunk_tiles;
  const int cm = (gm < tm - ch * gm) ? gm : (tm - ch * gm);
  n = r / cm;
  m = ch * gm + (r - n * cm);
  return true;
}

// Which tiles a scheduler (a CTA, or a CTA pair) takes: first, first + stride, ...
// Even rounds: with R = ceil(tiles / schedulers) rounds needed anyway, only ceil(tiles / R)
// schedulers take tiles, R each (the last ones maybe one fewer), instead of all of them taking
// R - 1 and a few taking one more.  The makespan in tiles is the same; when the kernel streams
// weights (few rows per expert) the last round no longer runs on a handful of SMs that cannot
// draw the full memory bandwidth.  Schedulers past the stride sit out (first = total).
__host__ __device__ __forceinline__ void tile_walk(int total, int schedulers, int sched_id, int& first,
                                                   int& stride) {
  const int rounds = (total + schedulers - 1) / schedulers;
  stride = rounds > 0 ? (total + rounds - 1) / rounds : schedulers;
  first = sched_id < stride ? sched_id : total;
}

}  // namespace b200
