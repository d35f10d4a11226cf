// The plan of a decode step whose launch shape depends on the batch size alone: which piece of which request's keys a
// workgroup computes, derived on the device from seq_lens.  Shared by the 16-bit / fp8 decode kernel (tmx_decode.hip)
// and the 4-bit one (tmx_fp4_decode.hip).
#pragma once

#include "tmx_common.h"

namespace tmx {

// ---- the fixed-grid form's plan (see DecodeParams): computed by every workgroup for itself ----
// Sum of v over the NT threads of the workgroup (sm: NT / 64 ints of LDS, free again on return).
template <int NT>
__device__ __forceinline__ int dc_block_sum(int v, int* sm, int tid) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if ((tid & 63) == 0) sm[tid >> 6] = v;
  __syncthreads();
  int tot = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) tot += sm[w];
  __syncthreads();
  return tot;
}
__device__ __forceinline__ int dc_tiles_of(int n) { return n > 0 ? (n + kBlockN - 1) / kBlockN : 0; }
// Piece length of the step: one piece per workgroup slot of the chip, at least 8 tiles.
__device__ __forceinline__ int dc_piece_len(long long total_tiles, int units, int slots) {
  const long long c = (total_tiles * units + slots - 1) / slots;
  return c < 8 ? 8 : (int)c;
}
struct DcPiece {
  int b, n, tile0, ntiles, pieces;  // request (-1: no such piece), its keys, the piece's tiles, the request's piece count
};
// The request that owns piece w of the step, and which of its tiles the piece covers.  All NT threads call it.
template <int NT>
__device__ __forceinline__ DcPiece dc_find_piece(const int32_t* seq_lens, int batch, int units, int slots, int w, int* sm, int tid) {
  const int per = (batch + NT - 1) / NT;  // requests per thread, a contiguous run
  const int j0 = imin(batch, tid * per), j1 = imin(batch, j0 + per);
  int mine = 0;
  for (int j = j0; j < j1; ++j) mine += dc_tiles_of(seq_lens[j]);
  const int total = dc_block_sum<NT>(mine, sm, tid);
  const int P = dc_piece_len(total, units, slots);
  int cnt = 0;
  for (int j = j0; j < j1; ++j) cnt += (dc_tiles_of(seq_lens[j]) + P - 1) / P;
  // exclusive prefix of cnt over the threads: inside the wave by shuffles, across waves through LDS
  int inc = cnt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int up = __shfl_up(inc, d, 64);
    if ((tid & 63) >= d) inc += up;
  }
  if ((tid & 63) == 63) sm[tid >> 6] = inc;
  if (tid == 0) sm[NT / 64] = -1;  // the answer's slot: (request, first piece of the request)
  __syncthreads();
  int start = inc - cnt;
  for (int x = 0; x < (tid >> 6); ++x) start += sm[x];
  if (w >= start && w < start + cnt) {
    int first = start;
    for (int j = j0; j < j1; ++j) {
      const int pj = (dc_tiles_of(seq_lens[j]) + P - 1) / P;
      if (w < first + pj) {
        sm[NT / 64] = j;
        sm[NT / 64 + 1] = first;
        break;
      }
      first += pj;
    }
  }
  __syncthreads();
  DcPiece r;
  r.b = sm[NT / 64];
  if (r.b < 0) return r;
  r.n = seq_lens[r.b];
  const int tiles = dc_tiles_of(r.n);
  r.pieces = (tiles + P - 1) / P;
  r.tile0 = (w - sm[NT / 64 + 1]) * P;
  r.ntiles = imin(P, tiles - r.tile0);
  return r;
}

}  // namespace tmx
