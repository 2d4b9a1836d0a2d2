// Group table of the grouped GEMMs: which rows of x go with which weight matrix.
//
// moe_grouped_gemm_plan_splits / _plan_ep write it into the caller's
// workspace on the device; the bf16 and the 8-bit grouped GEMM read it.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include "moe_common.cuh"

namespace moe {
namespace gg {

struct WsLayout {
  int32_t* err;
  int32_t* row_start;
  int32_t* rows;
  int32_t* widx;
  int32_t* tmp;
  int32_t* rows_body;   // whole 256-row tiles of each group (CTA-pair kernel)
  int32_t* tail_start;  // first row after them
  int32_t* rows_tail;   // remaining rows (single-CTA kernel)
};

inline size_t ws_array_bytes(int64_t G) {
  return (static_cast<size_t>(G) * 4 + 255) & ~static_cast<size_t>(255);
}
inline size_t ws_bytes(int64_t G) { return 256 + 7 * ws_array_bytes(G); }

inline WsLayout ws_layout(const void* ws, int64_t G) {
  char* b = static_cast<char*>(const_cast<void*>(ws));
  const size_t a = ws_array_bytes(G);
  WsLayout l;
  l.err = reinterpret_cast<int32_t*>(b);
  l.row_start = reinterpret_cast<int32_t*>(b + 256);
  l.rows = reinterpret_cast<int32_t*>(b + 256 + a);
  l.widx = reinterpret_cast<int32_t*>(b + 256 + 2 * a);
  l.tmp = reinterpret_cast<int32_t*>(b + 256 + 3 * a);
  l.rows_body = reinterpret_cast<int32_t*>(b + 256 + 4 * a);
  l.tail_start = reinterpret_cast<int32_t*>(b + 256 + 5 * a);
  l.rows_tail = reinterpret_cast<int32_t*>(b + 256 + 6 * a);
  return l;
}

struct Tile {
  int g;
  int m_idx;
  int n_idx;
};

// Maps a linear tile index to (group, M-tile, N-tile), kTileM rows per M-tile.
// Indices handed to one CTA (or CTA pair) only grow, so the walk only moves
// forward. n_chunk 0: inside a group, super-rows of `raster` M-tiles sweep all
// N-tiles.
// n_chunk > 0 replaces the super-rows by N-chunks: a group's tiles are walked
// chunk by chunk of n_chunk N-tiles, and inside a chunk M-tile by M-tile
// (every N-tile of the chunk for one M-tile, then the next M-tile). The CTA
// pairs running at once then share one M-tile of rows and one chunk of the
// weight slab, which is sized to stay in L2 while all of the group's M-tiles
// stream past it; rows are read once per chunk.
template <int kTileM>
struct WalkerRT {
  const int32_t* rows;
  int G;
  int n_tiles;
  int raster;
  int n_chunk;
  int above = 0;            // groups of more than `above` rows ...
  int most = 0x7fffffff;    // ... and at most `most` are walked
  int g = 0;
  int mt = -1;
  long long base = 0;

  __device__ bool locate(long long t, Tile& tile) {
    while (g < G) {
      if (mt < 0) {
        const int r = rows[g];
        mt = r > above && r <= most ? (r - 1) / kTileM + 1 : 0;
      }
      const long long cnt = static_cast<long long>(mt) * n_tiles;
      if (t < base + cnt) break;
      base += cnt;
      ++g;
      mt = -1;
    }
    if (g >= G) return false;
    const long long local = t - base;
    tile.g = g;
    if (n_chunk > 0) {
      const long long full = static_cast<long long>(mt) * n_chunk;  // tiles of a whole chunk
      const int ci = static_cast<int>(local / full);
      const int rem = static_cast<int>(local - ci * full);
      const int nc = min(n_chunk, n_tiles - ci * n_chunk);  // the last chunk may be narrower
      tile.m_idx = rem / nc;
      tile.n_idx = ci * n_chunk + rem % nc;
      return true;
    }
    const long long sr_tiles = static_cast<long long>(raster) * n_tiles;
    const int sr = static_cast<int>(local / sr_tiles);
    const int within = static_cast<int>(local - sr * sr_tiles);
    const int mg = min(raster, mt - sr * raster);
    tile.n_idx = within / mg;
    tile.m_idx = sr * raster + within % mg;
    return true;
  }
};

// Bounded wait for copies or MMAs in flight before a kernel gives up or ends.
MOE_DEVICE bool wait_drain(uint32_t bar, uint32_t parity) {
  const unsigned long long t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitTimeoutNs) return false;
  }
  return true;
}

MOE_DEVICE void raise_abort(volatile int* abort_flag, int32_t* err, int code) {
  atomicCAS(err, 0, code);
  *abort_flag = 1;
  __threadfence_block();
}

// cuTensorMapEncodeTiled of the installed driver (nullptr if it has none).
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

}  // namespace gg
}  // namespace moe
