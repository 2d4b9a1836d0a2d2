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

// cuTensorMapEncodeTiled of the installed driver (nullptr if it has none).
PFN_cuTensorMapEncodeTiled_v12000 get_encode_fn();

}  // namespace gg
}  // namespace moe
