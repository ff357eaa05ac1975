// The arguments of one ms_class_ce* call, and the narrow form's entry (ms_class_ce_narrow.hip) for the dispatch in ms_class_ce.hip.
#pragma once
#include "ms_common.h"

namespace ms {
struct CeArgs {
  const void *h, *w; const float* b; const int64_t* labels;
  float *loss, *nll, *lse; const float *lse_in, *grad; void *dh, *dw; float* db;
  float sign; int mean_valid; const float* scale_dev;
  int N, C, V, HW, types; void* ws; size_t ws_bytes; hipStream_t st;
};
bool ce_narrow_ok(int N, int C, int V, int HW);
size_t ce_narrow_ws_bytes(int N, int C, int V, int HW, int types, bool grad);
int ce_narrow_run(const CeArgs& a, bool grad, const char* who);
}  // namespace ms
