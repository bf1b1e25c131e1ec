// What the entry points (token_api.hip) hand to clip.hip: norms of gradients, and clipping.
#pragma once

#include "../../include/dci_hip.h"
#include "token_common.h"

namespace dcih {

int64_t clip_work_bytes(const dcih_span* spans, int64_t n);
bool clip_fits(const dcih_span* spans, int64_t n);          // in one grid
int grad_norm(const dcih_span* spans, int64_t n, double scale, float* norm, void* work, hipStream_t s);
int clip_grads(const dcih_span* spans, int64_t n, double max_norm, double scale, float* norm, void* work, hipStream_t s);

}  // namespace dcih
