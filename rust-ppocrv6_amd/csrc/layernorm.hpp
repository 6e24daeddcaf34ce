// LayerNorm over rows, forward and backward (layernorm.hip).
#pragma once
#include "common.hpp"

namespace ppocr {

constexpr int64_t kLayerNormMaxD = 16384;
// Workgroups of the backward pass, each with a sum of dw and db of its own.
int layernorm_parts(int64_t m, int64_t d);
int launch_layernorm_forward(const void* x, const float* w, const float* b, int64_t m, int d, float eps, int bf16, void* y,
                             float* mean, float* rstd, hipStream_t st);
// part: [layernorm_parts][2][d]; dx, dw, db may be null
int launch_layernorm_backward(const void* dy, const void* x, const float* w, const float* mean, const float* rstd, int64_t m,
                              int d, int bf16, void* dx, float* dw, float* db, float* part, hipStream_t st);

}  // namespace ppocr
