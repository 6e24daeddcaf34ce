// The global norm of many gradients and their clipping (grad_clip.hip).
#pragma once
#include <vector>

#include "common.hpp"

namespace ppocr {

struct GradTensor {
    const void* in;
    void* out;
    int64_t count;
    int bf16;
};
// Partial sums, 8 bytes each, that tensors of these sizes leave in the workspace at most.
int64_t grad_clip_most_parts(const int64_t* sizes, int64_t count);
int launch_grad_clip(const std::vector<GradTensor>& tensors, float most, float* norm, double* parts, hipStream_t st);

}  // namespace ppocr
