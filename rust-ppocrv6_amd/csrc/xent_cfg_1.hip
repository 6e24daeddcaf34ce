// Kernels of the vocabulary losses on bf16 tensors (one fp16 plane).
#include "xent_kernels.hpp"

namespace ppocr {
PPOCR_XENT_INSTANCES(1, 1)
PPOCR_XENT_INSTANCES(2, 1)
PPOCR_XENT_INSTANCES(3, 1)
PPOCR_XENT_INSTANCES(4, 1)
PPOCR_XENT_INSTANCES(6, 1)
PPOCR_XENT_INSTANCES(8, 1)
}  // namespace ppocr
