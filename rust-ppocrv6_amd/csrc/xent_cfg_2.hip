// Kernels of the vocabulary losses on 32-bit tensors (two fp16 planes).
#include "xent_kernels.hpp"

namespace ppocr {
PPOCR_XENT_INSTANCES(1, 2)
PPOCR_XENT_INSTANCES(2, 2)
PPOCR_XENT_INSTANCES(3, 2)
PPOCR_XENT_INSTANCES(4, 2)
PPOCR_XENT_INSTANCES(6, 2)
PPOCR_XENT_INSTANCES(8, 2)
}  // namespace ppocr
