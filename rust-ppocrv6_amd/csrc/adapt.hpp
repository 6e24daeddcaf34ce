// Low-rank adapters beside the vocabulary projection (adapt.hip), and merged into a weight (merge.hip).
#pragma once
#include "kernels.hpp"

namespace ppocr {

constexpr int kAdaptMostRank = 64;
constexpr int kAdaptMostSlots = 4096;

// What the kernels need of a slot's adapter (device memory, written when the slot is set).
struct AdapterMeta {
    int shift;  // the head's products are scaled by 2^-shift beside the adapter's
};

// The adapters of a head: records in device memory, one set a slot, and one of zeros behind the last slot
// for lines without an adapter.
struct Adapters {
    int slots = 0, max_rank = 0;
    int steps = 0;  // 16-rank steps of the records: 1, 2 or 4
    int G = 0, tiles = 0;
    uint8_t* down = nullptr;  // [slots + 1][tiles of 32 ranks] fragments of both halves
    uint8_t* up = nullptr;    // [slots + 1][class tiles][halves][steps][2][32][8]
    AdapterMeta* meta = nullptr;
    unsigned* range = nullptr;  // [slots + 1][2][kAdaptMostRank] sizes that a slot's powers of two come from
    // The head's fp16 records and the classes' units [n]: up is held divided by them, as the products of the
    // records are.  An INT8 head's own, or where its scales lie far apart others with nearer units; for an FP32 head
    // records of each class's weights over a power of two.
    const uint8_t* rec = nullptr;
    const float* unit = nullptr;
    uint8_t* own_rec = nullptr;
    float* own_unit = nullptr;
    size_t down_bytes() const;  // of a slot
    size_t up_bytes() const;
};

// Text lines and their slots on the device.
struct AdaptLines {
    const int64_t* off;
    int64_t lines;
    const int32_t* slot;
};

// Sets the zero records of every slot.
int launch_adapters_clear(const Adapters& ad, hipStream_t st);
// Records of a slot from its adapter, down [rank][k] and up [n][rank] of fp32 or bf16 (rank 0: none).
int launch_adapter_set(const Adapters& ad, int slot, const void* down, const void* up, int rank, float scale, int bf16, int64_t n,
                       int64_t k, hipStream_t st);

size_t adapt_workspace(const Adapters& ad, int64_t m);
// cfg: CFG_H2 (INT8 head) or CFG_HF3 (FP32 head).
int launch_adapt_logits(int cfg, const TileGeom& tg, const Adapters& ad, const AdaptLines& lines, const float* a, int64_t m,
                        int64_t n, int64_t k, float* out, uint8_t* ws, hipStream_t st);
int launch_adapt_decode(int cfg, const TileGeom& tg, const Adapters& ad, const AdaptLines& lines, const float* a, int64_t m,
                        int64_t n, int64_t k, int32_t* idx, float* maxprob, const CtcOut& ctc, uint8_t* ws,
                        hipStream_t st);

struct MergeArgs {
    const void* w;   // forward: the weight that the adapter is merged into
    const void* dw;  // backward: the merged weight's gradient
    const void* down;
    const void* up;
    int64_t n;
    int k, rank;
    float scale;
    int bf16;
    void* out;
};
int launch_merge(const MergeArgs& x, hipStream_t st);
// Groups of rows of the backward pass, each with a sum of ddown of its own: part [parts][rank][k].
int merge_parts(int64_t n, int64_t k);
int launch_merge_backward(const MergeArgs& x, void* ddown, void* dup, float* part, hipStream_t st);

}  // namespace ppocr
