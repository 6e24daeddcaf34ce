// Losses over the vocabulary without keeping the logits: host-side declarations (xent.hip,
// xent_kernels.hpp).
//
//   z = a W^T + b          a [m][k], W [n][k], b [n] (or none)
//   lse_r = log sum_j exp(z_rj / tau)
//   loss_r = sum_i q_ri (log q_ri - z_r,c(r,i) / tau + lse_r)
//   dz_rj = g_r / tau (p_rj - sum_{i: c(r,i) = j} q_ri),   p = exp(z / tau - lse)
//   da = dz W,  dW = dz^T a,  db = sum_r dz_r
//
// Cross entropy is the case of one target entry with q = 1 and tau = 1; distillation takes q
// as the softmax of a teacher's kept logits over tau.  The backward pass computes the logits
// again, tile by tile.
#pragma once
#include "common.hpp"

namespace ppocr {

constexpr int kXentMaxK = 256;       // inner dimension
constexpr int kXentMaxTargets = 64;  // target entries of a row
constexpr int64_t kXentMost = 1 << 24;  // rows and classes (a list key holds a class and 5 bits of row in 32)

// Operand images.  A tensor of `rows` entries (activation rows or classes) of k values becomes
// one record per 32 entries: every value times 2^e, e chosen so that the largest magnitude lies in
// [2^14, 2^15), as one fp16 plane (bf16 tensors: exact down to 2^-27 of an entry's largest value) or
// two (32-bit tensors: high and low halves, 22 bits down to 2^-12 of it, and below that to within 2^-35
// of it), in the order the MFMA fragments are read.  The entries share e where their own largest values are within 16 of each
// other; otherwise each has its own, so that a row of huge values, padding perhaps, takes no bits from
// its neighbours.
//   [plane][2 D steps of 16 k][lane][8]     entry lane % 32, k = 16 step + 8 (lane / 32) + j
//   [plane][D][2][lane][8]                  transposed: k = 32 d + lane % 32, and the entries
//                                           in the order an MFMA result holds its rows
//                                           (backward only)
//   float[32], float[32], float[16], float[32]   per entry: class: bias log2(e) / tau; row: lse
//                                           log2(e) and gradient factor times 2^-ge; then 2^-e, e (of
//                                           the largest entry), the largest L2 norm of an entry, the
//                                           largest finite magnitude among the first 32 values, the
//                                           exponent bound that XentGradSide::str_u holds, ge, and
//                                           whether the entries share e; per entry 2^-e
// D = the number of 32-wide pieces of k, one of 1, 2, 3, 4, 6, 8.
constexpr int kXentAux = 448;
constexpr int kXentNone = -1000;  // the exponent bound of a record without gradients
inline int xent_pieces(int64_t k) {
    const int d = (int)((k + 31) / 32);
    return d <= 4 ? (d < 1 ? 1 : d) : (d <= 6 ? 6 : 8);
}
inline int64_t xent_tiles(int64_t rows) { return (rows + 31) / 32; }
inline size_t xent_rec_bytes(int D, int planes, bool back) {
    return (size_t)planes * D * 2048 * (back ? 2 : 1) + kXentAux;
}

// The problem of a call.  target is set for cross entropy, teacher_idx / teacher_z for
// distillation (tn entries a row).
struct XentProblem {
    const void* a;
    const void* w;
    const float* bias;
    const int32_t* target;
    const int32_t* teacher_idx;
    const float* teacher_z;
    int tn;
    float tau;
    int64_t m, n;
    int k, bf16;
    const float* lse;   // backward
    const float* grad;  // backward, may be null (1)
    int planes() const { return bf16 ? 1 : 2; }
};

// Sizes and offsets of a call's workspace.
struct XentLayout {
    int D;
    int64_t row_tiles, class_tiles;
    int fblocks;             // blocks of 32 rows of a wave of the statistics pass
    int fsplit, fper;        // its chunks of class records, records of a chunk
    int split_a, per_a;      // chunks of class records for da
    int split_w, per_w;      // chunks of row records for dW
    // forward
    size_t f_row_rec, f_class_rec, f_class_u, f_part, f_total;
    // backward
    size_t b_row_rec, b_class_rec, b_row_u, b_class_u, b_keys, b_vals, b_offs, b_part_a, b_part_w, b_part_db, b_total;
    size_t total() const { return f_total > b_total ? f_total : b_total; }
};
XentLayout xent_layout(int64_t m, int64_t n, int64_t k, int tn, int planes);

int launch_xent_forward(const XentProblem& x, float* loss, float* lse, uint8_t* ws, hipStream_t st);
int launch_xent_backward(const XentProblem& x, void* da, void* dw, float* db, uint8_t* ws, hipStream_t st);
int launch_xent_zero(const XentProblem& x, void* dw, float* db, hipStream_t st);  // gradients of no rows

// ---------------------------------------------------------------- kernels by configuration
struct XentStatsArgs {
    const uint8_t* own;  // row records (forward form)
    const uint8_t* str;  // class records
    const int* str_u;    // as XentGradSide's; only the last bit is used
    int64_t m;
    int64_t tiles;  // class records
    int nsplit, per_split;
    float c0;     // log2(e) / tau
    float2* part;  // [nsplit][m]: reference and sum of exp2(t - reference)
};
struct XentGradSide {
    const uint8_t* own;  // owner records
    const uint8_t* str;  // stream records
    int64_t owners;     // rows or classes
    int64_t own_tiles;  // their records
    int64_t str_tiles;
    const int* str_u;  // per stream record: twice the exponent bound of what is summed over it (kXentNone:
                       // nothing), and 1 where its entries have scales of their own
    int nsplit, per_split;
    float* part;  // [nsplit][owners][32 D]
};
struct XentGradArgs {
    XentGradSide rows, classes;  // da, dW
    unsigned row_grid;           // workgroups of da, the others are dW's
    float c0;
    const uint32_t* keys;
    const float* vals;
    const uint16_t* offs;
    int list;     // entries of a row group's list
    int blocks;   // blocks of 128 classes; a group's offsets are blocks + 1
    float* part_db;  // [classes.nsplit][classes]
};
template <int D, int P>
int xent_stats_cfg(const XentStatsArgs& x, int blocks, unsigned grid, hipStream_t st);
template <int D, int P>
int xent_grad_cfg(const XentGradArgs& x, unsigned grid, hipStream_t st);
// Blocks of 32 rows of a wave of the statistics pass (registers allow two but for wide records of
// two planes), owners of a gradient workgroup, and how many workgroups of either a CU holds
// (registers and LDS).
constexpr int xent_stats_most_blocks(int D, int planes) { return planes == 2 && D > 4 ? 1 : 2; }
constexpr int kXentGradOwners = 128;
constexpr int xent_grad_per_cu(int D, int planes) {
    return planes == 1 ? (D <= 3 ? 4 : D == 4 ? 3 : 2) : (D <= 2 ? 4 : D == 3 ? 3 : D == 4 ? 2 : 1);
}

}  // namespace ppocr
