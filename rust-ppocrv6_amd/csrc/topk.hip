// The largest values of each row with their columns, largest first, equal values by column.
//
// Bound by one read of the rows.  A workgroup takes a row into registers (R values a thread, up to
// 1024 R columns; wider rows are read again where it says so).  Every value and its column make one
// 64-bit number, all different, in the order of the result.  The largest values of the 256 groups
// of four threads bound the result from below: their top-th largest is reached by at least `top` of
// the row's values, and in rows as they come by few more, which are collected and whose places are
// counted.  Where more reach it than there is memory for (rows of equal values, mostly), the
// largest are taken one after the other.
//
// 7680 rows of 18710, top 16: 121 us, 4.8 TB/s (a large copy moves 4.9 on the same card); 341 us
// with two reads of the row by 256 threads.  The register limit keeps two workgroups on a CU, so that
// one row loads while the other is searched; with one, 203 us.  120 rows: 8.6 us, latency.
#include <algorithm>

#include "kernels.hpp"

namespace ppocr {
namespace {

constexpr int kCandidates = 1024;
typedef unsigned long long u64;

// The order of values as that of unsigned numbers: NaN 0, below every value; -0 and 0 equal.
__device__ __forceinline__ unsigned rank_of(float x) {
    const unsigned u = x == 0.0f ? 0u : __float_as_uint(x);
    return x == x ? ((u >> 31) ? ~u : u | 0x80000000u) : 0u;
}
// The value of a rank (1: the lowest).
__device__ __forceinline__ float of_rank(unsigned k) {
    return k <= 0x007FFFFFu ? -INFINITY : __uint_as_float((k >> 31) ? k & 0x7FFFFFFFu : ~k);
}
__device__ __forceinline__ u64 order_of(float x, unsigned col) {
    const unsigned k = rank_of(x);
    return k ? ((u64)k << 32) | (0xFFFFFFFFu - col) : 0;
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const u64 w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// NT threads, R values each in registers; R = 0: the row is read from memory each time.
template <int NT, int R>
__global__ __launch_bounds__(NT, R <= 20 ? 8 : 4) void topk_kernel(const float* __restrict__ x, int64_t rows, unsigned cols, int top,
                                                  int32_t* __restrict__ idx, float* __restrict__ val) {
    constexpr int GROUPS = 256, SIZE = NT / GROUPS;
    __shared__ unsigned group_max[GROUPS];
    __shared__ u64 cand[kCandidates];
    __shared__ u64 wave_best[NT / 64];
    __shared__ unsigned bound;
    __shared__ int count;
    const unsigned tid = threadIdx.x;
    float v[R > 0 ? R : 1];
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float* p = x + row * (int64_t)cols;
        // each value of this thread with its column
        auto each = [&](auto&& f) {
            if constexpr (R > 0) {
#pragma unroll
                for (int i = 0; i < R; ++i) f(v[i], i * NT + tid);
            } else {
                for (unsigned c = tid; c < cols; c += NT) f(p[c], c);
            }
        };
        if constexpr (R > 0) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const float* q = p + i * NT;  // the same for the workgroup
                v[i] = i * NT + tid < cols ? q[tid] : NAN;
            }
        }
        float most = NAN;  // fmaxf leaves NaN out
        each([&](float a, unsigned) { most = fmaxf(most, a); });
        unsigned of_group = rank_of(most);
#pragma unroll
        for (int o = 1; o < SIZE; o <<= 1) of_group = max(of_group, (unsigned)__shfl_xor((int)of_group, o, 64));
        __syncthreads();  // the row before is done with the shared memory
        if (tid % SIZE == 0) group_max[tid / SIZE] = of_group;
        if (tid == 0) count = 0;
        __syncthreads();
        if (tid < 64) {
            // the top-th largest group, bit by bit: the largest number that at least `top` reach
            unsigned g[GROUPS / 64];
#pragma unroll
            for (int i = 0; i < GROUPS / 64; ++i) g[i] = group_max[i * 64 + tid];
            unsigned b = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned t = b | (1u << bit);
                int reach = 0;
#pragma unroll
                for (int i = 0; i < GROUPS / 64; ++i) reach += __popcll(__ballot(g[i] >= t));
                if (reach >= top) {
                    b = t;
                    if (reach == top) break;
                }
            }
            if (tid == 0) bound = b;
        } else if ((int)tid - 64 < top) {
            idx[row * top + tid - 64] = -1;
            val[row * top + tid - 64] = -INFINITY;
        }
        __syncthreads();
        const float b = of_rank(bound);  // rank 0: fewer groups with a value than `top`, so all values
        if (most >= b)
            each([&](float a, unsigned c) {
                if (a >= b) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kCandidates) cand[at] = order_of(a, c);
                }
            });
        __syncthreads();
        const int n = count;
        if (n <= kCandidates) {
            for (int i = (int)tid; i < n; i += NT) {
                const u64 o = cand[i];
                int place = 0;
                for (int j = 0; j < n; ++j) place += cand[j] > o;
                if (place < top) {
                    const unsigned c = 0xFFFFFFFFu - (unsigned)o;
                    idx[row * top + place] = (int32_t)c;
                    val[row * top + place] = p[c];
                }
            }
            continue;
        }
        u64 last = ~0ull;
        for (int t = 0; t < top; ++t) {
            u64 m = 0;
            if (most >= b)
                for (unsigned c = tid; c < cols; c += NT) {
                    const u64 o = order_of(p[c], c);
                    if (o < last && o > m) m = o;
                }
            m = wave_max64(m);
            __syncthreads();
            if ((tid & 63) == 0) wave_best[tid >> 6] = m;
            __syncthreads();
            for (int i = 0; i < NT / 64; ++i) m = wave_best[i] > m ? wave_best[i] : m;
            if (m == 0) break;
            if (tid == 0) {
                const unsigned c = 0xFFFFFFFFu - (unsigned)m;
                idx[row * top + t] = (int32_t)c;
                val[row * top + t] = p[c];
            }
            last = m;
        }
    }
}

template <int NT, int R>
int run(const float* x, int64_t rows, int64_t cols, int top, int32_t* idx, float* val, hipStream_t st) {
    topk_kernel<NT, R><<<(unsigned)std::min<int64_t>(rows, 1 << 20), NT, 0, st>>>(x, rows, (unsigned)cols, top, idx, val);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace

int launch_topk_rows(const float* x, int64_t rows, int64_t cols, int top, int32_t* idx, float* val, hipStream_t st) {
    if (cols <= 2048) return run<256, 8>(x, rows, cols, top, idx, val, st);
    if (cols <= 8192) return run<1024, 8>(x, rows, cols, top, idx, val, st);
    if (cols <= 20480) return run<1024, 20>(x, rows, cols, top, idx, val, st);
    if (cols <= 40960) return run<1024, 40>(x, rows, cols, top, idx, val, st);
    return run<1024, 0>(x, rows, cols, top, idx, val, st);
}

}  // namespace ppocr
