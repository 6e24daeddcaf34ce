// The largest values of each row with their columns, largest first, equal values by column.
//
// A workgroup per row.  Every value and its column make one 64-bit number, all different, in the
// order of the result.  Each thread takes the largest of its columns; the top-th largest of those
// is a bound that at least `top` of the row's values reach, and only the columns of `top`
// threads can, so one more look at the row leaves few candidates (for random rows not many more
// than `top`), whose places in the result are counted.  Where more reach the bound than LDS holds,
// the largest are taken one by one.
#include <algorithm>

#include "kernels.hpp"

namespace ppocr {
namespace {

constexpr int kThreads = 256, kCandidates = 2048;
typedef unsigned long long u64;

// NaN and missing columns give 0, below every value.  -0 and 0 are equal.
__device__ __forceinline__ u64 order_of(float x, unsigned col) {
    if (!(x == x)) return 0;
    const unsigned u = x == 0.0f ? 0u : __float_as_uint(x);
    const unsigned k = (u >> 31) ? ~u : u | 0x80000000u;
    return ((u64)k << 32) | (0xFFFFFFFFu - col);
}
__device__ __forceinline__ u64 wave_max64(u64 v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const u64 w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

__global__ __launch_bounds__(kThreads) void topk_kernel(const float* __restrict__ x, int64_t rows, int64_t cols, int top,
                                                        int32_t* __restrict__ idx, float* __restrict__ val) {
    __shared__ u64 best[kThreads];
    __shared__ u64 cand[kCandidates];
    __shared__ u64 bound;
    __shared__ int count;
    const int tid = threadIdx.x;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
        const float* p = x + row * cols;
        __syncthreads();  // the row before is done with the shared memory
        u64 mine = 0;
        for (int64_t c = tid; c < cols; c += kThreads) {
            const u64 o = order_of(p[c], (unsigned)c);
            mine = o > mine ? o : mine;
        }
        best[tid] = mine;
        if (tid == 0) {
            count = 0;
            bound = 1;
        }
        if (tid < top) {
            idx[row * top + tid] = -1;
            val[row * top + tid] = -INFINITY;
        }
        __syncthreads();
        int above = 0;
        for (int i = 0; i < kThreads; ++i) above += best[i] > mine;
        if (mine && above == top - 1) bound = mine;
        __syncthreads();
        const u64 b = bound;
        if (mine >= b)
            for (int64_t c = tid; c < cols; c += kThreads) {
                const u64 o = order_of(p[c], (unsigned)c);
                if (o >= b) {
                    const int at = atomicAdd(&count, 1);
                    if (at < kCandidates) cand[at] = o;
                }
            }
        __syncthreads();
        const int n = count;
        if (n <= kCandidates) {
            for (int i = tid; i < n; i += kThreads) {
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
            for (int64_t c = tid; c < cols; c += kThreads) {
                const u64 o = order_of(p[c], (unsigned)c);
                if (o < last && o > m) m = o;
            }
            m = wave_max64(m);
            __syncthreads();
            if ((tid & 63) == 0) best[tid >> 6] = m;
            __syncthreads();
            for (int i = 0; i < kThreads / 64; ++i) m = best[i] > m ? best[i] : m;
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

}  // namespace

int launch_topk_rows(const float* x, int64_t rows, int64_t cols, int top, int32_t* idx, float* val, hipStream_t st) {
    topk_kernel<<<(unsigned)std::min<int64_t>(rows, 1 << 20), kThreads, 0, st>>>(x, rows, cols, top, idx, val);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace ppocr
