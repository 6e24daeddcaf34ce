// A low-rank adapter merged into the weight that it is trained under, and its gradients.
//
//   forward   w = w0 + s up down                     w0 [n][k], up [n][rank], down [rank][k]
//   backward  ddown = s up^T dw, dup = s dw down^T   from the gradient dw of the merged weight
//
// Memory bound (the rank is far below n and k): w0 or dw is read once and w written once.  The products
// run on fp32 MFMA, exact products summed in 32 bits, of bf16 tensors too.  ddown sums over all
// n rows: each workgroup keeps the sum over its rows in registers and leaves it to a second kernel, which
// adds the workgroups' sums in a fixed order.
#include <algorithm>

#include "adapt.hpp"

namespace ppocr {
namespace {

__device__ __forceinline__ float up32(float v) { return v; }
__device__ __forceinline__ float up32(uint16_t v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ void put32(float* p, float v) { *p = v; }
__device__ __forceinline__ void put32(uint16_t* p, float v) { *p = __builtin_bit_cast(uint16_t, (__bf16)v); }

// Layout of v_mfma_f32_32x32x2_f32: lane l holds row l % 32 of A and column l % 32 of B at k = l / 32; the
// result's register r is row 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32.
__device__ __forceinline__ f32x16 mfma_f32(float a, float b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0);
}

// Each wave takes 32 rows of the weight: their up rows in registers, then 32 columns after the other.
template <typename T, int RANK>
__global__ __launch_bounds__(256) void merge_kernel(const T* w0, const T* __restrict__ down, const T* __restrict__ up, int64_t n,
                                                    int k, int rank, float s, T* w) {
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int64_t row0 = ((int64_t)blockIdx.x * 4 + (threadIdx.x >> 6)) * 32;
    if (row0 >= n) return;
    float a[RANK / 2];
    const T* ur = up + min(row0 + i, n - 1) * rank;
#pragma unroll
    for (int x = 0; x < RANK / 2; ++x) a[x] = 2 * x + h < rank ? up32(ur[2 * x + h]) : 0.0f;
    for (int c0 = 0; c0 < k; c0 += 32) {
        const int c = c0 + i, cc = min(c, k - 1);
        f32x16 acc = {};
#pragma unroll
        for (int x = 0; x < RANK / 2; ++x) {
            const int t = 2 * x + h;
            const float b = t < rank ? up32(down[(int64_t)t * k + cc]) : 0.0f;
            acc = mfma_f32(a[x], b, acc);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int64_t row = row0 + 8 * (r >> 2) + 4 * h + (r & 3);
            if (row < n && c < k) put32(w + row * k + c, fmaf(s, acc[r], up32(w0[row * k + c])));
        }
    }
}

// A workgroup takes every parts-th block of 32 rows: dw and up rows through LDS (beside the whole of
// down), dup of the block written at once, ddown summed over its blocks in registers.
constexpr int kPairs = 4;  // 32 x 32 pieces of ddown that a wave holds: at most 2 x 8 pieces on 4 waves
template <typename T>
__global__ __launch_bounds__(256) void merge_backward_kernel(const T* __restrict__ dw, const T* __restrict__ down,
                                                             const T* __restrict__ up, int64_t n, int k, int rank, float s,
                                                             T* dup, float* part) {
    extern __shared__ float lds[];
    const int kp = (k + 31) / 32 * 32, rp = (rank + 31) / 32 * 32;
    const int ks = kp + 1, rs = rp + 1;
    float* ldown = lds;                // [rp][ks]
    float* ldw = ldown + rp * ks;      // [32][ks]
    float* lup = ldw + 32 * ks;        // [32][rs]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 31, h = lane >> 5;
    const int nt = rp / 32, pieces = nt * (kp / 32);
    for (int x = tid; x < rp * kp; x += 256) {
        const int t = x / kp, c = x % kp;
        ldown[t * ks + c] = t < rank && c < k ? up32(down[(int64_t)t * k + c]) : 0.0f;
    }
    f32x16 acc[kPairs];
#pragma unroll
    for (int p = 0; p < kPairs; ++p) acc[p] = f32x16{};
    for (int64_t row0 = (int64_t)blockIdx.x * 32; row0 < n; row0 += (int64_t)gridDim.x * 32) {
        __syncthreads();
        for (int x = tid; x < 32 * kp; x += 256) {
            const int r = x / kp, c = x % kp;
            ldw[r * ks + c] = row0 + r < n && c < k ? up32(dw[(row0 + r) * k + c]) : 0.0f;
        }
        for (int x = tid; x < 32 * rp; x += 256) {
            const int r = x / rp, t = x % rp;
            lup[r * rs + t] = row0 + r < n && t < rank ? up32(up[(row0 + r) * rank + t]) : 0.0f;
        }
        __syncthreads();
        if (dup && wave < nt) {
            f32x16 d = {};
            for (int c = 0; c < kp; c += 2) d = mfma_f32(ldw[i * ks + c + h], ldown[(32 * wave + i) * ks + c + h], d);
            const int t = 32 * wave + i;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int64_t row = row0 + 8 * (r >> 2) + 4 * h + (r & 3);
                if (row < n && t < rank) put32(dup + row * rank + t, s * d[r]);
            }
        }
        if (part) {
#pragma unroll
            for (int p = 0; p < kPairs; ++p) {
                const int piece = wave + 4 * p;
                if (piece < pieces) {
                    const int t0 = 32 * (piece % nt), c0 = 32 * (piece / nt);
#pragma unroll
                    for (int j = 0; j < 32; j += 2)
                        acc[p] = mfma_f32(lup[(j + h) * rs + t0 + i], ldw[(j + h) * ks + c0 + i], acc[p]);
                }
            }
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * rank * k;
#pragma unroll
    for (int p = 0; p < kPairs; ++p) {
        const int piece = wave + 4 * p;
        if (piece < pieces) {
            const int t0 = 32 * (piece % nt), c = 32 * (piece / nt) + i;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = t0 + 8 * (r >> 2) + 4 * h + (r & 3);
                if (t < rank && c < k) out[t * k + c] = acc[p][r];
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void merge_sum_kernel(const float* __restrict__ part, int parts, int size, float s, T* out) {
    const int x = blockIdx.x * 256 + threadIdx.x;
    if (x >= size) return;
    float v = 0.0f;
    for (int p = 0; p < parts; ++p) v += part[(int64_t)p * size + x];
    put32(out + x, s * v);
}

template <typename T>
int merge(const MergeArgs& x, hipStream_t st) {
    const unsigned grid = (unsigned)((x.n + 127) / 128);
    auto go = [&]<int R>() {
        merge_kernel<T, R><<<grid, 256, 0, st>>>((const T*)x.w, (const T*)x.down, (const T*)x.up, x.n, x.k, x.rank, x.scale,
                                                 (T*)x.out);
    };
    if (x.rank <= 16) go.template operator()<16>();
    else if (x.rank <= 32) go.template operator()<32>();
    else go.template operator()<64>();
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

template <typename T>
int backward(const MergeArgs& x, void* ddown, void* dup, float* part, hipStream_t st) {
    const int kp = (x.k + 31) / 32 * 32, rp = (x.rank + 31) / 32 * 32, parts = merge_parts(x.n);
    const size_t lds = ((size_t)(rp + 32) * (kp + 1) + 32 * (size_t)(rp + 1)) * 4;
    auto kern = merge_backward_kernel<T>;
    PPOCR_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
    kern<<<parts, 256, lds, st>>>((const T*)x.dw, (const T*)x.down, (const T*)x.up, x.n, x.k, x.rank, x.scale, (T*)dup,
                                  ddown ? part : nullptr);
    PPOCR_HIP(hipGetLastError());
    if (!ddown) return PPOCR_OK;
    const int size = x.rank * x.k;
    merge_sum_kernel<T><<<(size + 255) / 256, 256, 0, st>>>(part, parts, size, x.scale, (T*)ddown);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace

int merge_parts(int64_t n) { return (int)std::min<int64_t>((n + 31) / 32, 256); }

int launch_merge(const MergeArgs& x, hipStream_t st) { return x.bf16 ? merge<uint16_t>(x, st) : merge<float>(x, st); }

int launch_merge_backward(const MergeArgs& x, void* ddown, void* dup, float* part, hipStream_t st) {
    return x.bf16 ? backward<uint16_t>(x, ddown, dup, part, st) : backward<float>(x, ddown, dup, part, st);
}

}  // namespace ppocr
