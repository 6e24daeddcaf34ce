// LayerNorm over rows of d values.
//
//   forward   mu = mean(x), v = mean((x - mu)^2), rstd = 1 / sqrt(v + eps), h = (x - mu) rstd,
//             y = h w + b
//   backward  t = dy w, dx = rstd (t - mean(t) - h mean(t h)), dw = sum over rows of dy h,
//             db = sum over rows of dy
//
// Memory bound: x in and y out, or dy and x in and dx out, once each.  A team of G lanes holds a
// row in registers (4 R values a lane), so the mean and the variance are two sums over
// registers, not two passes over memory.  The backward pass gives each team's lanes the same columns
// in every row it takes, so dw and db are summed in registers too; a workgroup's teams meet in LDS,
// the workgroups' sums in a second kernel, in a fixed order.
#include <algorithm>

#include "layernorm.hpp"

namespace ppocr {
namespace {

template <typename T>
__device__ __forceinline__ float up(T v);
template <>
__device__ __forceinline__ float up<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float up<uint16_t>(uint16_t v) {
    return __uint_as_float((unsigned)v << 16);
}
template <typename T>
__device__ __forceinline__ T down(float v);
template <>
__device__ __forceinline__ float down<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ uint16_t down<uint16_t>(float v) {
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// Column of value v (0..3) of chunk r of lane l: neighbouring quads of columns when rows can be read
// four values at a time, neighbouring columns otherwise.
template <int G, bool VEC>
__device__ __forceinline__ int column(int r, int v, int l) {
    return VEC ? (r * G + l) * 4 + v : (r * 4 + v) * G + l;
}

template <typename T, int G, int R, bool VEC>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int d, int l, float (&x)[4 * R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if constexpr (VEC) {
            struct alignas(4 * sizeof(T)) Q {
                T v[4];
            };
            const int c = (r * G + l) * 4;
            Q q{};
            if (c < d) q = *reinterpret_cast<const Q*>(p + c);
#pragma unroll
            for (int v = 0; v < 4; ++v) x[4 * r + v] = up<T>(q.v[v]);
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = column<G, VEC>(r, v, l);
                x[4 * r + v] = c < d ? up<T>(p[c]) : 0.0f;
            }
        }
    }
}
template <typename T, int G, int R, bool VEC>
__device__ __forceinline__ void store_row(T* __restrict__ p, int d, int l, const float (&x)[4 * R]) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if constexpr (VEC) {
            struct alignas(4 * sizeof(T)) Q {
                T v[4];
            };
            const int c = (r * G + l) * 4;
            Q q;
#pragma unroll
            for (int v = 0; v < 4; ++v) q.v[v] = down<T>(x[4 * r + v]);
            if (c < d) *reinterpret_cast<Q*>(p + c) = q;
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = column<G, VEC>(r, v, l);
                if (c < d) p[c] = down<T>(x[4 * r + v]);
            }
        }
    }
}

// Sums of two values over a team; for G > 64 through LDS (red: 2 per wave), every lane of the
// workgroup calling it.
template <int G>
__device__ __forceinline__ void team_sum(float& a, float& b, float2* red) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o >= 1; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (G > 64) {
        const int wave = threadIdx.x >> 6;
        __syncthreads();
        if ((threadIdx.x & 63) == 0) red[wave] = make_float2(a, b);
        __syncthreads();
        a = 0.0f;
        b = 0.0f;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) {
            a += red[i].x;
            b += red[i].y;
        }
    }
}

constexpr int threads_of(int G) { return G > 256 ? G : 256; }

template <typename T, int G, int R, bool VEC>
__global__ __launch_bounds__(threads_of(G)) void forward_kernel(const T* __restrict__ x, const float* __restrict__ w,
                                                                const float* __restrict__ b, int64_t m, int d, float eps,
                                                                T* __restrict__ y, float* __restrict__ mean,
                                                                float* __restrict__ rstd) {
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ float2 red[G > 64 ? G / 64 : 1];
    const int l = threadIdx.x % G;
    for (int64_t r0 = (int64_t)blockIdx.x * TEAMS; r0 < m; r0 += (int64_t)gridDim.x * TEAMS) {
        const int64_t row = r0 + threadIdx.x / G;
        const bool live = row < m;
        float v[4 * R];
        load_row<T, G, R, VEC>(x + (live ? row : m - 1) * d, d, l, v);
        float s = 0.0f, none = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) s += v[i];
        team_sum<G>(s, none, red);
        const float mu = s / (float)d;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) {
            const float c = column<G, VEC>(i >> 2, i & 3, l) < d ? v[i] - mu : 0.0f;
            v[i] = c;
            q = fmaf(c, c, q);
        }
        team_sum<G>(q, none, red);
        const float rs = 1.0f / sqrtf(q / (float)d + eps);
        if (live && l == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
        float wv[4 * R];
        load_row<float, G, R, VEC>(w, d, l, wv);
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) v[i] = (v[i] * rs) * wv[i];
        load_row<float, G, R, VEC>(b, d, l, wv);
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) v[i] += wv[i];
        if (live) store_row<T, G, R, VEC>(y + row * d, d, l, v);
    }
}

template <typename T, int G, int R, bool VEC>
__global__ __launch_bounds__(threads_of(G)) void backward_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, int64_t m, int d,
                                                                 T* __restrict__ dx, float* __restrict__ part) {
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ float2 red[G > 64 ? G / 64 : 1];
    __shared__ float cols[TEAMS > 1 ? TEAMS * 4 * R * G : 1];
    const int l = threadIdx.x % G, team = threadIdx.x / G;
    float wv[4 * R], dw[4 * R], db[4 * R];
    load_row<float, G, R, VEC>(w, d, l, wv);
#pragma unroll
    for (int i = 0; i < 4 * R; ++i) dw[i] = db[i] = 0.0f;
    for (int64_t r0 = (int64_t)blockIdx.x * TEAMS; r0 < m; r0 += (int64_t)gridDim.x * TEAMS) {
        const int64_t row = r0 + team;
        const bool live = row < m;
        const int64_t at = live ? row : m - 1;
        float g[4 * R], h[4 * R];
        load_row<T, G, R, VEC>(dy + at * d, d, l, g);
        load_row<T, G, R, VEC>(x + at * d, d, l, h);
        const float mu = mean[at], rs = rstd[at];
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * R; ++i) {
            // columns past d hold g = 0 and w = 0
            h[i] = column<G, VEC>(i >> 2, i & 3, l) < d ? (h[i] - mu) * rs : 0.0f;
            if (live) {
                dw[i] = fmaf(g[i], h[i], dw[i]);
                db[i] += g[i];
            }
            g[i] *= wv[i];
            c1 += g[i];
            c2 = fmaf(g[i], h[i], c2);
        }
        team_sum<G>(c1, c2, red);
        c1 /= (float)d;
        c2 /= (float)d;
        if (dx) {
#pragma unroll
            for (int i = 0; i < 4 * R; ++i) g[i] = rs * (g[i] - c1 - h[i] * c2);
            if (live) store_row<T, G, R, VEC>(dx + row * d, d, l, g);
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if constexpr (TEAMS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4 * R; ++i)
                cols[team * (4 * R * G) + column<G, VEC>(i >> 2, i & 3, l)] = which ? db[i] : dw[i];
            __syncthreads();
            for (int c = threadIdx.x; c < d; c += threads_of(G)) {
                float s = 0.0f;
#pragma unroll
                for (int t = 0; t < TEAMS; ++t) s += cols[t * (4 * R * G) + c];
                out[which * d + c] = s;
            }
        } else {
            store_row<float, G, R, VEC>(out + which * d, d, l, which ? db : dw);
        }
    }
}

// dw and db from the workgroups' sums: 32 columns of the 2 d per workgroup, 32 threads a column.
__global__ __launch_bounds__(1024) void columns_kernel(const float* __restrict__ part, int parts, int d,
                                                       float* __restrict__ dw, float* __restrict__ db) {
    __shared__ float red[32][33];
    const int c = threadIdx.x & 31, y = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + c;
    float s = 0.0f;
    if (col < 2 * (int64_t)d)
        for (int p = y; p < parts; p += 32) s += part[(int64_t)p * 2 * d + col];
    red[y][c] = s;
    __syncthreads();
    if (y == 0 && col < 2 * (int64_t)d) {
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) s += red[i][c];
        float* out = col < d ? dw : db;
        if (out) out[col < d ? col : col - d] = s;
    }
}

template <typename T, int G, int R>
int forward(const T* x, const float* w, const float* b, int64_t m, int d, float eps, bool vec, T* y, float* mean, float* rstd,
            hipStream_t st) {
    constexpr int NT = threads_of(G), TEAMS = NT / G;
    const unsigned grid = (unsigned)std::min<int64_t>((m + TEAMS - 1) / TEAMS, 1 << 20);
    if (vec) forward_kernel<T, G, R, true><<<grid, NT, 0, st>>>(x, w, b, m, d, eps, y, mean, rstd);
    else forward_kernel<T, G, R, false><<<grid, NT, 0, st>>>(x, w, b, m, d, eps, y, mean, rstd);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}
template <typename T, int G, int R>
int backward(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, int64_t m, int d, bool vec, T* dx,
             float* part, int parts, hipStream_t st) {
    constexpr int NT = threads_of(G);
    if (vec) backward_kernel<T, G, R, true><<<parts, NT, 0, st>>>(dy, x, w, mean, rstd, m, d, dx, part);
    else backward_kernel<T, G, R, false><<<parts, NT, 0, st>>>(dy, x, w, mean, rstd, m, d, dx, part);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

// Lanes of a row's team by its width.
int team_of(int64_t d) { return d <= 128 ? 16 : d <= 2048 ? 64 : d <= 8192 ? 256 : 1024; }

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

template <typename T>
int forward_of(const T* x, const float* w, const float* b, int64_t m, int d, float eps, T* y, float* mean, float* rstd,
               hipStream_t st) {
    const bool vec = d % 4 == 0 && aligned(x, 4 * sizeof(T)) && aligned(y, 4 * sizeof(T)) && aligned(w, 16) && aligned(b, 16);
    if (d <= 128) return forward<T, 16, 2>(x, w, b, m, d, eps, vec, y, mean, rstd, st);
    if (d <= 512) return forward<T, 64, 2>(x, w, b, m, d, eps, vec, y, mean, rstd, st);
    if (d <= 2048) return forward<T, 64, 8>(x, w, b, m, d, eps, vec, y, mean, rstd, st);
    if (d <= 8192) return forward<T, 256, 8>(x, w, b, m, d, eps, vec, y, mean, rstd, st);
    return forward<T, 1024, 4>(x, w, b, m, d, eps, vec, y, mean, rstd, st);
}
template <typename T>
int backward_of(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, int64_t m, int d, T* dx,
                float* part, int parts, hipStream_t st) {
    const bool vec = d % 4 == 0 && aligned(x, 4 * sizeof(T)) && aligned(dy, 4 * sizeof(T)) && aligned(dx, 4 * sizeof(T)) &&
                     aligned(w, 16);
    if (d <= 128) return backward<T, 16, 2>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, st);
    if (d <= 512) return backward<T, 64, 2>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, st);
    if (d <= 2048) return backward<T, 64, 8>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, st);
    if (d <= 8192) return backward<T, 256, 8>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, st);
    return backward<T, 1024, 4>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, st);
}

}  // namespace

int layernorm_parts(int64_t m, int64_t d) {
    const int g = team_of(d), teams = threads_of(g) / g;
    return (int)std::min<int64_t>((m + teams - 1) / teams, kLayerNormParts);
}

int launch_layernorm_forward(const void* x, const float* w, const float* b, int64_t m, int d, float eps, int bf16, void* y,
                             float* mean, float* rstd, hipStream_t st) {
    return bf16 ? forward_of((const uint16_t*)x, w, b, m, d, eps, (uint16_t*)y, mean, rstd, st)
                : forward_of((const float*)x, w, b, m, d, eps, (float*)y, mean, rstd, st);
}

int launch_layernorm_backward(const void* dy, const void* x, const float* w, const float* mean, const float* rstd, int64_t m,
                              int d, int bf16, void* dx, float* dw, float* db, float* part, hipStream_t st) {
    const int parts = layernorm_parts(m, d);
    float* p = dw || db ? part : nullptr;
    if (parts) {
        if (int e = bf16 ? backward_of((const uint16_t*)dy, (const uint16_t*)x, w, mean, rstd, m, d, (uint16_t*)dx, p, parts, st)
                         : backward_of((const float*)dy, (const float*)x, w, mean, rstd, m, d, (float*)dx, p, parts, st))
            return e;
    }
    if (dw || db) {
        columns_kernel<<<(unsigned)((2 * (int64_t)d + 31) / 32), 1024, 0, st>>>(part, parts, d, dw, db);
        PPOCR_HIP(hipGetLastError());
    }
    return PPOCR_OK;
}

}  // namespace ppocr
