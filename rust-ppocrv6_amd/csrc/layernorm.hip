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
// the workgroups' sums in a second kernel, in a fixed order.  A team reads its next row while it
// sums the present one.
//
// 16384 bf16 rows of 4096: forward 50 us (5.4 TB/s), backward 94 + 8 us (4.3 TB/s; the last 8 the
// workgroups' sums).  30720 fp32 rows of 120: 7.5 us (3.9 TB/s, tensors that the last-level cache holds
// from pass to pass), 9.6 + 3.5 us.  120 rows: 3.3 + 5.2 us.
// Above 8192 columns the backward pass keeps values in scratch, 20 registers and 72 to 86 where rows are
// not read in 16-byte chunks: 4096 rows of 16384: 106 us forward (fp32; bf16 57), 199 backward (152), and
// 378 (386) for rows of 16383.
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

// A lane holds R chunks of V values of a row, 16 bytes each: value v of chunk r of lane l is a
// column.  Rows that can be read 16 bytes at a time keep a chunk's columns together, others give
// neighbouring lanes neighbouring columns.
template <typename T>
constexpr int kV = 16 / (int)sizeof(T);
template <int V, int G, bool VEC>
__device__ __forceinline__ int column(int r, int v, int l) {
    return VEC ? (r * G + l) * V + v : (r * V + v) * G + l;
}

template <typename T, int R>
struct Raw {
    struct alignas(16) Chunk {
        T v[kV<T>];
    };
    Chunk c[R];
};

// The rows may be the output's own (y over x, dx over dy or x), each written after it was read: no
// pointer to them is __restrict__.
template <typename T, int G, int R, bool VEC>
__device__ __forceinline__ void load_raw(const T* p, int d, int l, Raw<T, R>& x) {
    constexpr int V = kV<T>;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if constexpr (VEC) {
            const int c = (r * G + l) * V;
            x.c[r] = typename Raw<T, R>::Chunk{};
            if (c < d) x.c[r] = *reinterpret_cast<const typename Raw<T, R>::Chunk*>(p + c);
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = column<V, G, VEC>(r, v, l);
                x.c[r].v[v] = c < d ? p[c] : T(0);
            }
        }
    }
}
template <typename T, int R, int E>
__device__ __forceinline__ void widen(const Raw<T, R>& x, float (&f)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) f[i] = up<T>(x.c[i / kV<T>].v[i % kV<T>]);
}
template <typename T, int G, int R, bool VEC, int E>
__device__ __forceinline__ void store_row(T* p, int d, int l, const float (&x)[E]) {
    constexpr int V = kV<T>;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if constexpr (VEC) {
            const int c = (r * G + l) * V;
            typename Raw<T, R>::Chunk q;
#pragma unroll
            for (int v = 0; v < V; ++v) q.v[v] = down<T>(x[V * r + v]);
            if (c < d) *reinterpret_cast<typename Raw<T, R>::Chunk*>(p + c) = q;
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c = column<V, G, VEC>(r, v, l);
                if (c < d) p[c] = down<T>(x[V * r + v]);
            }
        }
    }
}
// The fp32 weights of the columns that a lane holds of rows of type T.
template <typename T, int G, int R, bool VEC, int E>
__device__ __forceinline__ void load_weights(const float* __restrict__ p, int d, int l, float (&f)[E]) {
    constexpr int V = kV<T>;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        if constexpr (VEC) {
            const int c = column<V, G, VEC>(i / V, i % V, l);
            f32x4 q = {};
            if (c < d) q = *reinterpret_cast<const f32x4*>(p + c);
#pragma unroll
            for (int v = 0; v < 4; ++v) f[i + v] = q[v];
        } else {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = column<V, G, VEC>((i + v) / V, (i + v) % V, l);
                f[i + v] = c < d ? p[c] : 0.0f;
            }
        }
    }
}

// Sums of two values over a team; for G > 64 through LDS, every lane of the workgroup calling it.
// Two buffers in turn: a buffer is written again only after the barrier of the sum in between.
template <int G>
__device__ __forceinline__ void team_sum(float& a, float& b, float2 (*red)[G > 64 ? G / 64 : 1], int& turn) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o >= 1; o >>= 1) {
        a += __shfl_xor(a, o, 64);
        b += __shfl_xor(b, o, 64);
    }
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) red[turn][threadIdx.x >> 6] = make_float2(a, b);
        __syncthreads();
        a = 0.0f;
        b = 0.0f;
#pragma unroll
        for (int i = 0; i < G / 64; ++i) {
            a += red[turn][i].x;
            b += red[turn][i].y;
        }
        turn ^= 1;
    }
}

// Waves a CU holds of the forward kernel (its registers allow that many), so that a grid of them
// covers a large batch in one round: 8 per SIMD with 8 values a lane, 5 with 16, 4 in the widest
// rows.  16384 bf16 rows of 4096: 49.8 us so, 56.8 and 58.4 with 4 and 8 per SIMD.
template <typename T>
constexpr int forward_waves(int G, int R) {
    return G > 256 ? 16 : R * kV<T> <= 8 ? 32 : 20;
}
// Workgroups of the backward kernel: what the GPU holds at once (3 of 256 threads per CU where a
// lane holds 16 values: the rows above 93 us, 104 with 2 per CU, 113 with 4), fewer for the
// narrowest rows, whose sums the second kernel then has less of (30720 rows of 120: 13.8 us together
// with 512, 14.1 with 768).
constexpr int parts_of(int G) { return G == 1024 ? 256 : G == 16 || G == 512 ? 512 : 768; }

constexpr int threads_of(int G) { return G > 256 ? G : 256; }

template <typename T, int G, int R, bool VEC>
__global__ __launch_bounds__(threads_of(G)) void forward_kernel(const T* x, const float* __restrict__ w,
                                                                const float* __restrict__ b, int64_t m, int d, float eps,
                                                                T* y, float* __restrict__ mean,
                                                                float* __restrict__ rstd) {
    constexpr int TEAMS = threads_of(G) / G, V = kV<T>, E = V * R;
    constexpr bool AHEAD = G < 1024;  // its registers would not hold the next row beside this one
    __shared__ float2 red[2][G > 64 ? G / 64 : 1];
    int turn = 0;
    const int l = threadIdx.x % G;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    int64_t row = (int64_t)blockIdx.x * TEAMS + threadIdx.x / G;
    Raw<T, R> next;
    load_raw<T, G, R, VEC>(x + min(row, m - 1) * d, d, l, next);
    float wv[E], bv[E];
    load_weights<T, G, R, VEC>(w, d, l, wv);
    load_weights<T, G, R, VEC>(b, d, l, bv);
    for (int64_t r0 = (int64_t)blockIdx.x * TEAMS; r0 < m; r0 += step, row += step) {
        const bool live = row < m;
        float v[E];
        widen<T, R>(next, v);
        // the row after this one, while this one is summed
        if (AHEAD && r0 + step < m) load_raw<T, G, R, VEC>(x + min(row + step, m - 1) * d, d, l, next);
        float s = 0.0f, none = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) s += v[i];
        team_sum<G>(s, none, red, turn);
        const float mu = s / (float)d;
        float q = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float c = column<V, G, VEC>(i / V, i % V, l) < d ? v[i] - mu : 0.0f;
            v[i] = c;
            q = fmaf(c, c, q);
        }
        team_sum<G>(q, none, red, turn);
        const float rs = 1.0f / sqrtf(q / (float)d + eps);
        if (live && l == 0) {
            if (mean) mean[row] = mu;
            if (rstd) rstd[row] = rs;
        }
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = fmaf(v[i] * rs, wv[i], bv[i]);
        if (live) store_row<T, G, R, VEC>(y + row * d, d, l, v);
        if (!AHEAD && r0 + step < m) load_raw<T, G, R, VEC>(x + min(row + step, m - 1) * d, d, l, next);
    }
}

// A single workgroup (final: its sums are dw and db themselves) has no second kernel to wait for.
template <typename T, int G, int R, bool VEC, int NT>
__global__ __launch_bounds__(NT) void backward_kernel(const T* dy, const T* x,
                                                                 const float* __restrict__ w,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd, int64_t m, int d,
                                                                 T* dx, float* __restrict__ part, float* final_dw,
                                                                 float* final_db) {
    constexpr int TEAMS = NT / G, V = kV<T>, E = V * R;
    constexpr bool AHEAD = G < 1024;  // its registers would not hold the next row beside this one
    __shared__ float2 red[2][G > 64 ? G / 64 : 1];
    __shared__ float cols[TEAMS > 1 ? TEAMS * E * G : 1];
    int turn = 0;
    const int l = threadIdx.x % G, team = threadIdx.x / G;
    const int64_t step = (int64_t)gridDim.x * TEAMS;
    int64_t row = (int64_t)blockIdx.x * TEAMS + team;
    Raw<T, R> ng, nx;
    float nmu, nrs;
    auto fetch = [&](int64_t r) {
        const int64_t at = min(r, m - 1);
        load_raw<T, G, R, VEC>(dy + at * d, d, l, ng);
        load_raw<T, G, R, VEC>(x + at * d, d, l, nx);
        nmu = mean[at];
        nrs = rstd[at];
    };
    fetch(row);
    float wv[E], dw[E], db[E];
    load_weights<T, G, R, VEC>(w, d, l, wv);
#pragma unroll
    for (int i = 0; i < E; ++i) dw[i] = db[i] = 0.0f;
    for (int64_t r0 = (int64_t)blockIdx.x * TEAMS; r0 < m; r0 += step, row += step) {
        const bool live = row < m;
        float g[E], h[E];
        widen<T, R>(ng, g);
        widen<T, R>(nx, h);
        const float mu = nmu, rs = nrs;
        if (AHEAD && r0 + step < m) fetch(row + step);
        float c1 = 0.0f, c2 = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            // columns past d hold g = 0 and w = 0
            h[i] = column<V, G, VEC>(i / V, i % V, l) < d ? (h[i] - mu) * rs : 0.0f;
            if (live) {
                dw[i] = fmaf(g[i], h[i], dw[i]);
                db[i] += g[i];
            }
            g[i] *= wv[i];
            c1 += g[i];
            c2 = fmaf(g[i], h[i], c2);
        }
        team_sum<G>(c1, c2, red, turn);
        c1 /= (float)d;
        c2 /= (float)d;
        if (dx) {
#pragma unroll
            for (int i = 0; i < E; ++i) g[i] = rs * (g[i] - c1 - h[i] * c2);
            if (live) store_row<T, G, R, VEC>(dx + row * d, d, l, g);
        }
        if (!AHEAD && r0 + step < m) fetch(row + step);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        float* out = part ? part + ((int64_t)blockIdx.x * 2 + which) * d : which ? final_db : final_dw;
        if (!out) continue;  // the same for the workgroup
        if constexpr (TEAMS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; ++i)
                cols[team * (E * G) + column<V, G, VEC>(i / V, i % V, l)] = which ? db[i] : dw[i];
            __syncthreads();
            for (int c = threadIdx.x; c < d; c += NT) {
                float s = 0.0f;
#pragma unroll
                for (int t = 0; t < TEAMS; ++t) s += cols[t * (E * G) + c];
                out[c] = s;
            }
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const int c = column<V, G, VEC>(i / V, i % V, l);
                if (c < d) out[c] = which ? db[i] : dw[i];
            }
        }
    }
}

// dw and db from the workgroups' sums: C columns of the 2 d per workgroup, 1024 / C threads a column.
template <int C>
__global__ __launch_bounds__(1024) void columns_kernel(const float* __restrict__ part, int parts, int d,
                                                       float* __restrict__ dw, float* __restrict__ db) {
    constexpr int L = 1024 / C;
    __shared__ float red[L][C + 1];
    const int c = threadIdx.x % C, y = threadIdx.x / C;
    const int64_t col = (int64_t)blockIdx.x * C + c;
    float s = 0.0f;
    if (col < 2 * (int64_t)d)
        for (int p = y; p < parts; p += L) s += part[(int64_t)p * 2 * d + col];
    red[y][c] = s;
    __syncthreads();
    if (threadIdx.x < 64) {
        // lane (c, y) takes 16 of the column's sums, then the lanes of a column meet
        s = 0.0f;
#pragma unroll
        for (int i = 0; i < L * C / 64; ++i) s += red[y * (L * C / 64) + i][c];
#pragma unroll
        for (int o = C; o < 64; o <<= 1) s += __shfl_xor(s, o, 64);
        if (y == 0 && col < 2 * (int64_t)d) {
            float* out = col < d ? dw : db;
            if (out) out[col < d ? col : col - d] = s;
        }
    }
}

template <typename T, int G, int R>
int forward(const T* x, const float* w, const float* b, int64_t m, int d, float eps, bool vec, T* y, float* mean, float* rstd,
            hipStream_t st) {
    constexpr int NT = threads_of(G), TEAMS = NT / G;
    const unsigned grid = (unsigned)std::min<int64_t>((m + TEAMS - 1) / TEAMS, 256 * 64 * forward_waves<T>(G, R) / NT);
    if (vec) forward_kernel<T, G, R, true><<<grid, NT, 0, st>>>(x, w, b, m, d, eps, y, mean, rstd);
    else forward_kernel<T, G, R, false><<<grid, NT, 0, st>>>(x, w, b, m, d, eps, y, mean, rstd);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}
template <typename T, int G, int R, int NT = threads_of(G)>
int backward(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, int64_t m, int d, bool vec, T* dx,
             float* part, int parts, float* dw, float* db, hipStream_t st) {
    if (vec) backward_kernel<T, G, R, true, NT><<<parts, NT, 0, st>>>(dy, x, w, mean, rstd, m, d, dx, part, dw, db);
    else backward_kernel<T, G, R, false, NT><<<parts, NT, 0, st>>>(dy, x, w, mean, rstd, m, d, dx, part, dw, db);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

// Few narrow rows: one workgroup of 64 teams instead of a second kernel (120 rows of 120: 5.2 us, with
// the second kernel 3.6 + 2.5 and a launch more).
constexpr int kFewRows = 256;

// f.template operator()<G, C>(): the lanes of a row's team and the chunks of 8 values that each holds, by
// the row's width.
template <typename F>
auto by_width(int64_t d, F&& f) {
    if (d <= 128) return f.template operator()<16, 1>();
    if (d <= 512) return f.template operator()<64, 1>();
    if (d <= 1024) return f.template operator()<64, 2>();
    if (d <= 2048) return f.template operator()<256, 1>();
    if (d <= 4096) return f.template operator()<256, 2>();
    if (d <= 8192) return f.template operator()<512, 2>();
    return f.template operator()<1024, 2>();
}
int team_of(int64_t d) {
    return by_width(d, []<int G, int C>() { return G; });
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int forward_of(const T* x, const float* w, const float* b, int64_t m, int d, float eps, T* y, float* mean, float* rstd,
               hipStream_t st) {
    const bool vec = d % kV<T> == 0 && aligned(x) && aligned(y) && aligned(w) && aligned(b);
    return by_width(d, [&]<int G, int C>() { return forward<T, G, C * 8 / kV<T>>(x, w, b, m, d, eps, vec, y, mean, rstd, st); });
}
template <typename T>
int backward_of(const T* dy, const T* x, const float* w, const float* mean, const float* rstd, int64_t m, int d, T* dx,
                float* part, int parts, float* dw, float* db, hipStream_t st) {
    const bool vec = d % kV<T> == 0 && aligned(x) && aligned(dy) && aligned(dx) && aligned(w);
    if (d <= 128 && m <= kFewRows)
        return backward<T, 16, (sizeof(T) == 4 ? 2 : 1), 1024>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, dw, db, st);
    return by_width(d, [&]<int G, int C>() {
        return backward<T, G, C * 8 / kV<T>>(dy, x, w, mean, rstd, m, d, vec, dx, part, parts, dw, db, st);
    });
}

}  // namespace

int layernorm_parts(int64_t m, int64_t d) {
    const int g = team_of(d), teams = threads_of(g) / g;
    if (m > 0 && d <= 128 && m <= kFewRows) return 1;
    return (int)std::min<int64_t>((m + teams - 1) / teams, parts_of(g));
}

int launch_layernorm_forward(const void* x, const float* w, const float* b, int64_t m, int d, float eps, int bf16, void* y,
                             float* mean, float* rstd, hipStream_t st) {
    return bf16 ? forward_of((const uint16_t*)x, w, b, m, d, eps, (uint16_t*)y, mean, rstd, st)
                : forward_of((const float*)x, w, b, m, d, eps, (float*)y, mean, rstd, st);
}

int launch_layernorm_backward(const void* dy, const void* x, const float* w, const float* mean, const float* rstd, int64_t m,
                              int d, int bf16, void* dx, float* dw, float* db, float* part, hipStream_t st) {
    const int parts = layernorm_parts(m, d);
    const bool sums = (dw || db) && parts != 1;
    if (parts) {
        float* p = sums ? part : nullptr;
        float* fw = sums ? nullptr : dw;
        float* fb = sums ? nullptr : db;
        if (int e = bf16 ? backward_of((const uint16_t*)dy, (const uint16_t*)x, w, mean, rstd, m, d, (uint16_t*)dx, p, parts, fw,
                                       fb, st)
                         : backward_of((const float*)dy, (const float*)x, w, mean, rstd, m, d, (float*)dx, p, parts, fw, fb, st))
            return e;
    }
    if (sums) {
        // narrow rows: more workgroups (512 sums of 2 x 120 columns: 3.8 us, 4.4 with 16 columns each);
        // wide ones: whole lines (768 of 2 x 4096: 8.7 us, 16.5 with 8 columns each)
        if (d <= 512) columns_kernel<8><<<(unsigned)((2 * (int64_t)d + 7) / 8), 1024, 0, st>>>(part, parts, d, dw, db);
        else columns_kernel<32><<<(unsigned)((2 * (int64_t)d + 31) / 32), 1024, 0, st>>>(part, parts, d, dw, db);
        PPOCR_HIP(hipGetLastError());
    }
    return PPOCR_OK;
}

}  // namespace ppocr
