// A low-rank adapter merged into the weight that it is trained under, and its gradients.
//
//   forward   w = w0 + s up down                     w0 [n][k], up [n][rank], down [rank][k]
//   backward  ddown = s up^T dw, dup = s dw down^T   from the gradient dw of the merged weight
//
// Memory bound (the rank is far below n and k): w0 or dw is read once and w written once.  A block of 32
// rows is one contiguous piece of memory, whatever k is, and is read and written in 16-byte pieces; the
// products pass through LDS to meet it.  fp32 tensors are multiplied on fp32 MFMA, bf16 tensors on bf16 MFMA:
// exact products either way, summed in 32 bits.  ddown sums over all n rows: each workgroup keeps the sum
// over its rows in registers and leaves it to a second kernel, which adds the workgroups' sums in a fixed order.
#include <algorithm>

#include "adapt.hpp"

namespace ppocr {
namespace {

constexpr int kRows = 32;   // rows of a block
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;

__device__ __forceinline__ float wide(float v) { return v; }
__device__ __forceinline__ float wide(uint16_t v) { return __uint_as_float((unsigned)v << 16); }
template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ uint16_t narrow<uint16_t>(float v) {
    return __builtin_bit_cast(uint16_t, (__bf16)v);
}

// 16 bytes of a tensor.
template <typename T>
struct alignas(16) Piece {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

// Operands of one MFMA chain: per lane, Op<T>::N consecutive values along the contraction.  bf16: one
// v_mfma_f32_32x32x16_bf16, lane l holding row or column l % 32 at 8 (l / 32) .. + 7.  fp32: four
// v_mfma_f32_32x32x2_f32, product y taking value y of both lane halves.  The result's register r is row
// 8 (r / 4) + 4 (l / 32) + r % 4 of column l % 32.
template <typename T>
struct Op {
    static constexpr int N = Piece<T>::N;
    static constexpr int STEP = 2 * N;  // contraction covered by both halves
    T v[N];
};
__device__ __forceinline__ f32x16 multiply(const Op<uint16_t>& a, const Op<uint16_t>& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 multiply(const Op<float>& a, const Op<float>& b, f32x16 c) {
#pragma unroll
    for (int y = 0; y < 4; ++y) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[y], b.v[y], c, 0, 0, 0);
    return c;
}
__device__ __forceinline__ int result_row(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// Values p[0], p[stride] .. of an operand, those at `count` and above 0.
template <typename T>
__device__ __forceinline__ Op<T> gather(const T* p, int64_t stride, int count) {
    Op<T> o;
#pragma unroll
    for (int y = 0; y < Op<T>::N; ++y) o.v[y] = y < count ? p[y * stride] : T(0);
    return o;
}
template <typename T>
__device__ __forceinline__ Op<T> load_op(const T* p) {
    return __builtin_bit_cast(Op<T>, *reinterpret_cast<const Piece<T>*>(p));
}

// ---------------------------------------------------------------- forward
// A workgroup takes a block of rows.  Each wave multiplies the block's up rows with 32 columns of down at a
// time; w0's pieces are on their way meanwhile.
template <typename T, int RANK, bool VEC>
__global__ __launch_bounds__(kThreads) void merge_kernel(const T* w0, const T* __restrict__ down, const T* __restrict__ up,
                                                         int64_t n, int k, int rank, bool rank_vec, float s, T* w) {
    constexpr int V = Piece<T>::N, S = RANK / Op<T>::STEP;
    constexpr int PER = kRows * 256 / V / kThreads;  // pieces of a thread at the largest k
    extern __shared__ __align__(16) float sum[];    // [rows][k]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 31, h = lane >> 5;
    const int64_t row0 = (int64_t)blockIdx.x * kRows;
    const int rows = (int)min((int64_t)kRows, n - row0);
    const int size = rows * k, pieces = size / V;
    const T* src = w0 + row0 * k;
    T* dst = w + row0 * k;
    Piece<T> piece[PER];
    if constexpr (VEC) {
#pragma unroll
        for (int p = 0; p < PER; ++p)
            if (p * kThreads + tid < pieces) piece[p] = reinterpret_cast<const Piece<T>*>(src)[p * kThreads + tid];
    }
    Op<T> a[S];
    const T* ur = up + (row0 + min(i, rows - 1)) * rank;
#pragma unroll
    for (int x = 0; x < S; ++x) {
        const int t = x * Op<T>::STEP + h * V;
        if (rank_vec) a[x] = t < rank ? load_op(ur + t) : Op<T>{};
        else a[x] = gather(ur + min(t, rank - 1), 1, rank - t);
    }
    for (int c0 = 32 * wave; c0 < k; c0 += 32 * kWaves) {
        const int c = min(c0 + i, k - 1);
        f32x16 acc = {};
#pragma unroll
        for (int x = 0; x < S; ++x) {
            const int t = x * Op<T>::STEP + h * V;
            acc = multiply(a[x], gather(down + (int64_t)min(t, rank - 1) * k + c, k, rank - t), acc);
        }
        if (c0 + i < k) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sum[result_row(r, h) * k + c] = acc[r];
        }
    }
    __syncthreads();
    if constexpr (VEC) {
#pragma unroll
        for (int p = 0; p < PER; ++p) {
            const int at = p * kThreads + tid;
            if (at < pieces) {
                Piece<T> o;
#pragma unroll
                for (int v = 0; v < V; ++v) o.v[v] = narrow<T>(fmaf(s, sum[at * V + v], wide(piece[p].v[v])));
                reinterpret_cast<Piece<T>*>(dst)[at] = o;
            }
        }
        // the last rows' values behind whole pieces
        for (int x = pieces * V + tid; x < size; x += kThreads) dst[x] = narrow<T>(fmaf(s, sum[x], wide(src[x])));
    } else {
        for (int x = tid; x < size; x += kThreads) dst[x] = narrow<T>(fmaf(s, sum[x], wide(src[x])));
    }
}

// ---------------------------------------------------------------- backward
// LDS of a workgroup: rows of T at a pitch of an odd number of 16-byte pieces, which neighbouring rows' lanes
// read without bank conflicts.
__host__ __device__ constexpr int pitch_of(int cols, int v) { return ((cols + v - 1) / v | 1) * v; }

struct BackLayout {
    int kp, rp;      // columns and ranks, padded to 32
    int cpitch;      // values of a row of dw or down in LDS
    int rpitch;      // of up
    size_t down, dw, up, red, total;
};
template <typename T>
__host__ __device__ inline BackLayout back_layout(int k, int rank) {
    BackLayout L;
    constexpr int V = Piece<T>::N;
    L.kp = (k + 31) / 32 * 32;
    L.rp = (rank + 31) / 32 * 32;
    L.cpitch = pitch_of(L.kp, V);
    L.rpitch = pitch_of(L.rp, V);
    L.down = 0;
    L.dw = L.down + (size_t)L.rp * L.cpitch * sizeof(T);
    L.up = L.dw + (size_t)kRows * L.cpitch * sizeof(T);
    L.red = L.up + (size_t)kRows * L.rpitch * sizeof(T);
    L.total = L.red + (size_t)kWaves * 32 * 33 * 4;
    return L;
}

// Workgroup b takes blocks b, b + parts, ..: the next block's rows are on their way while this one's are
// multiplied.  dup: the waves share its 32-rank pieces and the contraction over the columns, and meet in
// LDS; ddown: each wave keeps up to kKeep 32 x 32 pieces of the sum over all of the workgroup's rows.
constexpr int kKeep = 4;  // at most 2 x 8 pieces on 4 waves
template <typename T, bool VEC>
__global__ __launch_bounds__(kThreads) void merge_backward_kernel(const T* __restrict__ dw, const T* __restrict__ down,
                                                                  const T* __restrict__ up, int64_t n, int k, int rank, float s,
                                                                  T* dup, float* part) {
    constexpr int V = Piece<T>::N, STEP = Op<T>::STEP;
    constexpr int PER = kRows * 256 / V / kThreads, UPER = kRows * 64 / V / kThreads;
    extern __shared__ __align__(16) uint8_t lds[];
    const BackLayout L = back_layout<T>(k, rank);
    T* ldown = reinterpret_cast<T*>(lds + L.down);
    T* ldw = reinterpret_cast<T*>(lds + L.dw);
    T* lup = reinterpret_cast<T*>(lds + L.up);
    float* red = reinterpret_cast<float*>(lds + L.red);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 31, h = lane >> 5;
    const int nt = L.rp / 32, nc = L.kp / 32, pieces = nt * nc;
    const int kv = k / V, rv = rank / V;  // VEC: pieces of a row

    u32x4 next[VEC ? PER : 1], unext[VEC ? UPER : 1];
    auto fetch = [&](int64_t row0) {
        if constexpr (VEC) {
            const int rows = (int)min((int64_t)kRows, n - row0);
            const u32x4* p = reinterpret_cast<const u32x4*>(dw + row0 * k);
            const u32x4* q = reinterpret_cast<const u32x4*>(up + row0 * rank);
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                next[x] = u32x4{0, 0, 0, 0};
                if (x * kThreads + tid < rows * kv) next[x] = p[x * kThreads + tid];
            }
#pragma unroll
            for (int x = 0; x < UPER; ++x) {
                unext[x] = u32x4{0, 0, 0, 0};
                if (x * kThreads + tid < rows * rv) unext[x] = q[x * kThreads + tid];
            }
        }
    };
    int64_t row0 = (int64_t)blockIdx.x * kRows;
    fetch(row0);
    // columns and ranks past the tensors' stay 0
    for (int x = tid; x < (int)((L.red - L.down) / 16); x += kThreads) reinterpret_cast<u32x4*>(lds)[x] = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (int x = tid; x < rank * k; x += kThreads) ldown[x / k * L.cpitch + x % k] = down[x];

    f32x16 acc[kKeep];
#pragma unroll
    for (int p = 0; p < kKeep; ++p) acc[p] = f32x16{};
    const int split = kWaves / nt;                       // waves that share a 32-rank piece of dup
    const int tt = wave % nt, part_of = wave / nt;       // this wave's piece, and its share of the columns
    const int steps = L.kp / STEP;
    for (; row0 < n; row0 += (int64_t)gridDim.x * kRows) {
        const int rows = (int)min((int64_t)kRows, n - row0);
        if constexpr (VEC) {
#pragma unroll
            for (int x = 0; x < PER; ++x) {
                const int at = x * kThreads + tid, r = at / kv;
                if (r < kRows) *reinterpret_cast<u32x4*>(ldw + r * L.cpitch + (at - r * kv) * V) = next[x];
            }
#pragma unroll
            for (int x = 0; x < UPER; ++x) {
                const int at = x * kThreads + tid, r = at / rv;
                if (r < kRows) *reinterpret_cast<u32x4*>(lup + r * L.rpitch + (at - r * rv) * V) = unext[x];
            }
        } else {
            for (int x = tid; x < kRows * k; x += kThreads) ldw[x / k * L.cpitch + x % k] = x < rows * k ? dw[row0 * k + x] : T(0);
            for (int x = tid; x < kRows * rank; x += kThreads)
                lup[x / rank * L.rpitch + x % rank] = x < rows * rank ? up[row0 * rank + x] : T(0);
        }
        __syncthreads();
        if (row0 + (int64_t)gridDim.x * kRows < n) fetch(row0 + (int64_t)gridDim.x * kRows);
        if (dup) {
            f32x16 d = {};
            for (int x = part_of; x < steps; x += split) {
                const int c = x * STEP + h * V;
                d = multiply(load_op(ldw + i * L.cpitch + c), load_op(ldown + (32 * tt + i) * L.cpitch + c), d);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) red[(wave * 32 + result_row(r, h)) * 33 + i] = d[r];
        }
        if (part) {
#pragma unroll
            for (int p = 0; p < kKeep; ++p) {
                const int piece = wave + kWaves * p;
                if (piece < pieces) {
                    const int t = 32 * (piece % nt) + i, c = 32 * (piece / nt) + i;
#pragma unroll
                    for (int x = 0; x < kRows / STEP; ++x) {
                        const int j = x * STEP + h * V;
                        acc[p] = multiply(gather(lup + j * L.rpitch + t, L.rpitch, V), gather(ldw + j * L.cpitch + c, L.cpitch, V),
                                          acc[p]);
                    }
                }
            }
        }
        __syncthreads();
        if (dup) {
            // the waves' shares of dup, one contiguous piece of memory
            for (int x = tid; x < rows * rank; x += kThreads) {
                const int r = x / rank, t = x - r * rank;
                float v = 0.0f;
                for (int y = 0; y < split; ++y) v += red[((y * nt + (t >> 5)) * 32 + r) * 33 + (t & 31)];
                dup[row0 * rank + x] = narrow<T>(s * v);
            }
        }
    }
    if (!part) return;
    float* out = part + (int64_t)blockIdx.x * rank * k;
#pragma unroll
    for (int p = 0; p < kKeep; ++p) {
        const int piece = wave + kWaves * p;
        if (piece < pieces) {
            const int t0 = 32 * (piece % nt), c = 32 * (piece / nt) + i;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int t = t0 + result_row(r, h);
                if (t < rank && c < k) out[t * k + c] = acc[p][r];
            }
        }
    }
}

// ddown from the workgroups' sums: 64 values a workgroup, the sums of a value on 16 threads.
__device__ __forceinline__ float part_sum(const float* __restrict__ part, int first, int parts, int64_t size, int64_t x) {
    float v = 0.0f;
#pragma unroll 8
    for (int p = first; p < parts; p += 16) v += part[p * size + x];
    return v;
}
template <typename T>
__global__ __launch_bounds__(1024) void merge_sum_kernel(const float* __restrict__ part, int parts, int size, float s, T* out) {
    __shared__ float red[16][65];
    const int c = threadIdx.x & 63, y = threadIdx.x >> 6;
    const int x = blockIdx.x * 64 + c;
    red[y][c] = x < size ? part_sum(part, y, parts, size, x) : 0.0f;
    __syncthreads();
    if (threadIdx.x < 64 && x < size) {
        float v = 0.0f;
#pragma unroll
        for (int p = 0; p < 16; ++p) v += red[p][c];
        out[x] = narrow<T>(s * v);
    }
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T>
int merge(const MergeArgs& x, hipStream_t st) {
    constexpr int V = Piece<T>::N;
    const unsigned grid = (unsigned)((x.n + kRows - 1) / kRows);
    const size_t lds = (size_t)kRows * x.k * 4;
    // a block of 32 rows starts at a multiple of 16 bytes wherever the tensor does
    const bool vec = aligned(x.w) && aligned(x.out);
    const bool rank_vec = aligned(x.up) && x.rank % V == 0;
    auto go = [&]<int R>() {
        auto kern = vec ? merge_kernel<T, R, true> : merge_kernel<T, R, false>;
        kern<<<grid, kThreads, lds, st>>>((const T*)x.w, (const T*)x.down, (const T*)x.up, x.n, x.k, x.rank, rank_vec, x.scale,
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
    constexpr int V = Piece<T>::N;
    const int parts = merge_parts(x.n);
    const size_t lds = back_layout<T>(x.k, x.rank).total;
    const bool vec = aligned(x.dw) && aligned(x.up) && x.k % V == 0 && x.rank % V == 0;
    auto kern = vec ? merge_backward_kernel<T, true> : merge_backward_kernel<T, false>;
    kern<<<parts, kThreads, lds, st>>>((const T*)x.dw, (const T*)x.down, (const T*)x.up, x.n, x.k, x.rank, x.scale, (T*)dup,
                                       ddown ? part : nullptr);
    PPOCR_HIP(hipGetLastError());
    if (!ddown) return PPOCR_OK;
    const int size = x.rank * x.k;
    merge_sum_kernel<T><<<(size + 63) / 64, 1024, 0, st>>>(part, parts, size, x.scale, (T*)ddown);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace

int merge_parts(int64_t n) { return (int)std::min<int64_t>((n + kRows - 1) / kRows, 256); }

int launch_merge(const MergeArgs& x, hipStream_t st) { return x.bf16 ? merge<uint16_t>(x, st) : merge<float>(x, st); }

int launch_merge_backward(const MergeArgs& x, void* ddown, void* dup, float* part, hipStream_t st) {
    return x.bf16 ? backward<uint16_t>(x, ddown, dup, part, st) : backward<float>(x, ddown, dup, part, st);
}

}  // namespace ppocr
