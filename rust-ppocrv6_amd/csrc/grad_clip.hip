// The global norm of many gradients, norm = sqrt(sum of all squares), and the gradients times
// min(1, most / norm).
//
// Memory bound: every gradient is read for the norm, then read again and written.  Two kernels: the first
// leaves one partial sum a workgroup, the second has each workgroup add all of them up in the same order
// (8 KB from L2) and scale its share, so no launch and no workgroup waits in between for a single value.
// Squares are exact in 64 bits and summed there: neither the squares of small gradients vanish nor those
// of large ones overflow.  34M bf16 gradients in 56 tensors: 15.8 us for the squares (4.3 TB/s; from the caches where
// the backward pass left them) and 22.5 for the second kernel (6 TB/s, its reads mostly from the caches), 44 us the call;
// a single adapter's two tensors 4 us each, which is what two launches take.
//
// The tensors' addresses and sizes go to the kernels as arguments, kTable tensors a launch: nothing is
// copied to the GPU, and a captured call holds its own table.
#include <algorithm>

#include "grad_clip.hpp"

namespace ppocr {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 120;          // tensors of a launch: 32 bytes each within the 4 KB of arguments
constexpr int kChunkBytes = 16384;   // of a workgroup's turn: 4 loads of 16 bytes a thread
constexpr int kMostParts = 1024;     // workgroups of a launch, each with a partial sum

struct Table {
    const void* in[kTable];
    void* out[kTable];
    int64_t count[kTable];    // values
    int first[kTable + 1];    // chunks of the tensors before this one
    uint8_t bf16[kTable];
    int tensors;
};
static_assert(sizeof(Table) + 64 <= 4096, "kernel arguments");

int64_t chunks_of(const GradTensor& t) {
    const int64_t per = kChunkBytes / (t.bf16 ? 2 : 4);
    return (t.count + per - 1) / per;
}

__device__ __forceinline__ float up(float v) { return v; }
__device__ __forceinline__ float up(uint16_t v) { return __uint_as_float((unsigned)v << 16); }
__device__ __forceinline__ float down(float v, float) { return v; }
__device__ __forceinline__ uint16_t down(float v, uint16_t) { return __builtin_bit_cast(uint16_t, (__bf16)v); }

template <typename T>
struct alignas(16) Wide {
    static constexpr int N = 16 / sizeof(T);
    T v[N];
};

// The tensor that a chunk belongs to.
__device__ __forceinline__ int tensor_of(const Table& t, int chunk) {
    int lo = 0, hi = t.tensors;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A chunk's values in a thread's registers: 16 bytes at a time where the tensor is aligned to that, else value by
// value.  All loads are issued together, from addresses held inside the chunk; values past its end count as 0.
template <typename T>
struct Chunk {
    static constexpr int V = Wide<T>::N, R = kChunkBytes / 16 / kThreads;
    Wide<T> w[R];
    // the values of piece r that are the chunk's own
    static __device__ __forceinline__ int place(bool wide, int r, int v) {
        const int x = r * kThreads + threadIdx.x;
        return wide ? x * V + v : (r * V + v) * kThreads + (int)threadIdx.x;
    }
    __device__ __forceinline__ void load(const T* p, int n, bool wide) {
        if (wide) {
            const int last = (n - 1) / V;  // the last piece may reach past the chunk: then value by value
            const bool whole = n % V == 0;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const int x = min(r * kThreads + (int)threadIdx.x, whole ? last : max(last - 1, 0));
                if (whole || last > 0) w[r] = reinterpret_cast<const Wide<T>*>(p)[x];
            }
            if (!whole) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    if (r * kThreads + (int)threadIdx.x == last) {
#pragma unroll
                        for (int v = 0; v < V; ++v) w[r].v[v] = p[min(last * V + v, n - 1)];
                    }
            }
        } else {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int v = 0; v < V; ++v) w[r].v[v] = p[min(place(false, r, v), n - 1)];
        }
    }
};

template <typename T>
__device__ __forceinline__ double chunk_squares(const void* in, int64_t at, int n) {
    using C = Chunk<T>;
    const bool wide = reinterpret_cast<uintptr_t>(in) % 16 == 0;
    C c;
    c.load((const T*)in + at, n, wide);
    double s = 0.0;
#pragma unroll
    for (int r = 0; r < C::R; ++r)
#pragma unroll
        for (int v = 0; v < C::V; ++v) {
            const double x = C::place(wide, r, v) < n ? (double)up(c.w[r].v[v]) : 0.0;
            s = fma(x, x, s);
        }
    return s;
}

template <typename T>
__device__ __forceinline__ void chunk_scale(const void* in, void* out, int64_t at, int n, float power, float scale) {
    using C = Chunk<T>;
    T* q = (T*)out + at;
    const bool wide = (reinterpret_cast<uintptr_t>(in) | reinterpret_cast<uintptr_t>(out)) % 16 == 0;
    C c;
    c.load((const T*)in + at, n, wide);
#pragma unroll
    for (int r = 0; r < C::R; ++r) {
#pragma unroll
        for (int v = 0; v < C::V; ++v) c.w[r].v[v] = down(up(c.w[r].v[v]) * power * scale, T());
        if (wide && C::place(true, r, C::V - 1) < n) {
            reinterpret_cast<Wide<T>*>(q)[r * kThreads + threadIdx.x] = c.w[r];
        } else {
#pragma unroll
            for (int v = 0; v < C::V; ++v)
                if (C::place(wide, r, v) < n) q[C::place(wide, r, v)] = c.w[r].v[v];
        }
    }
}

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ double block_sum(double s, double* red) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    s = 0.0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) s += red[i];
    return s;
}

// A workgroup takes chunks one behind the other, so that it looks for its tensor once: chunks `first` .. `last`.
__device__ __forceinline__ void share_of(int chunks, int* first, int* last) {
    const int each = chunks / (int)gridDim.x, more = chunks % (int)gridDim.x, b = blockIdx.x;
    *first = b * each + min(b, more);
    *last = *first + each + (b < more ? 1 : 0);
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Table t, double* __restrict__ parts) {
    __shared__ double red[kThreads / 64];
    int c, last;
    share_of(t.first[t.tensors], &c, &last);
    double s = 0.0;
    for (int i = c < last ? tensor_of(t, c) : 0; c < last; ++c) {
        if (c >= t.first[i + 1]) ++i;
        const int per = kChunkBytes / (t.bf16[i] ? 2 : 4);
        const int64_t at = (int64_t)(c - t.first[i]) * per;
        const int n = (int)min((int64_t)per, t.count[i] - at);
        s += t.bf16[i] ? chunk_squares<uint16_t>(t.in[i], at, n) : chunk_squares<float>(t.in[i], at, n);
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

// The chunks are taken from the last to the first: what the first kernel read last is what the caches
// still hold.
__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, const double* __restrict__ parts, int64_t nparts, float most,
                                                         float* __restrict__ norm_out) {
    __shared__ double red[kThreads / 64];
    double s = 0.0;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < nparts; i += kThreads) s += parts[i];
    const double norm = sqrt(block_sum(s, red));
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
    // gradients whose norm is no finite number stay as they are: the caller sees the norm
    const double factor = norm > (double)most && norm < (double)INFINITY ? (double)most / norm : 1.0;
    // Below the normal numbers 32 bits hold few bits of a factor, or none, while its products with values as large as
    // such a norm has are ordinary numbers.  The values meet a power of two first then, and what is left of the factor is
    // 2^-126 and more: the first product is exact wherever the second does not come to 0.
    const int below = factor < 0x1p-126 ? min(-126 - ilogb(factor), 149) : 0;
    const float power = (float)ldexp(1.0, -below), scale = (float)ldexp(factor, below);
    int first, last;
    share_of(t.first[t.tensors], &first, &last);
    int c = last - 1;
    for (int i = c >= first ? tensor_of(t, c) : 0; c >= first; --c) {
        if (c < t.first[i]) --i;
        if (scale == 1.0f && t.in[i] == t.out[i]) continue;
        const int per = kChunkBytes / (t.bf16[i] ? 2 : 4);
        const int64_t at = (int64_t)(c - t.first[i]) * per;
        const int n = (int)min((int64_t)per, t.count[i] - at);
        if (t.bf16[i]) chunk_scale<uint16_t>(t.in[i], t.out[i], at, n, power, scale);
        else chunk_scale<float>(t.in[i], t.out[i], at, n, power, scale);
    }
}

// f(table, workgroups of its first kernel) for the launches that cover the tensors.
template <typename F>
int for_tables(const std::vector<GradTensor>& tensors, F&& f) {
    size_t i = 0;
    do {
        Table t{};
        int64_t chunks = 0;
        for (; i < tensors.size() && t.tensors < kTable; ++i) {
            const int64_t c = chunks_of(tensors[i]);
            if (!c) continue;
            if (chunks + c > 0x7fffffffLL) break;
            t.in[t.tensors] = tensors[i].in;
            t.out[t.tensors] = tensors[i].out;
            t.count[t.tensors] = tensors[i].count;
            t.bf16[t.tensors] = tensors[i].bf16 ? 1 : 0;
            t.first[t.tensors++] = (int)chunks;
            chunks += c;
        }
        t.first[t.tensors] = (int)chunks;
        if (int e = f(t, (int)std::min<int64_t>(chunks, kMostParts))) return e;
    } while (i < tensors.size());
    return PPOCR_OK;
}

}  // namespace

int64_t grad_clip_most_parts(const int64_t* sizes, int64_t count) {
    // the widest type has the most chunks; a launch leaves no more sums than it has chunks
    int64_t chunks = 0;
    for (int64_t i = 0; i < count; ++i) chunks += chunks_of(GradTensor{nullptr, nullptr, sizes[i], 0});
    const int64_t launches = (count + kTable - 1) / kTable + (chunks >> 30);
    return std::min<int64_t>(chunks, launches * kMostParts) + 1;
}

int launch_grad_clip(const std::vector<GradTensor>& tensors, float most, float* norm, double* parts, hipStream_t st) {
    int64_t total = 0;
    if (int e = for_tables(tensors, [&](const Table& t, int blocks) {
            if (blocks) {
                squares_kernel<<<blocks, kThreads, 0, st>>>(t, parts + total);
                PPOCR_HIP(hipGetLastError());
            }
            total += blocks;
            return (int)PPOCR_OK;
        }))
        return e;
    float* out = norm;
    return for_tables(tensors, [&](const Table& t, int blocks) {
        scale_kernel<<<std::max(blocks, 1), kThreads, 0, st>>>(t, parts, total, most, out);
        PPOCR_HIP(hipGetLastError());
        out = nullptr;
        return (int)PPOCR_OK;
    });
}

}  // namespace ppocr
