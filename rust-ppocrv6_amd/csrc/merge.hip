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
//
// rank 16 of fp32 18710 x 120: forward 6.0 us (3.1 TB/s from and to the caches), backward 9.6 + 3.2.  rank 64 of bf16
// 32768 x 256: 13.5 us (2.8 TB/s), 17.5 + 4.0.  Latency bounds them, a round trip to memory and one through LDS for each
// block of rows, with few waves to cover it: the operands of the rank products take the registers.
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

__host__ __device__ __forceinline__ bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

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

// Values at, at + 1, .. of the `width` at p, 0 past them.
template <typename T>
__device__ __forceinline__ Op<T> gather_to(const T* p, int at, int width) {
    Op<T> o;
#pragma unroll
    for (int y = 0; y < Op<T>::N; ++y) {
        const T v = p[min(at + y, width - 1)];
        o.v[y] = at + y < width ? v : T(0);
    }
    return o;
}
template <typename T>
__device__ __forceinline__ Op<T> load_op(const T* p) {
    return __builtin_bit_cast(Op<T>, *reinterpret_cast<const Piece<T>*>(p));
}

// Two neighbouring values of a row.
template <typename T>
struct alignas(2 * sizeof(T)) Pair {
    T v[2];
};
// ---------------------------------------------------------------- forward
// A workgroup takes a block of rows.  Each wave multiplies the block's up rows with 32 columns of down at a
// time; w0's pieces are on their way meanwhile.  (Workgroups that kept down as operands over several blocks,
// half as many: 6.1 us instead of 5.3 for rank 16 of 18710 x 120, 19 instead of 12 for rank 64 of 32768 x 256.)
// FULL: the rank is RANK, no address to hold back and no value to clear.
template <typename T, int RANK, bool VEC, bool FULL>
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
    if (VEC && pieces > 0) {
#pragma unroll
        for (int p = 0; p < PER; ++p)
            piece[p] = reinterpret_cast<const Piece<T>*>(src)[min(p * kThreads + tid, pieces - 1)];
    }
    Op<T> a[S];
    const T* ur = up + (row0 + min(i, rows - 1)) * rank;
#pragma unroll
    for (int x = 0; x < S; ++x) {
        const int t = x * Op<T>::STEP + h * V;
        if (rank_vec) {
            a[x] = load_op(ur + min(t, rank - V));
            if (t >= rank) a[x] = Op<T>{};
        } else {
            a[x] = gather_to(ur, t, rank);
        }
    }
    for (int c0 = 32 * wave; c0 < k; c0 += 32 * kWaves) {
        const int c = min(c0 + i, k - 1);
        f32x16 acc = {};
        if constexpr (FULL) {
#pragma unroll
            for (int x = 0; x < S; ++x) {
                Op<T> b;
#pragma unroll
                for (int y = 0; y < V; ++y) b.v[y] = down[(x * Op<T>::STEP + h * V + y) * k + c];
                acc = multiply(a[x], b, acc);
            }
        } else {
            Op<T> b[S];
#pragma unroll
            for (int x = 0; x < S; ++x)
#pragma unroll
                for (int y = 0; y < V; ++y) b[x].v[y] = down[min(x * Op<T>::STEP + h * V + y, rank - 1) * k + c];
            // ranks that do not exist, behind the loads: a value that is looked at holds back the loads behind it
#pragma unroll
            for (int x = 0; x < S; ++x)
                if ((x + 1) * Op<T>::STEP > rank) {
#pragma unroll
                    for (int y = 0; y < V; ++y)
                        if (x * Op<T>::STEP + h * V + y >= rank) b[x].v[y] = T(0);
                }
#pragma unroll
            for (int x = 0; x < S; ++x) acc = multiply(a[x], b[x], acc);
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
// LDS of a dup workgroup: rows of T at a pitch of an odd number of 16-byte pieces, which neighbouring rows'
// lanes read without bank conflicts.
__host__ __device__ constexpr int pitch_of(int cols, int v) { return ((cols + v - 1) / v | 1) * v; }

struct BackLayout {
    int kp, rp;  // columns and ranks, padded to 32
    int cpitch;  // values of a row of dw or down in LDS
    size_t down, dw, red, total;
};
template <typename T>
__host__ __device__ inline BackLayout back_layout(int k, int rank) {
    BackLayout L;
    constexpr int V = Piece<T>::N;
    L.kp = (k + 31) / 32 * 32;
    L.rp = (rank + 31) / 32 * 32;
    L.cpitch = pitch_of(L.kp, V);
    L.down = 0;
    L.dw = L.down + (size_t)L.rp * L.cpitch * sizeof(T);
    L.red = L.dw + (size_t)kRows * L.cpitch * sizeof(T);
    L.total = L.red + (size_t)kWaves * 32 * 33 * 4;
    return L;
}

// Workgroup b of `workers` takes blocks b, b + workers, .. of 32 rows: the next block's rows are on their way while
// this one's are multiplied.  The waves share the 32-rank pieces and the contraction over the columns, and
// meet in LDS.
template <typename T, bool VEC>
__device__ __forceinline__ void dup_rows(const T* __restrict__ dw, const T* __restrict__ down, int64_t n, int k, int rank, float s,
                                         T* dup, int64_t worker, int64_t workers, uint8_t* lds) {
    constexpr int V = Piece<T>::N, STEP = Op<T>::STEP;
    constexpr int PER = kRows * 256 / V / kThreads;
    const BackLayout L = back_layout<T>(k, rank);
    T* ldown = reinterpret_cast<T*>(lds + L.down);
    T* ldw = reinterpret_cast<T*>(lds + L.dw);
    float* red = reinterpret_cast<float*>(lds + L.red);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 31, h = lane >> 5;
    const int nt = L.rp / 32;
    // where each piece of a block that this thread moves lies in LDS, the same for every block (past the
    // block's pieces: -1).  A block of 32 rows is whole pieces whatever k is; where k is not, a piece may reach into
    // the next row and is spread value by value.
    constexpr int PIECES = kRows / V;
    int at[PER], left[VEC ? 1 : PER];
#pragma unroll
    for (int x = 0; x < PER; ++x) {
        const int p = x * kThreads + tid, r = p * V / k, c = p * V - r * k;
        at[x] = p < PIECES * k ? r * L.cpitch + c : -1;
        if constexpr (!VEC) left[x] = k - c;  // values of the piece's first row
    }
    const bool whole = VEC || aligned16(dw);
    u32x4 next[PER];
    auto fetch = [&](int64_t row0) {
        const int rows = (int)min((int64_t)kRows, n - row0), last = rows * k / V - 1;
        if (VEC || (whole && last >= 0)) {
            const u32x4* p = reinterpret_cast<const u32x4*>(dw + row0 * k);
#pragma unroll
            for (int x = 0; x < PER; ++x) next[x] = p[min(x * kThreads + tid, last)];
        }
    };
    int64_t row0 = worker * kRows;
    if (row0 >= n) return;
    fetch(row0);
    // columns and ranks past the tensors' stay 0
    for (int x = tid; x < (int)((L.red - L.down) / 16); x += kThreads) reinterpret_cast<u32x4*>(lds)[x] = u32x4{0, 0, 0, 0};
    __syncthreads();
    if (const int kv = k / V; VEC && aligned16(down)) {
        for (int x = tid; x < rank * kv; x += kThreads) {
            const int t = x / kv;
            *reinterpret_cast<u32x4*>(ldown + t * L.cpitch + (x - t * kv) * V) = reinterpret_cast<const u32x4*>(down)[x];
        }
    } else {
        for (int x = tid; x < rank * k; x += kThreads) ldown[x / k * L.cpitch + x % k] = down[x];
    }
    const int split = kWaves / nt;                  // waves that share a 32-rank piece
    const int tt = wave % nt, part_of = wave / nt;  // this wave's piece, and its share of the columns
    const int steps = L.kp / STEP;
    for (; row0 < n; row0 += workers * kRows) {
        const int rows = (int)min((int64_t)kRows, n - row0);
        if constexpr (VEC) {
#pragma unroll
            for (int x = 0; x < PER; ++x)
                if (at[x] >= 0) *reinterpret_cast<u32x4*>(ldw + at[x]) = next[x];
        } else {
            // rows that do not exist hold whatever they held: their results are not written
            const int pieces = whole ? rows * k / V : 0;
#pragma unroll
            for (int x = 0; x < PER; ++x)
                if (x * kThreads + tid < pieces) {
                    const Piece<T> q = __builtin_bit_cast(Piece<T>, next[x]);
                    // (of narrow rows a piece may cover several)
                    int to = at[x], more = left[x];
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        ldw[to] = q.v[v];
                        const bool over = --more == 0;
                        to += over ? L.cpitch - k + 1 : 1;
                        more = over ? k : more;
                    }
                }
            for (int x = pieces * V + tid; x < rows * k; x += kThreads) ldw[x / k * L.cpitch + x % k] = dw[row0 * k + x];
        }
        __syncthreads();
        if (row0 + workers * kRows < n) fetch(row0 + workers * kRows);
        f32x16 d = {};
        for (int x = part_of; x < steps; x += split) {
            const int c = x * STEP + h * V;
            d = multiply(load_op(ldw + i * L.cpitch + c), load_op(ldown + (32 * tt + i) * L.cpitch + c), d);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) red[(wave * 32 + result_row(r, h)) * 33 + i] = d[r];
        __syncthreads();
        // the waves' shares, one contiguous piece of memory
        for (int x = tid; x < rows * rank; x += kThreads) {
            const int r = x / rank, t = x - r * rank;
            float v = 0.0f;
            for (int y = 0; y < split; ++y) v += red[((y * nt + (t >> 5)) * 32 + r) * 33 + (t & 31)];
            dup[row0 * rank + x] = narrow<T>(s * v);
        }
    }
}

// Sum over rows first .. last of up[j][.] dw[j][.] for 64 columns: the lanes read two neighbouring columns (and
// ranks, where there are more than 32) of a row at a time, straight into the operands; the even and the odd
// ones are a piece of the product each.  The waves take the rows in turn and meet in LDS.
constexpr int kGroupCols = 64;
constexpr int kAhead = 2;
template <typename T, int NT, bool VEC, bool PAIRS>
__device__ __forceinline__ void ddown_rows(const T* __restrict__ dw, const T* __restrict__ up, int k, int rank, int64_t first,
                                           int64_t last, int c0, float* __restrict__ out, float* lds) {
    constexpr int V = Piece<T>::N, STEP = Op<T>::STEP;
    const int lane = threadIdx.x & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    struct Rows {
        Pair<T> d[V], u[V];
    };
    // Loads are unconditional and their values untouched until they are used, so that they are on their way
    // together.  Columns and ranks that do not exist meet no others in the products, rows that do not are
    // cleared before their use.
    const int ci = min(c0 + 2 * i, VEC ? k - 2 : k - 1), cj = min(c0 + 2 * i + 1, k - 1);
    const int ti = NT == 2 ? min(2 * i, PAIRS ? rank - 2 : rank - 1) : min(i, rank - 1), tj = min(2 * i + 1, rank - 1);
    auto fetch = [&](Rows& w, int64_t j0) {
        if (j0 >= last) return;  // the same for the wave
        const T* dp = dw + j0 * k;
        const T* up_ = up + j0 * rank;
        const int left = (int)min(last - j0, (int64_t)STEP);
#pragma unroll
        for (int y = 0; y < V; ++y) {
            const int j = min(h * V + y, left - 1);
            if constexpr (VEC) w.d[y] = *reinterpret_cast<const Pair<T>*>(dp + j * k + ci);
            else w.d[y] = Pair<T>{{dp[j * k + ci], dp[j * k + cj]}};
            if constexpr (NT == 1) w.u[y].v[0] = up_[j * rank + ti];
            else if constexpr (PAIRS) w.u[y] = *reinterpret_cast<const Pair<T>*>(up_ + j * rank + ti);
            else w.u[y] = Pair<T>{{up_[j * rank + ti], up_[j * rank + tj]}};
        }
    };
    f32x16 acc[2][NT];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int q = 0; q < NT; ++q) acc[p][q] = f32x16{};
    // the rows of kAhead steps are on their way
    constexpr int TURN = kWaves * STEP;
    Rows w[kAhead];
    int64_t j = first + wave * STEP;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
        w[x] = Rows{};
        fetch(w[x], j + x * TURN);
    }
    for (; j < last; j += kAhead * TURN) {
#pragma unroll
        for (int x = 0; x < kAhead; ++x) {
            if (j + x * TURN >= last) break;
            Op<T> a[NT], b[2];
#pragma unroll
            for (int y = 0; y < V; ++y) {
                b[0].v[y] = w[x].d[y].v[0];
                b[1].v[y] = w[x].d[y].v[1];
#pragma unroll
                for (int q = 0; q < NT; ++q) a[q].v[y] = w[x].u[y].v[q];
            }
            if (j + x * TURN + STEP > last) {
#pragma unroll
                for (int y = 0; y < V; ++y)
                    if (j + x * TURN + h * V + y >= last) {
                        b[0].v[y] = b[1].v[y] = T(0);
#pragma unroll
                        for (int q = 0; q < NT; ++q) a[q].v[y] = T(0);
                    }
            }
            fetch(w[x], j + (x + kAhead) * TURN);
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int q = 0; q < NT; ++q) acc[p][q] = multiply(a[q], b[p], acc[p][q]);
        }
    }
    // the upper waves' sums to the lower ones, then the second's to the first
    constexpr int SIZE = 2 * NT * 16 * 64;
#pragma unroll
    for (int half = kWaves / 2; half >= 1; half /= 2) {
        __syncthreads();
        if (wave >= half && wave < 2 * half) {
            float* p = lds + (wave - half) * SIZE + lane;
#pragma unroll
            for (int x = 0; x < 2 * NT * 16; ++x) p[x * 64] = acc[x / (NT * 16)][x / 16 % NT][x % 16];
        }
        __syncthreads();
        if (wave < half) {
            const float* p = lds + wave * SIZE + lane;
#pragma unroll
            for (int x = 0; x < 2 * NT * 16; ++x) acc[x / (NT * 16)][x / 16 % NT][x % 16] += p[x * 64];
        }
    }
    if (wave) return;
#pragma unroll
    for (int q = 0; q < NT; ++q)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int t = NT == 2 ? 2 * result_row(r, h) + q : result_row(r, h);
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int c = c0 + 2 * i + p;
                if (t < rank && c < k) out[t * k + c] = acc[p][q][r];
            }
        }
}

// The first workgroups take ddown, by groups of rows and of 64 columns, the others dup: dw comes from memory
// once and from the caches the second time.  (One pass that kept both in a workgroup left a sum of ddown per
// workgroup: rank 64 of 32768 x 256, 512 sums of 64 KB beside 17 MB of dw, took 27 us where this takes 20.)
// VEC: rows of dw are read in pieces of 16 bytes, PAIRS: those of up in pairs.
template <typename T, int NT, bool VEC, bool PAIRS>
__global__ __launch_bounds__(kThreads) void merge_backward_kernel(const T* __restrict__ dw, const T* __restrict__ down,
                                                                  const T* __restrict__ up, int64_t n, int k, int rank, float s,
                                                                  T* dup, float* part, int parts, int64_t rows_each) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int groups = part ? (k + kGroupCols - 1) / kGroupCols : 0;
    const int b = blockIdx.x;
    if (b < groups * parts) {
        const int g = b / groups, c0 = (b - g * groups) * kGroupCols;
        const int64_t first = g * rows_each;
        ddown_rows<T, NT, VEC, PAIRS>(dw, up, k, rank, first, min(first + rows_each, n), c0, part + (int64_t)g * rank * k,
                               reinterpret_cast<float*>(lds));
    } else {
        dup_rows<T, VEC>(dw, down, n, k, rank, s, dup, b - groups * parts, (int)gridDim.x - groups * parts, lds);
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

constexpr int kDownWorkers = 256;
// Rows of a ddown workgroup, whole turns of its waves: about kDownWorkers of rows and columns together.
int64_t rows_of_part(int64_t n, int64_t k) {
    const int64_t most = std::max<int64_t>(kDownWorkers / ((k + kGroupCols - 1) / kGroupCols), 1);
    const int64_t turn = kWaves * Op<uint16_t>::STEP;
    return ((n + most - 1) / most + turn - 1) / turn * turn;
}

template <typename T>
int merge(const MergeArgs& x, hipStream_t st) {
    constexpr int V = Piece<T>::N;
    const unsigned grid = (unsigned)((x.n + kRows - 1) / kRows);
    const size_t lds = (size_t)kRows * x.k * 4;
    // a block of 32 rows starts at a multiple of 16 bytes wherever the tensor does
    const bool vec = aligned16(x.w) && aligned16(x.out);
    const bool rank_vec = aligned16(x.up) && x.rank % V == 0;
    auto go = [&]<int R>() {
        const bool full = x.rank == R;
        auto kern = vec ? (full ? merge_kernel<T, R, true, true> : merge_kernel<T, R, true, false>)
                        : (full ? merge_kernel<T, R, false, true> : merge_kernel<T, R, false, false>);
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
    const int parts = merge_parts(x.n, x.k);
    const int64_t rows_each = rows_of_part(x.n, x.k);
    const int groups = (x.k + kGroupCols - 1) / kGroupCols;
    const int nt = x.rank > 32 ? 2 : 1;
    const int64_t blocks = (x.n + kRows - 1) / kRows;
    const size_t lds = std::max(dup ? back_layout<T>(x.k, x.rank).total : 0, ddown ? (size_t)nt * kWaves / 2 * 2 * 16 * 64 * 4 : 0);
    // the workgroups that the GPU holds at once beside those of ddown (3 a CU at most by their registers;
    // rank 16 of 18710 x 120: 12.8 us with 512, 14.2 with 256)
    const int64_t held = 256 * std::min<int64_t>(3, 160 * 1024 / (int64_t)lds) - (ddown ? groups * parts : 0);
    const unsigned grid = (unsigned)((ddown ? groups * parts : 0) + (dup ? std::min(blocks, std::max<int64_t>(held, 256)) : 0));
    const bool vec = aligned16(x.dw) && x.k % V == 0, pairs = aligned16(x.up) && x.rank % 2 == 0;
    auto go = [&]<int NT>() {
        constexpr bool P = NT == 2;  // (up is read in pairs for two pieces of the product)
        auto kern = vec ? (P && pairs ? merge_backward_kernel<T, NT, true, P> : merge_backward_kernel<T, NT, true, false>)
                        : (P && pairs ? merge_backward_kernel<T, NT, false, P> : merge_backward_kernel<T, NT, false, false>);
        kern<<<grid, kThreads, lds, st>>>((const T*)x.dw, (const T*)x.down, (const T*)x.up, x.n, x.k, x.rank, x.scale, (T*)dup,
                                          ddown ? part : nullptr, parts, rows_each);
    };
    if (nt == 2) go.template operator()<2>();
    else go.template operator()<1>();
    PPOCR_HIP(hipGetLastError());
    if (!ddown) return PPOCR_OK;
    const int size = x.rank * x.k;
    merge_sum_kernel<T><<<(size + 63) / 64, 1024, 0, st>>>(part, parts, size, x.scale, (T*)ddown);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace

int merge_parts(int64_t n, int64_t k) { return (int)((n + rows_of_part(n, k) - 1) / rows_of_part(n, k)); }

int launch_merge(const MergeArgs& x, hipStream_t st) { return x.bf16 ? merge<uint16_t>(x, st) : merge<float>(x, st); }

int launch_merge_backward(const MergeArgs& x, void* ddown, void* dup, float* part, hipStream_t st) {
    return x.bf16 ? backward<uint16_t>(x, ddown, dup, part, st) : backward<float>(x, ddown, dup, part, st);
}

}  // namespace ppocr
