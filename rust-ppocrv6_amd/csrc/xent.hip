// Losses over the vocabulary without keeping the logits (xent.hpp): the operand records, the
// target lists, the merge of the forward pass, the sums of the backward pass, and the launches.
//
// All of these are small beside the matrix kernels and bound by latency or by what they read and
// write once (us at 30720 rows fp32 / one line or page): records 12 and 23 with the transposed form /
// 9.6; losses 8 / 5; sums of 3 to 28 chunks 18 / 11; lists of 16 teacher logits for a page 23.
#include <algorithm>

#include "xent.hpp"

namespace ppocr {
namespace {

constexpr int kThreads = 256;

// log2(e) and ln 2 in two floats: a logarithm of 16 times log2(e) rounded to 32 bits would be off by
// 2e-7, for every row in the same direction, and so would the sum of each row's probabilities.
constexpr float kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147182f, kLn2Rest = -1.90465432e-9f;
__device__ __forceinline__ float to_log2(float l) { return fmaf(l, kLog2e, l * kLog2eRest); }

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((unsigned)*p << 16); }

// The head and its rows: a [.][k], w [n][k].  VEC: k and both addresses are multiples of four values,
// so that rows can be read four at a time.
template <typename T, bool VEC>
struct HeadRef {
    typedef T type;
    static constexpr bool vec = VEC;
    const T* a;
    const T* w;
    const float* bias;
    int k;
};

// ---------------------------------------------------------------- target entries
// Entry i of row r: its class (-1: none) and, for distillation, the teacher's logit over tau.
struct Targets {
    const int32_t* target;
    const int32_t* idx;
    const float* z;
    int tn;
    float inv_tau;
    int64_t n;
    __device__ __forceinline__ int cls(int64_t r, int i) const {
        const int c = target ? target[r] : idx[r * tn + i];
        return c >= 0 && (int64_t)c < n ? c : -1;
    }
    __device__ __forceinline__ float logit(int64_t r, int i) const { return target ? 0.0f : z[r * tn + i] * inv_tau; }
};

template <typename T>
struct alignas(4 * sizeof(T)) Four {
    T v[4];
};
// Values j .. j + 3 of a row of k, zeros past its end.
template <bool VEC, typename T>
__device__ __forceinline__ Four<T> read_four(const T* __restrict__ p, int j, int k) {
    Four<T> q{};
    if constexpr (VEC) {
        if (j < k) q = *reinterpret_cast<const Four<T>*>(p + j);
    } else {
        // rows at any address: global memory is read in one piece from there too
        if (j + 4 <= k) {
            __builtin_memcpy(q.v, p + j, sizeof(q.v));
        } else {
#pragma unroll
            for (int u = 0; u < 3; ++u)
                if (j + u < k) q.v[u] = p[j + u];
        }
    }
    return q;
}

// a_r . w_c + b_c of N classes by 8 neighbouring lanes (all of them call it); 0 for c < 0, whose place
// class 0 is read for, so that the reads of all N are on their way at once.
template <int N, typename H>
__device__ __forceinline__ void logits_of(const H& h, int64_t r, const int (&c)[N], int l8, float (&out)[N]) {
    constexpr int PIECES = N == 1 ? 4 : 2;
    const auto* pa = h.a + r * h.k;
    float bias[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        bias[n] = h.bias ? h.bias[max(c[n], 0)] : 0.0f;
        out[n] = 0.0f;
    }
    for (int j = 4 * l8; j < h.k; j += 32 * PIECES) {
        Four<typename H::type> x[PIECES], y[N][PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) x[i] = read_four<H::vec>(pa, j + 32 * i, h.k);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < PIECES; ++i) y[n][i] = read_four<H::vec>(h.w + (int64_t)max(c[n], 0) * h.k, j + 32 * i, h.k);
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) out[n] = fmaf(value(x[i].v + u), value(y[n][i].v + u), out[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
        for (int o = 4; o >= 1; o >>= 1) out[n] += __shfl_xor(out[n], o, 64);
        out[n] = c[n] >= 0 ? out[n] + bias[n] : 0.0f;
    }
}
template <typename H>
__device__ __forceinline__ float logit_of(const H& h, int64_t r, int c, int l8) {
    const int cs[1] = {c};
    float z[1];
    logits_of(h, r, cs, l8, z);
    return z[0];
}

// One row by a wave: lane i holds the row's entry i, its class (-1: none, or past the last), the log of
// its weight and the weight (0 for none), and the head's logit for it.
struct RowTargets {
    int cls;
    float logq, q, z;
};
// MOST: entries of 8 lanes at a time (registers).
template <int MOST, typename H>
__device__ __forceinline__ RowTargets row_targets(const Targets& tg, const H& h, int64_t r, int lane) {
    RowTargets t;
    t.cls = lane < tg.tn ? tg.cls(r, lane) : -1;
    if (tg.target) {
        t.logq = 0.0f;
        t.q = t.cls >= 0 ? 1.0f : 0.0f;
    } else {
        const float x = t.cls >= 0 ? tg.logit(r, lane) : -INFINITY;
        float top = x;  // NaN is left out here and returns with the sum
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
        const float e = top == -INFINITY ? (x == x ? 0.0f : x) : expf(x - top);
        const float sum = wave_sum(e);
        t.logq = x - top - logf(sum);
        t.q = sum == 0.0f ? 0.0f : e / sum;
        if (!(t.q != 0.0f)) t.logq = 0.0f;
    }
    t.z = 0.0f;
    // 8 lanes an entry, N entries each at a time; lane i takes entry i's logit home
    auto round = [&]<int N>(int first) {
        int c[N];
        float z[N];
#pragma unroll
        for (int n = 0; n < N; ++n) c[n] = __shfl(t.cls, first + 8 * n + (lane >> 3), 64);
        logits_of(h, r, c, lane & 7, z);
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float here = __shfl(z[n], (lane & 7) * 8, 64);
            if ((lane & ~7) == first + 8 * n) t.z = here;
        }
    };
    if (tg.tn <= 8) round.template operator()<1>(0);
    else
        for (int i = 0; i < tg.tn; i += 8 * MOST) round.template operator()<MOST>(i);
    return t;
}

// A row's gradient factor, by 8 neighbouring lanes: g / tau when it has a target, 0 otherwise.
__device__ __forceinline__ float factor_of(const Targets& tg, const float* grad, int64_t r, int l8) {
    bool any = false;
    for (int i = l8; i < tg.tn; i += 8) any |= tg.cls(r, i) >= 0 && (tg.target || tg.logit(r, i) != -INFINITY);
    int n = any;
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) n |= __shfl_xor(n, o, 64);
    return n ? (grad ? grad[r] : 1.0f) * tg.inv_tau : 0.0f;
}

// ---------------------------------------------------------------- operand records
// One workgroup per record of 32 entries, rows of `a` first and then classes of `w`.
template <typename H>
struct RecordArgs {
    H h;
    Targets tg;
    const float* lse;
    const float* grad;
    int64_t m, n, row_tiles;
    uint8_t* row_rec;
    uint8_t* class_rec;
    int* row_u;
    int* class_u;
};

template <typename H, int D, int P, bool BACK>
__device__ void build_record(const RecordArgs<H>& x, int64_t t, bool rows, float* tile, float* red) {
    constexpr int LD = 32 * D + 1;
    const int tid = threadIdx.x, e = tid >> 3, l8 = tid & 7;  // 8 lanes an entry
    const int64_t first = t * 32, count = min((int64_t)32, (rows ? x.m : x.n) - first);
    float* gf = red + 12;  // 32 gradient factors
    float factor = 1.0f;
    if (BACK && rows) {
        factor = factor_of(x.tg, x.grad, first + min((int64_t)e, count - 1), l8);
        if (e >= count) factor = 0.0f;
        if (l8 == 0) gf[e] = factor;
    }
    // a row without gradient reaches no sum, whatever it holds
    const bool in = e < count && factor != 0.0f;
    const int k = x.h.k;
    const auto* src = (rows ? x.h.a : x.h.w) + (first + (e < count ? e : 0)) * k;
    Four<typename H::type> v[D];
#pragma unroll
    for (int i = 0; i < D; ++i) v[i] = read_four<H::vec>(src, 32 * i + 4 * l8, in ? k : 0);
    float first_aux = 0.0f;  // of entry `tid`
    if (tid < 32 && tid < count) {
        if (!rows) first_aux = x.h.bias ? x.h.bias[first + tid] * (kLog2e * x.tg.inv_tau) : 0.0f;
        else if (BACK) first_aux = x.lse[first + tid];
    }
    float top = 0.0f, ss = 0.0f;
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float f = value(v[i].v + u);
            ss = fmaf(f, f, ss);
            if (fabsf(f) < INFINITY) top = fmaxf(top, fabsf(f));
        }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) {
        ss += __shfl_xor(ss, o, 64);
        top = fmaxf(top, __shfl_xor(top, o, 64));
    }
    // the largest and the smallest of the entries' largest magnitudes (entries of zeros aside)
    const float most = wave_max(top), least = -wave_max(top > 0.0f ? -top : -INFINITY);
    const bool odd = __any(!(ss < INFINITY));
    ss = wave_max(ss);
    if ((tid & 63) == 0) {
        red[tid >> 6] = most;
        red[4 + (tid >> 6)] = odd ? INFINITY : ss;
        red[8 + (tid >> 6)] = least;
    }
    __syncthreads();
    const float largest = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const bool shared = largest <= 16.0f * fminf(fminf(red[8], red[9]), fminf(red[10], red[11]));
    // largest magnitude to [2^14, 2^15); 2^100 at most, so that 2^-e and the factors stay in range
    auto exponent = [](float t) { return t > 0.0f ? min(14 - ilogbf(t), 100) : 100; };
    const int ex = exponent(largest), own = shared ? ex : exponent(top);
#pragma unroll
    for (int i = 0; i < D; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) tile[e * LD + 32 * i + 4 * l8 + u] = ldexpf(value(v[i].v + u), own);
    __syncthreads();
    uint8_t* rec = (rows ? x.row_rec : x.class_rec) + t * (int64_t)((size_t)P * D * 2048 * (BACK ? 2 : 1) + kXentAux);
    constexpr int FORM = 2 * D * 64;  // 16-byte pieces of one plane of one form
#pragma unroll
    for (int tr = 0; tr < (BACK ? 2 : 1); ++tr) {
        f16x8* dst = reinterpret_cast<f16x8*>(rec + (tr ? (size_t)P * D * 2048 : 0));
#pragma unroll
        for (int c = tid; c < FORM; c += kThreads) {
            const int lane = c & 63, l = lane & 31, h = lane >> 5, step = c >> 6;
            f16x8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // transposed: step = 2 d + e, the entries of an MFMA result's rows
                const int en = tr ? 16 * (step & 1) + 8 * (j >> 2) + 4 * h + (j & 3) : l;
                const int kk = tr ? 32 * (step >> 1) + l : 16 * step + 8 * h + j;
                const float f = tile[en * LD + kk];
                hi[j] = (_Float16)f;
                if (P == 2) lo[j] = (_Float16)(f - (float)hi[j]);
            }
            dst[c] = hi;
            if (P == 2) dst[FORM + c] = lo;
        }
    }
    float* aux = reinterpret_cast<float*>(rec + (size_t)P * D * 2048 * (BACK ? 2 : 1));
    if (l8 == 0) aux[80 + e] = ldexpf(1.0f, -own);
    if (tid < 64) {
        const float bound = wave_max(!rows && fabsf(first_aux) < INFINITY ? fabsf(first_aux) : 0.0f);
        if (tid < 32) {
            if (!rows) {
                aux[tid] = tid < count ? first_aux : -INFINITY;
                aux[32 + tid] = 0.0f;
            } else if (BACK) {
                aux[tid] = gf[tid] != 0.0f ? to_log2(first_aux) : INFINITY;
            } else {
                aux[tid] = 0.0f;
                aux[32 + tid] = 0.0f;
            }
        } else if (tid < 48 && tid != 36 && tid != 37) {
            const float norm = sqrtf(fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7])));
            aux[32 + tid] = tid == 32 ? ldexpf(1.0f, -ex) : tid == 33 ? (float)ex : tid == 34 ? norm : tid == 35 ? bound : tid == 38 && shared ? 1.0f : 0.0f;
        }
    }
    if (!BACK && !rows && tid == 0) x.class_u[t] = !shared;
    if (BACK && tid < 64) {
        // The largest of what multiplies this record's values, as an exponent, against its own.
        float f = tid < 32 && rows ? fabsf(gf[tid]) : 0.0f;
        f = wave_max(f < INFINITY ? f : 0.0f);
        const int ge = f > 0.0f ? ilogbf(f) + 1 : 0;
        // an infinite one makes its sums NaN: P has a largest value
        if (rows && tid < 32) aux[32 + tid] = fabsf(gf[tid]) == INFINITY ? NAN : ldexpf(gf[tid], -ge);
        if (tid == 0) {
            const int u = !rows ? -ex : f > 0.0f ? ge - ex : kXentNone;
            (rows ? x.row_u : x.class_u)[t] = 2 * u + !shared;
            aux[68] = (float)u;
            aux[69] = (float)ge;
        }
    }
}

// ---------------------------------------------------------------- target lists (backward)
// One workgroup per group of 32 rows: every target entry's p - q in 32 bits, sorted by class (then
// row), entries of one row that name the same class joined, and where each block of 128 classes
// starts in the list.
template <typename H>
struct ListArgs {
    H h;
    Targets tg;
    const float* lse;
    const float* grad;
    int64_t m;
    int list, size, blocks;  // list = 32 tn entries, size = list rounded up to a power of two; blocks of 128 classes
    uint32_t* keys;
    float* vals;
    uint16_t* offs;
};
constexpr uint32_t kNoKey = 0xFFFFFFFFu;

// The value of lane ^ D, without memory: lane permutations within rows of 16, then swaps of halves.
template <int D>
__device__ __forceinline__ unsigned lane_xor(unsigned v) {
    if constexpr (D == 1) return __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false);        // quad 1 0 3 2
    else if constexpr (D == 2) return __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false);   // quad 2 3 0 1
    else if constexpr (D == 4) {
        const int t = __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false);                  // eight reversed: ^ 7
        return __builtin_amdgcn_update_dpp(0, t, 0x1B, 0xF, 0xF, false);                               // quad reversed: ^ 3
    } else if constexpr (D == 8) return __builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xF, 0xF, false);  // row rotated by 8
    else return (unsigned)__shfl_xor((int)v, D, 64);
}
template <int D>
__device__ __forceinline__ unsigned long long lane_xor64(unsigned long long v) {
    return ((unsigned long long)lane_xor<D>((unsigned)(v >> 32)) << 32) | lane_xor<D>((unsigned)v);
}

// Sorts `size` keys (a power of two from 32 to 2 NT; the last size - list count as largest): a bitonic
// network whose elements tid and tid + NT each thread keeps, so that the steps within a wave are
// exchanges of lanes and only the wider ones go through memory (2048 keys: 13 of 66).
template <int NT>
struct Sorter {
    unsigned long long v[2];
    unsigned long long* key;
    int tid, size;

    template <int W, int D>
    __device__ __forceinline__ void step() {
        if constexpr (D == NT) {
            if (v[0] > v[1]) {
                const unsigned long long t = v[0];
                v[0] = v[1];
                v[1] = t;
            }
        } else {
            unsigned long long other[2] = {~0ull, ~0ull};
            if constexpr (D >= 64) {
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (e * NT + tid < size) key[e * NT + tid] = v[e];
                __syncthreads();
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (e * NT + tid < size) other[e] = key[(e * NT + tid) ^ D];
                __syncthreads();
            } else {
                other[0] = lane_xor64<D>(v[0]);
                if (size > NT) other[1] = lane_xor64<D>(v[1]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int i = e * NT + tid;
                const bool low = ((i & D) == 0) == ((i & W) == 0);  // this place keeps the smaller one
                v[e] = (other[e] < v[e]) == low ? other[e] : v[e];
            }
        }
        if constexpr (D > 1) step<W, D / 2>();
    }
    template <int W>
    __device__ __forceinline__ void sort() {
        step<W, W / 2>();
        if constexpr (W < 2 * NT)
            if (W < size) sort<2 * W>();
    }
};
template <int NT>
__device__ void sort_keys(unsigned long long* key, int list, int size) {
    Sorter<NT> s;
    s.tid = threadIdx.x;
    s.key = key;
    s.size = size;
#pragma unroll
    for (int e = 0; e < 2; ++e) s.v[e] = e * NT + s.tid < list ? key[e * NT + s.tid] : ~0ull;
    __syncthreads();
    s.template sort<2>();
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (e * NT + s.tid < size) key[e * NT + s.tid] = s.v[e];
    __syncthreads();
}

template <typename H, int NT>
__device__ void build_list(const ListArgs<H>& x, int64_t g, unsigned long long* key, float* pv, float* qv) {
    const int tid = threadIdx.x, tn = x.tg.tn;
    auto put = [&](int s, int row, int c, float z, float q, float lse) {
        key[s] = c >= 0 ? ((unsigned long long)(((uint32_t)c << 5) | row) << 11) | s : ~0ull;
        const float p = expf(z * x.tg.inv_tau - lse);
        pv[s] = c >= 0 ? (p > 1.0f ? 1.0f : p) : 0.0f;  // more only by the roundings of large logits
        qv[s] = q;
    };
    if (x.tg.target) {
        // 8 lanes a row
        for (int row = tid >> 3; row < 32; row += NT / 8) {
            const int64_t r = g * 32 + row;
            const float f = factor_of(x.tg, x.grad, min(r, x.m - 1), tid & 7);
            const int c = r < x.m && f != 0.0f ? x.tg.cls(r, 0) : -1;
            const float z = logit_of(x.h, min(r, x.m - 1), c, tid & 7);
            if ((tid & 7) == 0) put(row, row, c, z, 1.0f, c >= 0 ? x.lse[r] : 0.0f);
        }
    } else {
        // a wave a row
        const int lane = tid & 63;
        for (int row = tid >> 6; row < 32; row += NT / 64) {
            const int64_t r = g * 32 + row;
            RowTargets t{-1, 0.0f, 0.0f, 0.0f};
            bool live = r < x.m && (!x.grad || x.grad[r] != 0.0f);
            if (live) {
                t = row_targets<sizeof(typename H::type) == 2 ? 2 : 1>(x.tg, x.h, r, lane);
                live = __any(t.q != 0.0f);
            }
            if (lane < tn) put(row * tn + lane, row, live ? t.cls : -1, t.z, t.q, live ? x.lse[r] : 0.0f);
        }
    }
    __syncthreads();
    sort_keys<NT>(key, x.list, x.size);
    for (int s = tid; s < x.list; s += NT) {
        const uint32_t kk = key[s] == ~0ull ? kNoKey : (uint32_t)(key[s] >> 11);
        float v = 0.0f;
        if (kk != kNoKey) {
            // the entries that name this class of this row, in their order
            int f = s;
            while (f > 0 && (uint32_t)(key[f - 1] >> 11) == kk) --f;
            v = pv[key[f] & 2047];
            float q = 0.0f;
            for (int i = f; i < x.list && key[i] != ~0ull && (uint32_t)(key[i] >> 11) == kk; ++i) q += qv[key[i] & 2047];
            v -= q;
        }
        x.keys[g * x.list + s] = kk;
        x.vals[g * x.list + s] = v;
    }
    for (int b = tid; b <= x.blocks; b += NT) {
        const unsigned long long lim = (unsigned long long)b << (7 + 5 + 11);
        int lo = 0, hi = x.list;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (key[mid] < lim) lo = mid + 1;
            else hi = mid;
        }
        x.offs[g * (x.blocks + 1) + b] = (uint16_t)lo;
    }
}

// Records, and with one target a row (a label) the lists too.
template <typename H, int D, int P, bool BACK>
__global__ __launch_bounds__(kThreads) void prep_kernel(RecordArgs<H> x, ListArgs<H> y, unsigned class_tiles) {
    __shared__ __align__(16) float lds[32 * (32 * D + 1) + 12 + 32];
    static_assert(sizeof(lds) >= 32 * 16, "a list of 32 entries");
    const unsigned b = blockIdx.x;
    if (b < x.row_tiles + class_tiles) {
        const bool rows = b < x.row_tiles;
        build_record<H, D, P, BACK>(x, rows ? b : b - x.row_tiles, rows, lds, lds + 32 * (32 * D + 1));
    } else if constexpr (BACK) {
        unsigned long long* key = reinterpret_cast<unsigned long long*>(lds);
        float* pv = reinterpret_cast<float*>(key + 32);
        build_list<H, kThreads>(y, b - x.row_tiles - class_tiles, key, pv, pv + 32);
    }
}
// Two workgroups on a CU, for which 2 to 8 registers go to scratch: 7 us less for 15360 rows of 32 entries
// than one without, 2 us more for a page's 71 groups.
constexpr int kListThreads = 1024;
template <typename H>
__global__ __launch_bounds__(kListThreads, 8) void list_kernel(ListArgs<H> y) {
    extern __shared__ __align__(16) uint8_t list_lds[];
    unsigned long long* key = reinterpret_cast<unsigned long long*>(list_lds);
    float* pv = reinterpret_cast<float*>(key + y.size);
    build_list<H, kListThreads>(y, blockIdx.x, key, pv, pv + y.size);
}

// ---------------------------------------------------------------- forward: merge and loss
// Joins two sums of exp2(t - reference).
__device__ __forceinline__ void join(float* ref, float* sum, float2 v) {
    const float nr = fmaxf(*ref, v.x);
    const float s = *ref == -INFINITY ? *sum : *sum * exp2f(*ref - nr);
    *sum = s + (v.x == -INFINITY ? v.y : v.y * exp2f(v.x - nr));
    *ref = nr;
}
// Their natural logarithm; a row whose classes are all -inf keeps reference -inf and sum 0.  The sum's
// exponent goes with the reference: logf of 18710 is off by half a step of 10 on average, one way.
__device__ __forceinline__ float log_sum(float ref, float sum) {
    if (!(sum > 0.0f && sum < INFINITY)) return ref == -INFINITY ? logf(sum) : ref + logf(sum);
    int e;
    const float m = frexpf(sum, &e);
    const float two = (ref == -INFINITY ? 0.0f : ref) + (float)e;
    return fmaf(two, kLn2, fmaf(two, kLn2Rest, logf(m)));
}

// Labels of many rows: 8 lanes a row (30720 fp32 rows: 7.8 us; 26 with a wave a row, when this took 9).
template <typename H>
__global__ __launch_bounds__(kThreads) void label_loss_kernel(H h, Targets tg, int64_t m, int nsplit,
                                                              const float2* __restrict__ part, float* loss,
                                                              float* lse) {
    const int l8 = threadIdx.x & 7;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 8) + (threadIdx.x >> 3), r = min(row, m - 1);
    const int c = tg.cls(r, 0);
    float ref = -INFINITY, sum = 0.0f;
    for (int s = l8; s < nsplit; s += 8) join(&ref, &sum, part[(int64_t)s * m + r]);
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) join(&ref, &sum, make_float2(__shfl_xor(ref, o, 64), __shfl_xor(sum, o, 64)));
    const float z = logit_of(h, r, c, l8);
    if (row < m && l8 == 0) {
        const float l = log_sum(ref, sum);
        loss[row] = c >= 0 ? l - z : 0.0f;
        lse[row] = l;
    }
}

// A wave per row: the chunks' statistics of the row, then its targets' logits.
template <typename H>
__global__ __launch_bounds__(kThreads) void loss_kernel(H h, Targets tg, int64_t m, int nsplit,
                                                        const float2* __restrict__ part, float* loss,
                                                        float* lse) {
    const int lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
    if (row >= m) return;
    const RowTargets t = row_targets<4>(tg, h, row, lane);
    float ref = -INFINITY, sum = 0.0f;
    for (int s = lane; s < nsplit; s += 64) join(&ref, &sum, part[(int64_t)s * m + row]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) join(&ref, &sum, make_float2(__shfl_xor(ref, o, 64), __shfl_xor(sum, o, 64)));
    const float l = log_sum(ref, sum);
    // entries without weight add nothing, whatever their class's logit
    const float total = wave_sum(t.q != 0.0f ? t.q * (t.logq - t.z * tg.inv_tau + l) : 0.0f);
    if (lane == 0) {
        loss[row] = total;
        lse[row] = l;
    }
}

// ---------------------------------------------------------------- backward: sums of the chunks
// out[o][j] = sum over chunks, for owners of k values held in rows of 32 D; then db.
template <typename T>
struct SumArgs {
    const float* part;
    int nsplit;
    int64_t owners;
    T* out;  // null: not asked for
    int vec;  // out's rows can be written four values at a time
};
template <typename T>
__device__ __forceinline__ void store(T* p, float v);
template <>
__device__ __forceinline__ void store<float>(float* p, float v) {
    *p = v;
}
template <>
__device__ __forceinline__ void store<uint16_t>(uint16_t* p, float v) {
    *p = __builtin_bit_cast(uint16_t, (__bf16)v);
}
template <typename T>
__device__ __forceinline__ void sum_chunks(const SumArgs<T>& x, int k, int ld, int64_t block, int64_t blocks) {
    const unsigned quads = (unsigned)(ld / 4);
    const int64_t all = x.owners * quads, plane = x.owners * ld;
    for (int64_t i = block * kThreads + threadIdx.x; i < all; i += blocks * kThreads) {
        const int64_t o = i / quads;
        const int j = (int)(i - o * quads) * 4;
        if (j >= k) continue;
        f32x4 s = {};
        for (int c0 = 0; c0 < x.nsplit; c0 += 8) {
            // eight chunks on their way at once, added in their order
            f32x4 v[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) v[c] = *reinterpret_cast<const f32x4*>(x.part + min(c0 + c, x.nsplit - 1) * plane + i * 4);
#pragma unroll
            for (int c = 0; c < 8; ++c)
#pragma unroll
                for (int u = 0; u < 4; ++u) s[u] += c0 + c < x.nsplit ? v[c][u] : 0.0f;
        }
        T* out = x.out + o * k + j;
        if (x.vec) {
            Four<T> q;
#pragma unroll
            for (int u = 0; u < 4; ++u) store<T>(q.v + u, s[u]);
            *reinterpret_cast<Four<T>*>(out) = q;
        } else {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (j + u < k) store<T>(out + u, s[u]);
        }
    }
}
// da by the first `grid_a` workgroups, dW and db by the others.
template <typename T>
__global__ __launch_bounds__(kThreads) void sum_kernel(SumArgs<T> a, SumArgs<T> w, int k, int ld, unsigned grid_a,
                                                       const float* __restrict__ part_db, float* db) {
    if (blockIdx.x < grid_a) {
        sum_chunks<T>(a, k, ld, blockIdx.x, grid_a);
        return;
    }
    const int64_t block = blockIdx.x - grid_a, blocks = gridDim.x - grid_a;
    if (w.out) sum_chunks<T>(w, k, ld, block, blocks);
    if (db)
        for (int64_t i = block * kThreads + threadIdx.x; i < w.owners; i += blocks * kThreads) {
            float s = 0.0f;
            for (int c = 0; c < w.nsplit; ++c) s += part_db[c * w.owners + i];
            db[i] = s;
        }
}

// ---------------------------------------------------------------- shapes and launches
int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int kBlockTiles = 4;  // records of a block of 128 classes
constexpr int kMostChunks = 256;
constexpr int64_t kMostGroups = 1 << 22;  // workgroups of a launch that is split further (grids count threads in 32 bits)

// Chunks of the class records for the statistics: the fewest records that any place of the GPU works
// through one after the other (a workgroup's start and end take about two records' time).
void pick_stats(XentLayout* L, int64_t m, int planes) {
    L->fblocks = m <= 128 ? 1 : xent_stats_most_blocks(L->D, planes);
    const int64_t blocks = div_up(m, 128 * L->fblocks), places = 512;
    int64_t best = -1;
    for (int s = 1; s <= 256; ++s) {
        const int64_t per = div_up(L->class_tiles, s);
        if (div_up(L->class_tiles, per) != s) continue;
        if (s > 1 && blocks * s > kMostGroups) break;
        const int64_t cost = 8 * div_up(blocks * s, places) * (per + 2) + s / 4;
        if (best < 0 || cost < best) {
            best = cost;
            L->fsplit = s;
            L->fper = (int)per;
        }
    }
}

// Chunks for the two gradients, whose workgroups share a launch: the same number of records for both,
// the fewest that any place works through; a further chunk costs the time its sums take to be written
// and read again (256 D bytes an owner at 5 TB/s, against 0.36 or 0.16 D us a record).
void pick_grads(XentLayout* L, int64_t m, int64_t n, int planes) {
    const int64_t places = 256 * xent_grad_per_cu(L->D, planes);
    const int64_t ba = div_up(m, kXentGradOwners), bw = div_up(n, kXentGradOwners);
    const double chunk_cost = 256.0 / 5e6 / (planes == 2 ? 0.36 : 0.16);
    double best = -1.0;
    // records of a chunk of a stream in `chunks`: da's walk the target lists from whole blocks of classes
    auto whole = [](int64_t tiles, int64_t chunks) { return div_up(div_up(tiles, chunks), kBlockTiles) * kBlockTiles; };
    for (int s = 1; s <= kMostChunks; ++s) {
        // s chunks of the shorter side's stream; the other's of the same length
        const bool by_a = L->class_tiles <= L->row_tiles;
        const int64_t per = whole(by_a ? L->class_tiles : L->row_tiles, s);
        const int64_t sa = div_up(L->class_tiles, per), sw = div_up(L->row_tiles, per);
        if (sa > kMostChunks || sw > kMostChunks || (s > 1 && ba * sa + bw * sw > kMostGroups)) break;
        const double cost = (double)div_up(ba * sa + bw * sw, places) * (double)(per + 2) +
                            chunk_cost * (double)(sa * m + sw * n);
        if (best < 0 || cost < best) {
            best = cost;
            L->split_a = (int)sa;
            L->split_w = (int)sw;
            L->per_a = L->per_w = (int)per;
        }
    }
    if (best < 0) {
        // Streams of very different lengths: each in the most chunks, but no more than keep the GPU busy
        // (each has sums of its own: 63 of them for 2000 rows under 600000 classes would be 19 GB).
        auto chunks = [&](int64_t blocks) { return std::clamp<int64_t>(8 * places / blocks, 1, kMostChunks); };
        L->per_a = (int)whole(L->class_tiles, chunks(ba));
        L->per_w = (int)div_up(L->row_tiles, chunks(bw));
        L->split_a = (int)div_up(L->class_tiles, L->per_a);
        L->split_w = (int)div_up(L->row_tiles, L->per_w);
    }
}

bool in_fours(const void* p, int k, bool bf16) { return k % 4 == 0 && reinterpret_cast<uintptr_t>(p) % (bf16 ? 8 : 16) == 0; }

// f(head) with the problem's head as it can be read.
template <typename T, typename F>
int with_head(const XentProblem& x, F&& f) {
    const T* a = static_cast<const T*>(x.a);
    const T* w = static_cast<const T*>(x.w);
    if (in_fours(x.a, x.k, x.bf16) && in_fours(x.w, x.k, x.bf16)) return f(HeadRef<T, true>{a, w, x.bias, x.k});
    return f(HeadRef<T, false>{a, w, x.bias, x.k});
}

Targets targets_of(const XentProblem& x) {
    return Targets{x.target, x.teacher_idx, x.teacher_z, x.tn, 1.0f / x.tau, x.n};
}

// f.template operator()<D>() for the layout's D.
template <typename F>
int by_pieces(int D, F&& f) {
    switch (D) {
        case 1: return f.template operator()<1>();
        case 2: return f.template operator()<2>();
        case 3: return f.template operator()<3>();
        case 4: return f.template operator()<4>();
        case 6: return f.template operator()<6>();
        default: return f.template operator()<8>();
    }
}

template <typename T, int P, bool BACK>
int prep(const XentProblem& x, const XentLayout& L, uint8_t* ws, hipStream_t st) {
    return with_head<T>(x, [&]<typename H>(const H& h) -> int {
        const Targets tg = targets_of(x);
        const RecordArgs<H> r{h, tg, x.lse, x.grad, x.m, x.n, L.row_tiles, ws + (BACK ? L.b_row_rec : L.f_row_rec),
                              ws + (BACK ? L.b_class_rec : L.f_class_rec), reinterpret_cast<int*>(ws + L.b_row_u),
                              reinterpret_cast<int*>(ws + (BACK ? L.b_class_u : L.f_class_u))};
        const int list = 32 * x.tn;
        int size = 32;
        while (size < list) size *= 2;
        const ListArgs<H> y{h, tg, x.lse, x.grad, x.m, list, size, (int)div_up(x.n, 128),
                            reinterpret_cast<uint32_t*>(ws + L.b_keys), reinterpret_cast<float*>(ws + L.b_vals),
                            reinterpret_cast<uint16_t*>(ws + L.b_offs)};
        const bool lists_here = BACK && x.target;
        const unsigned grid = (unsigned)(L.row_tiles * (lists_here ? 2 : 1) + L.class_tiles);
        by_pieces(L.D, [&]<int D>() {
            prep_kernel<H, D, P, BACK><<<grid, kThreads, 0, st>>>(r, y, (unsigned)L.class_tiles);
            return 0;
        });
        PPOCR_HIP(hipGetLastError());
        if (BACK && !x.target) {
            list_kernel<H><<<(unsigned)L.row_tiles, kListThreads, (size_t)size * 16, st>>>(y);
            PPOCR_HIP(hipGetLastError());
        }
        return PPOCR_OK;
    });
}

template <typename T>
int losses(const XentProblem& x, const Targets& tg, int nsplit, const float2* part, float* loss, float* lse, hipStream_t st) {
    return with_head<T>(x, [&]<typename H>(const H& h) -> int {
        if (x.target && x.m > 4096)
            label_loss_kernel<H><<<(unsigned)div_up(x.m, kThreads / 8), kThreads, 0, st>>>(h, tg, x.m, nsplit, part, loss, lse);
        else
            loss_kernel<H><<<(unsigned)div_up(x.m, kThreads / 64), kThreads, 0, st>>>(h, tg, x.m, nsplit, part, loss, lse);
        PPOCR_HIP(hipGetLastError());
        return PPOCR_OK;
    });
}

template <typename T>
int sums(const XentLayout& L, const float* pa, const float* pw, const float* pdb, int64_t m, int64_t n, int k, void* da,
         void* dw, float* db, hipStream_t st) {
    const bool bf16 = sizeof(T) == 2;
    const SumArgs<T> a{pa, L.split_a, m, (T*)da, in_fours(da, k, bf16)}, w{pw, L.split_w, n, (T*)dw, in_fours(dw, k, bf16)};
    auto blocks = [&](int64_t owners) { return (unsigned)std::min<int64_t>(div_up(owners * 8 * L.D, kThreads), 2048); };
    const unsigned ga = da ? blocks(m) : 0, gw = dw || db ? blocks(n) : 0;
    sum_kernel<T><<<ga + gw, kThreads, 0, st>>>(a, w, k, 32 * L.D, ga, pdb, db);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

}  // namespace

XentLayout xent_layout(int64_t m, int64_t n, int64_t k, int tn, int planes) {
    XentLayout L{};
    L.D = xent_pieces(k);
    L.row_tiles = xent_tiles(m);
    L.class_tiles = xent_tiles(n);
    pick_stats(&L, m, planes);
    pick_grads(&L, m, n, planes);
    auto put = [](size_t* at, size_t bytes) {
        const size_t here = *at;
        *at += (bytes + 255) / 256 * 256;
        return here;
    };
    // a workspace may also serve the head's calls, whose list header its first bytes hold
    size_t f = 256;
    L.f_row_rec = put(&f, (size_t)L.row_tiles * xent_rec_bytes(L.D, planes, false));
    L.f_class_rec = put(&f, (size_t)L.class_tiles * xent_rec_bytes(L.D, planes, false));
    L.f_class_u = put(&f, (size_t)L.class_tiles * 4);
    L.f_part = put(&f, (size_t)L.fsplit * m * sizeof(float2));
    L.f_total = f;
    size_t b = 256;
    L.b_row_rec = put(&b, (size_t)L.row_tiles * xent_rec_bytes(L.D, planes, true));
    L.b_class_rec = put(&b, (size_t)L.class_tiles * xent_rec_bytes(L.D, planes, true));
    L.b_row_u = put(&b, (size_t)L.row_tiles * 4);
    L.b_class_u = put(&b, (size_t)L.class_tiles * 4);
    L.b_keys = put(&b, (size_t)L.row_tiles * 32 * tn * 4);
    L.b_vals = put(&b, (size_t)L.row_tiles * 32 * tn * 4);
    L.b_offs = put(&b, (size_t)L.row_tiles * (div_up(n, 128) + 1) * 2);
    L.b_part_a = put(&b, (size_t)L.split_a * m * 32 * L.D * 4);
    L.b_part_w = put(&b, (size_t)L.split_w * n * 32 * L.D * 4);
    L.b_part_db = put(&b, (size_t)L.split_w * n * 4);
    L.b_total = b;
    return L;
}

int launch_xent_forward(const XentProblem& x, float* loss, float* lse, uint8_t* ws, hipStream_t st) {
    const XentLayout L = xent_layout(x.m, x.n, x.k, x.tn, x.planes());
    const Targets tg = targets_of(x);
    if (int e = x.bf16 ? prep<uint16_t, 1, false>(x, L, ws, st) : prep<float, 2, false>(x, L, ws, st)) return e;
    float2* part = reinterpret_cast<float2*>(ws + L.f_part);
    const XentStatsArgs s{ws + L.f_row_rec, ws + L.f_class_rec, reinterpret_cast<const int*>(ws + L.f_class_u), x.m, L.class_tiles, L.fsplit, L.fper, kLog2e / x.tau, part};
    const unsigned grid = (unsigned)(div_up(x.m, 128 * L.fblocks) * L.fsplit);
    if (int e = by_pieces(L.D, [&]<int D>() {
            return x.bf16 ? xent_stats_cfg<D, 1>(s, L.fblocks, grid, st) : xent_stats_cfg<D, 2>(s, L.fblocks, grid, st);
        }))
        return e;
    return x.bf16 ? losses<uint16_t>(x, tg, L.fsplit, part, loss, lse, st) : losses<float>(x, tg, L.fsplit, part, loss, lse, st);
}

int launch_xent_zero(const XentProblem& x, void* dw, float* db, hipStream_t st) {
    if (!dw && !db) return PPOCR_OK;
    XentLayout L{};
    L.D = xent_pieces(x.k);
    return x.bf16 ? sums<uint16_t>(L, nullptr, nullptr, nullptr, 0, x.n, x.k, nullptr, dw, db, st)
                  : sums<float>(L, nullptr, nullptr, nullptr, 0, x.n, x.k, nullptr, dw, db, st);
}

int launch_xent_backward(const XentProblem& x, void* da, void* dw, float* db, uint8_t* ws, hipStream_t st) {
    const XentLayout L = xent_layout(x.m, x.n, x.k, x.tn, x.planes());
    if (int e = x.bf16 ? prep<uint16_t, 1, true>(x, L, ws, st) : prep<float, 2, true>(x, L, ws, st)) return e;
    float* pa = reinterpret_cast<float*>(ws + L.b_part_a);
    float* pw = reinterpret_cast<float*>(ws + L.b_part_w);
    float* pdb = reinterpret_cast<float*>(ws + L.b_part_db);
    const uint8_t* rr = ws + L.b_row_rec;
    const uint8_t* cr = ws + L.b_class_rec;
    const unsigned ga = da ? (unsigned)(div_up(x.m, kXentGradOwners) * L.split_a) : 0;
    const unsigned gw = dw || db ? (unsigned)(div_up(x.n, kXentGradOwners) * L.split_w) : 0;
    const XentGradArgs s{{rr, cr, x.m, L.row_tiles, L.class_tiles, reinterpret_cast<const int*>(ws + L.b_class_u), L.split_a,
                          L.per_a, pa},
                         {cr, rr, x.n, L.class_tiles, L.row_tiles, reinterpret_cast<const int*>(ws + L.b_row_u), L.split_w,
                          L.per_w, pw},
                         ga,
                         kLog2e / x.tau,
                         reinterpret_cast<const uint32_t*>(ws + L.b_keys),
                         reinterpret_cast<const float*>(ws + L.b_vals),
                         reinterpret_cast<const uint16_t*>(ws + L.b_offs),
                         32 * x.tn,
                         (int)div_up(x.n, 128),
                         pdb};
    if (int e = by_pieces(L.D, [&]<int D>() {
            return x.bf16 ? xent_grad_cfg<D, 1>(s, ga + gw, st) : xent_grad_cfg<D, 2>(s, ga + gw, st);
        }))
        return e;
    return x.bf16 ? sums<uint16_t>(L, pa, pw, pdb, x.m, x.n, x.k, da, dw, db, st)
                  : sums<float>(L, pa, pw, pdb, x.m, x.n, x.k, da, dw, db, st);
}

}  // namespace ppocr
