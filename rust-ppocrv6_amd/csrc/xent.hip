// Losses over the vocabulary without keeping the logits (xent.hpp): the operand records, the
// target lists, the merge of the forward pass, the sums of the backward pass, and the launches.
#include <algorithm>

#include "xent.hpp"

namespace ppocr {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ float value(const uint16_t* p) { return __uint_as_float((unsigned)*p << 16); }

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

// The teacher's softmax over a row's entries, by 8 neighbouring lanes: the largest logit and the
// sum of exp(logit - largest); a row without entries (or with only -inf) has sum 0.
__device__ __forceinline__ void teacher_stats(const Targets& tg, int64_t r, bool live, int l8, float* top, float* sum) {
    float m = -INFINITY;
    bool bad = false;
    for (int i = l8; i < tg.tn; i += 8)
        if (live && tg.cls(r, i) >= 0) {
            const float t = tg.logit(r, i);
            bad |= !(t < INFINITY);
            m = fmaxf(m, t);
        }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    float s = bad ? NAN : 0.0f;
    for (int i = l8; i < tg.tn; i += 8)
        if (live && m > -INFINITY && tg.cls(r, i) >= 0) s += expf(tg.logit(r, i) - m);
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    *top = m;
    *sum = s;
}

// a_r . w_c + b_c, by 8 neighbouring lanes (all of them call it); 0 for c < 0.
template <typename T>
__device__ __forceinline__ float logit_of(const T* __restrict__ a, const T* __restrict__ w, const float* bias, int64_t r,
                                          int c, int k, int l8) {
    float s = 0.0f;
    if (c >= 0) {
        const T* pa = a + r * k;
        const T* pw = w + (int64_t)c * k;
        for (int j = l8; j < k; j += 8) s = fmaf(value(pa + j), value(pw + j), s);
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    return c >= 0 && bias ? s + bias[c] : s;
}

// A row's gradient factor: g / tau when it has a target, 0 otherwise.
__device__ __forceinline__ float factor_of(const Targets& tg, const float* grad, int64_t r) {
    bool any = false;
    for (int i = 0; i < tg.tn; ++i) any |= tg.cls(r, i) >= 0 && (tg.target || tg.logit(r, i) != -INFINITY);
    return any ? (grad ? grad[r] : 1.0f) * tg.inv_tau : 0.0f;
}

// ---------------------------------------------------------------- operand records
// One workgroup per record of 32 entries, rows of `a` first and then classes of `w`.
template <typename T>
struct RecordArgs {
    const T* a;
    const T* w;
    const float* bias;
    Targets tg;
    const float* lse;
    const float* grad;
    int64_t m, n, row_tiles;
    int k, D;
    uint8_t* row_rec;
    uint8_t* class_rec;
    int* row_u;
    int* class_u;
};

template <typename T, int P, bool BACK>
__device__ void build_record(const RecordArgs<T>& x, int64_t t, bool rows, float* tile, float* red) {
    const int tid = threadIdx.x, D = x.D, ld = 32 * D + 1;
    const int64_t first = t * 32, count = min((int64_t)32, (rows ? x.m : x.n) - first);
    const T* src = (rows ? x.a : x.w) + first * x.k;
    float* gf = red + 8;  // 32 gradient factors
    if (BACK && rows && tid < 32) gf[tid] = tid < count ? factor_of(x.tg, x.grad, first + tid) : 0.0f;
    __syncthreads();
    float top = 0.0f;
    for (int i = tid; i < 32 * 32 * D; i += kThreads) {
        const int e = i / (32 * D), j = i % (32 * D);
        // a row without gradient reaches no sum, whatever it holds
        const bool in = e < count && j < x.k && !(BACK && rows && gf[e] == 0.0f);
        const float v = in ? value(src + (int64_t)e * x.k + j) : 0.0f;
        tile[e * ld + j] = v;
        if (fabsf(v) < INFINITY) top = fmaxf(top, fabsf(v));
    }
    top = wave_max(top);
    if ((tid & 63) == 0) red[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    // largest magnitude to [2^14, 2^15); 2^100 at most, so that 2^-e and the factors stay in range
    const int ex = top > 0.0f ? min(14 - ilogbf(top), 100) : 100;
    uint8_t* rec = (rows ? x.row_rec : x.class_rec) + t * (int64_t)((size_t)P * D * 2048 * (BACK ? 2 : 1) + kXentAux);
    const int form = 2 * D * 64;  // 16-byte pieces of one plane of one form
    for (int i = tid; i < form * (BACK ? 2 : 1); i += kThreads) {
        const bool tr = i >= form;
        const int c = tr ? i - form : i, lane = c & 63, l = lane & 31, h = lane >> 5, step = c >> 6;
        f16x8 hi, lo;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // transposed: step = 2 d + e, the entries of an MFMA result's rows
            const int e = tr ? 16 * (step & 1) + 8 * (j >> 2) + 4 * h + (j & 3) : l;
            const int kk = tr ? 32 * (step >> 1) + l : 16 * step + 8 * h + j;
            const float v = ldexpf(tile[e * ld + kk], ex);
            hi[j] = (_Float16)v;
            if (P == 2) lo[j] = (_Float16)(v - (float)hi[j]);
        }
        f16x8* dst = reinterpret_cast<f16x8*>(rec + (tr ? (size_t)P * D * 2048 : 0));
        dst[c] = hi;
        if (P == 2) dst[form + c] = lo;
    }
    float* aux = reinterpret_cast<float*>(rec + (size_t)P * D * 2048 * (BACK ? 2 : 1));
    if (tid < 32) {
        if (!rows) {
            aux[tid] = tid < count ? (x.bias ? x.bias[first + tid] * (kLog2e * x.tg.inv_tau) : 0.0f) : -INFINITY;
            aux[32 + tid] = 0.0f;
        } else if (BACK) {
            aux[tid] = gf[tid] != 0.0f ? x.lse[first + tid] * kLog2e : INFINITY;
            aux[32 + tid] = gf[tid];
        } else {
            aux[tid] = 0.0f;
            aux[32 + tid] = 0.0f;
        }
    } else if (tid < 48) {
        aux[32 + tid] = tid == 32 ? ldexpf(1.0f, -ex) : tid == 33 ? (float)ex : 0.0f;
    }
    if (BACK && tid == 0) {
        float s = 0.0f;
        for (int i = 0; i < 32 && rows; ++i)
            if (fabsf(gf[i]) < INFINITY) s = fmaxf(s, fabsf(gf[i]));
        // the largest of what multiplies this record's values, as an exponent, against its own
        if (rows) x.row_u[t] = s > 0.0f ? max(ilogbf(s) + 1 - ex, -200) : -200;
        else x.class_u[t] = -ex;
    }
}

// ---------------------------------------------------------------- target lists (backward)
// One workgroup per group of 32 rows: every target entry's p - q in 32 bits, sorted by class (then
// row), entries of one row that name the same class joined, and where each block of 128 classes
// starts in the list.
template <typename T>
struct ListArgs {
    const T* a;
    const T* w;
    const float* bias;
    Targets tg;
    const float* lse;
    const float* grad;
    int64_t m;
    int k, list, size, blocks;  // list = 32 tn entries, size = list rounded up to a power of two
    uint32_t* keys;
    float* vals;
    uint16_t* offs;
};
constexpr uint32_t kNoKey = 0xFFFFFFFFu;

template <typename T>
__device__ void build_list(const ListArgs<T>& x, int64_t g, unsigned long long* key, float* pv, float* qv) {
    const int tid = threadIdx.x, l8 = tid & 7, row = tid >> 3, tn = x.tg.tn;
    const int64_t r = g * 32 + row;
    const bool live = r < x.m && factor_of(x.tg, x.grad, r) != 0.0f;
    float top = 0.0f, sum = 1.0f;
    if (!x.tg.target) teacher_stats(x.tg, r, live, l8, &top, &sum);
    for (int i = 0; i < tn; ++i) {
        const int c = live ? x.tg.cls(r, i) : -1;
        const float z = logit_of(x.a, x.w, x.bias, r, c, x.k, l8);
        if (l8 == 0) {
            const int s = row * tn + i;
            const float q = x.tg.target ? 1.0f : (c >= 0 ? expf(x.tg.logit(r, i) - top) / sum : 0.0f);
            key[s] = c >= 0 ? ((unsigned long long)(((uint32_t)c << 5) | row) << 11) | s : ~0ull;
            pv[s] = c >= 0 ? expf(z * x.tg.inv_tau - x.lse[r]) : 0.0f;
            qv[s] = q;
        }
    }
    for (int s = x.list + tid; s < x.size; s += kThreads) key[s] = ~0ull;
    __syncthreads();
    for (int w2 = 2; w2 <= x.size; w2 <<= 1)
        for (int d = w2 >> 1; d >= 1; d >>= 1) {
            for (int p = tid; p < x.size / 2; p += kThreads) {
                const int i = 2 * d * (p / d) + p % d, j = i + d;
                const bool up = (i & w2) == 0;
                const unsigned long long a = key[i], b = key[j];
                if ((a > b) == up) {
                    key[i] = b;
                    key[j] = a;
                }
            }
            __syncthreads();
        }
    for (int s = tid; s < x.list; s += kThreads) {
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
    for (int b = tid; b <= x.blocks; b += kThreads) {
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

// LDS: a record's tile, or a list's keys and values.
size_t prep_lds(int D, int size) {
    return std::max((size_t)(32 * (32 * D + 1) + 8 + 32) * 4, (size_t)size * 16);
}

template <typename T, int P, bool BACK>
__global__ __launch_bounds__(kThreads) void prep_kernel(RecordArgs<T> x, ListArgs<T> y, unsigned class_tiles) {
    extern __shared__ __align__(16) uint8_t lds[];
    const unsigned b = blockIdx.x;
    if (b < x.row_tiles + class_tiles) {
        float* tile = reinterpret_cast<float*>(lds);
        const bool rows = b < x.row_tiles;
        build_record<T, P, BACK>(x, rows ? b : b - x.row_tiles, rows, tile, tile + 32 * (32 * x.D + 1));
    } else if constexpr (BACK) {
        unsigned long long* key = reinterpret_cast<unsigned long long*>(lds);
        float* pv = reinterpret_cast<float*>(key + y.size);
        build_list<T>(y, b - x.row_tiles - class_tiles, key, pv, pv + y.size);
    }
}

// ---------------------------------------------------------------- forward: merge and loss
// Eight rows per wave, 8 lanes each: the chunks' statistics of a row, then its target's logits.
template <typename T>
__global__ __launch_bounds__(kThreads) void loss_kernel(const T* a, const T* w, const float* bias, Targets tg, int64_t m,
                                                        int k, int nsplit, const float2* __restrict__ part, float* loss,
                                                        float* lse) {
    const int l8 = threadIdx.x & 7;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 8) + (threadIdx.x >> 3);
    const bool live = row < m;
    const int64_t r = live ? row : m - 1;
    float ref = -INFINITY;
    for (int s = l8; s < nsplit; s += 8) ref = fmaxf(ref, part[(int64_t)s * m + r].x);
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) ref = fmaxf(ref, __shfl_xor(ref, o, 64));
    float sum = 0.0f;
    for (int s = l8; s < nsplit; s += 8) {
        const float2 v = part[(int64_t)s * m + r];
        sum += v.x == -INFINITY ? v.y : v.y * exp2f(v.x - ref);
    }
#pragma unroll
    for (int o = 4; o >= 1; o >>= 1) sum += __shfl_xor(sum, o, 64);
    // a row whose classes are all -inf keeps reference -inf and sum 0
    const float l = (ref == -INFINITY ? 0.0f : ref * (1.0f / kLog2e)) + logf(sum);
    float top = 0.0f, qs = 1.0f, total = 0.0f;
    if (!tg.target) teacher_stats(tg, r, true, l8, &top, &qs);
    const float logqs = logf(qs);
    for (int i = 0; i < tg.tn; ++i) {
        const int c = tg.cls(r, i);
        const float z = logit_of(a, w, bias, r, c, k, l8);
        if (c < 0) continue;
        if (tg.target) {
            total = l - z * tg.inv_tau;
        } else if (qs != 0.0f) {
            const float lq = tg.logit(r, i) - top - logqs;
            const float q = expf(lq);
            if (q != 0.0f) total += q * (lq - z * tg.inv_tau + l);
        }
    }
    if (live && l8 == 0) {
        loss[row] = total;
        lse[row] = l;
    }
}

// ---------------------------------------------------------------- backward: sums of the chunks
// out[o][j] = sum over chunks, for owners of k values held in rows of 32 D; then db.
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
__global__ __launch_bounds__(kThreads) void sum_kernel(const float* __restrict__ part, int nsplit, int64_t owners, int k, int ld,
                                                       T* out, const float* __restrict__ part_db, float* db) {
    const int64_t stride = (int64_t)gridDim.x * kThreads, base = (int64_t)blockIdx.x * kThreads + threadIdx.x;
    if (out) {
        for (int64_t i = base; i < owners * k; i += stride) {
            const int64_t at = i / k * ld + i % k;
            float s = 0.0f;
            for (int c = 0; c < nsplit; ++c) s += part[(int64_t)c * owners * ld + at];
            store<T>(out + i, s);
        }
    }
    if (db) {
        for (int64_t i = base; i < owners; i += stride) {
            float s = 0.0f;
            for (int c = 0; c < nsplit; ++c) s += part_db[(int64_t)c * owners + i];
            db[i] = s;
        }
    }
}

// Chunks of the streamed records, so that the workgroups fill the GPU's places in whole rounds: the
// fewest records in a row that any place works through, then the fewest chunks.
int pick_split(int64_t blocks, int64_t tiles, int per_cu, int multiple, int most) {
    const int64_t places = 256 * (int64_t)per_cu;
    int64_t best = -1;
    int pick = 1;
    for (int s = 1; s <= most; ++s) {
        int64_t per = (tiles + s - 1) / s;
        per = (per + multiple - 1) / multiple * multiple;
        if ((per * (s - 1)) >= tiles && s > 1) continue;  // an empty chunk
        const int64_t rounds = (blocks * s + places - 1) / places;
        const int64_t cost = rounds * (per + 2) + s / 16;  // a workgroup's start and end take about two records' time
        if (best < 0 || cost < best) {
            best = cost;
            pick = s;
        }
    }
    return pick;
}
int per_split(int64_t tiles, int split, int multiple) {
    const int64_t per = (tiles + split - 1) / split;
    return (int)((per + multiple - 1) / multiple * multiple);
}
constexpr int kBlockTiles = 4;  // records of a block of 128 classes

template <typename T, int P, bool BACK>
int prep(const XentProblem& x, const XentLayout& L, const Targets& tg, uint8_t* ws, hipStream_t st) {
    RecordArgs<T> r{static_cast<const T*>(x.a), static_cast<const T*>(x.w), x.bias, tg, x.lse, x.grad, x.m, x.n,
                    L.row_tiles, x.k, L.D, ws + (BACK ? L.b_row_rec : L.f_row_rec),
                    ws + (BACK ? L.b_class_rec : L.f_class_rec), reinterpret_cast<int*>(ws + L.b_row_u),
                    reinterpret_cast<int*>(ws + L.b_class_e)};
    const int list = 32 * x.tn;
    int size = 32;
    while (size < list) size *= 2;
    ListArgs<T> y{r.a, r.w, x.bias, tg, x.lse, x.grad, x.m, x.k, list, size, (int)((x.n + 127) / 128),
                  reinterpret_cast<uint32_t*>(ws + L.b_keys), reinterpret_cast<float*>(ws + L.b_vals),
                  reinterpret_cast<uint16_t*>(ws + L.b_offs)};
    const int64_t grid = L.row_tiles * (BACK ? 2 : 1) + L.class_tiles;
    prep_kernel<T, P, BACK><<<(unsigned)grid, kThreads, prep_lds(L.D, BACK ? size : 0), st>>>(r, y, (unsigned)L.class_tiles);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

template <int P>
int stats_pass(int D, const XentStatsArgs& s, unsigned grid, hipStream_t st) {
    switch (D) {
        case 1: return xent_stats_cfg<1, P>(s, grid, st);
        case 2: return xent_stats_cfg<2, P>(s, grid, st);
        case 3: return xent_stats_cfg<3, P>(s, grid, st);
        case 4: return xent_stats_cfg<4, P>(s, grid, st);
        case 6: return xent_stats_cfg<6, P>(s, grid, st);
        default: return xent_stats_cfg<8, P>(s, grid, st);
    }
}
template <int P, bool ROWS>
int grad_pass(int D, const XentGradArgs& s, unsigned grid, hipStream_t st) {
    switch (D) {
        case 1: return xent_grad_cfg<1, P, ROWS>(s, grid, st);
        case 2: return xent_grad_cfg<2, P, ROWS>(s, grid, st);
        case 3: return xent_grad_cfg<3, P, ROWS>(s, grid, st);
        case 4: return xent_grad_cfg<4, P, ROWS>(s, grid, st);
        case 6: return xent_grad_cfg<6, P, ROWS>(s, grid, st);
        default: return xent_grad_cfg<8, P, ROWS>(s, grid, st);
    }
}

Targets targets_of(const XentProblem& x) {
    return Targets{x.target, x.teacher_idx, x.teacher_z, x.tn, 1.0f / x.tau, x.n};
}

}  // namespace

XentLayout xent_layout(int64_t m, int64_t n, int64_t k, int tn, int planes) {
    XentLayout L{};
    L.D = xent_pieces(k);
    L.planes = planes;
    L.row_tiles = xent_tiles(m);
    L.class_tiles = xent_tiles(n);
    const int64_t frows = (m + xent_stats_rows(L.D, planes) - 1) / xent_stats_rows(L.D, planes),
                  arows = (m + kXentGradOwners - 1) / kXentGradOwners,
                  wrows = (n + kXentGradOwners - 1) / kXentGradOwners;
    L.fsplit = pick_split(frows, L.class_tiles, 2, 1, 128);
    const int occ = xent_grad_per_cu(L.D, planes);
    L.gsplit_a = pick_split(arows, L.class_tiles, occ, kBlockTiles, 64);
    L.gsplit_w = pick_split(wrows, L.row_tiles, occ, 1, 64);
    auto put = [](size_t* at, size_t bytes) {
        const size_t here = *at;
        *at += (bytes + 255) / 256 * 256;
        return here;
    };
    // a workspace may also serve the head's calls, whose list header its first bytes hold
    size_t f = 256;
    L.f_row_rec = put(&f, (size_t)L.row_tiles * xent_rec_bytes(L.D, planes, false));
    L.f_class_rec = put(&f, (size_t)L.class_tiles * xent_rec_bytes(L.D, planes, false));
    L.f_part = put(&f, (size_t)L.fsplit * m * sizeof(float2));
    L.f_total = f;
    size_t b = 256;
    L.b_row_rec = put(&b, (size_t)L.row_tiles * xent_rec_bytes(L.D, planes, true));
    L.b_class_rec = put(&b, (size_t)L.class_tiles * xent_rec_bytes(L.D, planes, true));
    L.b_row_u = put(&b, (size_t)L.row_tiles * 4);
    L.b_class_e = put(&b, (size_t)L.class_tiles * 4);
    L.b_keys = put(&b, (size_t)L.row_tiles * 32 * tn * 4);
    L.b_vals = put(&b, (size_t)L.row_tiles * 32 * tn * 4);
    L.b_offs = put(&b, (size_t)L.row_tiles * ((n + 127) / 128 + 1) * 2);
    const size_t pa = (size_t)L.gsplit_a * m * 32 * L.D * 4, pw = (size_t)L.gsplit_w * n * 32 * L.D * 4;
    L.b_part = put(&b, std::max(pa, pw));
    L.b_part_db = put(&b, (size_t)L.gsplit_w * n * 4);
    L.b_total = b;
    return L;
}

int launch_xent_forward(const XentProblem& x, float* loss, float* lse, uint8_t* ws, hipStream_t st) {
    const XentLayout L = xent_layout(x.m, x.n, x.k, x.tn, x.planes());
    const Targets tg = targets_of(x);
    if (int e = x.bf16 ? prep<uint16_t, 1, false>(x, L, tg, ws, st) : prep<float, 2, false>(x, L, tg, ws, st)) return e;
    float2* part = reinterpret_cast<float2*>(ws + L.f_part);
    const int per = per_split(L.class_tiles, L.fsplit, 1);
    XentStatsArgs s{ws + L.f_row_rec, ws + L.f_class_rec, x.m, L.class_tiles, L.fsplit, per, kLog2e / x.tau, part};
    const int rows = xent_stats_rows(L.D, L.planes);
    const unsigned grid = (unsigned)((x.m + rows - 1) / rows) * L.fsplit;
    if (int e = x.bf16 ? stats_pass<1>(L.D, s, grid, st) : stats_pass<2>(L.D, s, grid, st)) return e;
    const unsigned lg = (unsigned)((x.m + kThreads / 8 - 1) / (kThreads / 8));
    if (x.bf16)
        loss_kernel<uint16_t><<<lg, kThreads, 0, st>>>((const uint16_t*)x.a, (const uint16_t*)x.w, x.bias, tg, x.m, x.k,
                                                       L.fsplit, part, loss, lse);
    else
        loss_kernel<float><<<lg, kThreads, 0, st>>>((const float*)x.a, (const float*)x.w, x.bias, tg, x.m, x.k, L.fsplit,
                                                    part, loss, lse);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

static int sum_pass(const XentProblem& x, const float* part, int split, int64_t owners, int ld, void* out, const float* part_db,
                    float* db, hipStream_t st) {
    const unsigned grid = (unsigned)std::min<int64_t>((owners * x.k + kThreads - 1) / kThreads, 2048);
    if (x.bf16) sum_kernel<uint16_t><<<grid, kThreads, 0, st>>>(part, split, owners, x.k, ld, (uint16_t*)out, part_db, db);
    else sum_kernel<float><<<grid, kThreads, 0, st>>>(part, split, owners, x.k, ld, (float*)out, part_db, db);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

int launch_xent_zero(const XentProblem& x, void* dw, float* db, hipStream_t st) {
    return dw || db ? sum_pass(x, nullptr, 0, x.n, 0, dw, nullptr, db, st) : PPOCR_OK;
}

int launch_xent_backward(const XentProblem& x, void* da, void* dw, float* db, uint8_t* ws, hipStream_t st) {
    const XentLayout L = xent_layout(x.m, x.n, x.k, x.tn, x.planes());
    const Targets tg = targets_of(x);
    if (int e = x.bf16 ? prep<uint16_t, 1, true>(x, L, tg, ws, st) : prep<float, 2, true>(x, L, tg, ws, st)) return e;
    float* part = reinterpret_cast<float*>(ws + L.b_part);
    float* part_db = reinterpret_cast<float*>(ws + L.b_part_db);
    const int blocks = (int)((x.n + 127) / 128);
    auto pass = [&](bool rows) -> int {
        const int64_t owners = rows ? x.m : x.n, own_tiles = rows ? L.row_tiles : L.class_tiles,
                      str_tiles = rows ? L.class_tiles : L.row_tiles;
        const int split = rows ? L.gsplit_a : L.gsplit_w;
        const uint8_t* rr = ws + L.b_row_rec;
        const uint8_t* cr = ws + L.b_class_rec;
        XentGradArgs s{rows ? rr : cr, rows ? cr : rr, owners, own_tiles, str_tiles,
                       reinterpret_cast<const int*>(ws + (rows ? L.b_class_e : L.b_row_u)), split,
                       per_split(str_tiles, split, rows ? kBlockTiles : 1), kLog2e / x.tau,
                       reinterpret_cast<const uint32_t*>(ws + L.b_keys), reinterpret_cast<const float*>(ws + L.b_vals),
                       reinterpret_cast<const uint16_t*>(ws + L.b_offs), 32 * x.tn, blocks, part,
                       rows ? nullptr : part_db};
        const unsigned grid = (unsigned)((owners + kXentGradOwners - 1) / kXentGradOwners) * split;
        int e;
        if (rows) e = x.bf16 ? grad_pass<1, true>(L.D, s, grid, st) : grad_pass<2, true>(L.D, s, grid, st);
        else e = x.bf16 ? grad_pass<1, false>(L.D, s, grid, st) : grad_pass<2, false>(L.D, s, grid, st);
        if (e) return e;
        if (int e2 = sum_pass(x, part, split, owners, 32 * L.D, rows ? da : dw, part_db, rows ? nullptr : db, st)) return e2;
        return PPOCR_OK;
    };
    if (da)
        if (int e = pass(true)) return e;
    if (dw || db)
        if (int e = pass(false)) return e;
    return PPOCR_OK;
}

}  // namespace ppocr
