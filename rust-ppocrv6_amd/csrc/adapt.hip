// Low-rank adapters of many text lines beside the shared vocabulary projection:
//
//   z[r][j] = scale[j] (sum_c a[r][c] q[j][c]) + bias[j] + s (down a[r])[.] . up[j][.]
//
// with the adapter (down [rank][k], up [n][rank], s) of the slot that row r's line names, or none.  The head's
// weights are read once for rows of all adapters; only the rank products differ.
//
// Matrix bound at the head's own rate: 2 n k operations a row, of which an adapter of rank 16 adds 13%.
// Rows are put in order by slot (plan_kernel) and padded to units of 32, so that a wave's rows have one
// adapter; the four waves of a workgroup, each with a unit of its own, share the head's weight tiles through
// LDS, and each wave reads its adapter's tile from L2.  30720 rows of an INT8 head under 64 adapters of rank 32:
// 368 us in the statistics kernel, 386 GFLOP of halves at 1.05 PFLOP/s, the matrix units busy for 57% of them at 1.81 GHz
// (the head's own pass: 58%).  The plan before it takes 9 us, the join of the chunks behind it 8.
//
// Arithmetic: fp16 halves of both operands (22 bits), as the head's F16X2 mode, all in one fp32 accumulator: up is
// held divided by the class's unit (its scale, or where a head's lie far apart that times a power of two; of an FP32
// head a power of two above the class's weights).  Each row is scaled by the power of two that its largest value sets,
// so rows of any size keep their bits, whatever the rows beside them hold, and no row has to be computed again.  u =
// down a is computed by each wave before its first tile, from the rows it holds; the products' layout is that of the
// operand that the next product needs.
#include <algorithm>
#include <cmath>

#include "adapt.hpp"
#include "head_mfma.hpp"

namespace ppocr {

size_t Adapters::down_bytes() const { return (size_t)((steps + 1) / 2) * (2 * (size_t)G * 512 + 1024); }
size_t Adapters::up_bytes() const { return (size_t)tiles * 2 * steps * 1024; }

namespace {

constexpr int kWaves = 4;
constexpr int kDownShift = 10;  // down's halves are held 2^10 up: their low ones stay normal numbers
constexpr int kTop = 15;        // rows, and u, stay below 2^15
constexpr int kMostShift = 60;

// ---------------------------------------------------------------- setting a slot
__global__ __launch_bounds__(256) void clear_kernel(u32x4* p, int64_t count) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) p[i] = u32x4{0, 0, 0, 0};
}
__global__ void clear_meta_kernel(AdapterMeta* meta, int count) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < count; i += gridDim.x * blockDim.x) meta[i] = AdapterMeta{0};
}

template <typename T>
__device__ __forceinline__ float value(T v);
template <>
__device__ __forceinline__ float value<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float value<uint16_t>(uint16_t v) {
    return __uint_as_float((unsigned)v << 16);
}

// range[0][t]: the sum of |down[t]|; range[1][t]: cleared.
template <typename T>
__global__ __launch_bounds__(64) void down_range_kernel(const T* __restrict__ down, int rank, int k, unsigned* range) {
    const int t = blockIdx.x;
    float s = 0.0f;
    if (t < rank)
        for (int c = threadIdx.x; c < k; c += 64) s += __builtin_fabsf(value<T>(down[(int64_t)t * k + c]));
    s = wave_sum(s);
    if (threadIdx.x == 0) {
        range[t] = __float_as_uint(s);
        range[kAdaptMostRank + t] = 0u;
    }
}

// The value that the up records hold before their power of two.
__device__ __forceinline__ float up_value(float v, float scale, float unit) { return v * scale / unit; }

// range[1][t]: the largest |up[.][t]| over its class's unit (maxima of non-negative bits: any order gives the
// same).
template <typename T>
__global__ __launch_bounds__(256) void up_range_kernel(const T* __restrict__ up, int rank, float scale,
                                                       const float* __restrict__ unit, int64_t n, unsigned* range) {
    __shared__ unsigned top[kAdaptMostRank];
    if (threadIdx.x < kAdaptMostRank) top[threadIdx.x] = 0u;
    __syncthreads();
    const int64_t count = n * rank;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < count; x += (int64_t)gridDim.x * 256) {
        const int64_t j = x / rank;
        const float v = __builtin_fabsf(up_value(value<T>(up[x]), scale, unit[j]));
        if (v < INFINITY) atomicMax(&top[x - j * rank], __float_as_uint(v));
    }
    __syncthreads();
    if ((int)threadIdx.x < rank) atomicMax(&range[kAdaptMostRank + threadIdx.x], top[threadIdx.x]);
}

// Power of two above |down[t]|'s sum (1 where it is 0 or no finite number).
__device__ __forceinline__ int down_exp(const unsigned* range, int t) {
    const float s = __uint_as_float(range[t]);
    return s > 0.0f && s < INFINITY ? ilogbf(s) + 1 : 0;
}
// How far the head's products are scaled down beside the adapter's, so that the largest up value fits fp16: 0
// unless the adapter's largest products are 2^7 above the head's.
__device__ __forceinline__ int slot_shift(const unsigned* range, int rank) {
    int s = 0;
    for (int t = 0; t < rank; ++t) {
        const float b = __uint_as_float(range[kAdaptMostRank + t]);
        if (b > 0.0f) s = max(s, ilogbf(b) + 1 + down_exp(range, t) - (kTop - 1));
    }
    return min(s, kMostShift);
}

__device__ __forceinline__ unsigned short half_bits(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

// down record: per 32 ranks, as an FP32 head's tile (Geo<CFG_HF3, G>): [half][group][rank][8].
template <typename T>
__global__ __launch_bounds__(256) void down_record_kernel(const T* __restrict__ down, int rank, int k, int G, int steps,
                                                          const unsigned* __restrict__ range, uint8_t* rec, AdapterMeta* meta) {
    const int blocks = (steps + 1) / 2;
    const size_t stride = 2 * (size_t)G * 512 + 1024;
    for (int x = blockIdx.x * 256 + threadIdx.x; x < blocks * 32 * G * 8; x += gridDim.x * 256) {
        const int e = x % 8, i = x / 8 % 32, g = x / 256 % G, b = x / (256 * G);
        const int t = 32 * b + i, c = 8 * g + e;
        const float v = t < rank && c < k ? ldexpf(value<T>(down[(int64_t)t * k + c]), kDownShift - down_exp(range, t)) : 0.0f;
        unsigned short* p = reinterpret_cast<unsigned short*>(rec + b * stride);
        const unsigned short hi = half_bits(v);
        p[(g * 32 + i) * 8 + e] = hi;
        p[((G + g) * 32 + i) * 8 + e] = half_bits(v - (float)__builtin_bit_cast(_Float16, hi));
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) *meta = AdapterMeta{slot_shift(range, rank)};
}

// The rank that element e of lane half h holds in 16-rank step s of an operand: the order in which
// u = down a leaves the matrix unit (register r of a lane is row 8 (r / 4) + 4 h + r % 4).
__device__ __forceinline__ int rank_of(int s, int h, int e) { return 32 * (s >> 1) + 8 * (2 * (s & 1) + (e >> 2)) + 4 * h + (e & 3); }

// up record of a 32-class tile: [half][step][h][class][8].
template <typename T>
__global__ __launch_bounds__(256) void up_record_kernel(const T* __restrict__ up, int rank, float scale,
                                                        const float* __restrict__ unit, int64_t n, int steps,
                                                        const unsigned* __restrict__ range, uint8_t* rec) {
    __shared__ int exps[kAdaptMostRank];
    if (threadIdx.x < kAdaptMostRank) exps[threadIdx.x] = (int)threadIdx.x < rank ? down_exp(range, threadIdx.x) : 0;
    __shared__ int shift;
    if (threadIdx.x == 0) shift = slot_shift(range, rank);
    __syncthreads();
    const int per = steps * 512;  // values of a tile
    unsigned short* p = reinterpret_cast<unsigned short*>(rec) + (size_t)blockIdx.x * 2 * per;
    for (int x = threadIdx.x; x < per; x += 256) {
        const int e = x % 8, i = x / 8 % 32, h = x / 256 % 2, s = x / 512;
        const int t = rank_of(s, h, e);
        const int64_t j = (int64_t)blockIdx.x * 32 + i;
        float v = 0.0f;
        if (t < rank && j < n) v = ldexpf(up_value(value<T>(up[j * rank + t]), scale, unit[j]), exps[t] - shift);
        const unsigned short hi = half_bits(v);
        p[x] = hi;
        p[per + x] = half_bits(v - (float)__builtin_bit_cast(_Float16, hi));
    }
}

template <typename T>
int set_slot(const Adapters& ad, int slot, const T* down, const T* up, int rank, float scale, int64_t n, int64_t k,
             hipStream_t st) {
    unsigned* range = ad.range + (size_t)slot * 2 * kAdaptMostRank;
    down_range_kernel<T><<<kAdaptMostRank, 64, 0, st>>>(down, rank, (int)k, range);
    PPOCR_HIP(hipGetLastError());
    if (rank) {
        const unsigned grid = (unsigned)std::min<int64_t>((n * rank + 1023) / 1024, 1024);
        up_range_kernel<T><<<grid, 256, 0, st>>>(up, rank, scale, ad.unit, n, range);
        PPOCR_HIP(hipGetLastError());
    }
    down_record_kernel<T><<<16, 256, 0, st>>>(down, rank, (int)k, ad.G, ad.steps, range, ad.down + slot * ad.down_bytes(),
                                              ad.meta + slot);
    PPOCR_HIP(hipGetLastError());
    up_record_kernel<T><<<(unsigned)ad.tiles, 256, 0, st>>>(up, rank, scale, ad.unit, n, ad.steps, range,
                                                            ad.up + slot * ad.up_bytes());
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

// ---------------------------------------------------------------- rows in order of their slots
// Plan of a call: rows[units][unit], unit = 32 or 64 rows of a wave, the slot of each unit, the number of units.  Places
// that the last unit of a slot has no row for repeat the slot's first row: it is computed, and its results written,
// again, which are the same bits.
// A single line needs no lists: its rows are one run, the rows of no line before and behind it another.
struct Plan {
    int* units;
    int* rows;
    int* slot;
    const int64_t* one_off;  // a single line: its offsets and slot, the lists unused
    const int32_t* one_slot;
};
int64_t plan_units(int64_t m, int64_t groups, int unit) { return m / unit + groups; }

// One workgroup.  Rows of a group are placed in any order: no row's result depends on its place.  Rows of no
// line, and of lines that name no slot, form a group of their own.
//
// Where the offsets rise, whole lines are counted and placed (a wave a line, or a thread a line where they are
// short; the rows before the first and behind the last line are two lines more); the first kSpans are kept in LDS
// between the two.  Otherwise each row looks for its line, the last whose offset is not above it, so that each is
// placed once whatever the offsets hold.  Latency bound: 256 lines of 120 9 us (by rows 95), of which most is three
// memory round trips.
constexpr int kSpans = 1024;
struct Span {
    int lo, hi, g;
};
__global__ __launch_bounds__(1024) void plan_kernel(AdaptLines lines, int m, int slots, int unit, Plan plan) {
    extern __shared__ int groups[];
    __shared__ Span kept[kSpans];
    int* count = groups;                // [slots + 1] rows of a group
    int* some = groups + slots + 1;     // a row of it
    int* start = some + slots + 1;      // its first place
    int* cursor = start + slots + 1;    // its next place
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto group_of_line = [&](int64_t i) -> int {
        const int s = lines.slot[i];
        return s >= 0 && s < slots ? s : slots;
    };
    // Line i of lines.lines + 2; no rows where its offsets do not rise within [0, m].
    auto span = [&](int64_t i, bool& ok) {
        if (lines.lines == 0) return Span{0, i == 0 ? m : 0, slots};
        const bool inner = i < lines.lines;
        const int64_t a = i == lines.lines ? 0 : lines.off[inner ? i : lines.lines];
        const int64_t b = inner ? lines.off[i + 1] : i == lines.lines ? lines.off[0] : m;
        const bool good = a >= 0 && a <= b && b <= m;
        ok &= good;
        return Span{good ? (int)a : 0, good ? (int)b : 0, inner ? group_of_line(i) : slots};
    };
    const int64_t spans = lines.lines + 2;
    bool rising = true;
    for (int64_t i = tid; i < spans; i += 1024) {
        const Span s = span(i, rising);
        if (i < kSpans) kept[i] = s;
    }
    for (int g = tid; g <= slots; g += 1024) count[g] = some[g] = 0;
    rising = __syncthreads_and(rising);
    auto span_again = [&](int64_t i) {
        bool ok = true;
        return i < kSpans ? kept[i] : span(i, ok);
    };
    auto group_of = [&](int r) -> int {
        int64_t lo = 0, hi = lines.lines;  // off[lo] <= r < off[hi], if offsets rise
        if (hi == 0 || lines.off[0] > r) return slots;
        while (hi - lo > 1) {
            const int64_t mid = (lo + hi) >> 1;
            if (lines.off[mid] <= r) lo = mid;
            else hi = mid;
        }
        if (lines.off[lo + 1] <= r) return slots;
        return group_of_line(lo);
    };
    // a count of its group for each lane's row: lanes of one group together where the wave's rows all have it
    auto take = [&](int* counts, bool on, int g) -> int {
        const unsigned long long mask = __ballot(on);
        if (mask == 0ull) return 0;
        const int leader = __ffsll((long long)mask) - 1;
        const int g0 = __shfl(g, leader, 64);
        if (__ballot(on && g != g0) == 0ull) {
            int base = 0;
            if (lane == leader) base = atomicAdd(&counts[g0], __popcll(mask));
            return __shfl(base, leader, 64) + __popcll(mask & ((1ull << lane) - 1ull));
        }
        return on ? atomicAdd(&counts[g], 1) : 0;
    };
    if (rising) {
        for (int64_t i = tid; i < spans; i += 1024) {
            const Span s = span_again(i);
            if (s.hi > s.lo) {
                atomicAdd(&count[s.g], s.hi - s.lo);
                some[s.g] = s.lo;  // any of them
            }
        }
    } else {
        for (int r0 = 0; r0 < m; r0 += 1024) {
            const int r = r0 + tid, g = r < m ? group_of(r) : 0;
            (void)take(count, r < m, g);
            if (r < m) some[g] = r;
        }
    }
    __syncthreads();
    if (tid < 64) {
        int before = 0;
        for (int g0 = 0; g0 <= slots; g0 += 64) {
            const int g = g0 + lane;
            const int mine = g <= slots ? (count[g] + unit - 1) / unit : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(upto, o, 64);
                if (lane >= o) upto += v;
            }
            if (g <= slots) start[g] = cursor[g] = (before + upto - mine) * unit;
            before += __shfl(upto, 63, 64);
        }
        if (lane == 0) *plan.units = before;
    }
    __syncthreads();
    // the units' slots, and the places that the last unit of a group has no row for
    for (int g = tid; g <= slots; g += 1024) {
        const int n = count[g], first = start[g] / unit;
        for (int u = 0; u * unit < n; ++u) plan.slot[first + u] = g;
        for (int x = n; x % unit; ++x) plan.rows[start[g] + x] = some[g];
    }
    if (rising) {
        // a thread a line where they are short, a wave where they are not
        const int most = m / max(lines.lines, (int64_t)1) < 16 ? 1024 : 0;
        if (most)
            for (int64_t i = tid; i < spans; i += 1024) {
                const Span s = span_again(i);
                if (s.hi <= s.lo || s.hi - s.lo >= most) continue;
                int* to = plan.rows + atomicAdd(&cursor[s.g], s.hi - s.lo);
                for (int r = s.lo; r < s.hi; ++r) to[r - s.lo] = r;
            }
        for (int64_t i = wave; i < spans; i += 16) {
            const Span s = span_again(i);
            if (s.hi <= s.lo || s.hi - s.lo < most) continue;
            int at = 0;
            if (lane == 0) at = atomicAdd(&cursor[s.g], s.hi - s.lo);
            int* to = plan.rows + __shfl(at, 0, 64);
            for (int r = s.lo + lane; r < s.hi; r += 64) to[r - s.lo] = r;
        }
    } else {
        for (int r0 = 0; r0 < m; r0 += 1024) {
            const int r = r0 + tid;
            const int at = take(cursor, r < m, r < m ? group_of(r) : 0);
            if (r < m) plan.rows[at] = r;
        }
    }
}

// The plan as the kernels read it, for units of U rows.
template <int U>
struct PlanView {
    const Plan& plan;
    int m, slots, units;
    int lo = 0, len = 0, first = 0;  // a single line: its rows, and the units they take
    __device__ __forceinline__ PlanView(const Plan& p, int64_t rows, int slot_count) : plan(p), m((int)rows), slots(slot_count) {
        if (p.one_off) {
            const int64_t b = p.one_off[0], e = p.one_off[1];
            lo = (int)min(max(b, (int64_t)0), rows);
            len = (int)max(min(max(e, (int64_t)0), rows) - lo, (int64_t)0);
            first = (len + U - 1) / U;
            units = first + (m - len + U - 1) / U;
        } else {
            units = *p.units;
        }
    }
    __device__ __forceinline__ int slot_of(int unit) const {
        if (!plan.one_off) return plan.slot[unit];
        const int s = *plan.one_slot;
        return unit < first && s >= 0 && s < slots ? s : slots;
    }
    // row `i` of a unit; places past the rows repeat one of them
    __device__ __forceinline__ int row_of(int unit, int i) const {
        if (!plan.one_off) return plan.rows[unit * U + i];
        if (unit < first) return lo + min(unit * U + i, len - 1);
        const int k = min((unit - first) * U + i, m - len - 1);
        return k < lo ? k : k + len;
    }
};

// ---------------------------------------------------------------- rows and their u in registers
struct AdaptLaunch {
    const float* a;
    int64_t m;
    int k, vec;
    const uint8_t* rec;
    int tiles, n, nsplit, tpc, mblocks;
    Plan plan;
    int slots;
    const uint8_t* down;
    size_t down_stride;
    const uint8_t* up;
    size_t up_stride;
    const AdapterMeta* meta;
    Partial* part;
    float* out;
};

template <int C, int G, int NR>
struct RowOperands {
    u16x8 a[Geo<C, G>::S];
    u16x8 uhi[NR], ulo[NR];
    float inv;    // the row's power of two undone
    bool scaled;  // some row of the wave has one
};

// Row `row` (its lane's of 32) scaled, split, and multiplied with its adapter's down.
template <int C, int G, int NR>
__device__ __forceinline__ void load_rows(const AdaptLaunch& x, int64_t row, int slot, int i, int h, RowOperands<C, G, NR>& o) {
    using A = ActPlan<C, G>;
    using D = ActPlan<CFG_HF3, G>;
    static_assert(A::NL == D::NL, "both products read the rows in the same pieces");
    float raw[A::NL][8];
    act_issue<C, G>(x.a, row, x.k, x.vec, h, raw);
    const int shift = x.meta[slot].shift;
    float top = 0.0f;
    bool odd = false;
#pragma unroll
    for (int l = 0; l < A::NL; ++l)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            top = fmaxf(top, __builtin_fabsf(raw[l][e]));
            odd |= !(__builtin_fabsf(raw[l][e]) < INFINITY);
        }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    odd |= (bool)__shfl_xor((int)odd, 32, 64);
    // The row's largest value comes to below 2^kTop, in the head's products 2^-shift of it.  A row whose largest
    // value lies in [0.5, 2^kTop) is left as it is, whatever the rows beside it need, so that its bits do not depend on
    // them: the low halves, whose smallest step is 2^-24, then still hold 24 bits of that value.  Where that goes for
    // all of a wave's rows, no logit needs the power undone.
    const bool fits = shift == 0 && top >= 0.5f && top < (float)(1 << kTop);
    o.scaled = __any(!fits);
    int ex = 0;
    if (!fits && top > 0.0f && !odd) ex = max(min(kTop - 1 - ilogbf(top), 126), shift - 126);
    o.inv = ldexpf(1.0f, shift - ex);
    const float to = ldexpf(1.0f, ex), lower = ldexpf(1.0f, -shift);
#pragma unroll
    for (int l = 0; l < A::NL; ++l)
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[l][e] *= to;
    float none = 0.0f, none2 = 0.0f;
    {
        u16x8 d[Geo<CFG_HF3, G>::S];
        act_split_all<CFG_HF3, G>(raw, h, d, none, none2);
        const uint8_t* rec = x.down + (size_t)slot * x.down_stride;
#pragma unroll
        for (int b = 0; b < (NR + 1) / 2; ++b) {
            f32x16 u = {};
#pragma unroll
            for (int s = 0; s < Geo<CFG_HF3, G>::S; ++s)
                u = mfma16<true>(weight_frag<CFG_HF3, G>(rec + b * (2 * G * 512 + 1024), s, i * 16 + h * 512, i * 16, h), d[s], u);
#pragma unroll
            for (int y = 0; y < 2 && 2 * b + y < NR; ++y)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = u[8 * y + e] * (1.0f / (1 << kDownShift));
                    o.uhi[2 * b + y][e] = split_term<true>(v, 0);
                    o.ulo[2 * b + y][e] = split_term<true>(v, 1);
                }
        }
    }
#pragma unroll
    for (int l = 0; l < A::NL; ++l)
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[l][e] *= lower;
    act_split_all<C, G>(raw, h, o.a, none, none2);
}

// The adapter's fragments of a class tile: NR steps, both halves.
template <int NR>
__device__ __forceinline__ void load_up(const uint8_t* up, int tile, int lane, u16x8 (&hi)[NR], u16x8 (&lo)[NR]) {
    const u16x8* p = reinterpret_cast<const u16x8*>(up + (size_t)tile * (2 * NR * 1024)) + lane;
#pragma unroll
    for (int s = 0; s < NR; ++s) {
        hi[s] = p[s * 64];
        lo[s] = p[(NR + s) * 64];
    }
}

// ---------------------------------------------------------------- statistics
// A wave takes MB blocks of 32 rows (columns of the matrix product) of one slot, 32 classes a tile; the head's
// tiles go through a ring in LDS as in the head's statistics pass, the products of tile j + 1 interleaved with the
// epilogue of tile j.  PLAIN: the rows have no powers of two, and the sums no reference (no logit beyond 2^64 so far): a
// multiplication and a subtraction less for each logit.
template <int P, int MB, bool PLAIN>
__device__ __forceinline__ void adapt_piece(f32x16 (&t)[MB], const float (&inv)[MB], const float* __restrict__ ep, int h, int j,
                                            f32x4 (&cs)[2], f32x4 (&cb)[2], const float (&ref)[MB], float (&best)[MB],
                                            int (&bt)[MB], f32x4* save, EpiState<MB>& st) {
    if constexpr (!PLAIN && P < 12 * MB && P % (3 * MB) < MB) {
        constexpr int b = P % (3 * MB), q = P / (3 * MB);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[b][4 * q + e] *= inv[b];
    }
    epi_piece<P, MB, PLAIN>(t, ep, h, j, cs, cb, ref, best, bt, save, st);
    if constexpr (PLAIN && P == epi_pieces<MB>() - 1) {
#pragma unroll
        for (int b = 0; b < MB; ++b) st.need = st.need | ((best[b] != -INFINITY) & (__builtin_fabsf(best[b]) > 64.0f));
    }
}
template <int H, int x, int MB, bool PLAIN>
__device__ __forceinline__ void adapt_pieces(f32x16 (&t)[MB], const float (&inv)[MB], const float* __restrict__ ep, int h, int j,
                                             f32x4 (&cs)[2], f32x4 (&cb)[2], const float (&ref)[MB], float (&best)[MB],
                                             int (&bt)[MB], f32x4* save, EpiState<MB>& st) {
    constexpr int NP = epi_pieces<MB>();
    constexpr int p0 = x * NP / H, p1 = (x + 1) * NP / H;
    [&]<int... I>(std::integer_sequence<int, I...>) {
        (adapt_piece<p0 + I, MB, PLAIN>(t, inv, ep, h, j, cs, cb, ref, best, bt, save, st), ...);
    }(std::make_integer_sequence<int, p1 - p0>{});
}

constexpr int kAhead = 4;  // MFMA steps that a weight fragment is read ahead of its use

template <int C, int G, int NR, int MB, int OCC>
__global__ __launch_bounds__(64 * kWaves, OCC) void adapt_stats_kernel(AdaptLaunch x) {
    using GE = Geo<C, G>;
    constexpr int S = GE::S, NT = 64 * kWaves, UNIT = 32 * MB;
    constexpr int AHEAD = OCC == 1 ? kAhead : kPrefetch;
    extern __shared__ __align__(16) uint8_t lds[];
    int mbi, chunk;
    map_block<true>(blockIdx.x, x.nsplit, &mbi, &chunk);
    const PlanView<UNIT> plan(x.plan, x.m, x.slots);
    if (mbi * kWaves >= plan.units || chunk >= x.nsplit) return;
    const int t0 = chunk * x.tpc, t1 = min(t0 + x.tpc, x.tiles);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 31, h = lane >> 5;
    if (tid < 32 * kRing) reinterpret_cast<u32x4*>(lds + (tid >> 5) * GE::BUF + GE::REC)[tid & 31] = u32x4{0, 0, 0, 0};
    const int lb = i * 16 + h * 512;
    f32x4* save = reinterpret_cast<f32x4*>(lds + kRing * GE::BUF) + wave * (MB * 4 * 64) + lane;
    constexpr int kOps = stage_direct_min_ops<GE::REC, NT>();
    if (t0 < t1) {
#pragma unroll
        for (int y = 0; y < kRing - 1; ++y)
            stage_direct<GE::REC, NT>(x.rec + (size_t)min(t0 + y, t1 - 1) * GE::REC, lds + y * GE::BUF, tid);
    }
    const int unit = mbi * kWaves + wave;
    const bool live = unit < plan.units;
    const int slot = __builtin_amdgcn_readfirstlane(live ? plan.slot_of(unit) : x.slots);
    const uint8_t* up = x.up + (size_t)slot * x.up_stride;
    int row[MB];
    RowOperands<C, G, NR> o[MB];
    float inv[MB];
    bool plain = true;  // the same for the wave
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        row[b] = live ? plan.row_of(unit, 32 * b + i) : 0;
        load_rows<C, G, NR>(x, row[b], slot, i, h, o[b]);
        inv[b] = o[b].inv;
        plain = plain && !o[b].scaled;
    }

    float best[MB], ref[MB], sum[MB];
    int bt[MB];
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        best[b] = -INFINITY;
        ref[b] = sum[b] = 0.0f;
        bt[b] = -1;
    }
    // the loads of the newest staged tile may still be in flight at a barrier
    constexpr int kLead = (kRing - 3) * kOps;
    if (t0 < t1) {
        u16x8 whi[NR], wlo[NR];
        load_up<NR>(up, t0, lane, whi, wlo);
        ring_barrier<kLead>();  // tiles t0 and t0 + 1 are in LDS
        f32x16 acc_a[MB], acc_b[MB];
#pragma unroll
        for (int b = 0; b < MB; ++b) {
            acc_a[b] = f32x16{};
#pragma unroll
            for (int s = 0; s < NR; ++s) {
                acc_a[b] = mfma16<true>(whi[s], o[b].uhi[s], acc_a[b]);
                acc_a[b] = mfma16<true>(whi[s], o[b].ulo[s], acc_a[b]);
                acc_a[b] = mfma16<true>(wlo[s], o[b].uhi[s], acc_a[b]);
            }
        }
        load_up<NR>(up, min(t0 + 1, t1 - 1), lane, whi, wlo);
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const u16x8 wf = weight_frag<C, G>(lds, s, lb, i * 16, h);
#pragma unroll
            for (int b = 0; b < MB; ++b) acc_a[b] = mfma16<true>(wf, o[b].a[s], acc_a[b]);
        }
        auto step_as = [&]<int R, bool PLAIN>(int j, f32x16 (&accE)[MB], f32x16 (&accM)[MB]) __attribute__((always_inline)) {
            constexpr unsigned rel = (unsigned)R;  // (j - t0) % kRing
            const uint8_t* bufn = lds + ((rel + 1) & (kRing - 1)) * GE::BUF;
            const float* ep = reinterpret_cast<const float*>(lds + (rel & (kRing - 1)) * GE::BUF + GE::FRAG);
            f32x4 cs[2], cb[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                cs[q] = *reinterpret_cast<const f32x4*>(ep + 8 * q + 4 * h);
                cb[q] = *reinterpret_cast<const f32x4*>(ep + 32 + 8 * q + 4 * h);
            }
            EpiState<MB> st;
            st.need = false;
#pragma unroll
            for (int b = 0; b < MB; ++b) accM[b] = f32x16{};
            // products 0 .. 3 NR - 1: the adapter's, the rest the head's; the epilogue's pieces between them all
            constexpr int STEPS = S + 3 * NR;
            u16x8 wq[AHEAD];
            frag_prefetch_first<C, G, AHEAD>(wq, bufn, lb, i * 16, h);
            [&]<int... s>(std::integer_sequence<int, s...>) {
                ([&] {
                    constexpr int r = s / 3, y = s % 3;
                    const u16x8& wf = y == 2 ? wlo[r] : whi[r];
                    accM[0] = mfma16<true>(wf, y == 1 ? o[0].ulo[r] : o[0].uhi[r], accM[0]);
                    __builtin_amdgcn_sched_barrier(0);
                    adapt_pieces<2 * STEPS, 2 * s, MB, PLAIN>(accE, inv, ep, h, j, cs, cb, ref, best, bt, save, st);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int b = 1; b < MB; ++b) accM[b] = mfma16<true>(wf, y == 1 ? o[b].ulo[r] : o[b].uhi[r], accM[b]);
                    __builtin_amdgcn_sched_barrier(0);
                    adapt_pieces<2 * STEPS, 2 * s + 1, MB, PLAIN>(accE, inv, ep, h, j, cs, cb, ref, best, bt, save, st);
                    __builtin_amdgcn_sched_barrier(0);
                }(), ...);
            }(std::make_integer_sequence<int, 3 * NR>{});
            // The adapter's operands' registers take the next tile's, which has the rest of the step to arrive.  Those
            // loads are issued before the staged ones: the barrier's count of loads in flight stays that of the staged.
            load_up<NR>(up, min(j + 2, t1 - 1), lane, whi, wlo);
            stage_direct<GE::REC, NT>(x.rec + (size_t)min(j + kRing - 1, t1 - 1) * GE::REC,
                                      lds + ((rel + kRing - 1) & (kRing - 1)) * GE::BUF, tid);
            [&]<int... s>(std::integer_sequence<int, s...>) {
                ([&] {
                    constexpr int g = s + 3 * NR;
                    const u16x8& wf = frag_of<C, G, AHEAD, s>(wq);
                    accM[0] = mfma16<true>(wf, o[0].a[s], accM[0]);
                    __builtin_amdgcn_sched_barrier(0);
                    adapt_pieces<2 * STEPS, 2 * g, MB, PLAIN>(accE, inv, ep, h, j, cs, cb, ref, best, bt, save, st);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int b = 1; b < MB; ++b) accM[b] = mfma16<true>(wf, o[b].a[s], accM[b]);
                    frag_prefetch_after<C, G, AHEAD, s>(wq, bufn, lb, i * 16, h);
                    __builtin_amdgcn_sched_barrier(0);
                    adapt_pieces<2 * STEPS, 2 * g + 1, MB, PLAIN>(accE, inv, ep, h, j, cs, cb, ref, best, bt, save, st);
                    __builtin_amdgcn_sched_barrier(0);
                }(), ...);
            }(std::make_integer_sequence<int, S>{});
            if (__any(st.need)) {
                plain = false;
#pragma unroll
                for (int b = 0; b < MB; ++b)
                    if (best[b] != -INFINITY && __builtin_fabsf(best[b] - ref[b]) > 64.0f) {
                        const float nr = best[b];
                        sum[b] = (sum[b] == 0.0f) ? 0.0f : sum[b] * __builtin_amdgcn_exp2f(ref[b] - nr);
                        float v = 0.0f;
#pragma unroll
                        for (int r = 0; r < 16; ++r) v += __builtin_amdgcn_exp2f(accE[b][r] - nr);
                        st.tsum[b] = v;
                        ref[b] = nr;
                    }
            }
#pragma unroll
            for (int b = 0; b < MB; ++b) sum[b] += st.tsum[b];
            ring_barrier<kLead>();
        };
        auto step_of = [&]<int R>(int jj) __attribute__((always_inline)) {
            auto both = [&](f32x16 (&accE)[MB], f32x16 (&accM)[MB]) __attribute__((always_inline)) {
                if (plain) step_as.template operator()<R, true>(jj, accE, accM);
                else step_as.template operator()<R, false>(jj, accE, accM);
            };
            if constexpr (R % 2 == 0) both(acc_a, acc_b);
            else both(acc_b, acc_a);
        };
        int j = t0;
        for (; j + kRing - 1 < t1; j += kRing)
            [&]<int... R>(std::integer_sequence<int, R...>) {
                (step_of.template operator()<R>(j + R), ...);
            }(std::make_integer_sequence<int, kRing>{});
        [&]<int... R>(std::integer_sequence<int, R...>) {
            ((j + R < t1 ? step_of.template operator()<R>(j + R) : void()), ...);
        }(std::make_integer_sequence<int, kRing - 1>{});
        // the ring's last loads (repeats of the last tile) land before the workgroup ends
        vm_wait<0>();
    }

#pragma unroll
    for (int b = 0; b < MB; ++b) {
        int cls = 0;
        if (bt[b] >= 0) {
            int r0 = 16;
#pragma unroll
            for (int q = 3; q >= 0; --q) {
                const f32x4 v = save[(b * 4 + q) * 64];
#pragma unroll
                for (int e = 3; e >= 0; --e) r0 = (v[e] == best[b]) ? 4 * q + e : r0;
            }
            cls = bt[b] * 32 + (r0 < 16 ? 8 * (r0 >> 2) + 4 * h + (r0 & 3) : 0);
        }
        const RowStat mine{best[b], sum[b], ref[b], cls};
        const RowStat other{__shfl_xor(best[b], 32, 64), __shfl_xor(sum[b], 32, 64), __shfl_xor(ref[b], 32, 64),
                            __shfl_xor(cls, 32, 64)};
        const RowStat r = stat_merge(mine, other);
        if (h == 0 && live) x.part[(int64_t)chunk * x.m + row[b]] = Partial{r.best, r.sum, r.idx};
    }
}

// ---------------------------------------------------------------- logits
// Rows of the matrix product are the activation rows, columns the classes, so that a store writes 32
// consecutive classes of two rows.  Four waves multiply and store, one on a SIMD; a producer wave keeps a ring of
// tiles in LDS filled, the head's and those of the adapters of the workgroup's units.  The four load nothing: a
// wave's memory operations end in order, so that one which loaded its adapter's tiles itself waited for its own
// stores with them.  More waves on a CU write more pieces of rows at once and slower: rank 16 of 7680 rows of an INT8
// head 235 us, 258 with seven waves, 270 in two workgroups a CU (2.4 TB/s; the head's own logits 172).
//
// Units of a slot follow each other, so that a workgroup's units have few slots.  The ring holds those of kSets<NR>; a
// workgroup whose units have more (ranks above 32 only, where LDS holds no more) goes over its tiles again for the
// units behind.
constexpr int kLogitWaves = 4;
template <int NR>
constexpr int kSets = NR == 4 ? 3 : kLogitWaves;
constexpr int kLdsBytes = 160 * 1024;
template <int C, int G, int NR>
struct LogitRing {
    static constexpr int SET = 2 * NR * 1024;  // an adapter's tile
    static constexpr int SLOT = Geo<C, G>::BUF + kSets<NR> * SET;
    static constexpr int HEAD_OPS = stage_wave_ops<Geo<C, G>::REC>();
    // tiles held: LDS, and the loads that the producer's wait can count (those of all but two tiles)
    static constexpr int BY_LDS = kLdsBytes / SLOT, BY_WAIT = 2 + 63 / (HEAD_OPS + 2 * NR * kSets<NR>);
    static constexpr int R = BY_LDS < BY_WAIT ? BY_LDS : BY_WAIT;
    static_assert(R >= 3, "a tile in use, one behind it and one on its way");
};

template <int C, int G, int NR>
__global__ __launch_bounds__(64 * (kLogitWaves + 1), 1) void adapt_logits_kernel(AdaptLaunch x) {
    using GE = Geo<C, G>;
    using RING = LogitRing<C, G, NR>;
    constexpr int S = GE::S, R = RING::R, D = kSets<NR>;
    extern __shared__ __align__(16) uint8_t lds[];  // [R] x SLOT
    const int mbi = blockIdx.x / x.nsplit, chunk = blockIdx.x % x.nsplit;
    const PlanView<32> plan(x.plan, x.m, x.slots);
    if (mbi * kLogitWaves >= plan.units) return;
    const int t0 = chunk * x.tpc, t1 = min(t0 + x.tpc, x.tiles);
    if (t0 >= t1) return;
    const int ntiles = t1 - t0;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // workgroups start at tiles of their own, as in the head's writer
    const unsigned stride = x.nsplit == 1 ? kStartStepOne : kStartStepSeveral;
    const int rot = (int)(((int64_t)((blockIdx.x * stride) & 0xffffu) * ntiles) >> 16);
    // the slots of the workgroup's units, each run of units with one counted once
    int slot_of[kLogitWaves], set_of[kLogitWaves];
#pragma unroll
    for (int u = 0; u < kLogitWaves; ++u) {
        const int unit = mbi * kLogitWaves + u;
        slot_of[u] = unit < plan.units ? plan.slot_of(unit) : (u ? slot_of[u - 1] : x.slots);
        set_of[u] = u == 0 ? 0 : set_of[u - 1] + (slot_of[u] != slot_of[u - 1] ? 1 : 0);
    }
    const int sets = set_of[kLogitWaves - 1] + 1;
    const int passes = (sets + D - 1) / D;

    if (wave == kLogitWaves) {
        int pslot = 0;
        // N sets of adapters beside the head's tiles, from the first-th set on
        auto produce = [&]<int N>(int first) {
            constexpr int kOps = RING::HEAD_OPS + N * 2 * NR;
            const uint8_t* up[N];
#pragma unroll
            for (int d = 0; d < N; ++d) {
                int s = x.slots;
#pragma unroll
                for (int u = 0; u < kLogitWaves; ++u) s = set_of[u] == first + d ? slot_of[u] : s;
                up[d] = x.up + (size_t)s * x.up_stride;
            }
            int pt = t0 + rot;
            auto stage_next = [&] {
                uint8_t* to = lds + pslot * RING::SLOT;
                stage_wave<GE::REC>(x.rec + (size_t)pt * GE::REC, to, lane);
#pragma unroll
                for (int d = 0; d < N; ++d)
                    stage_wave<RING::SET>(up[d] + (size_t)pt * RING::SET, to + GE::BUF + d * RING::SET, lane);
                pt = pt + 1 == t1 ? t0 : pt + 1;
                pslot = pslot + 1 == R ? 0 : pslot + 1;
            };
#pragma unroll
            for (int g = 0; g < R - 1; ++g) stage_next();
            vm_wait<kOps*(R - 2)>();  // the first tile is in LDS
            barrier_lds();
            for (int g = 0; g < ntiles; ++g) {
                stage_next();
                vm_wait<kOps*(R - 2)>();  // tile g + 1 is in LDS
                barrier_lds();
            }
            vm_wait<0>();  // the ring's last loads land before the next pass, and before the workgroup ends
            barrier_lds();
        };
        for (int p = 0; p < passes; ++p) {
            const int n = min(sets - p * D, D);
            [&]<int... k>(std::integer_sequence<int, k...>) {
                ((n == k + 1 ? produce.template operator()<k + 1>(p * D) : void()), ...);
            }(std::make_integer_sequence<int, D>{});
            pslot = 0;
        }
        return;
    }

    for (int y = tid >> 5; y < R; y += 2 * kLogitWaves)
        reinterpret_cast<u32x4*>(lds + y * RING::SLOT + GE::REC)[tid & 31] = u32x4{0, 0, 0, 0};
    const int unit = mbi * kLogitWaves + wave;
    int slot = 0, set = 0;
#pragma unroll
    for (int u = 0; u < kLogitWaves; ++u) {
        slot = u == wave ? slot_of[u] : slot;
        set = u == wave ? set_of[u] : set;
    }
    const bool live = unit < plan.units;
    const int row = live ? plan.row_of(unit, i) : 0;
    RowOperands<C, G, NR> o;
    load_rows<C, G, NR>(x, row, slot, i, h, o);
    // where the rows of this lane's 16 accumulators begin in the output
    float* to[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) to[r] = x.out + (int64_t)__shfl(row, 8 * (r >> 2) + 4 * h + (r & 3), 64) * x.n;
    for (int p = 0; p < passes; ++p) {
        const bool mine = live && set / D == p;
        int pt = t0 + rot, cslot = 0;
        barrier_lds();  // zero blocks written; the first tile is in LDS
        for (int g = 0; g < ntiles; ++g) {
            const uint8_t* buf = lds + cslot * RING::SLOT;
            cslot = cslot + 1 == R ? 0 : cslot + 1;
            if (mine) {
                constexpr int AHEAD = S < kAhead ? S : kAhead;
                const u16x8* up = reinterpret_cast<const u16x8*>(buf + GE::BUF + (set % D) * RING::SET) + lane;
                u16x8 wq[AHEAD];
                f32x16 acc = {};
#pragma unroll
                for (int s = 0; s < NR; ++s) {
                    const u16x8 hi = up[s * 64], lo = up[(NR + s) * 64];
                    acc = mfma16<true>(o.uhi[s], hi, acc);
                    acc = mfma16<true>(o.ulo[s], hi, acc);
                    acc = mfma16<true>(o.uhi[s], lo, acc);
                }
                frag_prefetch_first<C, G, AHEAD>(wq, buf, i * 16 + h * 512, i * 16, h);
                [&]<int... st>(std::integer_sequence<int, st...>) {
                    ([&] {
                        acc = mfma16<true>(o.a[st], frag_of<C, G, AHEAD, st>(wq), acc);
                        frag_prefetch_after<C, G, AHEAD, st>(wq, buf, i * 16 + h * 512, i * 16, h);
                        __builtin_amdgcn_sched_barrier(0);
                    }(), ...);
                }(std::make_integer_sequence<int, S>{});
                const float* ep = reinterpret_cast<const float*>(buf + GE::FRAG);
                const float c0 = ep[64 + i], c1 = ep[96 + i];
                const int col = pt * 32 + i;
                float v[16];
                if (o.scaled) {
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        v[r] = fmaf(acc[r] * __shfl(o.inv, 8 * (r >> 2) + 4 * h + (r & 3), 64), c0, c1);
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) v[r] = fmaf(acc[r], c0, c1);
                }
                if (col < x.n) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) to[r][col] = v[r];
                }
            }
            pt = pt + 1 == t1 ? t0 : pt + 1;
            barrier_lds();  // this ring slot is read; the next tile is in LDS
        }
        barrier_lds();  // the ring is empty
    }
}

// ---------------------------------------------------------------- launches
int grid_of(int mblocks, int nsplit, bool rows_on_one_xcd) {
    if (nsplit >= 8) return mblocks * 8 * ((nsplit + 7) / 8);
    if (rows_on_one_xcd) return ((mblocks + 7) / 8) * nsplit * 8;
    const int r8 = 8 / nsplit;
    return ((mblocks + r8 - 1) / r8) * 8;
}

size_t align(size_t x) { return (x + 255) / 256 * 256; }

struct AdaptLayout {
    size_t units, rows, slot, part, total;
};
// Blocks of 32 rows of a wave of the statistics pass, and workgroups that a CU holds of it.  Ranks above 32 keep
// too many operands for two waves a SIMD: one wave then, with two blocks where there are rows enough (rank 64,
// 30720 rows in us: 539 so, 581 with one block, 728 in two spilling waves; 1200 rows: 60 and 56).  Up to rank 32 two
// waves with a block each are ahead of one with two (rank 16: 368 and 390, rank 32: 424 and 445).
int blocks_of(int64_t m, int steps) { return steps == 4 && m > 2048 ? 2 : 1; }
int per_cu_of(int steps) { return steps == 4 ? 1 : 2; }
// Vocabulary chunks of the statistics pass: the count with the fewest tile times, as the head's (stats_nsplit), of
// the row blocks that the plan is likely to make: half a unit lost for each slot and for the rows of none, and as many
// more as that is uncertain by (a row block too many makes a round of its own: a page under 8 adapters of rank 64
// 89 us in 16 chunks, 115 in 24, which would fill one round if every slot lost half a unit).
int chunks_of(const Adapters& ad, int64_t m) {
    const int64_t unit = 32 * blocks_of(m, ad.steps), slots = 32 * (int64_t)per_cu_of(ad.steps), fixed = 8;
    const double groups = (double)std::min<int64_t>(ad.slots + 1, (m + unit - 1) / unit);
    const int64_t units = (int64_t)std::ceil((double)m / (double)unit + groups / 2 + 1.3 * std::sqrt(groups / 12));
    const int64_t mblocks = (units + kWaves - 1) / kWaves;
    int best = 1;
    int64_t best_cost = -1;
    for (int cand = 1; cand <= 128; cand += cand < 2 ? 1 : cand < 8 ? cand : 8) {
        // the chunks that hold tiles; below 8 a count that divides 8
        int ns = (ad.tiles + (ad.tiles + cand - 1) / cand - 1) / ((ad.tiles + cand - 1) / cand);
        if (ns < 8) ns = ns <= 1 ? 1 : ns <= 2 ? 2 : ns <= 4 ? 4 : 8;
        const int64_t per_xcd = ns >= 8 ? mblocks * ((ns + 7) / 8) : (mblocks + 7) / 8 * ns;
        const int64_t rounds = (per_xcd + slots - 1) / slots;
        const int64_t cost = rounds * (fixed + (ad.tiles + ns - 1) / ns);
        if ((cand & (cand - 1)) != 0 && rounds > 1) continue;
        if (ns > 64 && per_xcd > 32) continue;
        if (best_cost < 0 || cost < best_cost) best = ns, best_cost = cost;
    }
    return best;
}
AdaptLayout layout_of(const Adapters& ad, int64_t m) {
    const int64_t units = plan_units(m, std::min<int64_t>(ad.slots, m) + 1, 32);  // of the smaller size: places of the larger one fit
    AdaptLayout L;
    L.units = 0;
    L.rows = 256;
    L.slot = L.rows + align((size_t)(units + std::min<int64_t>(ad.slots, m) + 1) * 32 * 4);
    L.part = L.slot + align((size_t)units * 4);
    L.total = L.part + align((size_t)chunks_of(ad, m) * (size_t)m * sizeof(Partial));
    return L;
}

int make_plan(const Adapters& ad, const AdaptLines& lines, int64_t m, int unit, const AdaptLayout& L, uint8_t* ws, Plan* plan, int64_t* units,
              hipStream_t st) {
    const bool one = lines.lines == 1;
    *plan = Plan{reinterpret_cast<int*>(ws + L.units), reinterpret_cast<int*>(ws + L.rows), reinterpret_cast<int*>(ws + L.slot),
                 one ? lines.off : nullptr, one ? lines.slot : nullptr};
    *units = plan_units(m, std::min<int64_t>(std::min<int64_t>(ad.slots, lines.lines) + 1, m), unit);
    if (one) return PPOCR_OK;
    plan_kernel<<<1, 1024, (size_t)(ad.slots + 1) * 16, st>>>(lines, (int)m, ad.slots, unit, *plan);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

AdaptLaunch launch_of(const TileGeom& tg, const Adapters& ad, const float* a, int64_t m, int64_t n, int64_t k,
                      int64_t units, int nsplit, const Plan& plan) {
    AdaptLaunch x{};
    x.a = a;
    x.m = m;
    x.k = (int)k;
    x.vec = k % 4 == 0 && reinterpret_cast<uintptr_t>(a) % 16 == 0 ? 1 : 0;
    x.rec = ad.rec;
    x.tiles = tg.tiles;
    x.n = (int)n;
    x.nsplit = nsplit;
    x.tpc = (tg.tiles + nsplit - 1) / nsplit;
    x.mblocks = (int)((units + kWaves - 1) / kWaves);
    x.plan = plan;
    x.slots = ad.slots;
    x.down = ad.down;
    x.down_stride = ad.down_bytes();
    x.up = ad.up;
    x.up_stride = ad.up_bytes();
    x.meta = ad.meta;
    return x;
}

// f.template operator()<C, G, NR>() for the head's configuration and the adapters' steps.
template <typename F>
int by_config(int cfg, int G, int steps, F&& f) {
    auto ranks = [&]<int C, int GG>() {
        if (steps == 1) return f.template operator()<C, GG, 1>();
        if (steps == 2) return f.template operator()<C, GG, 2>();
        return f.template operator()<C, GG, 4>();
    };
    if (cfg == CFG_H2) return G == 15 ? ranks.template operator()<CFG_H2, 15>() : ranks.template operator()<CFG_H2, 10>();
    return G == 15 ? ranks.template operator()<CFG_HF3, 15>() : ranks.template operator()<CFG_HF3, 10>();
}

}  // namespace

int launch_adapters_clear(const Adapters& ad, hipStream_t st) {
    const int64_t d = (int64_t)(ad.slots + 1) * ad.down_bytes() / 16, u = (int64_t)(ad.slots + 1) * ad.up_bytes() / 16;
    clear_kernel<<<1024, 256, 0, st>>>(reinterpret_cast<u32x4*>(ad.down), d);
    PPOCR_HIP(hipGetLastError());
    clear_kernel<<<4096, 256, 0, st>>>(reinterpret_cast<u32x4*>(ad.up), u);
    PPOCR_HIP(hipGetLastError());
    clear_meta_kernel<<<16, 256, 0, st>>>(ad.meta, ad.slots + 1);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

int launch_adapter_set(const Adapters& ad, int slot, const void* down, const void* up, int rank, float scale, int bf16, int64_t n,
                       int64_t k, hipStream_t st) {
    return bf16 ? set_slot(ad, slot, (const uint16_t*)down, (const uint16_t*)up, rank, scale, n, k, st)
                : set_slot(ad, slot, (const float*)down, (const float*)up, rank, scale, n, k, st);
}

size_t adapt_workspace(const Adapters& ad, int64_t m) { return m > 0 ? layout_of(ad, m).total : 0; }

int launch_adapt_decode(int cfg, const TileGeom& tg, const Adapters& ad, const AdaptLines& lines, const float* a,
                        int64_t m, int64_t n, int64_t k, int32_t* idx, float* maxprob, const CtcOut& ctc, uint8_t* ws,
                        hipStream_t st) {
    const AdaptLayout L = layout_of(ad, m);
    Plan plan;
    int64_t units;
    if (int e = make_plan(ad, lines, m, 32 * blocks_of(m, ad.steps), L, ws, &plan, &units, st)) return e;
    const int nsplit = chunks_of(ad, m);
    AdaptLaunch x = launch_of(tg, ad, a, m, n, k, units, nsplit, plan);
    x.part = reinterpret_cast<Partial*>(ws + L.part);
    const unsigned grid = (unsigned)grid_of(x.mblocks, nsplit, true);
    if (int e = by_config(cfg, tg.G, ad.steps, [&]<int C, int G, int NR>() {
            auto go = [&]<int MB, int OCC>() {
                constexpr int bytes = kRing * Geo<C, G>::BUF + kWaves * MB * 16 * 64 * 4;
                adapt_stats_kernel<C, G, NR, MB, OCC><<<grid, 64 * kWaves, bytes, st>>>(x);
            };
            if constexpr (NR < 4) go.template operator()<1, 2>();
            else if (blocks_of(m, ad.steps) == 2) go.template operator()<2, 1>();
            else go.template operator()<1, 1>();
            PPOCR_HIP(hipGetLastError());
            return (int)PPOCR_OK;
        }))
        return e;
    return launch_merge_ctc(x.part, m, nsplit, ctc, idx, maxprob, nullptr, st);
}

int launch_adapt_logits(int cfg, const TileGeom& tg, const Adapters& ad, const AdaptLines& lines, const float* a,
                        int64_t m, int64_t n, int64_t k, float* out, uint8_t* ws, hipStream_t st) {
    const AdaptLayout L = layout_of(ad, m);
    Plan plan;
    int64_t units;
    if (int e = make_plan(ad, lines, m, 32, L, ws, &plan, &units, st)) return e;
    const int64_t mblocks = (units + kLogitWaves - 1) / kLogitWaves;
    // The chunk count with the fewest tile times, a workgroup a CU at once and its start worth 8 tiles, of the row
    // blocks that the plan is likely to make; counts that keep an XCD at its own chunks (7680 rows in 8 and 16 chunks
    // 236 us, in 6 and 12 260 and 255).
    const int64_t whole = (m + 31) / 32;
    const int64_t likely = (whole + std::min<int64_t>(ad.slots, whole) / 2 + kLogitWaves - 1) / kLogitWaves;
    int nsplit = 1;
    int64_t best = -1;
    for (int ns = 1; ns <= 128 && ns <= tg.tiles; ns += ns < 8 ? ns : 8) {
        const int64_t cost = (likely * ns + 255) / 256 * (8 + (tg.tiles + ns - 1) / ns);
        if (best < 0 || cost < best) nsplit = ns, best = cost;
    }
    AdaptLaunch x = launch_of(tg, ad, a, m, n, k, units, nsplit, plan);
    x.out = out;
    const unsigned grid = (unsigned)(mblocks * nsplit);
    return by_config(cfg, tg.G, ad.steps, [&]<int C, int G, int NR>() {
        constexpr int bytes = LogitRing<C, G, NR>::R * LogitRing<C, G, NR>::SLOT;
        adapt_logits_kernel<C, G, NR><<<grid, 64 * (kLogitWaves + 1), bytes, st>>>(x);
        PPOCR_HIP(hipGetLastError());
        return (int)PPOCR_OK;
    });
}

}  // namespace ppocr
