// The matrix kernels of the vocabulary losses: the softmax statistics of the forward pass and
// the two gradient products of the backward pass (xent.hpp for the records they read).
//
// Why tiles of 32 x 32 and owners in registers: an MFMA result of the logits then is, lane by lane, a
// column of P, the operand of the second product, and a workgroup needs LDS only for the stream.
// 30720 rows, 18710 classes, k = 120: statistics 354 us (fp32, 1250 TFLOP/s of fp16 products) and 173
// (bf16, 850), both gradients 1672 (1055) and 750 (785).  The matrix pipe is busy 54% of the cycles in
// the fp32 gradients and 39% in the bf16 ones, at 1.81 and 1.95 GHz.  Earlier versions: fp32 5% less time
// without the LDS reads, none less for a fifth fewer vector instructions, which fits a limit by power
// (not measured); bf16 9-10% less without the exponentials, 12-15% without the staging loads.
#pragma once
#include "xent.hpp"

namespace ppocr {
namespace xent {

constexpr int kWaves = 4, kThreads = 64 * kWaves;
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// REC bytes of a record from global memory into LDS, 16 per lane, without registers: pieces of 1 KB, a
// wave each in turn, and the rest by the first lanes of the next.  Addresses are the piece's (the
// same for the wave) plus the lane's, so that a step of the stream costs no vector arithmetic.
template <int REC>
__device__ __forceinline__ void stage(const uint8_t* __restrict__ src, uint8_t* dst, int wave, unsigned lane16) {
    constexpr int FULL = REC / 1024, REST = REC % 1024;
    static_assert(REC % 16 == 0, "record size");
    auto piece = [&](int p) {
        const uint8_t* from = src + (size_t)p * 1024;
        asm volatile("" : "+s"(from));  // a scalar address: the lane's part stays an offset
        __builtin_amdgcn_global_load_lds(
            static_cast<const void*>(from + lane16),
            reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(dst + (size_t)p * 1024)), 16, 0,
            0);
    };
#pragma unroll
    for (int x = 0; x < (FULL + kWaves - 1) / kWaves; ++x)
        if (FULL % kWaves == 0 || x * kWaves + wave < FULL) piece(x * kWaves + wave);
    if (REST > 0 && wave == FULL % kWaves && lane16 < REST) piece(FULL);
}
__device__ __forceinline__ void wait_loads() {
    __builtin_amdgcn_s_waitcnt(0x0 | (0x7 << 4) | (0xF << 8));  // vmcnt(0)
}

// One record's logits for this lane's owner entry: 16 entries of the stream record (8 (r / 4)
// + 4 (lane / 32) + r % 4) against owner lane % 32.  With two planes the three products that
// fp32 sums keep: high x high, high x low, low x high.
template <int D, int P, int NB>
__device__ __forceinline__ void scores(const uint8_t* rec, const f16x8 (&own)[NB][P][2 * D], f32x16 (&s)[NB], int lane) {
    const f16x8* s0 = reinterpret_cast<const f16x8*>(rec) + lane;
#pragma unroll
    for (int b = 0; b < NB; ++b) s[b] = f32x16{};
#pragma unroll
    for (int ks = 0; ks < 2 * D; ++ks) {
        const f16x8 hi = s0[ks * 64];
#pragma unroll
        for (int b = 0; b < NB; ++b) s[b] = mma(hi, own[b][0][ks], s[b]);
        if constexpr (P == 2) {
            const f16x8 lo = s0[(2 * D + ks) * 64];
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = mma(hi, own[b][1][ks], s[b]);
#pragma unroll
            for (int b = 0; b < NB; ++b) s[b] = mma(lo, own[b][0][ks], s[b]);
        }
    }
}

// Are there records from t0 to t1 whose entries have scales of their own?  Those take another form of
// the loops: the branch in one form for all cost steps 4 to 13% of their time.  Steps whose rows or classes all do
// take 2% (fp32) to 10% (bf16) longer for either, 20% at k = 256 for rows.
__device__ __forceinline__ bool any_own(const int* __restrict__ u, int64_t t0, int64_t t1, int lane) {
    int any = 0;
    for (int64_t i = t0 + lane; i < t1; i += 64 * 8)
#pragma unroll
        for (int j = 0; j < 8; ++j) any |= u[min(i + 64 * j, t1 - 1)];
    return __any(any & 1);
}
// Where a stream record's entries have scales of their own (aux: its scalars and scales), the logits of
// this lane's owner (c: its own) take them here, and the factor that is left is 1.
__device__ __forceinline__ bool shared_scale(const float* aux) {
    return __builtin_amdgcn_readfirstlane(__float_as_int(aux[70])) != 0;
}
__device__ __forceinline__ float own_scales(const float* aux, float c, f32x16& s, int h) {
    if (shared_scale(aux)) return c * aux[64];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const f32x4 scale = *reinterpret_cast<const f32x4*>(aux + 80 + 8 * q + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[4 * q + e] *= c * scale[e];
        asm volatile("" ::: "memory");  // four scales at a time: this way is rare, its registers are not
    }
    return 1.0f;
}

template <int D, int P>
__device__ __forceinline__ void load_owner(const uint8_t* rec, f16x8 (&own)[P][2 * D], int lane) {
    const f16x8* s0 = reinterpret_cast<const f16x8*>(rec) + lane;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
        for (int ks = 0; ks < 2 * D; ++ks) own[p][ks] = s0[(p * 2 * D + ks) * 64];
}

// ---------------------------------------------------------------- forward: softmax statistics
// Streams the class records of a chunk past 32 NB rows per wave.  t = z log2(e) / tau, and a lane
// needs no other lane until the chunk ends.  Where |a| |w| + |b| (the records' largest norms)
// bounds |t| by 100, exp2(t) is summed as it is: no maximum and no reference, a third of the vector
// work.  Other records keep a reference that moves only when a maximum beats it by 16 (so sums stay
// below 2^16 n and lose nothing); a row that once needed one keeps it.
template <int D, int P, int NB, bool ODD>
__device__ __forceinline__ void statistics(const XentStatsArgs& x, uint8_t* lds) {
    constexpr int REC = P * D * 2048 + kXentAux;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lane16 = lane * 16;
    const int split = blockIdx.x % x.nsplit;
    const int64_t rb = blockIdx.x / x.nsplit;
    const int64_t t0 = (int64_t)split * x.per_split, t1 = min(t0 + x.per_split, x.tiles);
    const int64_t row0 = rb * (32 * NB * kWaves) + wave * (32 * NB);

    stage<REC>(x.str + t0 * REC, lds, wave, lane16);
    f16x8 own[NB][P][2 * D];
    float c[NB], norm[NB], ref[NB], sum[NB];
    bool shifted[NB];  // some row has a reference other than 0
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        const int64_t r = min(row0 + 32 * b, x.m - 1) / 32;  // a record that exists; unused rows are dropped at the end
        const uint8_t* rec = x.own + r * REC;
        const float* aux = reinterpret_cast<const float*>(rec + P * D * 2048);
        load_owner<D, P>(rec, own[b], lane);
        c[b] = x.c0 * aux[80 + (lane & 31)];
        norm[b] = x.c0 * aux[66];
        ref[b] = -INFINITY;
        sum[b] = 0.0f;
        shifted[b] = false;
    }
    for (int64_t t = t0; t < t1; ++t) {
        const uint8_t* cur = lds + ((t - t0) & 1) * REC;
        wait_loads();
        __syncthreads();
        if (t + 1 < t1) stage<REC>(x.str + (t + 1) * REC, lds + ((t + 1 - t0) & 1) * REC, wave, lane16);
        const float* aux = reinterpret_cast<const float*>(cur + P * D * 2048);
        const float ce = aux[64], cn = aux[66], cb = aux[67];
        f32x16 sc[NB];
        __builtin_amdgcn_s_setprio(1);
        scores<D, P, NB>(cur, own, sc, lane);
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x16& s = sc[b];
            const float cc = ODD ? own_scales(aux, c[b], s, h) : c[b] * ce;
            const bool plain = !shifted[b] && __builtin_amdgcn_readfirstlane(norm[b] * cn + cb <= 100.0f);
            if (plain) {
                if (ref[b] == -INFINITY) ref[b] = 0.0f;
                float add = 0.0f;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const f32x4 bias = *reinterpret_cast<const f32x4*>(aux + 8 * q + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) add += __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], cc, bias[e]));
                }
                sum[b] += add;
                continue;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 bias = *reinterpret_cast<const f32x4*>(aux + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * q + e] = fmaf(s[4 * q + e], cc, bias[e]);
                    mx = fmaxf(mx, s[4 * q + e]);
                }
            }
            if (__any(mx > ref[b] + 16.0f)) {
                const float nr = mx > ref[b] + 16.0f ? mx : ref[b];
                sum[b] = ref[b] == -INFINITY ? 0.0f : sum[b] * __builtin_amdgcn_exp2f(ref[b] - nr);
                ref[b] = nr;
                shifted[b] = true;
            }
            const float rf = ref[b] == -INFINITY ? 0.0f : ref[b];
            float add = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) add += __builtin_amdgcn_exp2f(s[r] - rf);
            sum[b] += add;
        }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        // the two halves of the wave hold the row's other classes
        const float r2 = __shfl_xor(ref[b], 32, 64), s2 = __shfl_xor(sum[b], 32, 64);
        const float nr = fmaxf(ref[b], r2);
        float s = 0.0f;
        s += ref[b] == -INFINITY ? sum[b] : sum[b] * __builtin_amdgcn_exp2f(ref[b] - nr);
        s += r2 == -INFINITY ? s2 : s2 * __builtin_amdgcn_exp2f(r2 - nr);
        const int64_t row = row0 + 32 * b + (lane & 31);
        if (h == 0 && row < x.m) x.part[(int64_t)split * x.m + row] = make_float2(nr, s);
    }
}
template <int D, int P, int NB>
__global__ __launch_bounds__(kThreads, 2) void stats_kernel(XentStatsArgs x) {
    extern __shared__ __align__(16) uint8_t lds[];
    const int64_t t0 = (int64_t)(blockIdx.x % x.nsplit) * x.per_split, t1 = min(t0 + x.per_split, x.tiles);
    if (any_own(x.str_u, t0, t1, threadIdx.x & 63)) statistics<D, P, NB, true>(x, lds);
    else statistics<D, P, NB, false>(x, lds);
}

// ---------------------------------------------------------------- backward: a gradient
// dX_o = sum_s P_os Y_s for the owners o of a workgroup (32 per wave), the stream records s of a
// chunk in turn: the logits of 32 x 32 pairs, p = exp2(t - lse), the target entries' places
// overwritten with p - q as the list holds it (exact in 32 bits, so that a nearly certain label
// leaves its small difference), then P as the second product's operand without leaving the
// registers: a result register's rows are the contraction's order, and the transposed part of
// the record holds the entries in that order.
//   ROWS: owners are activation rows, the stream is the classes (da).  P = p 2^(S - e).
//   else: owners are classes, the stream is the rows (dW, db).  P = p g 2^(S - e), g the row's
//   gradient factor.
// e is the stream record's (or its entry's) exponent and S the owner's: P's fp16 halves end at 2^-25, so an owner whose
// P are all small (a class that is improbable in every row) needs a larger S than others.  The first
// record's P set it, so that the largest is 2^4 to 2^5, and where a later one comes above 2^15, the
// owner's sums so far and its S go down with it: what a P loses is 2^-29 of the owner's largest.  S is
// never below F, where no P is above 2^14 (u is the records' bound of what multiplies p, F = 14 - max u).
// With bf16 tensors P is one half, 11 bits (a bf16 product of its own would keep 8): da and dW are off
// by 1.67e-3 of their norm, that being the rounding of the bf16 outputs; with a second half by 1.66e-3, and
// the step of 30720 rows takes 1117 us instead of 924.
// One S for all: 846 us a step of 30720 bf16 rows, 1981 fp32; so 892 and 2039 to 2058; the largest put to
// 2^8, more owners come above 2^15 (tiny head under 32 teacher logits 271 us, 254 so), to 2^0: 871 and 2011.
// The target lists are read 64 entries at a time, one a lane, and an entry's place is written by the
// lane that holds it, in the register that its row (or class) of the tile is: a wave-uniform number.
constexpr int kLargest = 4;
constexpr int kLow = 60;
__device__ __forceinline__ void set_entry(f32x16& p, int i, bool mine, float v) {
    const float old = p[i];
    p[i] = mine ? v : old;
}
__device__ __forceinline__ int lane_value(int v, int l) { return __builtin_amdgcn_readlane(v, l); }
// Has a loaded value here, where nothing younger is on its way: left to itself the compiler waits
// where the value is used, for everything loaded since.
__device__ __forceinline__ void arrive(int& a, int& b) { asm volatile("" : "+v"(a), "+v"(b)); }

// A row group's list, walked along with the classes.
struct ListWalk {
    const uint32_t* keys;
    const float* vals;
    int at, end;        // the next entry, the list's length
    int wkey, wval;     // this lane's entry of the window of 64 that holds `at`
    uint32_t key;       // the next entry's
    __device__ __forceinline__ void load(int lane) {
        const int i = (at & ~63) + lane;
        wkey = i < end ? (int)keys[i] : -1;
        wval = i < end ? __float_as_int(vals[i]) : 0;
        arrive(wkey, wval);
    }
    __device__ __forceinline__ void start(const XentGradArgs& x, bool have, int64_t group, int64_t tile, int lane) {
        keys = x.keys + (have ? group * x.list : 0);
        vals = x.vals + (have ? group * x.list : 0);
        end = have ? x.list : 0;
        at = have ? __builtin_amdgcn_readfirstlane(x.offs[group * (x.blocks + 1) + tile / 4]) : 0;
        load(lane);
        key = at < end ? (uint32_t)lane_value(wkey, at & 63) : 0xFFFFFFFFu;
    }
    __device__ __forceinline__ void step(int lane) {
        ++at;
        if ((at & 63) == 0) load(lane);
        key = at < end ? (uint32_t)lane_value(wkey, at & 63) : 0xFFFFFFFFu;
    }
};

// A row record's entries in a workgroup's 128 classes.
struct ListSlice {
    int from, to;  // where they are in the group's list
    int key, val;  // this lane's entry of a window of 64
    __device__ __forceinline__ void bounds(const XentGradArgs& x, int64_t t, int64_t ob) {
        const uint16_t* of = x.offs + t * (x.blocks + 1) + ob;
        from = of[0];
        to = of[1];
    }
    __device__ __forceinline__ void read(const XentGradArgs& x, int64_t t, int first, int lane) {
        const int i = first + lane;
        key = i < to ? (int)x.keys[t * x.list + i] : -1;
        val = i < to ? __float_as_int(x.vals[t * x.list + i]) : 0;
    }
};

template <int D, int P, bool ROWS, bool ODD>
__device__ __forceinline__ void gradient(const XentGradArgs& x, const XentGradSide& y, unsigned block, int um, uint8_t* lds) {
    constexpr int REC = 2 * P * D * 2048 + kXentAux, AUX = 2 * P * D * 2048;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const unsigned lane16 = lane * 16;
    const int split = block % y.nsplit;
    const int64_t ob = block / y.nsplit;
    const int64_t t0 = (int64_t)split * y.per_split, t1 = min(t0 + y.per_split, y.str_tiles);
    const int64_t og = ob * kWaves + wave;  // this wave's owner record
    const int64_t owner = og * 32 + (lane & 31);

    stage<REC>(y.str + t0 * REC, lds, wave, lane16);
    const int F = 14 - um, most = F + 86;  // 2^(S + u) stays a number
    int S = F;
    bool fresh = true;  // no record has set S

    const bool have = og < y.own_tiles;
    const uint8_t* orec = y.own + (have ? og : y.own_tiles - 1) * REC;
    f16x8 own[1][P][2 * D];
    load_owner<D, P>(orec, own[0], lane);
    const float* oaux = reinterpret_cast<const float*>(orec + AUX);
    const float c = x.c0 * oaux[80 + (lane & 31)];
    float own0 = oaux[lane & 31];                      // row: lse log2(e); class: bias log2(e) / tau
    float own1 = ROWS ? oaux[32 + (lane & 31)] : 0.0f;  // row: the gradient factor, times 2^-own_ge
    const int own_ge = ROWS ? __builtin_amdgcn_readfirstlane((int)oaux[69]) : 0;
    // da's lse to 2^-14, so that whole exponents add to it exactly; the rest multiplies the sums
    float rest = 1.0f;
    if (ROWS && fabsf(own0) < 1024.0f) {
        const float whole = rintf(own0 * 16384.0f) * (1.0f / 16384.0f);
        rest = exp2f(own0 - whole);
        own1 /= rest;
        own0 = whole;
    }
    f32x16 acc[D] = {};
    float dbias = 0.0f;
    float minus = -1.0f;  // a number the compiler does not know: it keeps the mixed-precision fma
    asm volatile("" : "+s"(minus));

    // the slice of the next record is read while a record's second product runs, its bounds one earlier
    ListWalk walk;
    ListSlice slice, after;
    if constexpr (ROWS) {
        walk.start(x, have, og, t0, lane);
    } else {
        slice.bounds(x, t0, ob);
        slice.read(x, t0, slice.from, lane);
        after.bounds(x, min(t0 + 1, y.str_tiles - 1), ob);
    }
    for (int64_t t = t0; t < t1; ++t) {
        const uint8_t* cur = lds + ((t - t0) & 1) * REC;
        wait_loads();
        if constexpr (!ROWS) {
            arrive(slice.key, slice.val);
            arrive(after.from, after.to);
        }
        __syncthreads();
        if (t + 1 < t1) stage<REC>(y.str + (t + 1) * REC, lds + ((t + 1 - t0) & 1) * REC, wave, lane16);
        f32x16 s[1];
        // the matrix instructions of one wave before the vector work of the CU's others
        __builtin_amdgcn_s_setprio(1);
        scores<D, P, 1>(cur, own, s, lane);
        __builtin_amdgcn_s_setprio(0);
        f32x16& p = s[0];
        const float* aux = reinterpret_cast<const float*>(cur + AUX);
        const float cc = ODD ? own_scales(aux, c, p, h) : c * aux[64];
        const int u = __builtin_amdgcn_readfirstlane((int)aux[68]);
        if constexpr (ROWS) {
            const float shift = own0 - (float)(S + u);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 bias = *reinterpret_cast<const f32x4*>(aux + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p[4 * q + e] = __builtin_amdgcn_exp2f(fmaf(p[4 * q + e], cc, bias[e]) - shift);
            }
            const uint32_t end = (uint32_t)((t + 1) * 1024);  // keys below: classes of this record
            while (walk.key < end) {
                const int cls = (int)(walk.key >> 5) & 31, row = (int)walk.key & 31;
                const float v = __int_as_float(lane_value(walk.wval, walk.at & 63));
                set_entry(p, (cls >> 3) * 4 + (cls & 3), lane == row + 32 * ((cls >> 2) & 1), ldexpf(v * rest, S + u));
                walk.step(lane);
            }
        } else {
            // The bias's sum does not weigh a row by its activations: a record whose activations are 2^60
            // smaller than others' keeps a scale of its own for it.
            const int at = ODD ? max(S + u, -46) : S + u;
            const float scale = ldexpf(1.0f, at);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 lse = *reinterpret_cast<const f32x4*>(aux + 8 * q + 4 * h);
                const f32x4 g = *reinterpret_cast<const f32x4*>(aux + 32 + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    p[4 * q + e] = __builtin_amdgcn_exp2f(fmaf(p[4 * q + e], cc, own0) - lse[e]) * (g[e] * scale);
            }
            const int from = __builtin_amdgcn_readfirstlane(slice.from), to = __builtin_amdgcn_readfirstlane(slice.to);
            for (int first = from; first < to; first += 64) {
                if (first != from) {
                    slice.read(x, t, first, lane);
                    arrive(slice.key, slice.val);
                }
                // each lane its entry: the lane and the register it goes to, and what goes there
                const int cls = (slice.key >> 5) & 31, row = slice.key & 31;
                const int lane_reg = cls + 32 * ((row >> 2) & 1) + (((row >> 3) * 4 + (row & 3)) << 8);
                const int v = __float_as_int(__int_as_float(slice.val) * aux[32 + row]);
                unsigned long long todo = __ballot((int64_t)((uint32_t)slice.key >> 10) == og && first + lane < to);
                while (todo) {
                    const int l = __builtin_ctzll(todo);
                    todo &= todo - 1;
                    const int place = lane_value(lane_reg, l);
                    set_entry(p, place >> 8, lane == (place & 63), __int_as_float(lane_value(v, l)) * scale);
                }
            }
            slice.from = after.from;
            slice.to = after.to;
            slice.read(x, min(t + 1, y.str_tiles - 1), slice.from, lane);
            after.bounds(x, min(t + 2, y.str_tiles - 1), ob);
            float add = 0.0f;
#pragma unroll
            for (int r = 0; r < 16; ++r) add += p[r];
            dbias += ldexpf(add, (int)aux[69] - at);
            if (u == kXentNone) continue;  // no row of the record has a gradient
        }
        if (ODD && !shared_scale(aux)) {
            // entries with scales of their own: what those are below the record's
            const int e0 = __builtin_amdgcn_readfirstlane((int)aux[65]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4 scale = *reinterpret_cast<const f32x4*>(aux + 80 + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[4 * q + e] *= ldexpf(scale[e], e0);
                asm volatile("" ::: "memory");
            }
        }
        const bool low = ODD && !ROWS && um - u > kLow;  // the same for all lanes
        float mx = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(p[r]));
        if (fresh || low || __any(mx > 32768.0f)) {
            const int off = low ? min(S + u + 46, 0) : 0;
            mx = ldexpf(fmaxf(mx, __shfl_xor(mx, 32, 64)), off);  // the owner's other half too
            int to = S;
            if (fresh || mx > 32768.0f) to = mx > 0.0f ? min(max(S + kLargest - ilogbf(mx), F), most) : most;
            const float by = ldexpf(1.0f, to - S), byp = ldexpf(1.0f, to - S + off);
            S = to;
            fresh = false;
#pragma unroll
            for (int r = 0; r < 16; ++r) p[r] *= byp;
#pragma unroll
            for (int d = 0; d < D; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[d][r] *= by;
            // still above at F: logits so large that their own roundings make p more than 1
            if (__any(mx * by > 32768.0f))
#pragma unroll
                for (int r = 0; r < 16; ++r) p[r] = fabsf(p[r]) > 32768.0f ? copysignf(16384.0f, p[r]) : p[r];
        }
        __builtin_amdgcn_s_setprio(1);
        const f16x8* tr = reinterpret_cast<const f16x8*>(cur + P * D * 2048) + lane;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            f16x8 ph, pl;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const f32x2 v = {p[8 * e + j], p[8 * e + j + 1]};
                const f16x2 hv = __builtin_convertvector(v, f16x2);
                ph[j] = hv[0];
                ph[j + 1] = hv[1];
                if constexpr (P == 2) {
                    // what the high half leaves, in one instruction each (exact)
                    const f32x2 r = {fmaf((float)hv[0], minus, v[0]), fmaf((float)hv[1], minus, v[1])};
                    const f16x2 lv = __builtin_convertvector(r, f16x2);
                    pl[j] = lv[0];
                    pl[j + 1] = lv[1];
                }
            }
#pragma unroll
            for (int d = 0; d < D; ++d) {
                const f16x8 hi = tr[(d * 2 + e) * 64];
                acc[d] = mma(hi, ph, acc[d]);
                if constexpr (P == 2) {
                    const f16x8 lo = tr[(D * 2 + d * 2 + e) * 64];
                    acc[d] = mma(hi, pl, acc[d]);
                    acc[d] = mma(lo, ph, acc[d]);
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
    }
    if (owner < y.owners) {
        float* out = y.part + ((int64_t)split * y.owners + owner) * (32 * D);
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = ldexpf(acc[d][4 * q + e], own_ge - S);
                    if (ROWS) v[e] = own1 == 0.0f ? 0.0f : v[e] * own1;  // no gradient, whatever the head holds
                }
                *reinterpret_cast<f32x4*>(out + 32 * d + 8 * q + 4 * h) = v;
            }
    }
    if constexpr (!ROWS) {
        dbias += __shfl_xor(dbias, 32, 64);
        if (h == 0 && owner < y.owners) x.part_db[(int64_t)split * y.owners + owner] = dbias;
    }
}

template <int D, int P, bool ROWS>
__device__ __forceinline__ void gradient(const XentGradArgs& x, const XentGradSide& y, unsigned block, uint8_t* lds) {
    // the largest and the smallest exponent bound of the stream, and whether entries have scales of their own
    int most = kXentNone, least = -kXentNone, own = 0;
    for (int64_t i = threadIdx.x & 63; i < y.str_tiles; i += 64 * 16) {
        int v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = y.str_u[min(i + 64 * j, y.str_tiles - 1)];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int u = v[j] >> 1;
            most = max(most, u);
            if (u != kXentNone) least = min(least, u);
            own |= v[j] & 1;
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        most = max(most, __shfl_xor(most, o, 64));
        least = min(least, __shfl_xor(least, o, 64));
    }
    const int um = __builtin_amdgcn_readfirstlane(most);
    const bool odd = __any(own) || (!ROWS && um - __builtin_amdgcn_readfirstlane(least) > kLow);
    if (odd) gradient<D, P, ROWS, true>(x, y, block, um, lds);
    else gradient<D, P, ROWS, false>(x, y, block, um, lds);
}

// Both gradients in one launch, so that the last workgroups of one fill up with the other's (and a
// page's step has a launch less).
template <int D, int P>
__global__ __launch_bounds__(kThreads, xent_grad_per_cu(D, P)) void grad_kernel(XentGradArgs x) {
    extern __shared__ __align__(16) uint8_t lds[];
    if (blockIdx.x < x.row_grid) gradient<D, P, true>(x, x.rows, blockIdx.x, lds);
    else gradient<D, P, false>(x, x.classes, blockIdx.x - x.row_grid, lds);
}

}  // namespace xent

template <int D, int P>
int xent_stats_cfg(const XentStatsArgs& x, int blocks, unsigned grid, hipStream_t st) {
    constexpr int lds = 2 * (P * D * 2048 + kXentAux);
    if constexpr (xent_stats_most_blocks(D, P) == 2) {
        if (blocks == 2) {
            xent::stats_kernel<D, P, 2><<<grid, xent::kThreads, lds, st>>>(x);
            PPOCR_HIP(hipGetLastError());
            return PPOCR_OK;
        }
    }
    xent::stats_kernel<D, P, 1><<<grid, xent::kThreads, lds, st>>>(x);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

template <int D, int P>
int xent_grad_cfg(const XentGradArgs& x, unsigned grid, hipStream_t st) {
    constexpr int lds = 2 * (2 * P * D * 2048 + kXentAux);
    xent::grad_kernel<D, P><<<grid, xent::kThreads, lds, st>>>(x);
    PPOCR_HIP(hipGetLastError());
    return PPOCR_OK;
}

#define PPOCR_XENT_INSTANCES(D, P)                                                       \
    template int xent_stats_cfg<D, P>(const XentStatsArgs&, int, unsigned, hipStream_t); \
    template int xent_grad_cfg<D, P>(const XentGradArgs&, unsigned, hipStream_t);

}  // namespace ppocr
