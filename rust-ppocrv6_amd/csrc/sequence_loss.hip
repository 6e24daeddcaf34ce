// Losses over text lines from the cross entropies of their steps, x = loss[r] = -log p(class of step r).
//
//   policy      rho = exp(old - x), v = -min(rho A, clip(rho, 1 - low, 1 + high) A) + beta (e^t - t - 1)
//               with t = x - ref; a line's loss is the mean of v over its steps that count, and
//               dv/dx = rho A where the clipped product is not the smaller one, + beta (e^t - 1)
//   preference  R = w sum (ref - x) over a line's steps that count (w: beta, over their number for means),
//               h = R of the chosen line - R of the other, L = -(1 - e) log s(h) - e log s(-h) with the
//               logistic s, dL/dh = e s(h) - (1 - e) s(-h), dR/dx = -w
//
// Each step's values are read once and its gradient written once.  A team of G lanes takes a line (or a pair of
// lines): the sums go through the team in a fixed order, and the gradient, which needs them, is written from what the
// lanes kept in registers; the steps beyond them are read again.  Sums are held in 64 bits.
//
// 4M steps in 32768 lines under a policy loss, 101 MB: 28.1 us, 3.6 TB/s (a copy: 5.1); in 16384 pairs, 68 MB: 19.5 us.
// Vector instructions bound the policy loss: some 400 a wave of 64 lanes and 4 steps a lane (the exponentials, the sums in
// 64 bits, the clipping's border), 21 us of issue, which is why loads are held back by nothing and sums use the
// registers' lane paths (34 and 22 us with shuffles and branches around the loads).  The preference loss has 12 us of
// them; the rest is memory's latency, of which a pair of more than 256 steps has two turns.  Small calls are bound by the
// launch: a page's 2245 steps 4 us.
//
// In 32 bits are a step's differences old - x and x - ref and what is taken from them: a difference is off by half a step
// of itself at most, which is no more than the rounding of the larger cross entropy put into it (both are positive, so
// the difference is the smaller), and the ratio and the divergence by that.  The logistic and its logarithm are in 32 bits
// too, with what the rounding of h lost put back.
#include <algorithm>
#include <cmath>

#include "sequence_loss.hpp"

namespace ppocr {
namespace {

// Steps of a line that a lane keeps in registers between the sums and the gradient.
constexpr int kKeep = 4;
constexpr int threads_of(int G) { return G > 256 ? G : 256; }

struct Sums {
    double a, b;
    int x, y;
};

// v plus the value of a lane of the same 16, through the registers' own lane paths.
template <int CTRL>
__device__ __forceinline__ double add_lane(double v) {
    const unsigned long long u = __builtin_bit_cast(unsigned long long, v);
    const int lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)u, CTRL, 0xF, 0xF, true);
    const int hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(u >> 32), CTRL, 0xF, 0xF, true);
    return v + __builtin_bit_cast(double, ((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}
// Sum over a team's lanes of the wave: neighbours, pairs, then the mirror images within 8 and 16 lanes, which hold the
// other half's sums.
template <int G>
__device__ __forceinline__ double lane_sum(double v) {
    v = add_lane<0xB1>(v);   // lanes 1 0 3 2
    v = add_lane<0x4E>(v);   // lanes 2 3 0 1
    v = add_lane<0x141>(v);  // mirrored in 8
    v = add_lane<0x140>(v);  // mirrored in 16
    if constexpr (G >= 32) v += __shfl_xor(v, 16, 64);
    if constexpr (G >= 64) v += __shfl_xor(v, 32, 64);
    return v;
}
// Lanes of this lane's team (of its wave, for larger teams) that hold `on`.
template <int G>
__device__ __forceinline__ int team_count(bool on) {
    const unsigned long long mask = __ballot(on);
    if constexpr (G >= 64) return __popcll(mask);
    else return __popcll((mask >> (threadIdx.x & 63 & ~(G - 1))) & ((1ull << G) - 1));
}

// Sums over the lanes of a team, the same in each lane; the counts are those of its waves already.  For G > 64
// through LDS, every lane of the workgroup (one team) calling it.
template <int G>
__device__ __forceinline__ Sums team_sum(Sums v, Sums* red) {
    v.a = lane_sum<G>(v.a);
    v.b = lane_sum<G>(v.b);
    if constexpr (G > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = Sums{0.0, 0.0, 0, 0};
#pragma unroll
        for (int i = 0; i < G / 64; ++i) {
            v.a += red[i].a;
            v.b += red[i].b;
            v.x += red[i].x;
            v.y += red[i].y;
        }
    }
    return v;
}

// Steps are numbered in 32 bits (the entry points take up to 2^30): an array's element is its base, the same for the
// wave, and a 32-bit offset.
__device__ __forceinline__ unsigned clamp_row(int64_t r, int64_t m) { return (unsigned)(r < 0 ? 0 : r > m ? m : r); }

// The steps that no line covers have no gradient: workgroup `part` of `parts` clears its share.
__device__ __forceinline__ void clear_uncovered(const LineSteps& s, float* row_grad, int part, int parts) {
    unsigned first = (unsigned)s.m, last = first;
    if (s.lines > 0) {
        first = clamp_row(s.off[0], s.m);
        last = max(clamp_row(s.off[s.lines], s.m), first);
    }
    const unsigned step = parts * blockDim.x;
    for (unsigned r = part * blockDim.x + threadIdx.x; r < first; r += step) row_grad[r] = 0.0f;
    for (unsigned r = last + part * blockDim.x + threadIdx.x; r < (unsigned)s.m; r += step) row_grad[r] = 0.0f;
}

// e^t - t - 1 (kl) and e^t - 1 (em1) to a few units of the last place.  Below 1 by the series of the first, whose terms up
// to t^13 / 13! leave less than 2^-26 of the value at |t| = 1, as the difference would lose all of it near 0; the
// second is the first plus t.
__device__ __forceinline__ void exp_tail(float t, float& kl, float& em1) {
    float p = 1.0f / 6227020800.0f;
    p = fmaf(p, t, 1.0f / 479001600.0f);
    p = fmaf(p, t, 1.0f / 39916800.0f);
    p = fmaf(p, t, 1.0f / 3628800.0f);
    p = fmaf(p, t, 1.0f / 362880.0f);
    p = fmaf(p, t, 1.0f / 40320.0f);
    p = fmaf(p, t, 1.0f / 5040.0f);
    p = fmaf(p, t, 1.0f / 720.0f);
    p = fmaf(p, t, 1.0f / 120.0f);
    p = fmaf(p, t, 1.0f / 24.0f);
    p = fmaf(p, t, 1.0f / 6.0f);
    p = fmaf(p, t, 0.5f);
    kl = p * t * t;
    em1 = kl + t;
    if (!(__builtin_fabsf(t) < 1.0f)) {
        const float e = expf(t);
        em1 = e - 1.0f;
        kl = em1 - t;
    }
}

struct PolicyRow {
    float x, old, ref, adv;
    int target;
};

// Which side of the clipping's border a step lies on is decided on the difference of the logarithms in 64
// bits, where it is exact: the ratio's own rounding would decide it next to the border.
struct Border {
    double above, below;  // log(1 + high), log(1 - low)
    float top, bottom;    // 1 + high, 1 - low
};

// REF: without a reference, with one whose divergence has a weight, with one that is only reported.
constexpr int kNoRef = 0, kWeighed = 1, kReported = 2;
// The arguments' structures are passed by value: by reference 4M steps take 28.4 us instead of 27.4.
// Loads that nothing stands between: of a step of the line in any case, what they hold is looked at later.
template <int REF>
__device__ __forceinline__ PolicyRow policy_fetch(LineSteps s, PolicyArgs a, float line_adv, unsigned r, unsigned hi) {
    const unsigned at = min(r, hi - 1);
    PolicyRow p{s.loss[at], a.old[at], 0.0f, line_adv, 0};
    if constexpr (REF) p.ref = a.ref[at];
    if (a.per_row) p.adv = a.adv[at];
    if (s.target) p.target = s.target[at];
    return p;
}
// The step's gradient; its value, divergence and clipping into v, kl and cut.
template <int REF>
__device__ __forceinline__ float policy_eval(PolicyRow p, Border bo, float beta, float& v, float& kl, bool& cut) {
    const double far = (double)p.old - (double)p.x;
    cut = p.adv > 0.0f ? far > bo.above : p.adv < 0.0f && far < bo.below;
    const float ratio = expf(p.old - p.x);
    // an advantage of 0 takes nothing from a ratio beyond every bound
    v = p.adv == 0.0f ? 0.0f : -(cut ? (p.adv > 0.0f ? bo.top : bo.bottom) : ratio) * p.adv;
    float slope = cut || p.adv == 0.0f ? 0.0f : ratio * p.adv;
    kl = 0.0f;
    if constexpr (REF) {
        float em1;
        exp_tail(p.x - p.ref, kl, em1);
        // a weight of 0 takes nothing from a divergence beyond every bound either
        if constexpr (REF == kWeighed) {
            v = fmaf(beta, kl, v);
            slope = fmaf(beta, em1, slope);
        }
    }
    return slope;
}
// Sums of a team's lanes over steps lo .. hi - 1; the slopes of the last turn, and which of its steps count, stay.
template <int G, int REF>
__device__ __forceinline__ Sums policy_sums(LineSteps s, PolicyArgs a, Border bo, float line_adv, unsigned lo,
                                            unsigned hi, int l, float (&slope)[kKeep], bool (&there)[kKeep]) {
    Sums sum{0.0, 0.0, 0, 0};
    for (unsigned base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = policy_fetch<REF>(s, a, line_adv, base + i * G + l, hi);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            there[i] = false;
            if (base + i * G >= hi) continue;  // the same for the team: places that no lane has a step for
            float v, kl;
            bool cut;
            slope[i] = policy_eval<REF>(p[i], bo, a.beta, v, kl, cut);
            there[i] = base + i * G + l < hi && p[i].target >= 0;
            sum.a += there[i] ? (double)v : 0.0;
            if constexpr (REF) sum.b += there[i] ? (double)kl : 0.0;
            sum.x += team_count<G>(there[i]);
            sum.y += team_count<G>(there[i] && cut);
        }
    }
    return sum;
}
__device__ __forceinline__ void policy_put(const PolicyArgs& a, float g, float share, unsigned r, unsigned hi, bool on, float d) {
    if (r < hi) a.row_grad[r] = on && g != 0.0f ? share * d : 0.0f;
}
// Gradients of steps lo .. hi - 1, each computed again.
template <int G, int REF>
__device__ __forceinline__ void policy_grads(LineSteps s, PolicyArgs a, Border bo, float line_adv, float g,
                                             float share, unsigned lo, unsigned hi, int l) {
    for (unsigned base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = policy_fetch<REF>(s, a, line_adv, base + i * G + l, hi);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            float v, kl;
            bool cut;
            const float d = policy_eval<REF>(p[i], bo, a.beta, v, kl, cut);
            policy_put(a, g, share, base + i * G + l, hi, p[i].target >= 0, d);
        }
    }
}
// The mean of `count` values; their sum may pass the largest 32-bit number where the mean does not.
__device__ __forceinline__ float mean_of(double sum, float count) {
    const float s = (float)sum;
    return __builtin_fabsf(s) < INFINITY ? s / count : (float)(sum / (double)count);
}
// A line's outputs, and what its gradients are multiplied with.
__device__ __forceinline__ float policy_line_outputs(const PolicyArgs& a, int64_t line, const Sums& sum, bool write, float* g) {
    const float count = (float)max(sum.x, 1);
    if (write) {
        if (a.loss) a.loss[line] = mean_of(sum.a, count);
        if (a.kl) a.kl[line] = mean_of(sum.b, count);
        if (a.clipped) a.clipped[line] = (float)sum.y / count;
    }
    *g = a.grad ? a.grad[line] : 1.0f;
    return *g / count;
}
template <int G, int REF>
__device__ __forceinline__ void policy_line(LineSteps s, PolicyArgs a, Border bo, int64_t line, unsigned lo,
                                            unsigned hi, int l, Sums* red) {
    const float line_adv = a.per_row ? 0.0f : a.adv[line];
    float slope[kKeep], g;
    bool there[kKeep];
    const Sums sum = team_sum<G>(policy_sums<G, REF>(s, a, bo, line_adv, lo, hi, l, slope, there), red);
    const float share = policy_line_outputs(a, line, sum, l == 0, &g);
    if (!a.row_grad) return;
    if (hi - lo <= kKeep * G) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i) policy_put(a, g, share, lo + i * G + l, hi, there[i], slope[i]);
    } else {
        policy_grads<G, REF>(s, a, bo, line_adv, g, share, lo, hi, l);
    }
}

template <int G, int REF>
__global__ __launch_bounds__(threads_of(G)) void policy_kernel(LineSteps s, PolicyArgs a, Border bo, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ Sums red[G > 64 ? G / 64 : 1];
    const int64_t line = (int64_t)blockIdx.x * TEAMS + threadIdx.x / G;
    if (line >= s.lines) return;  // G > 64: the same for the workgroup
    const unsigned lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    policy_line<G, REF>(s, a, bo, line, lo, hi, threadIdx.x % G, red);
}

// Steps of a pair whose counting a lane remembers as bits between the sums and the gradient.
constexpr int kBits = 32;

// Step t of a pair: the chosen line's steps, then the other's.
struct PairSteps {
    unsigned la, len, from_a, from_b;  // (from_b modulo 2^32)
    __device__ __forceinline__ PairSteps(const LineSteps& s, int64_t pair) {
        const unsigned o0 = clamp_row(s.off[2 * pair], s.m), o1 = clamp_row(s.off[2 * pair + 1], s.m);
        const unsigned o2 = clamp_row(s.off[2 * pair + 2], s.m);
        la = o1 > o0 ? o1 - o0 : 0;
        len = la + (o2 > o1 ? o2 - o1 : 0);
        from_a = o0;
        from_b = o1 - la;
    }
    __device__ __forceinline__ unsigned row_of(unsigned t) const { return (t < la ? from_a : from_b) + t; }
};
// Sums of a team's lanes over steps first .. last - 1 of a pair; whether a lane's first kBits steps count in `on`.
template <int G, bool REF>
__device__ __forceinline__ Sums preference_sums(const LineSteps& s, const PreferenceArgs& a, const PairSteps& ps, unsigned first,
                                                unsigned last, int l, unsigned& on) {
    Sums sum{0.0, 0.0, 0, 0};
    on = 0;
    int at = 0;
    for (unsigned base = first; base < last; base += kKeep * G) {
        float x[kKeep], ref[kKeep];
        int target[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const unsigned r = ps.row_of(min(base + i * G + l, last - 1));
            x[i] = s.loss[r];
            ref[i] = 0.0f;
            if constexpr (REF) ref[i] = a.ref[r];
            target[i] = s.target ? s.target[r] : 0;
        }
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            if (base + i * G >= last) break;  // the same for the team
            const bool there = base + i * G + l < last && target[i] >= 0;
            const double gain = there ? (double)ref[i] - (double)x[i] : 0.0;
            const bool chosen = base + i * G + l < ps.la;
            sum.a += chosen ? gain : 0.0;
            sum.b += chosen ? 0.0 : gain;
            sum.x += team_count<G>(there && chosen);
            sum.y += team_count<G>(there && !chosen);
            if (at < kBits) on |= (there ? 1u : 0u) << at;
            ++at;
        }
    }
    return sum;
}
// A pair's outputs, and the gradients of both lines' steps into da and db.
__device__ __forceinline__ void preference_pair_outputs(const PreferenceArgs& a, int64_t pair, const Sums& sum, bool write, float& da,
                                                        float& db) {
    double wa = a.beta, wb = wa;
    if (a.average) {
        // both weights from one division
        const double na = max(sum.x, 1), nb = max(sum.y, 1), each = wa / (na * nb);
        wa = each * nb;
        wb = each * na;
    }
    const double ra = wa * sum.a, rb = wb * sum.b, h = ra - rb;
    // s(-|h|) = e / (1 + e) with e = exp(-|h|), the rounding of |h| to 32 bits put back into the exponential
    const double big = __builtin_fabs(h);
    const float hf = (float)big;
    const float left = hf < INFINITY ? (float)(big - (double)hf) : 0.0f;
    const float e = expf(-hf) * (1.0f - left);
    const float small = e / (1.0f + e), large = 1.0f / (1.0f + e);
    // log(1 + e), what the sum lost put back
    const float one = 1.0f + e, soft = logf(one) + (e - (one - 1.0f)) / one;
    const float up = h >= 0.0 ? soft : hf + soft, down = h >= 0.0 ? hf + soft : soft;  // -log s(h), -log s(-h)
    const float keep = 1.0f - a.smoothing;
    if (write) {
        // a weight of 0 takes nothing from a loss beyond every bound
        if (a.loss) a.loss[pair] = a.smoothing == 0.0f ? up : keep == 0.0f ? down : fmaf(keep, up, a.smoothing * down);
        if (a.reward) {
            a.reward[2 * pair] = (float)ra;
            a.reward[2 * pair + 1] = (float)rb;
        }
    }
    if (!a.row_grad) return;
    const float g = a.grad ? a.grad[pair] : 1.0f;
    const float slope = a.smoothing * (h >= 0.0 ? large : small) - keep * (h >= 0.0 ? small : large);
    da = g == 0.0f ? 0.0f : -g * slope * (float)wa;
    db = g == 0.0f ? 0.0f : g * slope * (float)wb;
}
template <int G>
__device__ __forceinline__ void preference_grads(const LineSteps& s, const PreferenceArgs& a, const PairSteps& ps, unsigned first,
                                                 unsigned last, int l, unsigned on, float da, float db) {
    int at = 0;
    for (unsigned t = first + l; t < last; t += G, ++at) {
        const unsigned r = ps.row_of(t);
        const bool there = at < kBits ? (on >> at) & 1u : !s.target || s.target[r] >= 0;
        a.row_grad[r] = there ? (t < ps.la ? da : db) : 0.0f;
    }
}
template <int G, bool REF>
__device__ __forceinline__ void preference_pair(const LineSteps& s, const PreferenceArgs& a, const PairSteps& ps, int64_t pair, int l,
                                                Sums* red) {
    unsigned on;
    float da = 0.0f, db = 0.0f;
    const Sums sum = team_sum<G>(preference_sums<G, REF>(s, a, ps, 0, ps.len, l, on), red);
    preference_pair_outputs(a, pair, sum, l == 0, da, db);
    if (a.row_grad) preference_grads<G>(s, a, ps, 0, ps.len, l, on, da, db);
}

template <int G, bool REF>
__global__ __launch_bounds__(threads_of(G)) void preference_kernel(LineSteps s, PreferenceArgs a, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ Sums red[G > 64 ? G / 64 : 1];
    const int64_t pair = (int64_t)blockIdx.x * TEAMS + threadIdx.x / G;
    if (2 * pair >= s.lines) return;  // G > 64: the same for the workgroup
    preference_pair<G, REF>(s, a, PairSteps(s, pair), pair, threadIdx.x % G, red);
}

// ---------------------------------------------------------------- few, long lines
// Each line (or pair) is split over `parts` workgroups, in three kernels: the parts' sums, the line's outputs from
// them, the gradients.  In between the sums lie where the gradients will: each part's own first steps hold them, so
// that no workspace is needed and no part waits for another.  A line too short to split is left to the third
// kernel whole.  Without gradients there is no such place, and lines are not split.
constexpr int kWide = 256;           // lanes of a part
constexpr unsigned kLeastPart = 64;  // steps of one: above the kRecord values that it holds
constexpr int kRecord = 6;
static_assert(sizeof(Sums) == kRecord * 4);

// Part `part` of `len` steps in at most `most` parts.
struct PartOf {
    unsigned first, last;
    int count;  // parts that the steps are split in
    __device__ __forceinline__ PartOf(unsigned len, int most, int part) {
        const unsigned each = max((len + most - 1) / most, kLeastPart);
        count = (int)max(len / each, 1u);
        first = part * each;  // of part < count
        last = part + 1 == count ? len : first + each;
    }
};
// A value that the wave's lanes all loaded, its load waited for here.
__device__ __forceinline__ float read_now(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
template <typename ROW>
__device__ __forceinline__ void record_put(float* row_grad, const Sums& v, unsigned first, ROW&& row_of) {
    struct Words {
        float w[kRecord];
    };
    const Words words = __builtin_bit_cast(Words, v);
#pragma unroll
    for (int i = 0; i < kRecord; ++i) row_grad[row_of(first + i)] = words.w[i];
}
template <typename ROW>
__device__ __forceinline__ Sums record_get(const float* row_grad, unsigned first, ROW&& row_of) {
    struct Words {
        float w[kRecord];
    } words;
#pragma unroll
    for (int i = 0; i < kRecord; ++i) words.w[i] = row_grad[row_of(first + i)];
    return __builtin_bit_cast(Sums, words);
}
// The line's sums from its parts', the same in every thread; the parts are added in a fixed order.
template <typename ROW>
__device__ __forceinline__ Sums parts_sum(const float* row_grad, unsigned len, int most, int count, Sums* red, ROW&& row_of) {
    Sums v{0.0, 0.0, 0, 0};
    for (int p = threadIdx.x; p < count; p += kWide) {
        const Sums w = record_get(row_grad, PartOf(len, most, p).first, row_of);
        v.a += w.a;
        v.b += w.b;
        v.x += w.x;
        v.y += w.y;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        v.x += __shfl_xor(v.x, o, 64);
        v.y += __shfl_xor(v.y, o, 64);
    }
    return team_sum<kWide>(v, red);
}

template <int REF>
__global__ __launch_bounds__(kWide) void policy_parts_kernel(LineSteps s, PolicyArgs a, Border bo, int parts) {
    __shared__ Sums red[kWide / 64];
    const int64_t line = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const unsigned lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    const PartOf p(hi - lo, parts, part);
    if (p.count == 1 || part >= p.count) return;
    float slope[kKeep];
    bool there[kKeep];
    const Sums sum = team_sum<kWide>(policy_sums<kWide, REF>(s, a, bo, a.per_row ? 0.0f : a.adv[line], lo + p.first, lo + p.last,
                                                             threadIdx.x, slope, there),
                                     red);
    if (threadIdx.x == 0) record_put(a.row_grad, sum, p.first, [&](unsigned t) { return lo + t; });
}
__global__ __launch_bounds__(kWide) void policy_total_kernel(LineSteps s, PolicyArgs a, int parts) {
    __shared__ Sums red[kWide / 64];
    const int64_t line = blockIdx.x;
    const unsigned lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    const int count = PartOf(hi - lo, parts, 0).count;
    if (count == 1) return;
    const Sums sum = parts_sum(a.row_grad, hi - lo, parts, count, red, [&](unsigned t) { return lo + t; });
    float g;
    const float share = policy_line_outputs(a, line, sum, threadIdx.x == 0, &g);
    // (all records are read: the sum's barrier lies between)
    for (int p = threadIdx.x; p < count; p += kWide) {
        const unsigned first = lo + PartOf(hi - lo, parts, p).first;
        a.row_grad[first] = g;
        a.row_grad[first + 1] = share;
    }
}
template <int REF>
__global__ __launch_bounds__(kWide) void policy_grads_kernel(LineSteps s, PolicyArgs a, Border bo, int parts, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    __shared__ Sums red[kWide / 64];
    const int64_t line = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const unsigned lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    const PartOf p(hi - lo, parts, part);
    if (part >= p.count) return;
    if (p.count == 1) {
        policy_line<kWide, REF>(s, a, bo, line, lo, hi, threadIdx.x, red);
        return;
    }
    const float g = read_now(a.row_grad[lo + p.first]), share = read_now(a.row_grad[lo + p.first + 1]);
    __syncthreads();  // every wave has read them
    policy_grads<kWide, REF>(s, a, bo, a.per_row ? 0.0f : a.adv[line], g, share, lo + p.first, lo + p.last, threadIdx.x);
}

template <bool REF>
__global__ __launch_bounds__(kWide) void preference_parts_kernel(LineSteps s, PreferenceArgs a, int parts) {
    __shared__ Sums red[kWide / 64];
    const PairSteps ps(s, blockIdx.x / parts);
    const int part = blockIdx.x % parts;
    const PartOf p(ps.len, parts, part);
    if (p.count == 1 || part >= p.count) return;
    unsigned on;
    const Sums sum = team_sum<kWide>(preference_sums<kWide, REF>(s, a, ps, p.first, p.last, threadIdx.x, on), red);
    if (threadIdx.x == 0) record_put(a.row_grad, sum, p.first, [&](unsigned t) { return ps.row_of(t); });
}
__global__ __launch_bounds__(kWide) void preference_total_kernel(LineSteps s, PreferenceArgs a, int parts) {
    __shared__ Sums red[kWide / 64];
    const int64_t pair = blockIdx.x;
    const PairSteps ps(s, pair);
    const int count = PartOf(ps.len, parts, 0).count;
    if (count == 1) return;
    const Sums sum = parts_sum(a.row_grad, ps.len, parts, count, red, [&](unsigned t) { return ps.row_of(t); });
    float da = 0.0f, db = 0.0f;
    preference_pair_outputs(a, pair, sum, threadIdx.x == 0, da, db);
    // (all records are read: the sum's barrier lies between)
    for (int p = threadIdx.x; p < count; p += kWide) {
        const unsigned first = PartOf(ps.len, parts, p).first;
        a.row_grad[ps.row_of(first)] = da;
        a.row_grad[ps.row_of(first + 1)] = db;
    }
}
template <bool REF>
__global__ __launch_bounds__(kWide) void preference_grads_kernel(LineSteps s, PreferenceArgs a, int parts, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    __shared__ Sums red[kWide / 64];
    const int64_t pair = blockIdx.x / parts;
    const int part = blockIdx.x % parts;
    const PairSteps ps(s, pair);
    const PartOf p(ps.len, parts, part);
    if (part >= p.count) return;
    if (p.count == 1) {
        preference_pair<kWide, REF>(s, a, ps, pair, threadIdx.x, red);
        return;
    }
    const float da = read_now(a.row_grad[ps.row_of(p.first)]), db = read_now(a.row_grad[ps.row_of(p.first + 1)]);
    __syncthreads();  // every wave has read them
    for (unsigned t = p.first + threadIdx.x; t < p.last; t += kWide) {
        const unsigned r = ps.row_of(t);
        a.row_grad[r] = !s.target || s.target[r] >= 0 ? (t < ps.la ? da : db) : 0.0f;
    }
}

// Parts of a line (or pair), 1: not split.  Split where its steps keep a workgroup for longer than two more launches
// take, and there are too few of them for the GPU (policy in us, whole and split: one line of 12000 steps 17 and 16, of
// 16384 22 and 14, of 4M 5900 and 44; 64 lines of together 4M 150 and 57, 127 80 and 66, 256 47 and 71; pairs: one of
// 16384 11 and 13, of 32768 16 and 13, 64 of together 4M 73 and 36, 200 25 and 43).  Lines differ in length, so
// there are more parts where there are more lines (64 in 16 parts each: 84).
int parts_of(const float* row_grad, int64_t m, int64_t units) {
    if (!row_grad || units < 1 || units >= 128 || m / units < 16384) return 1;
    return (int)std::min({(int64_t)1024, 4096 / units, (m / units + 511) / 512});
}

// f.template operator()<G>(): the lanes of a team, by the steps that a line (or pair) has on average.
template <typename F>
int by_length(int64_t m, int64_t units, F&& f) {
    const int64_t mean = m / std::max<int64_t>(units, 1);
    if (mean <= 16) return f.template operator()<16>();
    if (mean <= 512) return f.template operator()<64>();
    if (mean <= 4096) return f.template operator()<256>();
    return f.template operator()<1024>();
}

// Workgroups that clear the steps of no line.
unsigned clear_blocks(const float* row_grad, int64_t m) {
    return row_grad ? (unsigned)std::min<int64_t>((m + 4095) / 4096, 64) : 0u;
}

template <int G>
unsigned team_blocks(int64_t units) {
    constexpr int TEAMS = threads_of(G) / G;
    return (unsigned)((units + TEAMS - 1) / TEAMS);
}

}  // namespace

int launch_policy_loss(const LineSteps& s, const PolicyArgs& a, hipStream_t st) {
    const Border bo{std::log1p((double)a.high), std::log1p(-(double)a.low), (float)(1.0 + (double)a.high),
                    (float)(1.0 - (double)a.low)};
    auto by_reference = [&](auto&& f) {
        if (!a.ref) return f.template operator()<kNoRef>();
        if (a.beta != 0.0f) return f.template operator()<kWeighed>();
        return f.template operator()<kReported>();
    };
    if (const int parts = parts_of(a.row_grad, s.m, s.lines); parts > 1) {
        const unsigned work = (unsigned)(s.lines * parts), grid = work + clear_blocks(a.row_grad, s.m);
        auto go = [&]<int REF>() {
            policy_parts_kernel<REF><<<work, kWide, 0, st>>>(s, a, bo, parts);
            PPOCR_HIP(hipGetLastError());
            policy_total_kernel<<<(unsigned)s.lines, kWide, 0, st>>>(s, a, parts);
            PPOCR_HIP(hipGetLastError());
            policy_grads_kernel<REF><<<grid, kWide, 0, st>>>(s, a, bo, parts, work);
            PPOCR_HIP(hipGetLastError());
            return (int)PPOCR_OK;
        };
        return by_reference(go);
    }
    return by_length(s.m, s.lines, [&]<int G>() {
        const unsigned work = team_blocks<G>(s.lines), grid = work + clear_blocks(a.row_grad, s.m);
        if (!grid) return (int)PPOCR_OK;
        return by_reference([&]<int REF>() {
            policy_kernel<G, REF><<<grid, threads_of(G), 0, st>>>(s, a, bo, work);
            PPOCR_HIP(hipGetLastError());
            return (int)PPOCR_OK;
        });
    });
}

int launch_preference_loss(const LineSteps& s, const PreferenceArgs& a, hipStream_t st) {
    if (const int parts = parts_of(a.row_grad, s.m, s.lines / 2); parts > 1) {
        const unsigned work = (unsigned)(s.lines / 2 * parts), grid = work + clear_blocks(a.row_grad, s.m);
        auto go = [&]<bool REF>() {
            preference_parts_kernel<REF><<<work, kWide, 0, st>>>(s, a, parts);
            PPOCR_HIP(hipGetLastError());
            preference_total_kernel<<<(unsigned)(s.lines / 2), kWide, 0, st>>>(s, a, parts);
            PPOCR_HIP(hipGetLastError());
            preference_grads_kernel<REF><<<grid, kWide, 0, st>>>(s, a, parts, work);
            PPOCR_HIP(hipGetLastError());
            return (int)PPOCR_OK;
        };
        return a.ref ? go.template operator()<true>() : go.template operator()<false>();
    }
    return by_length(s.m, s.lines / 2, [&]<int G>() {
        const unsigned work = team_blocks<G>(s.lines / 2), grid = work + clear_blocks(a.row_grad, s.m);
        if (grid) {
            if (a.ref) preference_kernel<G, true><<<grid, threads_of(G), 0, st>>>(s, a, work);
            else preference_kernel<G, false><<<grid, threads_of(G), 0, st>>>(s, a, work);
            PPOCR_HIP(hipGetLastError());
        }
        return (int)PPOCR_OK;
    });
}

}  // namespace ppocr
