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
// 4M steps in 32768 lines under a policy loss, 101 MB: 27.4 us, 3.7 TB/s (a copy: 5.1); in 16384 pairs, 68 MB: 19.8 us.
// Vector instructions bound both: some 400 a wave of 64 lanes and 4 steps a lane (the exponentials, the sums in 64 bits,
// the clipping's border), which is why loads are held back by nothing and sums use the registers' lane paths (34 and
// 22 us with shuffles and branches around the loads).  Small calls are bound by the launch: a page's 2245 steps 4 us.
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

template <int G, bool REF>
__global__ __launch_bounds__(threads_of(G)) void policy_kernel(LineSteps s, PolicyArgs a, Border bo, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ Sums red[G > 64 ? G / 64 : 1];
    const int l = threadIdx.x % G;
    const int64_t line = (int64_t)blockIdx.x * TEAMS + threadIdx.x / G;
    if (line >= s.lines) return;  // G > 64: the same for the workgroup
    const unsigned lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    const float line_adv = a.per_row ? 0.0f : a.adv[line];

    // loads that nothing stands between: of a step of the line in any case, what they hold is looked at later
    auto fetch = [&](unsigned r) {
        const unsigned at = min(r, hi - 1);
        PolicyRow p{s.loss[at], a.old[at], 0.0f, line_adv, 0};
        if constexpr (REF) p.ref = a.ref[at];
        if (a.per_row) p.adv = a.adv[at];
        if (s.target) p.target = s.target[at];
        return p;
    };
    // the step's gradient; its value, divergence and clipping into v, kl and cut
    auto eval = [&](const PolicyRow& p, float& v, float& kl, bool& cut) {
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
            v = fmaf(a.beta, kl, v);
            slope = fmaf(a.beta, em1, slope);
        }
        return slope;
    };

    Sums sum{0.0, 0.0, 0, 0};
    float slope[kKeep];
    bool there[kKeep];
    for (unsigned base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = fetch(base + i * G + l);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            there[i] = false;
            if (base + i * G >= hi) continue;  // the same for the team: places that no lane has a step for
            float v, kl;
            bool cut;
            slope[i] = eval(p[i], v, kl, cut);
            there[i] = base + i * G + l < hi && p[i].target >= 0;
            sum.a += there[i] ? (double)v : 0.0;
            if constexpr (REF) sum.b += there[i] ? (double)kl : 0.0;
            sum.x += team_count<G>(there[i]);
            sum.y += team_count<G>(there[i] && cut);
        }
    }
    sum = team_sum<G>(sum, red);
    const float count = (float)max(sum.x, 1);
    if (l == 0) {
        if (a.loss) a.loss[line] = (float)sum.a / count;
        if (a.kl) a.kl[line] = (float)sum.b / count;
        if (a.clipped) a.clipped[line] = (float)sum.y / count;
    }
    if (!a.row_grad) return;
    const float g = a.grad ? a.grad[line] : 1.0f;
    const float share = g / count;
    auto put = [&](unsigned r, bool on, float d) {
        if (r < hi) a.row_grad[r] = on && g != 0.0f ? share * d : 0.0f;
    };
    if (hi - lo <= kKeep * G) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i) put(lo + i * G + l, there[i], slope[i]);
        return;
    }
    for (unsigned base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = fetch(base + i * G + l);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            float v, kl;
            bool cut;
            put(base + i * G + l, p[i].target >= 0, eval(p[i], v, kl, cut));
        }
    }
}

// Steps of a pair whose counting a lane remembers as bits between the sums and the gradient.
constexpr int kBits = 32;

template <int G, bool REF>
__global__ __launch_bounds__(threads_of(G)) void preference_kernel(LineSteps s, PreferenceArgs a, unsigned work_blocks) {
    if (blockIdx.x >= work_blocks) {
        clear_uncovered(s, a.row_grad, (int)(blockIdx.x - work_blocks), (int)(gridDim.x - work_blocks));
        return;
    }
    constexpr int TEAMS = threads_of(G) / G;
    __shared__ Sums red[G > 64 ? G / 64 : 1];
    const int l = threadIdx.x % G;
    const int64_t pair = (int64_t)blockIdx.x * TEAMS + threadIdx.x / G;
    if (2 * pair >= s.lines) return;  // G > 64: the same for the workgroup
    const unsigned o0 = clamp_row(s.off[2 * pair], s.m), o1 = clamp_row(s.off[2 * pair + 1], s.m);
    const unsigned o2 = clamp_row(s.off[2 * pair + 2], s.m);
    // step t of the pair: the chosen line's steps, then the other's
    const unsigned la = o1 > o0 ? o1 - o0 : 0, len = la + (o2 > o1 ? o2 - o1 : 0);
    const unsigned from_a = o0, from_b = o1 - la;  // (modulo 2^32)
    auto row_of = [&](unsigned t) { return (t < la ? from_a : from_b) + t; };
    Sums sum{0.0, 0.0, 0, 0};
    unsigned on = 0;
    int at = 0;
    for (unsigned base = 0; base < len; base += kKeep * G) {
        float x[kKeep], ref[kKeep];
        int target[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const unsigned r = row_of(min(base + i * G + l, len - 1));
            x[i] = s.loss[r];
            ref[i] = 0.0f;
            if constexpr (REF) ref[i] = a.ref[r];
            target[i] = s.target ? s.target[r] : 0;
        }
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            if (base + i * G >= len) break;  // the same for the team
            const bool there = base + i * G + l < len && target[i] >= 0;
            const double gain = there ? (double)ref[i] - (double)x[i] : 0.0;
            const bool chosen = base + i * G + l < la;
            sum.a += chosen ? gain : 0.0;
            sum.b += chosen ? 0.0 : gain;
            sum.x += team_count<G>(there && chosen);
            sum.y += team_count<G>(there && !chosen);
            if (at < kBits) on |= (there ? 1u : 0u) << at;
            ++at;
        }
    }
    sum = team_sum<G>(sum, red);
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
    if (l == 0) {
        if (a.loss) a.loss[pair] = a.smoothing == 0.0f ? up : fmaf(keep, up, a.smoothing * down);
        if (a.reward) {
            a.reward[2 * pair] = (float)ra;
            a.reward[2 * pair + 1] = (float)rb;
        }
    }
    if (!a.row_grad) return;
    const float g = a.grad ? a.grad[pair] : 1.0f;
    const float slope = a.smoothing * (h >= 0.0 ? large : small) - keep * (h >= 0.0 ? small : large);
    const float da = g == 0.0f ? 0.0f : -g * slope * (float)wa, db = g == 0.0f ? 0.0f : g * slope * (float)wb;
    at = 0;
    for (unsigned t = l; t < len; t += G, ++at) {
        const unsigned r = row_of(t);
        const bool there = at < kBits ? (on >> at) & 1u : !s.target || s.target[r] >= 0;
        a.row_grad[r] = there ? (t < la ? da : db) : 0.0f;
    }
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
    return by_length(s.m, s.lines, [&]<int G>() {
        const unsigned work = team_blocks<G>(s.lines), grid = work + clear_blocks(a.row_grad, s.m);
        if (grid) {
            if (a.ref) policy_kernel<G, true><<<grid, threads_of(G), 0, st>>>(s, a, bo, work);
            else policy_kernel<G, false><<<grid, threads_of(G), 0, st>>>(s, a, bo, work);
            PPOCR_HIP(hipGetLastError());
        }
        return (int)PPOCR_OK;
    });
}

int launch_preference_loss(const LineSteps& s, const PreferenceArgs& a, hipStream_t st) {
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
