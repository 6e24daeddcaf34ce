// Losses over text lines from the cross entropies of their steps, x = loss[r] = -log p(class of step r).
//
//   policy      rho = exp(old - x), v = -min(rho A, clip(rho, 1 - low, 1 + high) A) + beta (e^t - t - 1)
//               with t = x - ref; a line's loss is the mean of v over its steps that count, and
//               dv/dx = rho A where the clipped product is not the smaller one, + beta (e^t - 1)
//   preference  R = w sum (ref - x) over a line's steps that count (w: beta, over their number for means),
//               h = R of the chosen line - R of the other, L = -(1 - e) log s(h) - e log s(-h) with the
//               logistic s, dL/dh = e s(h) - (1 - e) s(-h), dR/dx = -w
//
// Memory bound: each step's values are read once and its gradient written once.  A team of G lanes takes
// a line (or a pair of lines): the sums go through the team in a fixed order, and the gradient, which needs
// them, is written from what the lanes kept in registers; the steps beyond them are read again.
// Sums are held in 64 bits.
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

// Sums over the lanes of a team, the same in each lane.  For G > 64 through LDS, every lane of the
// workgroup (one team) calling it.
template <int G>
__device__ __forceinline__ Sums team_sum(Sums v, Sums* red) {
#pragma unroll
    for (int o = (G < 64 ? G : 64) / 2; o >= 1; o >>= 1) {
        v.a += __shfl_xor(v.a, o, 64);
        v.b += __shfl_xor(v.b, o, 64);
        v.x += __shfl_xor(v.x, o, 64);
        v.y += __shfl_xor(v.y, o, 64);
    }
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

__device__ __forceinline__ int64_t clamp_row(int64_t r, int64_t m) { return r < 0 ? 0 : r > m ? m : r; }

// The steps that no line covers have no gradient: workgroup `part` of `parts` clears its share.
__device__ __forceinline__ void clear_uncovered(const LineSteps& s, float* row_grad, int part, int parts) {
    int64_t first = s.m, last = s.m;
    if (s.lines > 0) {
        first = clamp_row(s.off[0], s.m);
        last = max(clamp_row(s.off[s.lines], s.m), first);
    }
    const int64_t step = (int64_t)parts * blockDim.x;
    for (int64_t r = (int64_t)part * blockDim.x + threadIdx.x; r < first; r += step) row_grad[r] = 0.0f;
    for (int64_t r = last + (int64_t)part * blockDim.x + threadIdx.x; r < s.m; r += step) row_grad[r] = 0.0f;
}

// e^t - t - 1 to a few units of the last place: near 0 by its series, whose terms up to t^13 / 13! leave
// less than 2^-26 of the value at |t| = 1, as the difference would lose all of it.
__device__ __forceinline__ float exp_tail(float t, float em1) {
    if (__builtin_fabsf(t) >= 1.0f) return em1 - t;
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
    return p * t * t;
}

struct PolicyRow {
    float x, old, ref, adv;
    bool there;
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
    const int64_t lo = clamp_row(s.off[line], s.m), hi = max(clamp_row(s.off[line + 1], s.m), lo);
    const float line_adv = a.per_row ? 0.0f : a.adv[line];

    auto fetch = [&](int64_t r) {
        PolicyRow p{0.0f, 0.0f, 0.0f, line_adv, false};
        if (r < hi) {
            p.there = !s.target || s.target[r] >= 0;
            p.x = s.loss[r];
            p.old = a.old[r];
            if constexpr (REF) p.ref = a.ref[r];
            if (a.per_row) p.adv = a.adv[r];
        }
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
            const float t = p.x - p.ref, em1 = expm1f(t);
            kl = exp_tail(t, em1);
            v = fmaf(a.beta, kl, v);
            slope = fmaf(a.beta, em1, slope);
        }
        return slope;
    };

    Sums sum{0.0, 0.0, 0, 0};
    float slope[kKeep];
    bool there[kKeep];
    for (int64_t base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = fetch(base + i * G + l);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            float v, kl;
            bool cut;
            slope[i] = eval(p[i], v, kl, cut);
            there[i] = p[i].there;
            if (there[i]) {
                sum.a += (double)v;
                sum.b += (double)kl;
                sum.x += 1;
                sum.y += cut ? 1 : 0;
            }
        }
    }
    sum = team_sum<G>(sum, red);
    const float count = (float)max(sum.x, 1);
    if (l == 0) {
        if (a.loss) a.loss[line] = (float)(sum.a / (double)count);
        if (a.kl) a.kl[line] = (float)(sum.b / (double)count);
        if (a.clipped) a.clipped[line] = (float)sum.y / count;
    }
    if (!a.row_grad) return;
    const float g = a.grad ? a.grad[line] : 1.0f;
    const float share = g / count;
    auto put = [&](int64_t r, bool on, float d) {
        if (r < hi) a.row_grad[r] = on && g != 0.0f ? share * d : 0.0f;
    };
    if (hi - lo <= kKeep * G) {
#pragma unroll
        for (int i = 0; i < kKeep; ++i) put(lo + i * G + l, there[i], slope[i]);
        return;
    }
    for (int64_t base = lo; base < hi; base += kKeep * G) {
        PolicyRow p[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) p[i] = fetch(base + i * G + l);
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            float v, kl;
            bool cut;
            put(base + i * G + l, p[i].there, eval(p[i], v, kl, cut));
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
    const int64_t o0 = clamp_row(s.off[2 * pair], s.m), o1 = clamp_row(s.off[2 * pair + 1], s.m);
    const int64_t o2 = clamp_row(s.off[2 * pair + 2], s.m);
    // step t of the pair: the chosen line's steps, then the other's
    const int64_t la = max(o1 - o0, (int64_t)0), len = la + max(o2 - o1, (int64_t)0);
    auto row_of = [&](int64_t t) { return t < la ? o0 + t : o1 + (t - la); };
    Sums sum{0.0, 0.0, 0, 0};
    unsigned on = 0;
    int at = 0;
    for (int64_t base = 0; base < len; base += kKeep * G) {
        float x[kKeep], ref[kKeep];
        bool there[kKeep];
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const int64_t t = base + i * G + l;
            x[i] = ref[i] = 0.0f;
            there[i] = false;
            if (t < len) {
                const int64_t r = row_of(t);
                there[i] = !s.target || s.target[r] >= 0;
                x[i] = s.loss[r];
                if constexpr (REF) ref[i] = a.ref[r];
            }
        }
#pragma unroll
        for (int i = 0; i < kKeep; ++i) {
            const double gain = there[i] ? (double)ref[i] - (double)x[i] : 0.0;
            if (base + i * G + l < la) {
                sum.a += gain;
                sum.x += there[i] ? 1 : 0;
            } else {
                sum.b += gain;
                sum.y += there[i] ? 1 : 0;
            }
            if (at < kBits) on |= (there[i] ? 1u : 0u) << at;
            ++at;
        }
    }
    sum = team_sum<G>(sum, red);
    const double wa = a.average ? (double)a.beta / max(sum.x, 1) : (double)a.beta;
    const double wb = a.average ? (double)a.beta / max(sum.y, 1) : (double)a.beta;
    const double ra = wa * sum.a, rb = wb * sum.b, h = ra - rb;
    // s(-|h|) = e / (1 + e) with e = exp(-|h|), the rounding of |h| to 32 bits put back into the exponential
    const double big = __builtin_fabs(h);
    const float hf = (float)big;
    const float left = hf < INFINITY ? (float)(big - (double)hf) : 0.0f;
    const float e = expf(-hf) * (1.0f - left);
    const float small = e / (1.0f + e), large = 1.0f / (1.0f + e);
    const float soft = log1pf(e);
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
    for (int64_t t = l; t < len; t += G, ++at) {
        const int64_t r = row_of(t);
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
