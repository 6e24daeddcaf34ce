// Losses over text lines from the cross entropies of their steps (sequence_loss.hip).
#pragma once
#include "common.hpp"

namespace ppocr {

// Lines of steps, packed: line i is steps off[i] .. off[i + 1] of m, clamped into [0, m].  A step whose
// target is negative does not count (target null: all count).
struct LineSteps {
    const float* loss;      // [m] cross entropies: minus the log probabilities of the steps' classes
    const int32_t* target;  // [m] or null
    const int64_t* off;     // [lines + 1]
    int64_t lines, m;
};

struct PolicyArgs {
    const float* old;  // [m] the same under the policy that sampled the steps
    const float* ref;  // [m] under the reference, or null
    const float* adv;  // [m] (per_row) or [lines]
    int per_row;
    float low, high, beta;
    const float* grad;  // [lines] or null
    float* loss;        // the outputs may be null
    float* kl;
    float* clipped;
    float* row_grad;
};
int launch_policy_loss(const LineSteps& s, const PolicyArgs& a, hipStream_t st);

struct PreferenceArgs {
    const float* ref;  // [m] or null
    float beta, smoothing;
    int average;
    const float* grad;  // [pairs] or null
    float* loss;        // the outputs may be null
    float* reward;
    float* row_grad;
};
// s.lines is twice the number of pairs
int launch_preference_loss(const LineSteps& s, const PreferenceArgs& a, hipStream_t st);

}  // namespace ppocr
