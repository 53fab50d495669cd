// camal_act.hpp — the 8-bit activation checkpoints as the library's other parts call them: the camal_act_* entry points of
// include/camal_hip.h without their checks.
#pragma once
#include "camal_common.hpp"

namespace camal {

// rows of one call: row indices are 32-bit and run up to a tile past the last
constexpr long long ACT_MAX_ROWS = (1LL << 31) - 4096;

// A train-mode BatchNorm: batch statistics, scale and shift
struct ActNorm {
    const float *mean, *invstd, *gamma, *beta;
};

// A checkpoint's two tensors
struct ActCodes {
    unsigned* codes = nullptr;
    unsigned char* scales = nullptr;
};

// A layer's input held as checkpoint(s); codes_r null: no skip branch
struct ActIn {
    const unsigned* codes; const unsigned char* scales; const float *gamma, *beta;
    const unsigned* codes_r; const unsigned char* scales_r; const float *gamma_r, *beta_r;
    int e4m3, relu, zero_pad;
};

// How the weight gradient is cut up: windows B of L steps (one tap: all rows as one window), co co tiles per workgroup, tap groups
// (the first n_hi take nhi taps, the others nhi - 1), splits of `units` units each, gx of them side by side.  want = the splits
// aimed at, at least nsplit
struct ActPlan { int B, L, co, groups, n_hi, nhi, nsplit, units, want, gx; };
#define ACT_UNIT 64   // timesteps of a unit
#define ACT_WAVES 8   // waves of a workgroup
// Taps a wave takes at most.  With 8 their accumulators leave too few registers for the rest: 23 to 71 spilled, with 7 none, 8 or
// 26 (four, two, one co tile).  15 taps as 5 + 5 + 5 / as 8 + 7, us: 64 -> 128 channels, 37 x 333: 21.5 / 26.5; 128 x 510: 55.8 / 58.4; 64 -> 64, 128 x 510: 36.0 / 33.8.
#define ACT_TAPS 7

// Rows that a wave sums in one chain (plan: camal_act.hip)
#define ACT_CHAIN_ROWS 4096

// Where the sums go, in floats: partial sums [split][tap][co][ci], or with one split the gradient [co][ci][tap] itself
struct ActOut { int split, tap, co, ci; };

template <int CO>  // 1, 2 or 4
int act_wgrad_launch(hipStream_t s, const ActPlan& p, const float* dz, const ActIn& in, float* sums, ActOut out, float* bias_grad, int cin,
                     int cout, int ks);

// zr null: no skip branch
int act_write(hipStream_t s, const float* z, ActNorm n, bool relu, const float* zr, ActNorm nr, size_t rows, int channels, int format,
              float* out, ActCodes kept, ActCodes kept_r);
// gamma null: the normalised values
int act_read(hipStream_t s, const ActIn& in, size_t rows, int channels, float* out);

size_t act_norm_bwd_bytes(size_t rows, int channels);
int act_norm_bwd(hipStream_t s, const float* da, bool pooled, ActCodes kept, int format, int B, int L, int channels,
                 const float* invstd, const float* gamma, const float* beta, bool relu, float* dz, float* dgamma, float* dbeta,
                 void* workspace);

// bytes of partial sums for one shape, and for any shape of at most B windows of at most L steps
size_t act_wgrad_bytes(int B, int L, int cin, int cout, int ks);
size_t act_wgrad_max_bytes(int B, int L, int cin, int cout, int ks);
// bias_grad [cout] is set to 0 (null: not written)
int act_wgrad(hipStream_t s, const float* dz, const ActIn& in, int B, int L, int cin, int cout, int ks, float* dw, float* bias_grad,
              float* part);

}  // namespace camal
