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
