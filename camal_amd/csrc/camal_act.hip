// camal_act.hip — host side of the 8-bit activation checkpoints: argument checks, launch shapes and the camal_act_* entry
// points.  A translation unit of its own, so that it compiles beside camal_hip.hip.
#include "camal_act.hpp"
#include "camal_act_kernels.hpp"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "../../include/camal_hip.h"

using namespace camal;

namespace {

inline bool act_channels_ok(int c) { return c == 32 || c == 64 || c == 128 || c == 256; }
inline bool act_aligned(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }
inline bool act_format_ok(int f) { return f == CAMAL_ACT_INT8 || f == CAMAL_ACT_E4M3; }

// Run-time choices as template arguments: f(constant ...)
template <typename Fn>
int with_format(int format, Fn&& f) { return format == CAMAL_ACT_INT8 ? f(ActI8()) : f(ActE4M3()); }
template <typename Fn>
int with_flag(bool b, Fn&& f) { return b ? f(std::true_type()) : f(std::false_type()); }
template <typename Fn>
int with_channels(int c, Fn&& f) {
    switch (c) {
        case 32: return f(std::integral_constant<int, 32>());
        case 64: return f(std::integral_constant<int, 64>());
        case 128: return f(std::integral_constant<int, 128>());
        case 256: return f(std::integral_constant<int, 256>());
    }
    return fail(CAMAL_ERR_ARG, "channels must be 32, 64, 128 or 256");
}

// What the entry points share: the shape, null pointers, alignment of the float rows (16-byte loads) and of the rest (4-byte)
int act_check(std::initializer_list<const void*> floats, std::initializer_list<const void*> words,
              std::initializer_list<const void*> bytes, long long rows, int channels, int format) {
    if (rows < 1 || rows > ACT_MAX_ROWS) return fail(CAMAL_ERR_ARG, "the number of rows must be in 1 .. 2^31 - 4096");
    if (!act_channels_ok(channels)) return fail(CAMAL_ERR_ARG, "channels must be 32, 64, 128 or 256");
    if (!act_format_ok(format)) return fail(CAMAL_ERR_ARG, "format must be CAMAL_ACT_INT8 or CAMAL_ACT_E4M3");
    for (const void* p : floats) {
        if (!p) return fail(CAMAL_ERR_ARG, "null argument");
        if (!act_aligned(p, 16)) return fail(CAMAL_ERR_ARG, "float tensors must be 16-byte aligned");
    }
    for (const void* p : words) {
        if (!p) return fail(CAMAL_ERR_ARG, "null argument");
        if (!act_aligned(p, 4)) return fail(CAMAL_ERR_ARG, "codes must be 4-byte aligned");
    }
    for (const void* p : bytes)
        if (!p) return fail(CAMAL_ERR_ARG, "null argument");
    return 0;
}

inline int act_blocks(size_t work, size_t per_block, int cap) { return (int)std::min<size_t>((work + per_block - 1) / per_block, (size_t)cap); }

// whether an fp32 output of n4 quads goes past the L3
inline bool act_streams(size_t n4) { return n4 * 16 >= ACT_STREAM_BYTES; }

inline size_t act_bwd_blocks(size_t rows) { return std::min<size_t>((rows + ACT_BWD_ROWS - 1) / ACT_BWD_ROWS, ACT_BWD_BLOCKS); }

template <typename F, int C, bool RELU, bool BCAST>
int act_norm_bwd_impl(hipStream_t s, const float* da, ActCodes k, const float* invstd, const float* gamma, const float* beta, int N,
                      int L, float* dz, float* dgamma, float* dbeta, void* ws) {
    if (N <= ACT_SMALL_ROWS) {
        hipLaunchKernelGGL((act_bwd_small_kernel<F, RELU, BCAST>), dim3(C / 32), dim3(1024), 0, s, da, k.codes, k.scales, invstd, gamma,
                           beta, N, L, C, dz, dgamma, dbeta);
        HIP_TRY(hipGetLastError());
        return 0;
    }
    const int nb = (int)act_bwd_blocks(N);
    double* partial = (double*)ws;
    float* means = (float*)(partial + (size_t)nb * C * 2);
    const size_t n4 = (size_t)N * (C / 4);
    hipLaunchKernelGGL((act_bwd_partial_kernel<F, C, RELU, BCAST>), dim3(nb), dim3(256), 0, s, da, k.codes, k.scales, gamma, beta, N,
                       L, partial);
    hipLaunchKernelGGL(act_bwd_final_kernel<C>, dim3(C / ACT_FINAL_CPB), dim3(ACT_FINAL_THREADS), 0, s, partial, nb, N, means,
                       dgamma, dbeta);
    with_flag(act_streams(n4), [&](auto st) {
        hipLaunchKernelGGL((act_bwd_apply_kernel<F, C, RELU, BCAST, decltype(st)::value>), dim3(act_blocks(n4, 256, 4096)), dim3(256), 0,
                           s, da, k.codes, k.scales, invstd, gamma, beta, means, n4, L, dz);
        return 0;
    });
    HIP_TRY(hipGetLastError());
    return 0;
}

// How the weight gradient is cut up, fixed by the shapes alone: the sums have the same order on every call.
// Tap groups of nearly equal size (9 = 5 + 4, 25 = 7 + 6 + 6 + 6); splits for one workgroup on each of 256 CUs.  (Two ci tiles
// a wave, which halves the cutting of dz, is slower where the taps leave room for it: 3 taps on 128 x 510, 128 -> 128 channels
// 31.0 instead of 27.8 us, 64 -> 64 19.2 instead of 16.0.)
// A long call gets gx of them at a time, one set after the other (the tiles of a set read the same rows), so that a wave's chain of
// fp32 sums stays near ACT_CHAIN_ROWS rows: twice that at most, where long and short units alternate.  A matrix product cuts its
// sum off instead of rounding it, an error of one sign that grows with the chain: dz and input of one sign, 100 x 10080, 256 -> 256
// channels, 63 taps 1.3e-4 in two chains and 2.6e-6 here (a plain fp32 product 2.0e-6).  us, one set of longer chains / sets of
// 8192 / 4096 rows: that case 24600 / 17430 / 17840 (one set leaves CUs idle); 7 taps, 400 x 10080, 128 -> 128: 1957 / 2024 / 2064;
// 3 taps, 800 x 10080, 256 -> 256: 9480 / 9260 / 9330.
// CO = co tiles of a workgroup, as many as there are up to 4: they share the decoding of their input.  (Two of four tiles leave
// half the partial sums: 25 taps on 37 x 333 33.4 instead of 34.4 us, but 20.7 instead of 20.3 for one tap on 128 x 510 and 186
// instead of 177 for 7 taps on 8 x 10080.)
ActPlan act_wgrad_plan(int B, int L, int cin, int cout, int ks) {
    ActPlan p;
    p.B = ks == 1 ? 1 : B;  // one tap knows no window edges
    p.L = ks == 1 ? B * L : L;
    p.groups = (ks + ACT_TAPS - 1) / ACT_TAPS;
    const int base = ks / p.groups, rem = ks % p.groups;
    p.nhi = rem ? base + 1 : base;
    p.n_hi = rem ? rem : p.groups;
    const int total = p.B * ((p.L + ACT_UNIT - 1) / ACT_UNIT);
    p.co = std::min(4, cout / 32);
    const int tiles = p.groups * (cin / 32) * (cout / (32 * p.co)), wk = ACT_WAVES / p.co;
    p.gx = std::min(std::max(1, 256 / tiles), (total + wk - 1) / wk);
    const long long rows = (long long)p.gx * wk * ACT_CHAIN_ROWS;
    p.want = p.gx * (int)(((long long)p.B * p.L + rows - 1) / rows);
    p.units = (total + p.want - 1) / p.want;
    p.nsplit = (total + p.units - 1) / p.units;
    if (p.want == p.gx) p.gx = p.nsplit;
    p.nsplit = (p.nsplit + p.gx - 1) / p.gx * p.gx;  // at most want, which never falls as B and L grow
    return p;
}

}  // namespace

int camal::act_write(hipStream_t s, const float* z, ActNorm n, bool relu, const float* zr, ActNorm nr, size_t rows, int channels,
                     int format, float* out, ActCodes k, ActCodes kr) {
    const size_t n4 = rows * (size_t)(channels / 4);
    with_format(format, [&](auto f) { return with_flag(relu, [&](auto re) { return with_flag(zr != nullptr, [&](auto res) {
        hipLaunchKernelGGL((act_write_kernel<decltype(f), decltype(re)::value, decltype(res)::value>),
                           dim3(act_blocks(n4, 256 * ACT_ROWS, 4096)), dim3(256), 0, s, z, n, zr, nr, out, k.codes, k.scales,
                           kr.codes, kr.scales, n4, channels / 4 - 1);
        return 0;
    }); }); });
    HIP_TRY(hipGetLastError());
    return 0;
}

int camal::act_read(hipStream_t s, const ActIn& in, size_t rows, int channels, float* out) {
    const size_t n4 = rows * (size_t)(channels / 4);
    with_format(in.e4m3 ? CAMAL_ACT_E4M3 : CAMAL_ACT_INT8, [&](auto f) {
        auto launch = [&](auto affine, auto relu, auto res) {
            hipLaunchKernelGGL((act_read_kernel<decltype(f), decltype(affine)::value, decltype(relu)::value, decltype(res)::value>),
                               dim3(act_blocks(n4, 256, 4096)), dim3(256), 0, s, in.codes, in.scales, in.gamma, in.beta, in.codes_r,
                               in.scales_r, in.gamma_r, in.beta_r, out, n4, channels / 4 - 1);
            return 0;
        };
        if (!in.gamma) return launch(std::false_type(), std::false_type(), std::false_type());
        return with_flag(in.relu != 0, [&](auto relu) {
            return with_flag(in.codes_r != nullptr, [&](auto res) { return launch(std::true_type(), relu, res); }); });
    });
    HIP_TRY(hipGetLastError());
    return 0;
}

// partial sums [blocks][channels][2] in 64 bits, then the two rows of means
size_t camal::act_norm_bwd_bytes(size_t rows, int channels) {
    return act_bwd_blocks(rows) * channels * 2 * sizeof(double) + 2 * (size_t)channels * sizeof(float);
}

int camal::act_norm_bwd(hipStream_t s, const float* da, bool pooled, ActCodes k, int format, int B, int L, int channels,
                        const float* invstd, const float* gamma, const float* beta, bool relu, float* dz, float* dgamma,
                        float* dbeta, void* ws) {
    return with_format(format, [&](auto f) { return with_channels(channels, [&](auto c) { return with_flag(relu, [&](auto re) {
        return with_flag(pooled, [&](auto po) {
            return act_norm_bwd_impl<decltype(f), decltype(c)::value, decltype(re)::value, decltype(po)::value>(
                s, da, k, invstd, gamma, beta, B * L, L, dz, dgamma, dbeta, ws);
        }); }); }); });
}

size_t camal::act_wgrad_bytes(int B, int L, int cin, int cout, int ks) {
    const ActPlan p = act_wgrad_plan(B, L, cin, cout, ks);
    return (size_t)p.nsplit * ks * cout * cin * sizeof(float);
}

size_t camal::act_wgrad_max_bytes(int B, int L, int cin, int cout, int ks) {
    const ActPlan p = act_wgrad_plan(B, L, cin, cout, ks);
    return (size_t)p.want * ks * cout * cin * sizeof(float);
}

int camal::act_wgrad(hipStream_t s, const float* dz, const ActIn& in, int B, int L, int cin, int cout, int ks, float* dw,
                     float* bias_grad, float* part) {
    const ActPlan p = act_wgrad_plan(B, L, cin, cout, ks);
    const bool direct = p.nsplit == 1;
    float* sums = direct ? dw : part;
    const ActOut out = direct ? ActOut{0, 1, cin * ks, ks} : ActOut{cout * cin * ks, cout * cin, cin, 1};
    const auto launch = p.co == 4 ? act_wgrad_launch<4> : (p.co == 2 ? act_wgrad_launch<2> : act_wgrad_launch<1>);
    if (int r = launch(s, p, dz, in, sums, out, bias_grad, cin, cout, ks)) return r;
    if (direct) return 0;
    const int quads = cout * cin * ks / 4;
    hipLaunchKernelGGL(act_wgrad_reduce_kernel, dim3((quads + 15) / 16), dim3(256), 0, s, part, p.nsplit, cout, cin, ks, dw);
    HIP_TRY(hipGetLastError());
    return 0;
}

extern "C" {

int camal_act_write(const float* z, const float* mean, const float* invstd, const float* gamma, const float* beta, int relu,
                    const float* zr, const float* mean_r, const float* invstd_r, const float* gamma_r, const float* beta_r,
                    long long rows, int channels, int format, float* out, void* codes, unsigned char* scales, void* codes_r,
                    unsigned char* scales_r, void* stream) {
    if (int r = act_check({z, mean, invstd, gamma, beta, out}, {codes}, {scales}, rows, channels, format)) return r;
    if (zr)
        if (int r = act_check({mean_r, invstd_r, gamma_r, beta_r, zr}, {codes_r}, {scales_r}, rows, channels, format)) return r;
    return act_write((hipStream_t)stream, z, {mean, invstd, gamma, beta}, relu != 0, zr, {mean_r, invstd_r, gamma_r, beta_r},
                     (size_t)rows, channels, format, out, {(unsigned*)codes, scales}, {(unsigned*)codes_r, scales_r});
}

int camal_act_read(const void* codes, const unsigned char* scales, int format, long long rows, int channels, const float* gamma,
                   const float* beta, int relu, const void* codes_r, const unsigned char* scales_r, const float* gamma_r,
                   const float* beta_r, float* out, void* stream) {
    if (int r = act_check({out}, {codes}, {scales}, rows, channels, format)) return r;
    if ((gamma != nullptr) != (beta != nullptr)) return fail(CAMAL_ERR_ARG, "gamma and beta come together");
    if (!gamma && (relu || codes_r)) return fail(CAMAL_ERR_ARG, "the activation needs gamma and beta");
    if (gamma)
        if (int r = act_check({gamma, beta}, {}, {}, rows, channels, format)) return r;
    if (codes_r)
        if (int r = act_check({gamma_r, beta_r}, {codes_r}, {scales_r}, rows, channels, format)) return r;
    return act_read((hipStream_t)stream,
                    {(const unsigned*)codes, scales, gamma, beta, (const unsigned*)codes_r, scales_r, gamma_r, beta_r,
                     format == CAMAL_ACT_E4M3, relu != 0, 0},
                    (size_t)rows, channels, out);
}

size_t camal_act_norm_bwd_workspace_bytes(long long rows, int channels) {
    return rows < 1 || rows > ACT_MAX_ROWS || !act_channels_ok(channels) ? 0 : act_norm_bwd_bytes((size_t)rows, channels);
}

int camal_act_norm_bwd(const float* da, int pooled, const void* codes, const unsigned char* scales, int format, int B, int L,
                       int channels, const float* invstd, const float* gamma, const float* beta, int relu, float* dz,
                       float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, void* stream) {
    if (B < 1 || L < 1) return fail(CAMAL_ERR_ARG, "B and L must be >= 1");
    const long long rows = (long long)B * L;
    if (int r = act_check({da, invstd, gamma, beta, dz, workspace}, {codes, dgamma, dbeta}, {scales}, rows, channels, format)) return r;
    if (workspace_bytes < act_norm_bwd_bytes((size_t)rows, channels))
        return fail(CAMAL_ERR_ARG, "workspace smaller than camal_act_norm_bwd_workspace_bytes(B * L, channels)");
    return act_norm_bwd((hipStream_t)stream, da, pooled != 0, {(unsigned*)codes, (unsigned char*)scales}, format, B, L, channels, invstd,
                        gamma, beta, relu != 0, dz, dgamma, dbeta, workspace);
}

static bool act_wgrad_shape_ok(int B, int L, int cin, int cout, int ks) {
    return B >= 1 && L >= 1 && (long long)B * L <= ACT_MAX_ROWS && act_channels_ok(cin) && act_channels_ok(cout) && ks >= 1 && ks <= 63 && (ks & 1);
}

size_t camal_act_wgrad_workspace_bytes(int B, int L, int cin, int cout, int ks) {
    return act_wgrad_shape_ok(B, L, cin, cout, ks) ? act_wgrad_bytes(B, L, cin, cout, ks) : 0;
}

int camal_act_wgrad(const float* dz, const void* codes, const unsigned char* scales, int format, int B, int L, int cin, int cout,
                    int ks, const float* gamma, const float* beta, int relu, const void* codes_r, const unsigned char* scales_r,
                    const float* gamma_r, const float* beta_r, int zero_pad, float* dw, void* workspace, size_t workspace_bytes,
                    void* stream) {
    if (!act_wgrad_shape_ok(B, L, cin, cout, ks))
        return fail(CAMAL_ERR_ARG, "B, L >= 1, cin and cout in {32, 64, 128, 256}, ks odd and in 1..63");
    const long long rows = (long long)B * L;
    if (int r = act_check({dz, gamma, beta, workspace}, {codes, dw}, {scales}, rows, cin, format)) return r;
    if (codes_r)
        if (int r = act_check({gamma_r, beta_r}, {codes_r}, {scales_r}, rows, cin, format)) return r;
    if (workspace_bytes < act_wgrad_bytes(B, L, cin, cout, ks))
        return fail(CAMAL_ERR_ARG, "workspace smaller than camal_act_wgrad_workspace_bytes(B, L, cin, cout, ks)");
    return act_wgrad((hipStream_t)stream, dz,
                     {(const unsigned*)codes, scales, gamma, beta, (const unsigned*)codes_r, scales_r, gamma_r, beta_r,
                      format == CAMAL_ACT_E4M3, relu != 0, zero_pad != 0},
                     B, L, cin, cout, ks, dw, nullptr, (float*)workspace);
}

}  // extern "C"
