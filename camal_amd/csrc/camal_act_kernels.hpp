// camal_act_kernels.hpp — gfx950 device code of the 8-bit activation checkpoints: what the training step keeps of its
// forward pass for its backward pass.
//
// A checkpoint holds the normalised values x = (z - mean) * invstd of one BatchNorm, [row][channel], as 8-bit codes, and
// one scale byte e per 32 channels of a row: value = code * 2^(e - 127).  The scale is the smallest power of two under
// which the block's largest |x| fits the format (int8: 127, e4m3: 448), so a code is exact in bf16 and x needs no
// division.  A block with an infinity, a NaN or a value beyond largest code * 2^121 (int8) or 2^119 (e4m3) has e = 255 and
// codes 0: it reads back as NaN (0 * inf).
//
// Behind a ReLU the code keeps the side of the threshold that x is on: where rounding alone would put
// fma(value, gamma, beta) on the other side than fma(x, gamma, beta), the other neighbour of x is taken.  fma is monotone
// in its first argument and x lies between the two neighbours, so that one is always right.  The backward pass then has
// the forward pass's mask element for element; rounding alone flips the 1 to 2 % of the elements that lie within half a
// step of the threshold, an error of about 10 % in the gradient's norm.
#pragma once
#include "camal_train_kernels.hpp"

namespace camal {

struct ActI8 {   // codes -127 .. 127
    static constexpr unsigned CARRY = 0x1FFFFu;  // added to the bits of the largest |x|: carries into the exponent past 127/64
    static constexpr int OFFSET = 6;             // 2^(E - 127 - 6) holds 1.f * 2^(E - 127) for 1.f <= 127/64
    static __device__ __forceinline__ float nearest(float y, float& step) { step = 1.f; return rintf(y); }
    static __device__ __forceinline__ unsigned pack(const float (&v)[4]) {
        unsigned w = 0;  // byte inserts of v + 128, then back to two's complement
#pragma unroll
        for (int k = 0; k < 4; ++k) w = __builtin_amdgcn_cvt_pk_u8_f32(v[k] + 128.f, k, w);
        return w ^ 0x80808080u;
    }
    static __device__ __forceinline__ void unpack(unsigned w, float (&v)[4]) {
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = (float)(int)(signed char)(w >> (8 * k));
    }
};

struct ActE4M3 {  // OCP e4m3: largest 448, step 2^-9 below 2^-6
    static constexpr unsigned CARRY = 0x1FFFFFu;  // past 448/256 = 1.75
    static constexpr int OFFSET = 8;
    static __device__ __forceinline__ float nearest(float y, float& step) {
        const unsigned e = __builtin_bit_cast(unsigned, y) & 0x7F800000u;
        step = __builtin_bit_cast(float, (e > (121u << 23) ? e : (121u << 23)) - (3u << 23));
        return __builtin_amdgcn_cvt_f32_fp8(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false), 0);
    }
    static __device__ __forceinline__ unsigned pack(const float (&v)[4]) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
        return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true);
    }
    static __device__ __forceinline__ void unpack(unsigned w, float (&v)[4]) {
        v[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        v[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        v[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        v[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
};

__device__ __forceinline__ float act_scale(unsigned e) { return __builtin_bit_cast(float, e << 23); }

// max over the 8 lanes that share a scale block (lanes 8k .. 8k + 7), on the VALU's lane permutations
__device__ __forceinline__ unsigned act_block_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
    return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));  // row_half_mirror
}

// ReLU that lets a NaN through
__device__ __forceinline__ float act_relu(float u) { return u <= 0.f ? 0.f : u; }

// 4 channels of a lane -> their codes and the block's scale byte (the same in the block's 8 lanes, which all take part)
template <typename F, bool RELU>
__device__ __forceinline__ unsigned act_encode(const float (&x)[4], const float (&u)[4], const float (&g)[4],
                                               const float (&b)[4], unsigned& e) {
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) m = max(m, __builtin_bit_cast(unsigned, x[k]) & 0x7FFFFFFFu);
    m = act_block_max(m);
    const bool bad = m + F::CARRY >= 0x7F800000u;  // the next scale's codes would decode past the largest float
    e = bad ? 255u : (unsigned)max((int)((m + F::CARRY) >> 23) - F::OFFSET, 1);
    const float s = act_scale(e), inv = __builtin_bit_cast(float, (254u - min(e, 253u)) << 23);
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const float y = x[k] * inv;
        float step;
        v[k] = F::nearest(y, step);
        if (RELU) {
            const float back = v[k] * s;  // exact; y may have underflowed, so the side is taken from x itself
            const bool same = (fmaf(back, g[k], b[k]) > 0.f) == (u[k] > 0.f);
            v[k] = same ? v[k] : (back < x[k] ? v[k] + step : v[k] - step);
        }
        if (bad) v[k] = 0.f;
    }
    return F::pack(v);
}

// ---- write: a = relu(bn(z)) [+ bn_r(zr)] in fp32, and the checkpoint(s) --------------------------------------------
// A lane owns 4 channels for the whole launch (the stride between its rows is a multiple of the row), so the statistics
// stay in registers; ACT_ROWS of its rows are in flight at once.
struct ActNorm {
    const float *mean, *invstd, *gamma, *beta;
};
#define ACT_ROWS 4

template <typename F, bool RELU, bool RES>
__global__ __launch_bounds__(256) void act_write_kernel(const float* __restrict__ z, ActNorm n, const float* __restrict__ zr,
                                                        ActNorm nr, float* __restrict__ out, unsigned* __restrict__ codes,
                                                        unsigned char* __restrict__ scales, unsigned* __restrict__ codes_r,
                                                        unsigned char* __restrict__ scales_r, size_t n4, int c4mask) {
    const int c = (int)(threadIdx.x & c4mask) * 4;
    float m[4], is[4], g[4], b[4], mr[4], isr[4], gr[4], br[4];
    load4(n.mean + c, m); load4(n.invstd + c, is); load4(n.gamma + c, g); load4(n.beta + c, b);
    if constexpr (RES) { load4(nr.mean + c, mr); load4(nr.invstd + c, isr); load4(nr.gamma + c, gr); load4(nr.beta + c, br); }
    const size_t step = (size_t)gridDim.x * 256 * ACT_ROWS;
    for (size_t base = (size_t)blockIdx.x * 256 * ACT_ROWS; base < n4; base += step) {
        float v[ACT_ROWS][4], vr[ACT_ROWS][4];
#pragma unroll
        for (int q = 0; q < ACT_ROWS; ++q) {
            const size_t i = base + q * 256 + threadIdx.x, ic = i < n4 ? i : n4 - 1;
            load4(z + ic * 4, v[q]);
            if constexpr (RES) load4(zr + ic * 4, vr[q]);
        }
#pragma unroll
        for (int q = 0; q < ACT_ROWS; ++q) {
            // n4 is a multiple of 8 lanes (a row has 8 lanes per scale block): a block is stored whole or not at all
            const size_t i = base + q * 256 + threadIdx.x;
            float x[4], u[4], o[4];
            unsigned e;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                x[k] = (v[q][k] - m[k]) * is[k];
                u[k] = fmaf(x[k], g[k], b[k]);
                o[k] = RELU ? act_relu(u[k]) : u[k];
            }
            const unsigned w = act_encode<F, RELU>(x, u, g, b, e);
            if (i < n4) {
                codes[i] = w;
                if ((threadIdx.x & 7) == 0) scales[i >> 3] = (unsigned char)e;
            }
            if constexpr (RES) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    x[k] = (vr[q][k] - mr[k]) * isr[k];
                    u[k] = fmaf(x[k], gr[k], br[k]);
                    o[k] += u[k];
                }
                const unsigned wr = act_encode<F, false>(x, u, gr, br, e);
                if (i < n4) {
                    codes_r[i] = wr;
                    if ((threadIdx.x & 7) == 0) scales_r[i >> 3] = (unsigned char)e;
                }
            }
            if (i < n4) store4(out + i * 4, o[0], o[1], o[2], o[3]);
        }
    }
}

// ---- read back: the normalised values (gamma null), or the activation relu(gamma x + beta) [+ gamma_r x_r + beta_r] ----
template <typename F>
__device__ __forceinline__ void act_load(const unsigned* codes, const unsigned char* scales, size_t i, float (&x)[4]) {
    F::unpack(codes[i], x);
    const float s = act_scale(scales[i >> 3]);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] *= s;
}

template <typename F, bool AFFINE, bool RELU, bool RES>
__global__ __launch_bounds__(256) void act_read_kernel(const unsigned* __restrict__ codes, const unsigned char* __restrict__ scales,
                                                       const float* __restrict__ gamma, const float* __restrict__ beta,
                                                       const unsigned* __restrict__ codes_r,
                                                       const unsigned char* __restrict__ scales_r,
                                                       const float* __restrict__ gamma_r, const float* __restrict__ beta_r,
                                                       float* __restrict__ out, size_t n4, int c4mask) {
    const int c = (int)(threadIdx.x & c4mask) * 4;
    float g[4], b[4], gr[4], br[4];
    if constexpr (AFFINE) { load4(gamma + c, g); load4(beta + c, b); }
    if constexpr (RES) { load4(gamma_r + c, gr); load4(beta_r + c, br); }
    const size_t step = (size_t)gridDim.x * 256;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += step) {
        float x[4], o[4];
        act_load<F>(codes, scales, i, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            o[k] = AFFINE ? fmaf(x[k], g[k], b[k]) : x[k];
            if (RELU) o[k] = act_relu(o[k]);
        }
        if constexpr (RES) {
            act_load<F>(codes_r, scales_r, i, x);
#pragma unroll
            for (int k = 0; k < 4; ++k) o[k] += fmaf(x[k], gr[k], br[k]);
        }
        store4(out + i * 4, o[0], o[1], o[2], o[3]);
    }
}

// ---- backward of norm + ReLU from the checkpoint -----------------------------------------------------------------------
//   dy = da * [fma(x, gamma, beta) > 0],  s1 = sum dy,  s2 = sum dy x,  dz = gamma invstd (dy - s1/N - x s2/N)
// The sums come first, so the input is read twice by nature.  BCAST: da[b][t][c] = dpool[b][c] / L.
template <typename F, int C, bool RELU, bool BCAST>
__global__ __launch_bounds__(256) void act_bwd_partial_kernel(const float* __restrict__ da, const unsigned* __restrict__ codes,
                                                              const unsigned char* __restrict__ scales,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              int N, int L, double* __restrict__ partial) {
    constexpr int Q = C / 4, G = 256 / Q, RPL = BN_ROWS_PER_BLOCK / G;
    __shared__ float sh[G][C][2];
    const int q4 = threadIdx.x % Q, c4 = q4 * 4, g = threadIdx.x / Q;
    const int r0 = blockIdx.x * BN_ROWS_PER_BLOCK;
    float ga[4], be[4];
    load4(gamma + c4, ga); load4(beta + c4, be);
    unsigned w[RPL], e[RPL];
    float dv[RPL][4];
#pragma unroll
    for (int u = 0; u < RPL; ++u) {
        const int r = r0 + g + u * G;
        const int rc = r < N ? r : N - 1;  // a row past the end loads a valid address and counts for nothing
        w[u] = codes[(size_t)rc * Q + q4];
        e[u] = scales[(size_t)rc * (C / 32) + (q4 >> 3)];
        load4(BCAST ? da + (size_t)(rc / L) * C + c4 : da + (size_t)rc * C + c4, dv[u]);
    }
    const float len = (float)L;
    float s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < RPL; ++u) {
        const bool live = r0 + g + u * G < N;
        float x[4];
        F::unpack(w[u], x);
        const float s = act_scale(e[u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float xh = x[k] * s;
            float d = BCAST ? dv[u][k] / len : dv[u][k];
            if (RELU) d = fmaf(xh, ga[k], be[k]) > 0.f ? d : 0.f;
            s1[k] += live ? d : 0.f;
            s2[k] += live ? d * xh : 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) { sh[g][c4 + k][0] = s1[k]; sh[g][c4 + k][1] = s2[k]; }
    __syncthreads();
    if (threadIdx.x < C) {
        const int c = threadIdx.x;
        double a = 0.0, b = 0.0;
#pragma unroll
        for (int k = 0; k < G; ++k) { a += (double)sh[k][c][0]; b += (double)sh[k][c][1]; }
        partial[((size_t)blockIdx.x * C + c) * 2 + 0] = a;
        partial[((size_t)blockIdx.x * C + c) * 2 + 1] = b;
    }
}

// means[0][c] = s1 / N, means[1][c] = s2 / N for the apply pass
template <int C>
__global__ __launch_bounds__(BN_FINAL_THREADS) void act_bwd_final_kernel(const double* __restrict__ partial, int nblocks, int N,
                                                                         float* __restrict__ means, float* __restrict__ dgamma,
                                                                         float* __restrict__ dbeta) {
    double a, b;
    int c;
    if (!bn_final_reduce<C>(partial, nblocks, c, a, b)) return;
    means[c] = (float)(a / N);
    means[C + c] = (float)(b / N);
    dbeta[c] = (float)a;
    dgamma[c] = (float)b;
}

template <typename F, int C, bool RELU, bool BCAST>
__global__ __launch_bounds__(256) void act_bwd_apply_kernel(const float* __restrict__ da, const unsigned* __restrict__ codes,
                                                            const unsigned char* __restrict__ scales,
                                                            const float* __restrict__ invstd, const float* __restrict__ gamma,
                                                            const float* __restrict__ beta, const float* __restrict__ means,
                                                            size_t n4, int L, float* __restrict__ dz) {
    constexpr int Q = C / 4;
    const int c = (int)(threadIdx.x % Q) * 4;
    float is[4], g[4], b[4], a1[4], a2[4];
    load4(invstd + c, is); load4(gamma + c, g); load4(beta + c, b); load4(means + c, a1); load4(means + C + c, a2);
    const float len = (float)L;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < n4; i += (size_t)gridDim.x * 256) {
        float x[4], d[4], o[4];
        act_load<F>(codes, scales, i, x);
        load4(BCAST ? da + (size_t)((int)(i / Q) / L) * C + c : da + i * 4, d);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float dy = BCAST ? d[k] / len : d[k];
            if (RELU) dy = fmaf(x[k], g[k], b[k]) > 0.f ? dy : 0.f;
            o[k] = g[k] * is[k] * (dy - a1[k] - x[k] * a2[k]);
        }
        store4(dz + i * 4, o[0], o[1], o[2], o[3]);
    }
}

// ---- weight gradient from the checkpoint ---------------------------------------------------------------------------------
//   dw[co][ci][j] = sum_{b,t} dz[b][t][co] a[b][clamp(t + j - ks/2)][ci],  a = bf16(relu(gamma x + beta) [+ skip])
// a holds 8 significant bits: the code behind it has 7 (int8) or 4 (e4m3).
// Partial sums of each split go to part[split][j][co][ci]; wgrad_reduce_kernel adds them in a fixed order.
struct ActIn {  // the layer's input as checkpoint(s)
    const unsigned* codes; const unsigned char* scales; const float *gamma, *beta;
    const unsigned* codes_r; const unsigned char* scales_r; const float *gamma_r, *beta_r;
};

// 4 channels (c .. c + 3) of row r of the layer's input, as it takes part in the product
template <typename F, bool RELU, bool RES>
__device__ __forceinline__ void act_input(const ActIn& in, size_t r, int cin, int c, float (&a)[4]) {
    const size_t i = r * (size_t)(cin / 4) + c / 4;
    float x[4], g[4], b[4];
    act_load<F>(in.codes, in.scales, i, x);
    load4(in.gamma + c, g); load4(in.beta + c, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) { a[k] = fmaf(x[k], g[k], b[k]); if (RELU) a[k] = act_relu(a[k]); }
    if constexpr (RES) {
        act_load<F>(in.codes_r, in.scales_r, i, x);
        load4(in.gamma_r + c, g); load4(in.beta_r + c, b);
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] += fmaf(x[k], g[k], b[k]);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) a[k] = (float)(__bf16)a[k];
}

#define ACT_WG_TT 32
template <typename F, bool RELU, bool RES>
__global__ __launch_bounds__(256) void act_wgrad_simple_kernel(const float* __restrict__ dz, ActIn in, float* __restrict__ part,
                                                               int B, int L, int cin, int cout, int ks, int tiles_per_split,
                                                               bool zero_pad) {
    __shared__ float s_dz[ACT_WG_TT][32], s_a[ACT_WG_TT][32];
    const int ci0 = (blockIdx.y % (cin / 32)) * 32, co0 = (blockIdx.y / (cin / 32)) * 32, j = blockIdx.z;
    const int tpw = (L + ACT_WG_TT - 1) / ACT_WG_TT, total = B * tpw;
    const int lo = min(total, (int)blockIdx.x * tiles_per_split), hi = min(total, lo + tiles_per_split);
    const int q = (threadIdx.x & 7) * 4, row = threadIdx.x >> 3;  // 4 columns, one of 32 rows
    float acc[4] = {0.f, 0.f, 0.f, 0.f};  // dw[co0 + row][ci0 + q ..]
    for (int tile = lo; tile < hi; ++tile) {
        const int b = tile / tpw, t = (tile - b * tpw) * ACT_WG_TT + row, p = t + j - (ks >> 1);
        const int pc = p < 0 ? 0 : (p > L - 1 ? L - 1 : p);
        float d[4] = {0.f, 0.f, 0.f, 0.f}, a[4] = {0.f, 0.f, 0.f, 0.f};
        if (t < L) {
            load4(dz + ((size_t)b * L + t) * cout + co0 + q, d);
            if (!(zero_pad && p != pc)) act_input<F, RELU, RES>(in, (size_t)b * L + pc, cin, ci0 + q, a);
        }
        __syncthreads();
        store4(&s_dz[row][q], d[0], d[1], d[2], d[3]);
        store4(&s_a[row][q], a[0], a[1], a[2], a[3]);
        __syncthreads();
        for (int k = 0; k < ACT_WG_TT; ++k)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[c] = fmaf(s_dz[k][row], s_a[k][q + c], acc[c]);
    }
    store4(part + (((size_t)blockIdx.x * ks + j) * cout + co0 + row) * cin + ci0 + q, acc[0], acc[1], acc[2], acc[3]);
}

}  // namespace camal
