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
#include "camal_act_codes.hpp"

namespace camal {

// max over the 8 lanes that share a scale block (lanes 8k .. 8k + 7), on the VALU's lane permutations
__device__ __forceinline__ unsigned act_block_max(unsigned m) {
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, true));   // quad_perm 1,0,3,2
    m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, true));   // quad_perm 2,3,0,1
    return max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, true));  // row_half_mirror
}

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
// First stage.  A block takes chunks of ACT_BWD_ROWS rows, one after another; a lane 4 channels of every G-th row of a chunk,
// all of them in flight.  fp32 sums run over a lane's rows of one chunk (2 to 16) and are then carried in 64 bits; at most
// ACT_BWD_BLOCKS blocks, so that the second stage has little to read: 128 x 510 x 128 takes 23.1 us with 512, 24.8 with 1024,
// 23.4 with 256 (first stage 9 us = 4.7 TB/s, second 4, apply 12.5 = 6 TB/s).
#define ACT_BWD_ROWS 64
#define ACT_BWD_BLOCKS 512

template <typename F, int C, bool RELU, bool BCAST>
__global__ __launch_bounds__(256) void act_bwd_partial_kernel(const float* __restrict__ da, const unsigned* __restrict__ codes,
                                                              const unsigned char* __restrict__ scales,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              int N, int L, double* __restrict__ partial) {
    constexpr int Q = C / 4, G = 256 / Q, RPL = ACT_BWD_ROWS / G;
    __shared__ double sh[G][C][2];
    const int q4 = threadIdx.x % Q, c4 = q4 * 4, g = threadIdx.x / Q;
    const int chunks = (N + ACT_BWD_ROWS - 1) / ACT_BWD_ROWS;
    float ga[4], be[4];
    load4(gamma + c4, ga); load4(beta + c4, be);
    const float len = (float)L;
    double t1[4] = {0., 0., 0., 0.}, t2[4] = {0., 0., 0., 0.};
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int r0 = chunk * ACT_BWD_ROWS + g;
        unsigned w[RPL], e[RPL];
        float dv[RPL][4];
#pragma unroll
        for (int u = 0; u < RPL; ++u) {
            const int rc = min(r0 + u * G, N - 1);  // a row past the end loads a valid address and counts for nothing
            w[u] = codes[(size_t)rc * Q + q4];
            e[u] = scales[(size_t)rc * (C / 32) + (q4 >> 3)];
            load4(BCAST ? da + (size_t)(rc / L) * C + c4 : da + (size_t)rc * C + c4, dv[u]);
        }
        float s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < RPL; ++u) {
            const bool live = r0 + u * G < N;
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
        for (int k = 0; k < 4; ++k) { t1[k] += (double)s1[k]; t2[k] += (double)s2[k]; }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) { sh[g][c4 + k][0] = t1[k]; sh[g][c4 + k][1] = t2[k]; }
    __syncthreads();
    if (threadIdx.x < C) {
        const int c = threadIdx.x;
        double a = 0.0, b = 0.0;
#pragma unroll
        for (int k = 0; k < G; ++k) { a += sh[k][c][0]; b += sh[k][c][1]; }
        partial[((size_t)blockIdx.x * C + c) * 2 + 0] = a;
        partial[((size_t)blockIdx.x * C + c) * 2 + 1] = b;
    }
}

// Second stage: ACT_FINAL_CPB channels per workgroup, each lane a fixed strided subset of the partial sums, combined in a fixed
// order (xor shuffles inside the wave, LDS across the waves).
#define ACT_FINAL_CPB 8
#define ACT_FINAL_THREADS 1024
template <int C>
__device__ __forceinline__ bool act_final_reduce(const double* __restrict__ partial, int nblocks, int& c, double& a, double& b) {
    constexpr int G = ACT_FINAL_THREADS / ACT_FINAL_CPB, NW = ACT_FINAL_THREADS / 64;
    static_assert(C % ACT_FINAL_CPB == 0 && 64 % ACT_FINAL_CPB == 0, "channels per workgroup");
    __shared__ double sh[NW][ACT_FINAL_CPB][2];
    const int cl = threadIdx.x % ACT_FINAL_CPB, g = threadIdx.x / ACT_FINAL_CPB;
    c = blockIdx.x * ACT_FINAL_CPB + cl;
    double s = 0.0, ss = 0.0;
#pragma unroll 4
    for (int i = g; i < nblocks; i += G) {
        const double2 t = *reinterpret_cast<const double2*>(partial + ((size_t)i * C + c) * 2);
        s += t.x;
        ss += t.y;
    }
#pragma unroll
    for (int m = ACT_FINAL_CPB; m < 64; m <<= 1) {
        s += __shfl_xor(s, m, 64);
        ss += __shfl_xor(ss, m, 64);
    }
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    if (lane < ACT_FINAL_CPB) { sh[wave][lane][0] = s; sh[wave][lane][1] = ss; }
    __syncthreads();
    a = 0.0; b = 0.0;
    if (threadIdx.x >= ACT_FINAL_CPB) return false;
#pragma unroll
    for (int k = 0; k < NW; ++k) { a += sh[k][cl][0]; b += sh[k][cl][1]; }
    return true;
}

// means[0][c] = s1 / N, means[1][c] = s2 / N for the apply pass
template <int C>
__global__ __launch_bounds__(ACT_FINAL_THREADS) void act_bwd_final_kernel(const double* __restrict__ partial, int nblocks, int N,
                                                                         float* __restrict__ means, float* __restrict__ dgamma,
                                                                         float* __restrict__ dbeta) {
    double a, b;
    int c;
    if (!act_final_reduce<C>(partial, nblocks, c, a, b)) return;
    means[c] = (float)(a / N);
    means[C + c] = (float)(b / N);
    dbeta[c] = (float)a;
    dgamma[c] = (float)b;
}

// From half the 256 MiB L3 on, dz is stored past it (STREAM): left there, its lines push out what the next kernels read and are
// written out under their reads.  us of 128 channels and dz of 140 / 180 / 220 / 300 / 500 MiB, kept in the L3 -> stored past it:
//   the call alone                       104 -> 88   132 -> 109   163 -> 134   226 -> 195   377 -> 350
//   with a 1-tap weight gradient of dz   157 -> 147  201 -> 185   249 -> 229   336 -> 320   559 -> 552
//   with a 3-tap one                     182 -> 177  230 -> 224   281 -> 275   383 -> 382   639 -> 646
//   with an elementwise pass over dz     135 -> 141  186 -> 182   235 -> 228   330 -> 325   558 -> 556
// so its reader gains, too, but for an elementwise one at the lower end.  The same stores in the write and read kernels change
// nothing (83.0 and 47.3 us either way on 124 and 189 MB).
#define ACT_STREAM_BYTES (128u << 20)
template <bool STREAM>
__device__ __forceinline__ void act_store4(float* p, const float (&o)[4]) {  // (a run-time choice: hipcc merges the two stores)
    const f32x4 v = {o[0], o[1], o[2], o[3]};
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
    else *reinterpret_cast<f32x4*>(p) = v;
}

template <typename F, int C, bool RELU, bool BCAST, bool STREAM>
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
        act_store4<STREAM>(dz + i * 4, o);
    }
}

// All of it in one launch for at most ACT_SMALL_ROWS rows, where three launches cost more than the work: a workgroup has 32
// channels (a scale block) and keeps its rows in registers between the sums and their use.  A call in a stream of calls /
// alone: 14.7 / 28.1 us here and 19.5 / 31.2 us there at 384 rows, 14.8 / 30.7 at 1024, 15.8 / 38.2 at 2048 (32 to 256
// channels alike).  fp32 sums run over the at most 8 rows of a lane and are then carried in 64 bits.
#define ACT_SMALL_ROWS 1024
template <typename F, bool RELU, bool BCAST>
__global__ __launch_bounds__(1024) void act_bwd_small_kernel(const float* __restrict__ da, const unsigned* __restrict__ codes,
                                                             const unsigned char* __restrict__ scales,
                                                             const float* __restrict__ invstd, const float* __restrict__ gamma,
                                                             const float* __restrict__ beta, int N, int L, int C,
                                                             float* __restrict__ dz, float* __restrict__ dgamma,
                                                             float* __restrict__ dbeta) {
    constexpr int U = ACT_SMALL_ROWS / 128;
    __shared__ double sh[16][32][2];
    __shared__ __align__(16) float mean[2][32];
    const int q = threadIdx.x & 7, g = threadIdx.x >> 3, c = blockIdx.x * 32 + 4 * q, wave = threadIdx.x >> 6;
    float ga[4], be[4], is[4];
    load4(gamma + c, ga); load4(beta + c, be); load4(invstd + c, is);
    const float len = (float)L;
    float x[U][4], dy[U][4], s1[4] = {0.f, 0.f, 0.f, 0.f}, s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u * 128 >= N) break;
        const int r = g + u * 128, rc = min(r, N - 1);
        F::unpack(codes[(size_t)rc * (C / 4) + c / 4], x[u]);
        const float s = act_scale(scales[(size_t)rc * (C / 32) + blockIdx.x]);
        load4(da + (size_t)(BCAST ? rc / L : rc) * C + c, dy[u]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            x[u][k] *= s;
            if (BCAST) dy[u][k] /= len;
            if (RELU) dy[u][k] = fmaf(x[u][k], ga[k], be[k]) > 0.f ? dy[u][k] : 0.f;
            s1[k] += r < N ? dy[u][k] : 0.f;
            s2[k] += r < N ? dy[u][k] * x[u][k] : 0.f;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        double a = (double)s1[k], b = (double)s2[k];
#pragma unroll
        for (int m = 8; m < 64; m <<= 1) { a += __shfl_xor(a, m, 64); b += __shfl_xor(b, m, 64); }
        if ((threadIdx.x & 63) < 8) { sh[wave][4 * q + k][0] = a; sh[wave][4 * q + k][1] = b; }
    }
    __syncthreads();
    if (threadIdx.x < 64) {
        const int ch = threadIdx.x & 31, which = threadIdx.x >> 5;
        double a = 0.0;
#pragma unroll
        for (int w = 0; w < 16; ++w) a += sh[w][ch][which];
        mean[which][ch] = (float)(a / N);
        (which ? dgamma : dbeta)[blockIdx.x * 32 + ch] = (float)a;
    }
    __syncthreads();
    float a1[4], a2[4];
    load4(&mean[0][4 * q], a1); load4(&mean[1][4 * q], a2);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u * 128 >= N) break;
        const int r = g + u * 128;
        float o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = ga[k] * is[k] * (dy[u][k] - a1[k] - x[u][k] * a2[k]);
        if (r < N) store4(dz + (size_t)r * C + c, o[0], o[1], o[2], o[3]);
    }
}

// ---- weight gradient: the second stage of what camal_act_wgrad.hpp leaves ------------------------------------------------
// dw[co][ci][j] = sum_split part[split][j][co][ci].  Four ci per lane; the splits are dealt to 16 groups of lanes, each with
// independent 16-byte loads, combined in a fixed order.  29 MB (64 splits of 7 taps, 128 -> 128): 6.2 us, 4.7 TB/s; with 4
// groups the same, but 7.8 instead of 6.7 us on 16 splits of 7 taps, 256 -> 256.
__global__ __launch_bounds__(256) void act_wgrad_reduce_kernel(const float* __restrict__ part, int nsplit, int cout, int cin, int ks,
                                                               float* __restrict__ dw) {
    constexpr int GRP = 16, QB = 256 / GRP;
    __shared__ float4 red[GRP][QB];
    const int total = cout * cin * ks;
    const int q = threadIdx.x % QB, g = threadIdx.x / QB;
    const int idx = (blockIdx.x * QB + q) * 4;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (idx < total) {
#pragma unroll 8
        for (int s = g; s < nsplit; s += GRP) {
            const float4 v = *reinterpret_cast<const float4*>(part + (size_t)s * total + idx);
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
    }
    red[g][q] = a;
    __syncthreads();
    if (g == 0 && idx < total) {
#pragma unroll
        for (int k = 1; k < GRP; ++k) {
            const float4 v = red[k][q];
            a.x += v.x; a.y += v.y; a.z += v.z; a.w += v.w;
        }
        const int ci = idx % cin, co = (idx / cin) % cout, j = idx / (cin * cout);
        float* o = dw + ((size_t)co * cin + ci) * ks + j;
        o[0] = a.x;
        o[ks] = a.y;
        o[2 * ks] = a.z;
        o[3 * ks] = a.w;
    }
}

}  // namespace camal
