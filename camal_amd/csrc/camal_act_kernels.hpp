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
#include "camal_act.hpp"

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
// ACT_BWD_FLIGHT of them in flight.  fp32 sums run over a lane's rows of one chunk (at most 64) and are then carried in 64
// bits; at most ACT_BWD_BLOCKS blocks, so that the second stage has little to read whatever the number of rows.
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

// A dz that the 256 MiB L3 cannot hold for its reader is stored past it (STREAM): left there, its lines are written out under
// the next kernel's reads.  24 x 10080 x 256 (248 MB): 179 -> 150 us, all of it in the first stage's reads.  The same stores in
// the write and read kernels change nothing (83.0 and 47.3 us either way on 124 and 189 MB).
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
// channels alike).
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

// ---- weight gradient from the checkpoint, on MFMA ------------------------------------------------------------------------
//   dw[co][ci][j] = sum_{b,t} dz[b][t][co] a[b][clamp(t + j - ks/2)][ci],  a = bf16(relu(gamma x + beta) [+ skip])
// GEMM view: M = co, N = ci, K = time, for every tap j.  v_mfma_f32_32x32x16_bf16 takes 16 timesteps per instruction: lane
// (i = l & 31, h = l >> 5) feeds 8 consecutive times of channel co_i (A) and ci_i (B).
//   a holds 8 significant bits (the code behind it has 7 or 4), so it is a bf16 operand without loss.  dz is cut into three
//   bf16 pieces, each the leading 8 bits of what is left: they add up to it exactly, so the three products, summed in the
//   instruction's fp32, are an fp32 product sum at a third of the bf16 rate, 5 times the rate of fp32 MFMA.
// One wave = 32 co x CIW * 32 ci x NTAP taps on a unit of 64 timesteps.  The 8 waves of a workgroup are CO co tiles x WK units:
// the CO waves of a unit share its decoded input, and the WK sums of a tile are added in LDS before they leave the workgroup
// (what the partial sums weigh is what bounds a short call).
//   A: dz straight from global memory into registers, as the fragment wants it: no other wave needs these values; rows past
//      the window's end are out of the buffer's range and come back as zeros;
//   B: the unit's input, decoded into LDS as plain rows [time][32 channels] of bf16, read with the transposing
//      ds_read_b64_tr_b16 (4 times of a channel per lane): a tap is a row offset, and a row is 64 bytes, so neither side
//      has bank conflicts.
// On these SIMDs a vector instruction hides behind a matrix product only up to about three per product (measured: 15.9 ns a
// product alone, 16.3 with 2, 18.1 with 4, 23.3 with 8 vector instructions to each, two waves), so what counts beside the
// products is the number of vector instructions: cutting dz takes 44 per 24 products of 8 taps, decoding is shared.
// Each split's sums go to part[split][j][co][ci]; act_wgrad_reduce_kernel adds them in a fixed order.
#define ACT_UNIT 64   // timesteps of a unit
#define ACT_WAVES 8   // waves of a workgroup
#define ACT_TAPS 8    // taps a wave takes at most

typedef short s16x4 __attribute__((ext_vector_type(4)));

// How a workgroup is made up, and the passes in which the CO waves of a unit fill its input tile (4 channels per lane)
template <int CO, int CIW, int NTAP> struct ActTile {
    static constexpr int WK = ACT_WAVES / CO;
    static constexpr int RPW = 8 / CIW, RPP = RPW * CO, ROWS = (ACT_UNIT + NTAP + 6) / 8 * 8, PASS = (ROWS + RPP - 1) / RPP;
    static constexpr int TILE = CIW * ROWS * 32;  // halfwords
    // LDS: two tiles per unit, then the waves' sums: ACT_WAVES * (16 - 16 / WK) registers per accumulator, CHUNK of them at once
    static constexpr int SUMS = ACT_WAVES * (16 - 16 / WK) * 64 * 4, FIT = 128 * 1024 / SUMS;
    static constexpr int CHUNK = NTAP * CIW < FIT ? NTAP * CIW : FIT;
    static constexpr int BYTES = 2 * WK * 2 * TILE > CHUNK * SUMS ? 2 * WK * 2 * TILE : CHUNK * SUMS;
};

// Where the sums go, in floats: partial sums [split][tap][co][ci], or with one split the gradient [co][ci][tap] itself
struct ActOut {
    int split, tap, co, ci;
};

template <int COUT, int CO, int CIW, int NTAP>
__device__ __forceinline__ void act_wgrad_body(unsigned short* lds, const float* __restrict__ dz, const ActIn& in,
                                               float* __restrict__ part, ActOut out, int B, int L, int cin, int ks,
                                               int units_per_split, int j0) {
    using T = ActTile<CO, CIW, NTAP>;
    constexpr int WK = T::WK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave / CO, col = wave % CO;
    const int i = lane & 31, h = lane >> 5, co0 = (blockIdx.z * CO + col) * 32, ci0 = blockIdx.y % (cin / (32 * CIW)) * 32 * CIW;
    const int tpw = (L + ACT_UNIT - 1) / ACT_UNIT, total = B * tpw;
    const int lo = min(total, (int)blockIdx.x * units_per_split), hi = min(total, lo + units_per_split);

    f32x16 acc[NTAP][CIW];
#pragma unroll
    for (int j = 0; j < NTAP; ++j)
#pragma unroll
        for (int w = 0; w < CIW; ++w)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[j][w][k] = 0.f;

    // ---- the input tile: a lane has 4 channels of every RPP-th row ----
    const int cq = lane % (8 * CIW), r0 = col * T::RPW + lane / (8 * CIW), lgc = 31 - __builtin_clz(cin);
    float g[4], b[4], gr[4] = {0.f, 0.f, 0.f, 0.f}, br[4] = {0.f, 0.f, 0.f, 0.f};
    load4(in.gamma + ci0 + 4 * cq, g); load4(in.beta + ci0 + 4 * cq, b);
    if (in.codes_r) { load4(in.gamma_r + ci0 + 4 * cq, gr); load4(in.beta_r + ci0 + 4 * cq, br); }
    const float floor = in.relu ? 0.f : -__builtin_inff();
    // The tile's codes travel in registers a whole unit ahead.  The tile at (bb, tt): rows relative to its first one, edges
    // clamped, so that offsets are small.
    unsigned cw[T::PASS], cs[T::PASS], rw[T::PASS], rs[T::PASS];
    struct Source { __amdgpu_buffer_rsrc_t codes, scales, codes_r, scales_r; int tb, rb; };
    auto source = [&](int bb, int tt) {
        Source o;
        o.tb = tt * ACT_UNIT + j0 - (ks >> 1);
        o.rb = max(0, min(o.tb, L - 1));
        const int rows = min(L - o.rb, 2 * ACT_UNIT);
        const size_t first = (size_t)bb * L + o.rb;
        auto rsrc = [&](const void* p, int lg) {
            return __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)p + (first << lg)), 0, rows << lg, 0x00027000);
        };
        o.codes = rsrc(in.codes, lgc);
        o.scales = rsrc(in.scales, lgc - 5);
        o.codes_r = rsrc(in.codes_r, lgc);  // not read from without a skip branch
        o.scales_r = rsrc(in.scales_r, lgc - 5);
        return o;
    };
    auto fetch = [&](const Source& o, int p) {
        if (col * T::RPW + p * T::RPP >= T::ROWS) return;
        const int rel = max(-o.rb, min(o.tb - o.rb + r0 + p * T::RPP, L - 1 - o.rb));
        const int oc = (rel << lgc) + ci0 + 4 * cq, os = (rel << (lgc - 5)) + ci0 / 32 + cq / 8;
        cw[p] = __builtin_amdgcn_raw_buffer_load_b32(o.codes, oc, 0, 0);
        cs[p] = __builtin_amdgcn_raw_buffer_load_b8(o.scales, os, 0, 0);
        if (in.codes_r) {
            rw[p] = __builtin_amdgcn_raw_buffer_load_b32(o.codes_r, oc, 0, 0);
            rs[p] = __builtin_amdgcn_raw_buffer_load_b8(o.scales_r, os, 0, 0);
        }
    };
    auto stash = [&](unsigned short* tile, int tb, int p) {
        if (col * T::RPW + p * T::RPP >= T::ROWS) return;
        float a[4];
        if (in.e4m3) ActE4M3::unpack(cw[p], a); else ActI8::unpack(cw[p], a);
        const float sc = act_scale(cs[p]);
#pragma unroll
        for (int k = 0; k < 4; ++k) a[k] = __builtin_elementwise_maximum(fmaf(a[k] * sc, g[k], b[k]), floor);
        if (in.codes_r) {
            float x[4];
            if (in.e4m3) ActE4M3::unpack(rw[p], x); else ActI8::unpack(rw[p], x);
            const float sr = act_scale(rs[p]);
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] += fmaf(x[k] * sr, gr[k], br[k]);
        }
        const int row = r0 + p * T::RPP;
        if (in.zero_pad) {
            const bool inside = (unsigned)(tb + row) < (unsigned)L;
#pragma unroll
            for (int k = 0; k < 4; ++k) a[k] = inside ? a[k] : 0.f;
        }
        *reinterpret_cast<uint2*>(tile + ((cq / 8) * T::ROWS + row) * 32 + 4 * (cq % 8)) = make_uint2(pk_bf16(a[0], a[1]), pk_bf16(a[2], a[3]));
    };

    // ---- dz: 8 times of this lane's channel per step, loaded two steps before it is cut, cut a step before it is used ----
    unsigned d[2][8];
    u32x4 pc[2][3];
    const int voff = (8 * h * COUT + co0 + i) * 4;
    auto load_dz = [&](__amdgpu_buffer_rsrc_t src, int s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[s & 1][e] = __builtin_amdgcn_raw_buffer_load_b32(src, voff + (16 * s + e) * COUT * 4, 0, 0);
    };
    auto cut = [&](int s, int e) {  // times 2 e, 2 e + 1 of step s
        unsigned q[2][3];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float v = __builtin_bit_cast(float, d[s & 1][2 * e + k]);
            q[k][0] = d[s & 1][2 * e + k];
            const float r1 = v - __builtin_bit_cast(float, q[k][0] & 0xFFFF0000u);
            q[k][1] = __builtin_bit_cast(unsigned, r1);
            q[k][2] = __builtin_bit_cast(unsigned, r1 - __builtin_bit_cast(float, q[k][1] & 0xFFFF0000u));
        }
#pragma unroll
        for (int p = 0; p < 3; ++p) pc[s & 1][p][e] = __builtin_amdgcn_perm(q[1][p], q[0][p], 0x07060302u);
    };

    // ---- the B operand: lane's place in a transposing read is rows 8 h + (l % 16) / 4 (+ 4), channels 16 ((l / 16) & 1) +
    // 4 (l % 4) .. + 3 ----
    constexpr int TRIOS = NTAP * CIW;
    const int bp = (8 * h + (lane & 15) / 4) * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    auto operand = [&](const unsigned short* tile, int s, int n) {  // trio n = tap * CIW + ci tile
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const unsigned short* q = tile + bp + ((n % CIW) * T::ROWS + 16 * s + n / CIW) * 32;
        const s16x4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)q);
        const s16x4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(q + 4 * 32));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    // The positions of the unit at hand, the next one (whose tile is decoded meanwhile) and the one after it (whose codes are
    // fetched).  Past the split's end the last unit repeats, and counts for nothing: no rows of dz.
    auto dz_source = [&](int bb, int tt, bool live) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(dz + ((size_t)bb * L + tt * ACT_UNIT) * COUT), 0,
                                                 live ? min(ACT_UNIT, L - tt * ACT_UNIT) * COUT * 4 : 0, 0x00027000);
    };
    int u = min(lo + wk, hi - 1), bb = u / tpw, tt = u - bb * tpw;
    auto advance = [&]() {
        const int step = min(WK, hi - 1 - u);
        u += step;
        tt += step;
        while (tt >= tpw) { tt -= tpw; ++bb; }
    };
    unsigned short* mine = lds + wk * 2 * T::TILE;  // two tiles: one is read, the other filled
    if (lo < hi) {
        Source at = source(bb, tt);
#pragma unroll
        for (int p = 0; p < T::PASS; ++p) fetch(at, p);
        __amdgpu_buffer_rsrc_t dsrc = dz_source(bb, tt, lo + wk < hi);
        load_dz(dsrc, 0);
        load_dz(dsrc, 1);
#pragma unroll
        for (int p = 0; p < T::PASS; ++p) stash(mine, at.tb, p);
        advance();
        at = source(bb, tt);
#pragma unroll
        for (int p = 0; p < T::PASS; ++p) fetch(at, p);
#pragma unroll
        for (int e = 0; e < 4; ++e) cut(0, e);
        load_dz(dsrc, 2);
        int cur = 0;
        for (int u0 = lo; u0 < hi; u0 += WK, cur ^= 1) {
            unsigned short *now = mine + cur * T::TILE, *next = mine + (cur ^ 1) * T::TILE;
            const int tb_next = at.tb;
            const __amdgpu_buffer_rsrc_t dnext = dz_source(bb, tt, u0 + WK + wk < hi);
            advance();
            at = source(bb, tt);
            __syncthreads();
            bf16x8 bt = operand(now, 0, 0);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                // Between the products of step s: the next step's dz is cut and its registers loaded again, a quarter of the
                // next tile decoded and its codes fetched again.  In clumps of their own these would leave the matrix pipe
                // idle (the two waves of a SIMD share it evenly, reach their clumps together and overlap nothing).
                constexpr int STASH = (T::PASS + 3) / 4, TASKS = 5 + STASH;
#pragma unroll
                for (int n = 0; n < TRIOS; ++n) {
                    bf16x8 bn;
                    if (n + 1 < TRIOS) bn = operand(now, s, n + 1);
                    else if (s < 3) bn = operand(now, s + 1, 0);
#pragma unroll
                    for (int p = 2; p >= 0; --p)
                        acc[n / CIW][n % CIW] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, pc[s & 1][p]), bt,
                                                                                       acc[n / CIW][n % CIW], 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < TASKS; ++t) {
                        if (t * TRIOS / TASKS != n) continue;
                        if (t < 4) cut(s + 1, t);
                        else if (t == 4) { if (s == 0) load_dz(dsrc, 3); else load_dz(dnext, s - 1); }
                        else {
                            const int p = (t - 5) * 4 + s;
                            if (p < T::PASS) { stash(next, tb_next, p); fetch(at, p); }
                        }
                    }
                    bt = bn;
                }
            }
            dsrc = dnext;
        }
    }
    // acc[j][w][reg] of lane l: row co = co0 + (reg & 3) + 8 (reg >> 2) + 4 h, column ci = ci0 + 32 w + i.  Of a tile's 16
    // registers each of its WK waves adds OWN and hands the others out through LDS, as many tiles at once as fit: the
    // workgroup has the CU to itself.
    constexpr int OWN = 16 / WK, V = OWN < 4 ? OWN : 4, CHUNK = T::CHUNK;
    typedef float fv __attribute__((ext_vector_type(V)));
    fv* red = reinterpret_cast<fv*>(lds);
    auto slot = [&](int tile, int owner, int from, int k) {  // registers k V .. of what `from` gives `owner`
        return ((((tile * WK + owner) * (WK - 1) + (from < owner ? from : from - 1)) * CO + col) * (OWN / V) + k) * 64 + lane;
    };
#pragma unroll
    for (int n0 = 0; n0 < TRIOS; n0 += CHUNK) {
        __syncthreads();
#pragma unroll
        for (int n = n0; n < n0 + CHUNK && n < TRIOS; ++n)
#pragma unroll
            for (int owner = 0; owner < WK; ++owner)
                if (owner != wk)
#pragma unroll
                    for (int k = 0; k < OWN / V; ++k) {
                        fv v;
#pragma unroll
                        for (int c = 0; c < V; ++c) v[c] = acc[n / CIW][n % CIW][owner * OWN + k * V + c];
                        red[slot(n - n0, owner, wk, k)] = v;
                    }
        __syncthreads();
#pragma unroll
        for (int owner = 0; owner < WK; ++owner)
            if (owner == wk)
#pragma unroll
                for (int n = n0; n < n0 + CHUNK && n < TRIOS; ++n) {
                    float* po = part + (size_t)blockIdx.x * out.split + (j0 + n / CIW) * out.tap + (co0 + 4 * h) * out.co + (ci0 + 32 * (n % CIW) + i) * out.ci;
#pragma unroll
                    for (int k = 0; k < OWN / V; ++k) {
                        fv v;
#pragma unroll
                        for (int c = 0; c < V; ++c) v[c] = acc[n / CIW][n % CIW][owner * OWN + k * V + c];
#pragma unroll
                        for (int from = 0; from < WK; ++from)
                            if (from != owner) v += red[slot(n - n0, owner, from, k)];
#pragma unroll
                        for (int c = 0; c < V; ++c) {
                            const int reg = owner * OWN + k * V + c;
                            po[((reg & 3) + 8 * (reg >> 2)) * out.co] = v[c];
                        }
                    }
                }
    }
}

// grid = (splits, tap groups x ci tiles, groups of CO co tiles); the first n_hi tap groups take NHI taps, the others NHI - 1
template <int COUT, int CO, int CIW, int NHI>
__global__ __launch_bounds__(64 * ACT_WAVES, 2) void act_wgrad_kernel(const float* __restrict__ dz, ActIn in, float* __restrict__ part,
                                                                      ActOut out, float* __restrict__ bias_grad, int B, int L,
                                                                      int cin, int ks, int units_per_split, int n_hi) {
    using T = ActTile<CO, CIW, NHI>;
    __shared__ __align__(16) unsigned short lds[T::BYTES / 2];
    const int y = blockIdx.y / (cin / (32 * CIW));
    if (bias_grad && blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x < COUT) bias_grad[threadIdx.x] = 0.f;
    if (y < n_hi) {
        act_wgrad_body<COUT, CO, CIW, NHI>(lds, dz, in, part, out, B, L, cin, ks, units_per_split, y * NHI);
    } else {
        if constexpr (NHI > 1)
            act_wgrad_body<COUT, CO, CIW, NHI - 1>(lds, dz, in, part, out, B, L, cin, ks, units_per_split, n_hi * NHI + (y - n_hi) * (NHI - 1));
    }
}

// dw[co][ci][j] = sum_split part[split][j][co][ci].  Four ci per lane; the splits are dealt
// to GRP groups of lanes, each with independent 16-byte loads, combined in a fixed order.  A small dw needs many groups to
// have enough loads in flight.
template <int GRP>
__global__ __launch_bounds__(256) void act_wgrad_reduce_kernel(const float* __restrict__ part, int nsplit, int cout, int cin, int ks,
                                                               float* __restrict__ dw) {
    constexpr int QB = 256 / GRP;
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
