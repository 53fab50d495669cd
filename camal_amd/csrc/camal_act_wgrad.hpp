// camal_act_wgrad.hpp — the weight gradient from 8-bit activation checkpoints.  Included by one translation unit for each number
// of co tiles a workgroup takes (camal_act_wgrad1.hip, 2, 4), so that they compile side by side.
#pragma once
#include <type_traits>

#include "../../include/camal_hip.h"
#include "camal_act_codes.hpp"

namespace camal {

// ---- weight gradient from the checkpoint, on MFMA ------------------------------------------------------------------------
//   dw[co][ci][j] = sum_{b,t} dz[b][t][co] a[b][clamp(t + j - ks/2)][ci],  a = bf16(relu(gamma x + beta) [+ skip])
// GEMM view: M = co, N = ci, K = time, for every tap j.  v_mfma_f32_32x32x16_bf16 takes 16 timesteps per instruction: lane
// (i = l & 31, h = l >> 5) feeds 8 consecutive times of channel co_i (A) and ci_i (B).
//   A code and its scale are exact in bf16, the activation made of them is not: it is computed in fp32 and rounded to bf16, by at
//   most 2^-8 of itself.  dz is cut into three bf16 pieces, each the leading 8 bits of what is
//   left: they add up to it exactly, so the three products, summed in the instruction's fp32, are an fp32 product sum of dz and
//   the rounded activation at a third of the bf16 rate, 5 times the rate of fp32 MFMA.  (Pieces and products below 2^-126 count
//   as zero: a dz under about 2^-104 keeps fewer of its bits.)
// One wave = 32 co x 32 ci x NTAP taps on a unit of 64 timesteps.  The 8 waves of a workgroup are CO co tiles x WK units:
// the CO waves of a unit share its decoded input, and the WK sums of a tile are added in LDS before they leave the workgroup
// (what the partial sums weigh is what bounds a short call).
//   A: dz straight from global memory into registers, as the fragment wants it: no other wave needs these values; rows past
//      the window's end are out of the buffer's range and come back as zeros;
//   B: the unit's input, decoded into LDS as plain rows [time][32 channels] of bf16, read with the transposing
//      ds_read_b64_tr_b16 (4 times of a channel per lane): a tap is a row offset, and a row is 64 bytes, so neither side
//      has bank conflicts.
// On these SIMDs a vector instruction hides behind a matrix product only up to about three per product (measured: 15.9 ns a
// product alone, 16.3 with 2, 18.1 with 4, 23.3 with 8 vector instructions to each, two waves), so what counts beside the
// products is the number of vector instructions: cutting dz takes 44 per 21 products of 7 taps, decoding is shared.  The source
// deals cutting and decoding out between the products; the compiled loop keeps to that in part only, since format, skip branch
// and zero padding are run-time choices and each ends a basic block: a step of <4, 7> is 20 products, the decoding (4 + 17 or 4 +
// 36 vector instructions) without one, 38 to 42 of cutting with one to three in between, and so on.  Registers that find no place,
// per lane: 4, 12 and 26 with one co tile and 5, 6 and 7 taps, 8 with two and 7, else none.
// 256 -> 256 channels, 7 taps, 8 x 10080: 173 to 180 us, 1240 to 1290 TF of bf16 products (MFMA busy 0.71, the clock at 1.74 GHz under this load;
// a large library product reaches 1130 TF here); 128 -> 128, 7 taps, 128 x 510: 43 us (and 6 of the
// second stage), of which about 7 until the first product,
// 25 in the products and 6 in writing 29 MB of sums at the end.  Error against 64 bits on that case, norm-wise, dz of either sign:
// 2.7e-7 (8 x 10080 of 256 channels 4.9e-7 to 5.9e-7); with two pieces of dz instead of three 2.5e-6 in 0.8 of the time: not taken.
// Where all terms have one sign 8e-8 and 1.1e-6, and 2.6e-6 at any length (the chains of sums are bounded: camal_act.hip).
// Each split's sums go to part[split][j][co][ci]; act_wgrad_reduce_kernel adds them in a fixed order.
typedef short s16x4 __attribute__((ext_vector_type(4)));

// How a workgroup is made up, and the passes in which the CO waves of a unit fill its input tile (4 channels per lane)
template <int CO, int NTAP> struct ActTile {
    static constexpr int WK = ACT_WAVES / CO;
    static constexpr int RPP = 8 * CO, ROWS = (ACT_UNIT + NTAP + 6) / 8 * 8, PASS = (ROWS + RPP - 1) / RPP;
    static constexpr int TILE = ROWS * 32;  // halfwords
    // LDS: two tiles per unit, then the waves' sums: ACT_WAVES * (16 - 16 / WK) registers per accumulator, CHUNK of them at once
    static constexpr int SUMS = ACT_WAVES * (16 - 16 / WK) * 64 * 4, FIT = 128 * 1024 / SUMS;
    static constexpr int CHUNK = NTAP < FIT ? NTAP : FIT;
    static constexpr int BYTES = 2 * WK * 2 * TILE > CHUNK * SUMS ? 2 * WK * 2 * TILE : CHUNK * SUMS;
};

template <int CO, int NTAP>
__device__ __forceinline__ void act_wgrad_body(unsigned short* lds, const float* __restrict__ dz, const ActIn& in,
                                               float* __restrict__ part, ActOut out, int B, int L, int cin, int cout,
                                               int ks, int units_per_split, int split, int z, int j0) {
    using T = ActTile<CO, NTAP>;
    constexpr int WK = T::WK;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wk = wave / CO, col = wave % CO;
    const int i = lane & 31, h = lane >> 5, co0 = (z * CO + col) * 32, ci0 = blockIdx.y % (cin / 32) * 32;
    const int tpw = (L + ACT_UNIT - 1) / ACT_UNIT, total = B * tpw;
    const int lo = min(total, split * units_per_split), hi = min(total, lo + units_per_split);

    f32x16 acc[NTAP];
#pragma unroll
    for (int j = 0; j < NTAP; ++j)
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[j][k] = 0.f;

    // ---- the input tile: a lane has 4 channels of every RPP-th row ----
    const int cq = lane % 8, r0 = col * 8 + lane / 8, lgc = 31 - __builtin_clz(cin);
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
        if (col * 8 + p * T::RPP >= T::ROWS) return;
        const int rel = max(-o.rb, min(o.tb - o.rb + r0 + p * T::RPP, L - 1 - o.rb));
        const int oc = (rel << lgc) + ci0 + 4 * cq, os = (rel << (lgc - 5)) + ci0 / 32;
        cw[p] = __builtin_amdgcn_raw_buffer_load_b32(o.codes, oc, 0, 0);
        cs[p] = __builtin_amdgcn_raw_buffer_load_b8(o.scales, os, 0, 0);
        if (in.codes_r) {
            rw[p] = __builtin_amdgcn_raw_buffer_load_b32(o.codes_r, oc, 0, 0);
            rs[p] = __builtin_amdgcn_raw_buffer_load_b8(o.scales_r, os, 0, 0);
        }
    };
    auto stash = [&](unsigned short* tile, int tb, int p) {
        if (col * 8 + p * T::RPP >= T::ROWS) return;
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
        *reinterpret_cast<uint2*>(tile + row * 32 + 4 * cq) = make_uint2(pk_bf16(a[0], a[1]), pk_bf16(a[2], a[3]));
    };

    // ---- dz: 8 times of this lane's channel per step, loaded two steps before it is cut, cut a step before it is used ----
    unsigned d[2][8];
    u32x4 pc[2][3];
    const int voff = (8 * h * cout + co0 + i) * 4;
    auto load_dz = [&](__amdgpu_buffer_rsrc_t src, int s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[s & 1][e] = __builtin_amdgcn_raw_buffer_load_b32(src, voff + (16 * s + e) * cout * 4, 0, 0);
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
    const int bp = (8 * h + (lane & 15) / 4) * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    auto operand = [&](const unsigned short* tile, int s, int tap) {
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const unsigned short* q = tile + bp + (16 * s + tap) * 32;
        const s16x4 b0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)q);
        const s16x4 b1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(q + 4 * 32));
        return __builtin_bit_cast(bf16x8, __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7));
    };

    // The positions of the unit at hand, the next one (whose tile is decoded meanwhile) and the one after it (whose codes are
    // fetched).  Past the split's end the last unit repeats, and counts for nothing: no rows of dz.
    auto dz_source = [&](int bb, int tt, bool live) {
        return __builtin_amdgcn_make_buffer_rsrc((void*)(dz + ((size_t)bb * L + tt * ACT_UNIT) * cout), 0,
                                                 live ? min(ACT_UNIT, L - tt * ACT_UNIT) * cout * 4 : 0, 0x00027000);
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
                // next tile decoded and its codes fetched again.  In clumps of their own these leave the matrix pipe idle (the
                // two waves of a SIMD share it evenly, reach their clumps together and overlap nothing); what the compiler
                // makes of this order is said above.
                constexpr int STASH = (T::PASS + 3) / 4, TASKS = 5 + STASH;
#pragma unroll
                for (int n = 0; n < NTAP; ++n) {
                    bf16x8 bn;
                    if (n + 1 < NTAP) bn = operand(now, s, n + 1);
                    else if (s < 3) bn = operand(now, s + 1, 0);
#pragma unroll
                    for (int p = 2; p >= 0; --p)
                        acc[n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, pc[s & 1][p]), bt, acc[n], 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < TASKS; ++t) {
                        if (t * NTAP / TASKS != n) continue;
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
    // acc[j][reg] of lane l: row co = co0 + (reg & 3) + 8 (reg >> 2) + 4 h, column ci = ci0 + i.  Of a tile's 16
    // registers each of its WK waves adds OWN and hands the others out through LDS, as many tiles at once as fit: the
    // workgroup has the CU to itself.
    constexpr int OWN = 16 / WK, V = OWN < 4 ? OWN : 4, CHUNK = T::CHUNK;
    typedef float fv __attribute__((ext_vector_type(V)));
    fv* red = reinterpret_cast<fv*>(lds);
    auto slot = [&](int tile, int owner, int from, int k) {  // registers k V .. of what `from` gives `owner`
        return ((((tile * WK + owner) * (WK - 1) + (from < owner ? from : from - 1)) * CO + col) * (OWN / V) + k) * 64 + lane;
    };
#pragma unroll
    for (int n0 = 0; n0 < NTAP; n0 += CHUNK) {
        __syncthreads();
#pragma unroll
        for (int n = n0; n < n0 + CHUNK && n < NTAP; ++n)
#pragma unroll
            for (int owner = 0; owner < WK; ++owner)
                if (owner != wk)
#pragma unroll
                    for (int k = 0; k < OWN / V; ++k) {
                        fv v;
#pragma unroll
                        for (int c = 0; c < V; ++c) v[c] = acc[n][owner * OWN + k * V + c];
                        red[slot(n - n0, owner, wk, k)] = v;
                    }
        __syncthreads();
#pragma unroll
        for (int owner = 0; owner < WK; ++owner)
            if (owner == wk)
#pragma unroll
                for (int n = n0; n < n0 + CHUNK && n < NTAP; ++n) {
                    float* po = part + (size_t)split * out.split + (j0 + n) * out.tap + (co0 + 4 * h) * out.co + (ci0 + i) * out.ci;
#pragma unroll
                    for (int k = 0; k < OWN / V; ++k) {
                        fv v;
#pragma unroll
                        for (int c = 0; c < V; ++c) v[c] = acc[n][owner * OWN + k * V + c];
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

// grid = (splits side by side, tap groups x ci tiles, sets of splits x groups of CO co tiles); the first n_hi tap groups take NHI taps, the others NHI - 1
template <int CO, int NHI>
__global__ __launch_bounds__(64 * ACT_WAVES, 2) void act_wgrad_kernel(const float* __restrict__ dz, ActIn in, float* __restrict__ part,
                                                                      ActOut out, float* __restrict__ bias_grad, int B, int L,
                                                                      int cin, int cout, int ks, int units_per_split,
                                                                      int n_hi) {
    using T = ActTile<CO, NHI>;
    __shared__ __align__(16) unsigned short lds[T::BYTES / 2];
    const int y = blockIdx.y / (cin / 32), nz = cout / (32 * CO), z = blockIdx.z % nz, split = blockIdx.z / nz * gridDim.x + blockIdx.x;
    if (bias_grad && blockIdx.x + blockIdx.y + blockIdx.z == 0 && threadIdx.x < cout) bias_grad[threadIdx.x] = 0.f;
    if (y < n_hi) {
        act_wgrad_body<CO, NHI>(lds, dz, in, part, out, B, L, cin, cout, ks, units_per_split, split, z, y * NHI);
    } else {
        if constexpr (NHI > 1)
            act_wgrad_body<CO, NHI - 1>(lds, dz, in, part, out, B, L, cin, cout, ks, units_per_split, split, z, n_hi * NHI + (y - n_hi) * (NHI - 1));
    }
}

// The kernel for the plan's tap groups
template <int CO>
int act_wgrad_launch(hipStream_t s, const ActPlan& p, const float* dz, const ActIn& in, float* sums, ActOut out, float* bias_grad, int cin,
                     int cout, int ks) {
    const dim3 grid(p.gx, p.groups * (cin / 32), p.nsplit / p.gx * (cout / (32 * CO)));
    auto launch = [&](auto taps) {
        hipLaunchKernelGGL((act_wgrad_kernel<CO, decltype(taps)::value>), grid, dim3(64 * ACT_WAVES), 0, s, dz, in, sums, out, bias_grad,
                           p.B, p.L, cin, cout, ks, p.units, p.n_hi);
        HIP_TRY(hipGetLastError());
        return 0;
    };
    switch (p.nhi) {
        case 1: return launch(std::integral_constant<int, 1>());
        case 3: return launch(std::integral_constant<int, 3>());
        case 5: return launch(std::integral_constant<int, 5>());
        case 6: return launch(std::integral_constant<int, 6>());
        case 7: return launch(std::integral_constant<int, 7>());
    }
    return fail(CAMAL_ERR_STATE, "no weight-gradient kernel for this kernel size");
}

}  // namespace camal
