// camal_act_codes.hpp — the two code formats of the 8-bit activation checkpoints on the device.
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

// ReLU that lets a NaN through
__device__ __forceinline__ float act_relu(float u) { return u <= 0.f ? 0.f : u; }

}  // namespace camal
