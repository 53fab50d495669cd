// camal_common.hpp — what every translation unit of the library shares: vector types, 4-channel loads and stores, errors.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>

namespace camal {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
}
// two floats -> one dword of two bf16 (round to nearest even) in ONE v_cvt_pk_bf16_f32: hipcc turns a 4-vector
// conversion into four single-value converts and two v_perm_b32 (3x the instructions; the bf16 epilogues are
// VALU-issue bound), a 2-vector conversion into the packed instruction
__device__ __forceinline__ unsigned pk_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const f32x2 v = {a, b};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ void store4(__bf16* p, float a, float b, float c, float d) {
    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 v = {pk_bf16(a, b), pk_bf16(c, d)};
    *reinterpret_cast<u32x2*>(p) = v;
}

__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
    float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void load4(const __bf16* p, float (&v)[4]) {
    bf16x4 t = *reinterpret_cast<const bf16x4*>(p);
    v[0] = (float)t[0]; v[1] = (float)t[1]; v[2] = (float)t[2]; v[3] = (float)t[3];
}

// Sets camal_last_error() of this thread and returns the code
int fail(int code, const std::string& msg);

}  // namespace camal

#define HIP_TRY(expr)                                                                               \
    do {                                                                                            \
        hipError_t e__ = (expr);                                                                    \
        if (e__ != hipSuccess)                                                                      \
            return camal::fail(CAMAL_ERR_HIP, std::string(#expr) + ": " + hipGetErrorString(e__));  \
    } while (0)
