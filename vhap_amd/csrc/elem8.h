// Eight consecutive elements of a float32 / bfloat16 / float16 array to and from fp32 registers, by a VHAP_DTYPE_* code that is a constant where the kernel
// is built per type.  The pointer needs the element's own alignment only: 16-byte accesses at any address are legal on this target, so an odd row length or
// a view into a flat buffer costs no scalar path.
#pragma once
#include <hip/hip_fp16.h>

#include "common.h"

struct __attribute__((packed, aligned(4))) VhapVec16a4 { unsigned w[4]; };
struct __attribute__((packed, aligned(2))) VhapVec16a2 { unsigned w[4]; };

__device__ __forceinline__ void vhap_load8(const void* p, long long i, int dt, int valid, float (&v)[8]) {
    if (dt == VHAP_DTYPE_F32) {
        const float* q = static_cast<const float*>(p) + i;
        if (valid >= 8) {
            const VhapVec16a4 a = *reinterpret_cast<const VhapVec16a4*>(q), b = *reinterpret_cast<const VhapVec16a4*>(q + 4);
#pragma unroll
            for (int k = 0; k < 4; k++) { v[k] = __uint_as_float(a.w[k]); v[4 + k] = __uint_as_float(b.w[k]); }
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = k < valid ? q[k] : 0.f;
        }
        return;
    }
    const unsigned short* q = static_cast<const unsigned short*>(p) + i;
    unsigned w[4];
    if (valid >= 8) {
        const VhapVec16a2 a = *reinterpret_cast<const VhapVec16a2*>(q);
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = a.w[k];
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = (2 * k < valid ? (unsigned)q[2 * k] : 0u) | (2 * k + 1 < valid ? (unsigned)q[2 * k + 1] << 16 : 0u);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if (dt == VHAP_DTYPE_BF16) {
            v[2 * k] = __uint_as_float(w[k] << 16);
            v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
        } else {
            v[2 * k] = __half2float(__ushort_as_half((unsigned short)(w[k] & 0xffff)));
            v[2 * k + 1] = __half2float(__ushort_as_half((unsigned short)(w[k] >> 16)));
        }
    }
}

// to nearest, halves to even; a NaN stays one (the target's own conversion, two numbers an instruction)
typedef __bf16 vhap_bf16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ unsigned vhap_bf16_pair(float lo, float hi) {
    const vhap_bf16x2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned vhap_bf16_bits(float f) { return vhap_bf16_pair(f, f) & 0xffffu; }

__device__ __forceinline__ void vhap_store8(void* p, long long i, int dt, int valid, const float (&v)[8]) {
    if (dt == VHAP_DTYPE_F32) {
        float* q = static_cast<float*>(p) + i;
        if (valid >= 8) {
            VhapVec16a4 a, b;
#pragma unroll
            for (int k = 0; k < 4; k++) { a.w[k] = __float_as_uint(v[k]); b.w[k] = __float_as_uint(v[4 + k]); }
            *reinterpret_cast<VhapVec16a4*>(q) = a;
            *reinterpret_cast<VhapVec16a4*>(q + 4) = b;
        } else {
#pragma unroll
            for (int k = 0; k < 8; k++)
                if (k < valid) q[k] = v[k];
        }
        return;
    }
    unsigned h[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
        h[k] = dt == VHAP_DTYPE_BF16 ? vhap_bf16_pair(v[2 * k], v[2 * k + 1])
                                     : (unsigned)__half_as_ushort(__float2half_rn(v[2 * k])) | (unsigned)__half_as_ushort(__float2half_rn(v[2 * k + 1])) << 16;
    unsigned short* q = static_cast<unsigned short*>(p) + i;
    if (valid >= 8) {
        VhapVec16a2 a;
#pragma unroll
        for (int k = 0; k < 4; k++) a.w[k] = h[k];
        *reinterpret_cast<VhapVec16a2*>(q) = a;
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++)
            if (k < valid) q[k] = (unsigned short)(h[k >> 1] >> 16 * (k & 1));
    }
}
