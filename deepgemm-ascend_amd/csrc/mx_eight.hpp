// Eight values of a lane and their codes under a block's scale (mx_quant.hip, norm.hip, swiglu.hip): four lanes side by side hold a
// block of 32.
#pragma once

#include "mx_scale.hpp"

namespace dg {
namespace {

typedef unsigned int u32;

// (rows need no alignment: global memory takes 16 bytes at any address)
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef int i32x4_half __attribute__((ext_vector_type(4), aligned(2)));

// Largest of a value's over a block's four lanes and the partner block's value: lane exchanges within a row of the wave
// (xor 1, xor 2; in a half row mirrored, which is xor 4 for what four lanes share), cheaper than through LDS.
template <int CTRL>
__device__ __forceinline__ u32 dpp(u32 v) { return (u32)__builtin_amdgcn_mov_dpp((int)v, CTRL, 0xf, 0xf, true); }
constexpr int kXor1 = 0xb1, kXor2 = 0x4e, kMirror8 = 0x141;   // quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror

// Eight values of a lane: as loaded, their largest magnitude's fp32 bits, and their codes under the scale 2^(s - 127).
template <typename E> struct Eight;
template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* x) {
        const f32x4 a = *reinterpret_cast<const f32x4_any*>(x), b = *reinterpret_cast<const f32x4_any*>(x + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
    __device__ __forceinline__ u32 top() const {
        u32 a = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = max(a, __builtin_bit_cast(u32, v[i]) & 0x7fffffffu);
        return a;
    }
    __device__ __forceinline__ u32 e2m1(float s) const {
        u32 w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], s, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], s, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], s, 3);
    }
    __device__ __forceinline__ i32x2 e4m3(float inv) const {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
        return i32x2{lo, hi};
    }
};

// bf16 stays packed: the maximum on pairs of 16-bit integers, e2m1 from pairs of bf16.
template <>
struct Eight<uint16_t> {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    i32x4 w;
    __device__ __forceinline__ void load(const uint16_t* x) { w = *reinterpret_cast<const i32x4_half*>(x); }
    __device__ __forceinline__ void zero() { w = i32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ u32 top() const {
        u16x2 a = __builtin_bit_cast(u16x2, w[0] & 0x7fff7fff);
#pragma unroll
        for (int i = 1; i < 4; ++i) a = __builtin_elementwise_max(a, __builtin_bit_cast(u16x2, w[i] & 0x7fff7fff));
        return (u32)max(a[0], a[1]) << 16;
    }
    // (through a value of its own: the compiler takes element 0 of any element that is bit-cast in place)
    __device__ __forceinline__ bf16x2 pair(int i) const {
        const int v = w[i];
        return __builtin_bit_cast(bf16x2, v);
    }
    __device__ __forceinline__ u32 e2m1(float s) const {
        u32 c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(0), s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(1), s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(2), s, 2);
        return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, pair(3), s, 3);
    }
    __device__ __forceinline__ i32x2 e4m3(float inv) const {
        Eight<float> f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f.v[2 * i] = __builtin_bit_cast(float, (u32)w[i] << 16);
            f.v[2 * i + 1] = __builtin_bit_cast(float, (u32)w[i] & 0xffff0000u);
        }
        return f.e4m3(inv);
    }
};

// Exponent byte of the block whose values four lanes side by side hold, `top` the largest magnitude of a lane's.
template <bool FP4>
__device__ __forceinline__ u32 block_scale(u32 top) {
    top = max(top, dpp<kXor1>(top));
    top = max(top, dpp<kXor2>(top));
    return scale_byte<FP4>(top);
}

// Codes of eight fp32 values under the exponent byte s, which blocks of 255 (NaN) have zeros for.
__device__ __forceinline__ u32 codes_e2m1(const Eight<float>& v, u32 s) {
    const u32 c = v.e2m1(__builtin_bit_cast(float, s << 23));
    return s == 255u ? 0u : c;
}
__device__ __forceinline__ i32x2 codes_e4m3(const Eight<float>& v, u32 s) {
    const i32x2 c = v.e4m3(__builtin_bit_cast(float, (254u - s) << 23));
    return s == 255u ? i32x2{0, 0} : c;
}

// 2^(s - 127); exponent byte 0 is 2^-127, 255 is NaN.
__device__ __forceinline__ float scale_value(u32 s) {
    return __builtin_bit_cast(float, s == 255u ? 0x7fc00000u : s == 0u ? 0x00400000u : s << 23);
}

// Eight values of a row as they lie in memory, zeros behind the n-th; 16-byte accesses where all eight are there.
template <typename E> struct Raw;
template <>
struct Raw<float> {
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* x, int n) {
        a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        if (n >= 8) {
            a = reinterpret_cast<const f32x4_any*>(x)[0];
            b = reinterpret_cast<const f32x4_any*>(x)[1];
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < n) (i < 4 ? a : b)[i & 3] = x[i];
        }
    }
    __device__ __forceinline__ void values(Eight<float>& v) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v.v[i] = a[i];
            v.v[4 + i] = b[i];
        }
    }
};
template <>
struct Raw<uint16_t> {
    i32x4 w;
    __device__ __forceinline__ void load(const uint16_t* x, int n) {
        w = i32x4{0, 0, 0, 0};
        if (n >= 8) {
            w = *reinterpret_cast<const i32x4_half*>(x);
        } else {
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (i < n) w[i >> 1] |= (int)((u32)x[i] << (i & 1 ? 16 : 0));
        }
    }
    __device__ __forceinline__ void values(Eight<float>& v) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v.v[2 * i] = __builtin_bit_cast(float, (u32)w[i] << 16);
            v.v[2 * i + 1] = __builtin_bit_cast(float, (u32)w[i] & 0xffff0000u);
        }
    }
};
template <typename E>
__device__ __forceinline__ void load_eight(Eight<float>& v, const E* x, int n) {
    Raw<E> r;
    r.load(x, n);
    r.values(v);
}

// The first n of eight values to a row of E (one rounding, to nearest even, for bf16).
template <typename E>
__device__ __forceinline__ void store_eight(E* x, const Eight<float>& v, int n) {
    if (n >= 8) {
        if constexpr (sizeof(E) == 4) {
            reinterpret_cast<f32x4_any*>(x)[0] = f32x4{v.v[0], v.v[1], v.v[2], v.v[3]};
            reinterpret_cast<f32x4_any*>(x)[1] = f32x4{v.v[4], v.v[5], v.v[6], v.v[7]};
        } else {
            *reinterpret_cast<i32x4_half*>(x) = i32x4{(int)pack_bf16x2(v.v[0], v.v[1]), (int)pack_bf16x2(v.v[2], v.v[3]),
                                                      (int)pack_bf16x2(v.v[4], v.v[5]), (int)pack_bf16x2(v.v[6], v.v[7])};
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i < n) {
            if constexpr (sizeof(E) == 4) x[i] = v.v[i];
            else x[i] = f32_to_bf16_rne(v.v[i]);
        }
    }
}

}  // namespace
}  // namespace dg
