// The 8-bit cache format shared by the kernels that write and read it: codes and scales, and the checks of its shape.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

// Shape rules of the cache, common to every entry point that takes one.
inline int vkc_q8_check(vkc_ctx *ctx, const char *who, int64_t B, int64_t Hkv, int64_t Lmax, int64_t D, int64_t block, int cache_dtype) {
    VKC_REQUIRE(ctx, cache_dtype == VKC_E4M3 || cache_dtype == VKC_I8, "%s: the cache type is %d, not VKC_E4M3 or VKC_I8", who, cache_dtype);
    if (D != 64 && D != 128 && D != 256) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "%s: head dim %lld not in {64,128,256}", who, (long long) D);
    if (block != 32 && block != 64 && block != 128) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "%s: block of %lld tokens not in {32,64,128}", who, (long long) block);
    VKC_REQUIRE(ctx, Lmax % block == 0, "%s: Lmax=%lld is not a multiple of the block of %lld tokens", who, (long long) Lmax, (long long) block);
    VKC_REQUIRE(ctx, Lmax <= INT32_MAX - 1024 && B <= 65535 && Hkv <= 65535, "%s: extents too large", who);
    return VKC_OK;
}

#ifdef __CUDACC__
namespace q8 {

    __device__ __forceinline__ float nan_value() { return __int_as_float(0x7fc00000); }

    // Scale of a block whose largest magnitude has the fp32 bits `top` (sign cleared).
    template <bool kE4m3> __device__ __forceinline__ float scale_of(uint32_t top) {
        if (top >= 0x7f800000u) return nan_value();
        if (top == 0) return 0.f;
        if (kE4m3) {
            // top = 1.m * 2^(E-127); 448 = 1.75 * 2^8: the exponent of the scale is E - 8, one more when 1.m > 1.75, at least 1 (2^-126)
            int e = (int) (top >> 23) - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
            e     = e < 1 ? 1 : e;
            return __uint_as_float((uint32_t) e << 23);
        }
        return fmaxf(__fdiv_rn(__uint_as_float(top), 127.0f), __uint_as_float(1u << 23));
    }

    __device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
        return (uint32_t) (a & 0xff) | (uint32_t) (b & 0xff) << 8 | (uint32_t) (c & 0xff) << 16 | (uint32_t) d << 24;
    }
    __device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
    __device__ __forceinline__ float e4m3_value(uint32_t code) { // low 8 bits
        return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t) (code & 0xff), __NV_E4M3)));
    }
    __device__ __forceinline__ int clamp127(int v) { return v > 127 ? 127 : (v < -127 ? -127 : v); }

    // `q`, the quotient that was asked for cut off towards zero, with its last bit set when something was cut off. Rounded to fewer bits
    // (two at least) from there it gives what the exact quotient gives: a value in the middle between two codes has that bit clear,
    // so one beside the middle keeps its side.
    __device__ __forceinline__ float odd(float q, bool cut) { return __uint_as_float(__float_as_uint(q) | (cut ? 1u : 0u)); }

    // x / s to the nearest code, ties to even. A scale that this library wrote is a power of two for e4m3, so that the product with
    // its reciprocal is exact; any other one (a caller's own cache) takes the quotient cut off to fp32 (odd; the product that tells
    // whether something was cut off is exact in double: 24 bits by 24). int8: the product with the
    // rounded reciprocal names a code k that is at most one off, and the remainder x - k * s, which is exact in fp32 (both terms
    // are multiples of 2^-24 of the power of two above s, and their difference is below s), says whether it is the nearest.
    template <bool kE4m3> struct Quant {
        float s, inv;
        bool  none, exact; // none: every code is 0 (the scale is 0 or NaN; one below 2^-126 only goes with zeros); exact: inv is exactly 1 / s
        __device__ __forceinline__ explicit Quant(float scale) : s(scale) {
            const uint32_t bits = __float_as_uint(scale);
            none                = !(scale >= __uint_as_float(1u << 23));
            exact               = (bits & 0x7fffffu) == 0 && (bits >> 23) >= 1 && (bits >> 23) <= 253;
            inv                 = kE4m3 && exact ? __uint_as_float(0x7f000000u - bits) : __fdiv_rn(1.0f, scale);
        }
        // Eight values. int8: adding 1.5 * 2^23 leaves the nearest integer in the low bits of the sum.
        __device__ __forceinline__ uint2 eight(const float (&x)[8]) const {
            if (none) return make_uint2(0u, 0u);
            if (kE4m3) {
                if (exact)
                    return make_uint2(e4m3x4(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv), e4m3x4(x[4] * inv, x[5] * inv, x[6] * inv, x[7] * inv));
                return make_uint2(e4m3x4(quotient(x[0]), quotient(x[1]), quotient(x[2]), quotient(x[3])),
                                  e4m3x4(quotient(x[4]), quotient(x[5]), quotient(x[6]), quotient(x[7])));
            }
            constexpr float kMagic = 12582912.0f;
            const float     half   = 0.5f * s;
            uint32_t        z[8];
            float           rest[8], most = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float f = fmaf(x[e], inv, kMagic);
                z[e]          = __float_as_uint(f);
                rest[e]       = fmaf(kMagic - f, s, x[e]);
                most          = fmaxf(most, fabsf(rest[e]));
            }
            if (most >= half) { // some value lies in the middle between two codes, or its code is one off
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float a = fabsf(rest[e]);
                    if (a > half || (a == half && (z[e] & 1u))) z[e] += rest[e] > 0.f ? 1u : ~0u;
                }
            }
            return make_uint2(bytes(z[0], z[1], z[2], z[3]), bytes(z[4], z[5], z[6], z[7]));
        }
        __device__ __forceinline__ float quotient(float x) const {
            const float q = __fdiv_rz(x, s);
            return odd(q, (double) q * (double) s != (double) x);
        }
        static __device__ __forceinline__ uint32_t bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) { // the low byte of each
            return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
        }
    };

    // code * s_old / s to the nearest code, s > s_old >= 0. e4m3 with powers of two: the product is exact; with others the quotient of
    // the product (28 bits) is cut off in double, whose remainder is exact, and then to fp32. int8: as above, the
    // close cases in double, where the quotient of the 31-bit product by the 24-bit scale keeps its side of the middle.
    template <bool kE4m3> struct Requant {
        float  ratio;
        double s_old, s;
        bool   exact;
        __device__ __forceinline__ Requant(float old_scale, float scale) : s_old(old_scale), s(scale) {
            exact = ((__float_as_uint(old_scale) | __float_as_uint(scale)) & 0x7fffffu) == 0;
            ratio = __fdiv_rn(old_scale, scale);
        }
        __device__ __forceinline__ int int8(int c) const {
            const float y = (float) c * ratio, r = rintf(y);
            if (fabsf(fabsf(y - r) - 0.5f) < 3.0517578125e-5f) return clamp127((int) rint((double) c * s_old / s));
            return clamp127((int) r);
        }
        __device__ __forceinline__ float e4m3(uint32_t code) const {
            const float v = e4m3_value(code);
            if (exact) return v * ratio;
            const double p = (double) v * s_old, q = __ddiv_rz(p, s);
            const float  f = __double2float_rz(q);
            return odd(f, (double) f != q || fma(-q, s, p) != 0.0);
        }
        __device__ __forceinline__ uint32_t four(uint32_t c) const {
            if (kE4m3) return e4m3x4(e4m3(c), e4m3(c >> 8), e4m3(c >> 16), e4m3(c >> 24));
            return pack4(int8((int8_t) c), int8((int8_t) (c >> 8)), int8((int8_t) (c >> 16)), int8((int8_t) (c >> 24)));
        }
    };

} // namespace q8
#endif
