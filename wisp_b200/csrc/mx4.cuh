// Microscaled 4-bit floating point (MXFP4), as the kernels see it.
//
// A matrix [rows][K], K a multiple of 32, is held as codes [rows][K / 2] --
// two E2M1 values (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5,
// 2, 3, 4, 6) a byte, the even column in the low nibble -- and scale bytes
// [rows][K / 32], E8M0: byte b stands for 2^(b - 127), 255 for NaN.  The
// value of a code is its E2M1 value times its block's scale.  This is the
// layout of MXFP4 checkpoints; every kernel reads it as it is, so that a page
// of expert weights needs no rearrangement after its copy.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace wisp {

// Rows of `bytes` bytes, `stride` bytes apart.
struct ByteRows {
    uintptr_t at;
    int64_t rows, stride, bytes;
    // Whether one of them has a byte of the `n` bytes at `p`.
    bool meets(uintptr_t p, int64_t n) const {
        const int64_t lo = (int64_t)(p - at), hi = lo + n;  // relative to the first row
        if (hi <= 0) return false;
        if (stride == 0 || rows == 1) return lo < bytes;
        const int64_t i = lo < bytes ? 0 : (lo - bytes) / stride + 1;  // the first row that ends behind lo
        return i < rows && i * stride < hi;
    }
};
inline bool meets(const void *p, int64_t bytes, const void *q, int64_t more) {
    return ByteRows{reinterpret_cast<uintptr_t>(p), 1, 0, bytes}.meets(reinterpret_cast<uintptr_t>(q), more);
}

namespace mx4 {

constexpr int kBlock = 32;  // values that share a scale

// 2^(b - 127) (b = 0 is a subnormal float, b = 255 NaN).
__device__ __forceinline__ float scale_value(uint32_t b) {
    return __uint_as_float(b == 0 ? 0x00400000u : b == 255 ? 0x7FFFFFFFu : b << 23);
}

// Two E2M1 codes (one byte, low nibble first) as fp16, exact.
__device__ __forceinline__ uint32_t e2m1x2_to_f16x2(uint32_t byte) {
    uint32_t r;
    asm("{\n .reg .b8 b;\n cvt.u8.u32 b, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}" : "=r"(r) : "r"(byte));
    return r;
}
// Eight codes (one 32-bit word, low nibble first) as four fp16 pairs.
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n cvt.rn.f16x2.e2m1x2 %0, b0;\n"
        " cvt.rn.f16x2.e2m1x2 %1, b1;\n cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// Eight floats as codes, to nearest even, saturating at 6.
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&v)[8]) {
    uint32_t r;
    asm("{\n .reg .b8 b0, b1, b2, b3;\n cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n mov.b32 %0, {b0, b1, b2, b3};\n}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}

// Eight consecutive values, rounded once from fp32.
template <typename T>
struct Vec8;
template <>
struct Vec8<float> {
    static __device__ __forceinline__ void store(float *p, const float (&v)[8]) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
};
template <>
struct Vec8<__nv_bfloat16> {
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const float (&v)[8]) {
        uint4 a;
        __nv_bfloat162 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&a, h, 16);
        *reinterpret_cast<uint4 *>(p) = a;
    }
};
template <>
struct Vec8<__half> {
    static __device__ __forceinline__ void store(__half *p, const float (&v)[8]) {
        uint4 a;
        __half2 h[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        memcpy(&a, h, 16);
        *reinterpret_cast<uint4 *>(p) = a;
    }
};

}  // namespace mx4
}  // namespace wisp
