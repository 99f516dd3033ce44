// Quantising a matrix to MXFP4 and reading it back (layout: mx4.cuh).
//
// A block of 32 values has m = max |x| and the scale 2^s, s = floor(log2 m)
// - 2 (the OCP microscaling rule: 2 is E2M1's largest exponent), held to
// [-127, 127]; its codes are x * 2^-s rounded to nearest even, saturating at
// 6.  Read off fp32 bits the scale byte is m's exponent field less 2, not
// below 0; a block with an infinity or a NaN gets byte 255 and codes 0, so it
// reads back as NaN.  The product by a power of two is exact (or so far below
// 0.25 that its rounding does not matter), hence one rounding a value.
//
// Bound by HBM: 2.53 bytes a bf16 value each way.  Four threads share a
// block: each holds 8 values (one 16-byte load of 16-bit types), the maximum
// takes two shuffles, and the codes leave as one 32-bit store a thread, so a
// warp's loads and stores are whole lines.  The values stay as loaded until
// they are rounded: widened at once they took twice the registers, and the
// loads in flight of half as many threads.  In a graph of calls whose inputs, in
// turn, exceed L2: 49152 x 2048 bf16 36 us to MXFP4 and 41 back, 255 MB each, 6.6
// TB/s together, what a copy has; rows that lie apart 48 (a division of 64 bits
// for 8 values); fp32 64 and 108 back (456 MB, 7.1 and 4.2 TB/s); 1021 x 4096 fp16
// 6.1 us for both (21 MB, 3.5 TB/s); one row of 2048: 1.2 us each, a launch.
#include "mx4.cuh"

namespace wisp {
namespace mx4 {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // 8-value pieces of a thread: loads in flight

// Eight values as they were loaded; the largest magnitude as fp32 bits with
// NaN above infinity above every number.  16-bit types compare two values an
// instruction and are widened only when they are rounded.
template <typename T>
struct Raw8;
template <>
struct Raw8<float> {
    uint4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = ld_stream16(p), b = ld_stream16(p + 4);
    }
    __device__ __forceinline__ void zero() { a = b = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ uint32_t block_max() const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        return max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
    }
};
template <typename T2>
__device__ __forceinline__ T2 as2(uint32_t w) {
    T2 r;
    memcpy(&r, &w, 4);
    return r;
}
template <typename T, typename T2>
struct Raw8x16 {
    uint4 a;
    __device__ __forceinline__ void load(const T *p) { a = ld_stream16(p); }
    __device__ __forceinline__ void zero() { a = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ T2 pair_max() const {
        T2 m = __hmax2_nan(__hmax2_nan(__habs2(as2<T2>(a.x)), __habs2(as2<T2>(a.y))),
                           __hmax2_nan(__habs2(as2<T2>(a.z)), __habs2(as2<T2>(a.w))));
        m = __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
        return __hmax2_nan(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    }
};
template <>
struct Raw8<__nv_bfloat16> : Raw8x16<__nv_bfloat16, __nv_bfloat162> {
    __device__ __forceinline__ uint32_t block_max() const {
        const __nv_bfloat162 m = pair_max();
        return __float_as_uint(__bfloat162float(__hmax_nan(m.x, m.y)));
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        v[0] = bf16lo(a.x), v[1] = bf16hi(a.x), v[2] = bf16lo(a.y), v[3] = bf16hi(a.y);
        v[4] = bf16lo(a.z), v[5] = bf16hi(a.z), v[6] = bf16lo(a.w), v[7] = bf16hi(a.w);
    }
};
template <>
struct Raw8<__half> : Raw8x16<__half, __half2> {
    __device__ __forceinline__ uint32_t block_max() const {
        const __half2 m = pair_max();
        return __float_as_uint(__half2float(__hmax_nan(m.x, m.y)));
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = __half22float2(as2<__half2>(w[i]));
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
    }
};

// Piece p of the matrix: columns 8 (p % (cols / 8)) .. of row p / (cols / 8).
template <typename T, bool CONTIGUOUS>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(const T *x, int64_t pieces, int64_t cols, int64_t row_stride, uint32_t *codes, uint8_t *scales) {
    const int64_t first = (int64_t)blockIdx.x * kThreads * kUnroll + threadIdx.x;
    Raw8<T> v[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        if (p < pieces)
            v[i].load(x + (CONTIGUOUS ? p * 8 : p * 8 / cols * row_stride + p * 8 % cols));
        else
            v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        const uint32_t field = v[i].block_max() >> 23;
        const uint32_t byte = field == 255 ? 255 : field > 2 ? field - 2 : 0;
        const float inv = __uint_as_float((254 - byte) << 23);  // 2^(127 - byte) = 2^-s
        float f[8];
        v[i].widen(f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= inv;
        if (p < pieces) {
            codes[p] = byte == 255 ? 0 : f32x8_to_e2m1(f);
            if ((p & 3) == 0) scales[p >> 2] = (uint8_t)byte;
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads)
    dequantize_kernel(const uint32_t *codes, const uint8_t *scales, int64_t pieces, T *out) {
    const int64_t first = (int64_t)blockIdx.x * kThreads * kUnroll + threadIdx.x;
    uint32_t c[kUnroll], b[kUnroll];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        c[i] = p < pieces ? __ldg(codes + p) : 0;
        b[i] = p < pieces ? __ldg(scales + (p >> 2)) : 0;
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        if (p >= pieces) return;
        const float s = scale_value(b[i]);
        uint32_t h[4];
        e2m1x8_to_f16(c[i], h);
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<__half2 *>(&h[j]));
            v[2 * j] = f.x * s, v[2 * j + 1] = f.y * s;
        }
        Vec8<T>::store(out + p * 8, v);
    }
}

int check_matrix(const char *who, int32_t dtype, int64_t rows, int64_t cols) {
    if (dtype < WISP_BF16 || dtype > WISP_FP32) return set_error(std::string(who) + ": unknown dtype"), WISP_ERR_INVALID;
    if (rows < 0 || cols < kBlock || cols % kBlock || rows > (int64_t(1) << 38) / cols)
        return set_error(std::string(who) + ": need rows >= 0, columns a multiple of 32, at most 2^38 values"),
               WISP_ERR_INVALID;
    return WISP_OK;
}

}  // namespace
}  // namespace mx4
}  // namespace wisp

using namespace wisp;
using namespace wisp::mx4;

extern "C" int wisp_mx4_quantize(const void *x, int32_t dtype, int64_t rows, int64_t cols, int64_t row_stride,
                                 void *codes, void *scales, void *stream) {
    if (const int rc = check_matrix("wisp_mx4_quantize", dtype, rows, cols)) return rc;
    if (rows == 0) return WISP_OK;
    if (!x || !codes || !scales) return set_error("wisp_mx4_quantize: NULL tensor"), WISP_ERR_INVALID;
    const int64_t size = dtype == WISP_FP32 ? 4 : 2;
    if (rows == 1) row_stride = cols;
    if (row_stride < cols || row_stride * size % 16 || reinterpret_cast<uintptr_t>(x) % 16 ||
        reinterpret_cast<uintptr_t>(codes) % 4)
        return set_error("wisp_mx4_quantize: rows must not overlap and must start on 16-byte boundaries"),
               WISP_ERR_INVALID;
    const int64_t code_bytes = rows * (cols / 2), scale_bytes = rows * (cols / kBlock);
    const ByteRows in{reinterpret_cast<uintptr_t>(x), rows, row_stride * size, cols * size};
    if (in.meets(reinterpret_cast<uintptr_t>(codes), code_bytes) ||
        in.meets(reinterpret_cast<uintptr_t>(scales), scale_bytes) || meets(codes, code_bytes, scales, scale_bytes))
        return set_error("wisp_mx4_quantize: codes, scales and x overlap"), WISP_ERR_INVALID;
    const int64_t pieces = rows * (cols / 8);
    const unsigned grid = (unsigned)((pieces + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint32_t *c = reinterpret_cast<uint32_t *>(codes);
    uint8_t *b = reinterpret_cast<uint8_t *>(scales);
    const auto run = [&](auto zero) {
        using T = decltype(zero);
        const T *in = reinterpret_cast<const T *>(x);
        if (row_stride == cols)
            quantize_kernel<T, true><<<grid, kThreads, 0, s>>>(in, pieces, cols, row_stride, c, b);
        else
            quantize_kernel<T, false><<<grid, kThreads, 0, s>>>(in, pieces, cols, row_stride, c, b);
    };
    if (dtype == WISP_BF16)
        run(__nv_bfloat16());
    else if (dtype == WISP_FP16)
        run(__half());
    else
        run(float());
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}

extern "C" int wisp_mx4_dequantize(const void *codes, const void *scales, int64_t rows, int64_t cols, void *out,
                                   int32_t dtype, void *stream) {
    if (const int rc = check_matrix("wisp_mx4_dequantize", dtype, rows, cols)) return rc;
    if (rows == 0) return WISP_OK;
    if (!codes || !scales || !out) return set_error("wisp_mx4_dequantize: NULL tensor"), WISP_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(codes) % 4 || reinterpret_cast<uintptr_t>(out) % 16)
        return set_error("wisp_mx4_dequantize: codes must be aligned to 4 bytes, out to 16"), WISP_ERR_INVALID;
    const int64_t out_bytes = rows * cols * (dtype == WISP_FP32 ? 4 : 2);
    if (meets(codes, rows * (cols / 2), out, out_bytes) || meets(scales, rows * (cols / kBlock), out, out_bytes))
        return set_error("wisp_mx4_dequantize: out overlaps codes or scales"), WISP_ERR_INVALID;
    const int64_t pieces = rows * (cols / 8);
    const unsigned grid = (unsigned)((pieces + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const uint32_t *c = reinterpret_cast<const uint32_t *>(codes);
    const uint8_t *b = reinterpret_cast<const uint8_t *>(scales);
    if (dtype == WISP_BF16)
        dequantize_kernel<<<grid, kThreads, 0, s>>>(c, b, pieces, reinterpret_cast<__nv_bfloat16 *>(out));
    else if (dtype == WISP_FP16)
        dequantize_kernel<<<grid, kThreads, 0, s>>>(c, b, pieces, reinterpret_cast<__half *>(out));
    else
        dequantize_kernel<<<grid, kThreads, 0, s>>>(c, b, pieces, reinterpret_cast<float *>(out));
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}
