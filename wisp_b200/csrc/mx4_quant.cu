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
// warp's loads and stores are whole lines.
#include "mx4.cuh"

namespace wisp {
namespace mx4 {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // 8-value pieces of a thread: loads in flight

__device__ __forceinline__ uint32_t quantize_piece(const float (&v)[8], uint32_t &byte) {
    // |x| compared as integers: NaN above infinity above every number
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 1));
    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 2));
    const uint32_t field = m >> 23;
    byte = field == 255 ? 255 : field > 2 ? field - 2 : 0;
    if (byte == 255) return 0;
    const float inv = __uint_as_float((254 - byte) << 23);  // 2^(127 - byte) = 2^-s
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = v[i] * inv;
    return f32x8_to_e2m1(q);
}

// Piece p of the matrix: columns 8 (p % (cols / 8)) .. of row p / (cols / 8).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    quantize_kernel(const T *x, int64_t pieces, int64_t cols, int64_t row_stride, uint32_t *codes, uint8_t *scales) {
    const int64_t first = (int64_t)blockIdx.x * kThreads * kUnroll + threadIdx.x;
    float v[kUnroll][8];
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        if (p < pieces) {
            int64_t at = p * 8;
            if (row_stride != cols) at = at / cols * row_stride + at % cols;
            Vec8<T>::load(x + at, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
    }
#pragma unroll
    for (int i = 0; i < kUnroll; ++i) {
        const int64_t p = first + i * kThreads;
        uint32_t byte;
        const uint32_t c = quantize_piece(v[i], byte);
        if (p < pieces) {
            codes[p] = c;
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
    const int64_t pieces = rows * (cols / 8);
    const unsigned grid = (unsigned)((pieces + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    uint32_t *c = reinterpret_cast<uint32_t *>(codes);
    uint8_t *b = reinterpret_cast<uint8_t *>(scales);
    if (dtype == WISP_BF16)
        quantize_kernel<<<grid, kThreads, 0, s>>>(reinterpret_cast<const __nv_bfloat16 *>(x), pieces, cols, row_stride, c, b);
    else if (dtype == WISP_FP16)
        quantize_kernel<<<grid, kThreads, 0, s>>>(reinterpret_cast<const __half *>(x), pieces, cols, row_stride, c, b);
    else
        quantize_kernel<<<grid, kThreads, 0, s>>>(reinterpret_cast<const float *>(x), pieces, cols, row_stride, c, b);
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
