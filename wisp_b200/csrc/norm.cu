// The step between two blocks of a decoder layer, in one pass over the rows:
//
//   z  = y                                      (post_weight NULL)
//      = y * rsqrt(mean(y^2) + eps) * post      (a norm after the block)
//   r' = residual + scale * gate * z            (gate NULL: 1)
//   n  = r' * rsqrt(mean(r'^2) + eps) * pre     (the norm before the next block)
//
// All of it in fp32; r' and n are rounded once each, n from the unrounded r'.
//
// Bound by HBM: y and the residual are read once, r' and n written once.  The
// CTAs are persistent; a thread copies the pieces of its CTA's next two rows
// to shared memory (cp.async, its own pieces only, so nothing but its own
// copies has to be waited for) while the present row lies in registers, which
// covers the two reductions of a row without the registers of a second row.
// The weights, which every row shares, stay in L1.  A thread's pieces of a row
// are VEC values wide: 8 where the width and every address allow 16-byte
// accesses, else 2, else 1 (2-byte pieces have no asynchronous copy and are
// loaded where they are used); NV of them, so that a row takes 256 threads or
// fewer where it can (more rows in flight, fewer warps in a reduction).
#include <type_traits>

#include "mx4.cuh"

namespace wisp {
namespace {

struct NormArgs {
    const void *y, *residual, *pre, *post, *gate;
    void *normed, *residual_out;
    int64_t rows, y_stride, res_stride, gate_stride;
    int cols, gate_kind;
    float scale, eps;
    int ahead;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
    return (float)v;
}
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f<__half>(float v) {
    return __float2half_rn(v);
}

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};
// VEC values through accesses of at most 16 bytes.
template <typename T, int VEC>
struct Piece {
    static constexpr int kPer = VEC * sizeof(T) > 16 ? 16 / sizeof(T) : VEC, kN = VEC / kPer;
    Pack<T, kPer> p[kN];
    __device__ __forceinline__ void load(const T *at) {
#pragma unroll
        for (int i = 0; i < kN; ++i) p[i] = reinterpret_cast<const Pack<T, kPer> *>(at)[i];
    }
    __device__ __forceinline__ void store(T *at) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) reinterpret_cast<Pack<T, kPer> *>(at)[i] = p[i];
    }
    // the piece to shared memory, asynchronously
    static __device__ __forceinline__ void copy(unsigned char *dst, const T *at) {
        constexpr int kBytes = kPer * sizeof(T);
#pragma unroll
        for (int i = 0; i < kN; ++i)
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                             (uint32_t)__cvta_generic_to_shared(dst + i * kBytes)),
                         "l"(at + i * kPer), "n"(kBytes < 4 ? 4 : kBytes)
                         : "memory");
    }
    __device__ __forceinline__ float get(int i) const { return to_f<T>(p[i / kPer].v[i % kPer]); }
    __device__ __forceinline__ void set(int i, float v) { p[i / kPer].v[i % kPer] = from_f<T>(v); }
};

// Sum over the block, the same in every thread.  Two buffers in turn: a
// thread that is already at the next sum does not overwrite this one.
__device__ __forceinline__ float block_sum(float v, float *buf) {
    v = warp_sum(v);
    const int warps = (blockDim.x + 31) >> 5;
    if (warps == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < warps; ++w) s += buf[w];
    return s;
}

constexpr int kRowsAhead = 2;  // 1 where the memory of two rows is more than an SM has

template <typename T, typename R, typename W, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS) block_norm_kernel(const NormArgs a) {
    constexpr bool kAsync = VEC * sizeof(T) >= 4;
    constexpr int kPieceT = VEC * sizeof(T), kPieceR = VEC * sizeof(R);
    extern __shared__ __align__(16) unsigned char rows[];  // [ahead][y, residual][NV][threads]
    __shared__ float sums[2][32];
    const int units = a.cols / VEC;
    const T *y = reinterpret_cast<const T *>(a.y);
    const R *res = reinterpret_cast<const R *>(a.residual);
    const W *pre = reinterpret_cast<const W *>(a.pre), *post = reinterpret_cast<const W *>(a.post);
    const T *gate = reinterpret_cast<const T *>(a.gate);
    T *normed = reinterpret_cast<T *>(a.normed);
    R *res_out = reinterpret_cast<R *>(a.residual_out);
    const float inv_cols = 1.f / (float)a.cols;
    const int slot_bytes = NV * blockDim.x * (kPieceT + kPieceR);
    unsigned char *my_y = rows + threadIdx.x * kPieceT, *my_r = rows + NV * blockDim.x * kPieceT + threadIdx.x * kPieceR;
    auto copy_row = [&](int64_t row, int slot) {
        if (row < a.rows)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = threadIdx.x + i * blockDim.x;
                if (c >= units) break;
                Piece<T, VEC>::copy(my_y + slot * slot_bytes + i * blockDim.x * kPieceT, y + row * a.y_stride + c * VEC);
                Piece<R, VEC>::copy(my_r + slot * slot_bytes + i * blockDim.x * kPieceR,
                                    res + row * a.res_stride + c * VEC);
            }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (kAsync)
        for (int i = 0; i < a.ahead; ++i) copy_row(blockIdx.x + (int64_t)i * gridDim.x, i);
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Piece<T, VEC> py[NV];
        Piece<R, VEC> pr[NV];
        if (kAsync) {
            if (a.ahead == kRowsAhead)
                asm volatile("cp.async.wait_group %0;" ::"n"(kRowsAhead - 1) : "memory");
            else
                asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= units) continue;
            if (kAsync) {
                py[i].load(reinterpret_cast<const T *>(my_y + slot * slot_bytes + i * blockDim.x * kPieceT));
                pr[i].load(reinterpret_cast<const R *>(my_r + slot * slot_bytes + i * blockDim.x * kPieceR));
            } else {
                py[i].load(y + row * a.y_stride + c * VEC);
                pr[i].load(res + row * a.res_stride + c * VEC);
            }
        }
        if (kAsync) {
            copy_row(row + (int64_t)a.ahead * gridDim.x, slot);
            slot = slot + 1 == a.ahead ? 0 : slot + 1;
        }
        const float token_gate =
            a.gate_kind == WISP_GATE_TOKEN ? a.scale * to_f<T>(gate[row * a.gate_stride]) : a.scale;
        float rms = 1.f;
        if (post) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (threadIdx.x + i * blockDim.x < units)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum += py[i].get(j) * py[i].get(j);
            rms = rsqrtf(block_sum(sum, sums[0]) * inv_cols + a.eps);
        }
        float r[NV][VEC];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= units) continue;
            float z[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[j] = py[i].get(j);
            if (post) {
                Piece<W, VEC> w;
                w.load(post + c * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[j] *= rms * w.get(j);
            }
            if (a.gate_kind >= WISP_GATE_CHANNEL) {
                Piece<T, VEC> g;
                g.load(gate + (a.gate_kind == WISP_GATE_FULL ? row * a.gate_stride : 0) + c * VEC);
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[j] *= g.get(j);
            }
            Piece<R, VEC> ro;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                r[i][j] = fmaf(token_gate, z[j], pr[i].get(j));
                sum += r[i][j] * r[i][j];
                ro.set(j, r[i][j]);
            }
            ro.store(res_out + row * a.cols + c * VEC);
        }
        rms = rsqrtf(block_sum(sum, sums[1]) * inv_cols + a.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = threadIdx.x + i * blockDim.x;
            if (c >= units) continue;
            Piece<W, VEC> w;
            w.load(pre + c * VEC);
            Piece<T, VEC> no;
#pragma unroll
            for (int j = 0; j < VEC; ++j) no.set(j, r[i][j] * rms * w.get(j));
            no.store(normed + row * a.cols + c * VEC);
        }
        if (!post) __syncthreads();  // sums[1] of this row is read before the next row's sum goes there
    }
    if (kAsync) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, typename R, typename W, int VEC, int NV, int THREADS>
int launch(NormArgs a, cudaStream_t stream) {
    constexpr bool kAsync = VEC * sizeof(T) >= 4;
    const int units = a.cols / VEC;
    const int threads = ((units + NV - 1) / NV + 31) / 32 * 32;
    const size_t row_bytes = (size_t)NV * threads * VEC * (sizeof(T) + sizeof(R));
    a.ahead = row_bytes * kRowsAhead <= 200 * 1024 ? kRowsAhead : 1;
    const size_t smem = kAsync ? a.ahead * row_bytes : 0;
    auto kernel = block_norm_kernel<T, R, W, VEC, NV, THREADS>;
    int dev = 0, sms = 0, per = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    if (a.rows > 148) {
        WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        if (smem > 48 * 1024)
            WISP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        WISP_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem));
        // without copies ahead, the next row starts when a CTA ends
        if (!kAsync) per *= 8;
    } else if (smem > 48 * 1024) {
        WISP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    }
    const int64_t most = (int64_t)sms * per;
    const unsigned grid = (unsigned)(a.rows <= 148 || a.rows < most ? a.rows : most);
    kernel<<<grid, threads, smem, stream>>>(a);
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}

template <typename T, typename R, typename W>
int dispatch(const NormArgs &a, cudaStream_t stream) {
    // the widest piece that every row start allows
    const auto fits = [&](int vec) {
        const auto ok = [&](const void *p, int64_t stride, size_t size) {
            const size_t w = vec * size > 16 ? 16 : vec * size;
            return reinterpret_cast<uintptr_t>(p) % w == 0 && (stride * (int64_t)size) % (int64_t)w == 0;
        };
        return a.cols % vec == 0 && ok(a.y, a.y_stride, sizeof(T)) && ok(a.residual, a.res_stride, sizeof(R)) &&
               ok(a.pre, 0, sizeof(W)) && (!a.post || ok(a.post, 0, sizeof(W))) &&
               (a.gate_kind < WISP_GATE_CHANNEL ||
                ok(a.gate, a.gate_kind == WISP_GATE_FULL ? a.gate_stride : 0, sizeof(T))) &&
               ok(a.normed, a.cols, sizeof(T)) && ok(a.residual_out, a.cols, sizeof(R));
    };
    if (fits(8)) {
        if (a.cols <= 8 * 256) return launch<T, R, W, 8, 1, 256>(a, stream);
        if (a.cols <= 8 * 512) return launch<T, R, W, 8, 2, 256>(a, stream);
        return launch<T, R, W, 8, 2, 1024>(a, stream);
    }
    if (fits(2)) {
        if (a.cols <= 2 * 512) return launch<T, R, W, 2, 2, 256>(a, stream);
        if (a.cols <= 2 * 2048) return launch<T, R, W, 2, 8, 256>(a, stream);
        return launch<T, R, W, 2, 8, 1024>(a, stream);
    }
    if (a.cols <= 1024) return launch<T, R, W, 1, 4, 256>(a, stream);
    if (a.cols <= 4096) return launch<T, R, W, 1, 16, 256>(a, stream);
    return launch<T, R, W, 1, 16, 1024>(a, stream);
}

template <typename T>
int dispatch_types(const NormArgs &a, int32_t residual_dtype, int32_t weight_dtype, cudaStream_t stream) {
    const bool rf = residual_dtype == WISP_FP32, wf = weight_dtype == WISP_FP32;
    if (std::is_same<T, float>::value) return dispatch<T, float, float>(a, stream);
    if (rf) return wf ? dispatch<T, float, float>(a, stream) : dispatch<T, float, T>(a, stream);
    return wf ? dispatch<T, T, float>(a, stream) : dispatch<T, T, T>(a, stream);
}

}  // namespace
}  // namespace wisp

using namespace wisp;

extern "C" int wisp_block_norm(const void *y, int64_t y_stride, const void *residual, int64_t residual_stride,
                               const void *pre_weight, const void *post_weight, const void *gate, int32_t gate_kind,
                               int64_t gate_stride, int32_t dtype, int32_t residual_dtype, int32_t weight_dtype,
                               int64_t rows, int32_t cols, float scale, float eps, void *normed, void *residual_out,
                               void *stream) {
    if (dtype < WISP_BF16 || dtype > WISP_FP32 || (residual_dtype != dtype && residual_dtype != WISP_FP32) ||
        (weight_dtype != dtype && weight_dtype != WISP_FP32))
        return set_error("wisp_block_norm: the residual and the weights have y's type or fp32"), WISP_ERR_INVALID;
    if (rows < 0 || rows > (int64_t(1) << 40) || cols < 1 || cols > 16384)
        return set_error("wisp_block_norm: need rows >= 0 and 1 <= columns <= 16384"), WISP_ERR_INVALID;
    if (gate_kind < WISP_GATE_NONE || gate_kind > WISP_GATE_FULL || (gate_kind != WISP_GATE_NONE) != (gate != nullptr))
        return set_error("wisp_block_norm: gate_kind and gate do not go together"), WISP_ERR_INVALID;
    if (rows == 0) return WISP_OK;
    if (!y || !residual || !pre_weight || !normed || !residual_out)
        return set_error("wisp_block_norm: NULL tensor"), WISP_ERR_INVALID;
    if (rows > 1 && (y_stride < 0 || residual_stride < 0 || gate_stride < 0))
        return set_error("wisp_block_norm: negative stride"), WISP_ERR_INVALID;
    const NormArgs a{y,    residual,        pre_weight, post_weight, gate, normed, residual_out, rows, y_stride,
                     residual_stride, gate_stride, cols,       gate_kind,   scale, eps, 0};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == WISP_BF16) return dispatch_types<__nv_bfloat16>(a, residual_dtype, weight_dtype, s);
    if (dtype == WISP_FP16) return dispatch_types<__half>(a, residual_dtype, weight_dtype, s);
    return dispatch_types<float>(a, residual_dtype, weight_dtype, s);
}
