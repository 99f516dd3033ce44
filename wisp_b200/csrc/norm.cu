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
// loaded where they are used); NV of them, so that a row takes 256 threads
// where it can (more rows in flight, fewer warps in a reduction).  Threads and
// pieces are constants of the kernel, which makes every address of a row one
// register and a constant: with 2-value pieces the instructions, not the
// memory, set the time (8191 rows of 2050: 80 us with the number of threads a
// variable, 935 instructions a warp and row).
//
// Measured: a row of 2048 bf16 2.0 us, a launch; 2048 x 4096 bf16 with both
// norms and a gate 16.3 us (67 MB, 4.1 TB/s; 4 to 5 rows a CTA, whose first
// loads and last reductions nothing hides); 8191 x 2050 bf16 with a fp32
// residual, 2-value pieces, 48 us (201 MB, 4.2 TB/s), by its instructions (60 %
// of the issue slots).  An odd width goes value by value with twice those
// instructions, at four to five times what its bytes take.
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
template <int WARPS>
__device__ __forceinline__ float block_sum(float v, float *buf) {
    v = warp_sum(v);
    if (WARPS == 1) return v;
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) s += buf[w];
    return s;
}

constexpr int kRowsAhead = 2;  // 1 where the memory of two rows is more than an SM has

template <typename T, typename R, typename W, int VEC, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS) block_norm_kernel(const NormArgs a) {
    constexpr bool kAsync = VEC * sizeof(T) >= 4;
    constexpr int kPieceT = VEC * sizeof(T), kPieceR = VEC * sizeof(R);
    extern __shared__ __align__(16) unsigned char rows[];  // [ahead][y, residual][NV][threads]
    __shared__ float sums[2][32];
    constexpr int kStep = THREADS * VEC;  // values between a thread's pieces
    constexpr int kSlotBytes = NV * THREADS * (kPieceT + kPieceR);
    const int col = threadIdx.x * VEC, mine = a.cols - col;  // piece i is in the row where mine > i * kStep
    const T *y = reinterpret_cast<const T *>(a.y) + col;
    const R *res = reinterpret_cast<const R *>(a.residual) + col;
    const W *pre = reinterpret_cast<const W *>(a.pre) + col, *post = reinterpret_cast<const W *>(a.post) + col;
    const T *gate = reinterpret_cast<const T *>(a.gate) + (a.gate_kind >= WISP_GATE_CHANNEL ? col : 0);
    T *normed = reinterpret_cast<T *>(a.normed) + col;
    R *res_out = reinterpret_cast<R *>(a.residual_out) + col;
    const bool has_post = a.post != nullptr;
    const float inv_cols = 1.f / (float)a.cols;
    unsigned char *my_y = rows + threadIdx.x * kPieceT, *my_r = rows + NV * THREADS * kPieceT + threadIdx.x * kPieceR;
    auto copy_row = [&](int64_t row, int slot) {
        if (row < a.rows) {
            const T *py = y + row * a.y_stride;
            const R *pr = res + row * a.res_stride;
            unsigned char *sy = my_y + slot * kSlotBytes, *sr = my_r + slot * kSlotBytes;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (mine > i * kStep) {
                    Piece<T, VEC>::copy(sy + i * THREADS * kPieceT, py + i * kStep);
                    Piece<R, VEC>::copy(sr + i * THREADS * kPieceR, pr + i * kStep);
                }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto token_gate_of = [&](int64_t row) {
        return a.gate_kind == WISP_GATE_TOKEN && row < a.rows ? a.scale * to_f<T>(gate[row * a.gate_stride]) : a.scale;
    };
    if (kAsync)
        for (int i = 0; i < a.ahead; ++i) copy_row(blockIdx.x + (int64_t)i * gridDim.x, i);
    float next_gate = token_gate_of(blockIdx.x);
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
        {
            const T *sy = kAsync ? reinterpret_cast<const T *>(my_y + slot * kSlotBytes) : y + row * a.y_stride;
            const R *sr = kAsync ? reinterpret_cast<const R *>(my_r + slot * kSlotBytes) : res + row * a.res_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (mine > i * kStep) {
                    py[i].load(sy + i * kStep);
                    pr[i].load(sr + i * kStep);
                }
        }
        if (kAsync) {
            copy_row(row + (int64_t)a.ahead * gridDim.x, slot);
            slot = slot + 1 == a.ahead ? 0 : slot + 1;
        }
        const float token_gate = next_gate;
        next_gate = token_gate_of(row + gridDim.x);
        float rms = 1.f;
        if (has_post) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (mine > i * kStep)
#pragma unroll
                    for (int j = 0; j < VEC; ++j) sum += py[i].get(j) * py[i].get(j);
            rms = rsqrtf(block_sum<THREADS / 32>(sum, sums[0]) * inv_cols + a.eps);
        }
        float r[NV][VEC];
        float sum = 0.f;
        R *ro_row = res_out + row * a.cols;
        const T *gate_row = gate + (a.gate_kind == WISP_GATE_FULL ? row * a.gate_stride : 0);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (mine <= i * kStep) continue;
            float z[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) z[j] = py[i].get(j);
            if (has_post) {
                Piece<W, VEC> w;
                w.load(post + i * kStep);
#pragma unroll
                for (int j = 0; j < VEC; ++j) z[j] *= rms * w.get(j);
            }
            if (a.gate_kind >= WISP_GATE_CHANNEL) {
                Piece<T, VEC> g;
                g.load(gate_row + i * kStep);
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
            ro.store(ro_row + i * kStep);
        }
        rms = rsqrtf(block_sum<THREADS / 32>(sum, sums[1]) * inv_cols + a.eps);
        T *no_row = normed + row * a.cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (mine <= i * kStep) continue;
            Piece<W, VEC> w;
            w.load(pre + i * kStep);
            Piece<T, VEC> no;
#pragma unroll
            for (int j = 0; j < VEC; ++j) no.set(j, r[i][j] * rms * w.get(j));
            no.store(no_row + i * kStep);
        }
        if (!has_post) __syncthreads();  // sums[1] of this row is read before the next row's sum goes there
    }
    if (kAsync) asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, typename R, typename W, int VEC, int THREADS, int NV>
int launch(NormArgs a, cudaStream_t stream) {
    constexpr bool kAsync = VEC * sizeof(T) >= 4;
    const size_t row_bytes = (size_t)NV * THREADS * VEC * (sizeof(T) + sizeof(R));
    a.ahead = row_bytes * kRowsAhead <= 200 * 1024 ? kRowsAhead : 1;
    const size_t smem = kAsync ? a.ahead * row_bytes : 0;
    auto kernel = block_norm_kernel<T, R, W, VEC, THREADS, NV>;
    int dev = 0, sms = 0, per = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    if (a.rows > 148) {
        WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        if (smem > 47 * 1024)
            WISP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        WISP_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, THREADS, smem));
        // without copies ahead, the next row starts when a CTA ends
        if (!kAsync) per *= 8;
    } else if (smem > 47 * 1024) {
        WISP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    }
    const int64_t most = (int64_t)sms * per;
    const unsigned grid = (unsigned)(a.rows <= 148 || a.rows < most ? a.rows : most);
    kernel<<<grid, THREADS, smem, stream>>>(a);
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
    const int cols = a.cols;
    if (fits(8)) {
        if (cols <= 8 * 64) return launch<T, R, W, 8, 64, 1>(a, stream);
        if (cols <= 8 * 256) return launch<T, R, W, 8, 256, 1>(a, stream);
        if (cols <= 8 * 512) return launch<T, R, W, 8, 256, 2>(a, stream);
        return launch<T, R, W, 8, 1024, 2>(a, stream);
    }
    if (fits(2)) {
        if (cols <= 2 * 256) return launch<T, R, W, 2, 64, 4>(a, stream);
        if (cols <= 2 * 768) return launch<T, R, W, 2, 256, 3>(a, stream);
        if (cols <= 2 * 1280) return launch<T, R, W, 2, 256, 5>(a, stream);
        if (cols <= 2 * 2048) return launch<T, R, W, 2, 256, 8>(a, stream);
        return launch<T, R, W, 2, 1024, 8>(a, stream);
    }
    if (cols <= 512) return launch<T, R, W, 1, 64, 8>(a, stream);
    if (cols <= 2048) return launch<T, R, W, 1, 256, 8>(a, stream);
    if (cols <= 4096) return launch<T, R, W, 1, 256, 16>(a, stream);
    return launch<T, R, W, 1, 1024, 16>(a, stream);
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
