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
// The weights, which every row shares, stay in L1.  Where the width and every
// address allow it a thread's pieces are 8 values wide, in 16-byte accesses,
// and NV of them, so that a row takes 256 threads where it can (more rows in
// flight, fewer warps in a reduction).  Threads and pieces are constants of the
// kernel, which makes every address of a row one register and a constant.
//
// Rows of any other width or alignment would go in accesses of 2 or 4 bytes,
// whose instructions set the time.  Pairs of values do for shorter rows; the
// others are copied as the 16-byte granules that hold them, shifted into place
// on the way from shared memory to registers, and the results go the same way
// back (4000 x 2803 fp16, fp32 residual, a full gate: 49 us, 114 value by
// value; 3000 x 6221 fp32: 106, 160).
//
// Measured (in a graph of calls whose inputs, in turn, exceed L2): a row of 2048
// bf16 2.2 us, a launch; 2048 x 4096 bf16 with both norms and a gate 16.7 us (67
// MB, 4.0 TB/s; 4 to 5 rows a CTA, whose first loads and last reductions nothing
// hides; on one input 16.3, with 512 threads 16.7, with 128 threads 20.9); 8191 x
// 2050 bf16 with a fp32 residual, pairs of values, 48.6 us (201 MB, 4.1 TB/s), by
// its instructions (60 % of the issue slots).
#include <algorithm>
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
                         "l"(at + i * kPer), "n"(kBytes)
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

constexpr size_t kMostShared = 226 * 1024;  // beside the sums
constexpr int kRowsAhead = 2;  // 1 where the memory of two rows is more than an SM has

template <typename T, typename R, typename W, int VEC, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS) block_norm_kernel(const NormArgs a) {
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
    for (int i = 0; i < a.ahead; ++i) copy_row(blockIdx.x + (int64_t)i * gridDim.x, i);
    float next_gate = token_gate_of(blockIdx.x);
    int slot = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        Piece<T, VEC> py[NV];
        Piece<R, VEC> pr[NV];
        if (a.ahead == kRowsAhead)
            asm volatile("cp.async.wait_group %0;" ::"n"(kRowsAhead - 1) : "memory");
        else
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        {
            const T *sy = reinterpret_cast<const T *>(my_y + slot * kSlotBytes);
            const R *sr = reinterpret_cast<const R *>(my_r + slot * kSlotBytes);
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (mine > i * kStep) {
                    py[i].load(sy + i * kStep);
                    pr[i].load(sr + i * kStep);
                }
        }
        copy_row(row + (int64_t)a.ahead * gridDim.x, slot);
        slot = slot + 1 == a.ahead ? 0 : slot + 1;
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
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---- rows of any width and alignment --------------------------------------------
// Eight values as 32-bit words.
template <typename T>
constexpr int kWords = 8 * sizeof(T) / 4;
__device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&v)[8], __nv_bfloat16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack(const uint32_t (&w)[4], float (&v)[8], __half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void unpack(const uint32_t (&w)[8], float (&v)[8], float) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
// Words of a row in shared memory from `off` (below 16) bytes behind `at` on.
// `off` is the same for a whole row: two rounds of selects and a funnel shift.
template <int N>
__device__ __forceinline__ void load_shifted(const uint4 *at, int off, uint32_t (&w)[N]) {
    uint32_t x[N + 4];
#pragma unroll
    for (int i = 0; i <= N / 4; ++i) {
        const uint4 v = at[i];
        x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < N + 2; ++i) x[i] = off & 8 ? x[i + 2] : x[i];
#pragma unroll
    for (int i = 0; i < N + 1; ++i) x[i] = off & 4 ? x[i + 1] : x[i];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(x[i], x[i + 1], (off & 3) * 8);
}
template <typename T>
__device__ __forceinline__ void store_shared(unsigned char *at, const float (&v)[8]) {
    Piece<T, 8> p;
#pragma unroll
    for (int i = 0; i < 8; ++i) p.set(i, v[i]);
    p.store(reinterpret_cast<T *>(at));
}
// Eight values of a vector that all rows share, `left` of them in it.
template <typename T>
__device__ __forceinline__ void load_shared_vector(const T *at, bool aligned, int left, float (&v)[8]) {
    if (aligned && left >= 8) {
        Piece<T, 8> p;
        p.load(at);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = p.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f<T>(at[i]) : 0.f;
    }
}
// A row's buffer in shared memory: its 16-byte granules (one more than its
// bytes fill where it is not aligned), and one that reads ahead of a shift.
__host__ __device__ constexpr size_t row_buffer(int cols, size_t size) {
    return ((size_t)(cols + 7) / 8 * 8 * size / 16 + 2) * 16;
}
// The granules that hold a row, asynchronously.  The bytes beside the row in
// its first and last granule come along and are not looked at.
template <int THREADS, typename T>
__device__ __forceinline__ void copy_granules(unsigned char *dst, const T *row, int cols, int tid) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    const int n = (int)((at & 15) + cols * sizeof(T) + 15) / 16;
    const unsigned char *src = reinterpret_cast<const unsigned char *>(at & ~(uintptr_t)15);
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(dst);
    for (int g = tid; g < n; g += THREADS)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + g * 16), "l"(src + g * 16) : "memory");
}
// A row from shared memory (it begins at `src`): whole granules of the
// destination, and value by value what it has of its first and last one.
template <int THREADS, typename T>
__device__ __forceinline__ void write_row(T *row, const unsigned char *src, int cols, int tid) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(row);
    const int off = (int)(at & 15), bytes = cols * (int)sizeof(T), end = (off + bytes) / 16;
    unsigned char *dst = reinterpret_cast<unsigned char *>(at - off);
    for (int g = (off ? 1 : 0) + tid; g < end; g += THREADS) {
        const int p = g * 16 - off;
        uint32_t w[4];
        load_shifted(reinterpret_cast<const uint4 *>(src) + p / 16, p & 15, w);
        *reinterpret_cast<uint4 *>(dst + g * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (tid < 16 / (int)sizeof(T)) {
        const int head = off ? min(16 - off, bytes) / (int)sizeof(T) : 0;
        const int tail = max(end * 16 - off, head * (int)sizeof(T)) / (int)sizeof(T) + tid;
        const T *values = reinterpret_cast<const T *>(src);
        if (tid < head) row[tid] = values[tid];
        if (tail < cols) row[tail] = values[tail];
    }
}

// THREADS threads have a row, each NV pieces of eight columns of it; a row of one
// warp shares the CTA with three others.
template <int THREADS>
constexpr int kRowsOfCta = THREADS == 32 ? 4 : 1;
template <typename T, typename R, typename W, int THREADS, int NV>
__global__ void __launch_bounds__(THREADS * kRowsOfCta<THREADS>) any_row_kernel(const NormArgs a) {
    extern __shared__ __align__(16) unsigned char memory[];  // a row's: [ahead][y, residual, gate], normed, new residual
    __shared__ float sums[2][32];
    const int tid = threadIdx.x % THREADS, cols = a.cols, chunks = (cols + 7) / 8;
    const int64_t row0 = (int64_t)blockIdx.x * kRowsOfCta<THREADS> + threadIdx.x / THREADS;
    const int64_t row_step = (int64_t)gridDim.x * kRowsOfCta<THREADS>;
    auto sync = [] {
        if (THREADS == 32)
            __syncwarp();
        else
            __syncthreads();
    };
    const bool full_gate = a.gate_kind == WISP_GATE_FULL;
    const int t_bytes = (int)row_buffer(cols, sizeof(T)), r_bytes = (int)row_buffer(cols, sizeof(R));
    const int slot_bytes = t_bytes + r_bytes + (full_gate ? t_bytes : 0);
    unsigned char *rows = memory + threadIdx.x / THREADS * (a.ahead * slot_bytes + t_bytes + r_bytes);
    unsigned char *normed_row = rows + a.ahead * slot_bytes, *res_row = normed_row + t_bytes;
    const T *y = reinterpret_cast<const T *>(a.y), *gate = reinterpret_cast<const T *>(a.gate);
    const R *res = reinterpret_cast<const R *>(a.residual);
    const W *pre = reinterpret_cast<const W *>(a.pre), *post = reinterpret_cast<const W *>(a.post);
    const auto aligned = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const bool has_post = a.post != nullptr, w_aligned = aligned(pre) && aligned(post), g_aligned = aligned(gate);
    const float inv_cols = 1.f / (float)cols;
    auto offset = [](const void *p) { return (int)(reinterpret_cast<uintptr_t>(p) & 15); };
    auto copy_row = [&](int64_t row, int slot) {
        if (row < a.rows) {
            unsigned char *at = rows + slot * slot_bytes;
            copy_granules<THREADS>(at, y + row * a.y_stride, cols, tid);
            copy_granules<THREADS>(at + t_bytes, res + row * a.res_stride, cols, tid);
            if (full_gate) copy_granules<THREADS>(at + t_bytes + r_bytes, gate + row * a.gate_stride, cols, tid);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto token_gate_of = [&](int64_t row) {
        return a.gate_kind == WISP_GATE_TOKEN && row < a.rows ? a.scale * to_f<T>(gate[row * a.gate_stride]) : a.scale;
    };
    for (int i = 0; i < a.ahead; ++i) copy_row(row0 + i * row_step, i);
    float next_gate = token_gate_of(row0);
    int slot = 0;
    for (int64_t row = row0; row < a.rows; row += row_step) {
        if (a.ahead == kRowsAhead)
            asm volatile("cp.async.wait_group %0;" ::"n"(kRowsAhead - 1) : "memory");
        else
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        sync();  // every thread's copies of this row; and the last row has left the output buffers
        const unsigned char *sy = rows + slot * slot_bytes, *sr = sy + t_bytes, *sg = sr + r_bytes;
        const int y_off = offset(y + row * a.y_stride), r_off = offset(res + row * a.res_stride);
        const int g_off = full_gate ? offset(gate + row * a.gate_stride) : 0;
        const float token_gate = next_gate;
        next_gate = token_gate_of(row + row_step);
        uint32_t yw[NV][kWords<T>];
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (const int c = tid + i * THREADS; c < chunks)
                load_shifted(reinterpret_cast<const uint4 *>(sy) + c * (kWords<T> / 4), y_off, yw[i]);
        float rms = 1.f;
        if (has_post) {
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = tid + i * THREADS;
                if (c >= chunks) continue;
                float v[8];
                unpack(yw[i], v, T());
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += c * 8 + j < cols ? v[j] * v[j] : 0.f;
            }
            rms = rsqrtf(block_sum<THREADS / 32>(sum, sums[0]) * inv_cols + a.eps);
        }
        float r[NV][8];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = tid + i * THREADS, left = cols - c * 8;
            if (c >= chunks) continue;
            float z[8], v[8];
            unpack(yw[i], z, T());
            if (has_post) {
                load_shared_vector(post + c * 8, w_aligned, left, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] *= rms * v[j];
            }
            if (a.gate_kind >= WISP_GATE_CHANNEL) {
                if (full_gate) {
                    uint32_t w[kWords<T>];
                    load_shifted(reinterpret_cast<const uint4 *>(sg) + c * (kWords<T> / 4), g_off, w);
                    unpack(w, v, T());
                } else {
                    load_shared_vector(gate + c * 8, g_aligned, left, v);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) z[j] *= v[j];
            }
            uint32_t w[kWords<R>];
            load_shifted(reinterpret_cast<const uint4 *>(sr) + c * (kWords<R> / 4), r_off, w);
            unpack(w, v, R());
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                r[i][j] = fmaf(token_gate, z[j], v[j]);
                sum += j < left ? r[i][j] * r[i][j] : 0.f;
            }
            store_shared<R>(res_row + c * 8 * sizeof(R), r[i]);
        }
        rms = rsqrtf(block_sum<THREADS / 32>(sum, sums[1]) * inv_cols + a.eps);
        copy_row(row + a.ahead * row_step, slot);  // every thread has read the slot
        slot = slot + 1 == a.ahead ? 0 : slot + 1;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = tid + i * THREADS;
            if (c >= chunks) continue;
            float v[8];
            load_shared_vector(pre + c * 8, w_aligned, cols - c * 8, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= r[i][j] * rms;
            store_shared<T>(normed_row + c * 8 * sizeof(T), v);
        }
        sync();
        write_row<THREADS>(reinterpret_cast<R *>(a.residual_out) + row * cols, res_row, cols, tid);
        write_row<THREADS>(reinterpret_cast<T *>(a.normed) + row * cols, normed_row, cols, tid);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename K>
int launch_rows(K kernel, int threads, int rows_of_cta, size_t smem, const NormArgs &a, cudaStream_t stream) {
    int dev = 0, sms = 0, per = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    // the limit is the same in every call: another thread's launch of this kernel may come between it and this one
    if (smem > 47 * 1024)
        WISP_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared));
    int64_t grid = (a.rows + rows_of_cta - 1) / rows_of_cta;
    if (grid > 148) {  // fewer than SMs need no count of what runs together
        WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
        WISP_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem));
        grid = std::min<int64_t>(grid, (int64_t)sms * per);
    }
    kernel<<<(unsigned)grid, threads, smem, stream>>>(a);
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}

template <typename T, typename R, typename W, int VEC, int THREADS, int NV>
int launch(NormArgs a, cudaStream_t stream) {
    const size_t row_bytes = (size_t)NV * THREADS * VEC * (sizeof(T) + sizeof(R));
    a.ahead = row_bytes * kRowsAhead <= 200 * 1024 ? kRowsAhead : 1;
    return launch_rows(block_norm_kernel<T, R, W, VEC, THREADS, NV>, THREADS, 1, a.ahead * row_bytes, a, stream);
}

template <typename T, typename R, typename W, int THREADS, int NV>
int launch_any(NormArgs a, cudaStream_t stream) {
    const size_t t = row_buffer(a.cols, sizeof(T)), r = row_buffer(a.cols, sizeof(R));
    const size_t in = t + r + (a.gate_kind == WISP_GATE_FULL ? t : 0);
    a.ahead = in * kRowsAhead + t + r <= kMostShared ? kRowsAhead : 1;
    constexpr int kRows = kRowsOfCta<THREADS>;
    return launch_rows(any_row_kernel<T, R, W, THREADS, NV>, THREADS * kRows, kRows, (a.ahead * in + t + r) * kRows, a,
                       stream);
}

template <typename T, typename R, typename W>
int dispatch(const NormArgs &a, cudaStream_t stream) {
    // whether every row start allows pieces of `vec` values, in accesses of at most 16 bytes
    const int cols = a.cols;
    const auto fits = [&](int vec) {
        const auto ok = [&](const void *p, int64_t stride, size_t size) {
            const size_t w = std::min<size_t>(vec * size, 16);
            return reinterpret_cast<uintptr_t>(p) % w == 0 && stride * (int64_t)size % (int64_t)w == 0;
        };
        return cols % vec == 0 && ok(a.y, a.y_stride, sizeof(T)) && ok(a.residual, a.res_stride, sizeof(R)) &&
               ok(a.pre, 0, sizeof(W)) && ok(a.post, 0, sizeof(W)) &&
               (a.gate_kind < WISP_GATE_CHANNEL ||
                ok(a.gate, a.gate_kind == WISP_GATE_FULL ? a.gate_stride : 0, sizeof(T))) &&
               ok(a.normed, cols, sizeof(T)) && ok(a.residual_out, cols, sizeof(R));
    };
    if (fits(8)) {
        if (cols <= 8 * 64) return launch<T, R, W, 8, 64, 1>(a, stream);
        if (cols <= 8 * 256) return launch<T, R, W, 8, 256, 1>(a, stream);
        if (cols <= 8 * 512) return launch<T, R, W, 8, 256, 2>(a, stream);
        // more threads a row cost more in the reductions, more pieces a thread registers (of fp32 first): 4000 x 7168 bf16
        // 42 us with 256 x 4, 48 with 512 x 2, 67 with 1024 x 2; 2863 x 7296 fp32 90, 78, 95; 3000 x 12288 bf16 54 with
        // 512 x 3, 75 with 1024 x 2
        if (sizeof(T) == 4) {
            if (cols <= 8 * 1024) return launch<T, R, W, 8, 512, 2>(a, stream);
        } else {
            if (cols <= 8 * 768) return launch<T, R, W, 8, 256, 3>(a, stream);
            if (cols <= 8 * 1024) return launch<T, R, W, 8, 256, 4>(a, stream);
        }
        if (cols <= 8 * 1536) return launch<T, R, W, 8, 512, 3>(a, stream);
        return launch<T, R, W, 8, 1024, 2>(a, stream);
    }
    // Pairs of values against shifted granules (us for 100 MB, floor 15.3, both norms and a token gate; bf16 | bf16 with a
    // fp32 residual | fp32): 258 columns 40.5, 56.3 | 28.9, 42.0 | 23.2, 34.5; 514 67.0, 43.9 | 46.4, 35.2 | 36.1, 32.4;
    // 770 48.5, 39.7 | 34.7, 33.1 | 27.6, 35.2; 900 43.6, 38.0 | 31.6, 38.0 | 25.8; 1026 39.9, 41.2 | 28.9, 31.9 | 24.3, 29.6;
    // 1538 35.1, 35.8 | 25.6, 30.5 | 23.0, 29.5; 2558 28.3, 35.4 | 21.8, 30.1 | 21.8, 31.1.  So pairs, but for 16-bit rows from
    // 513 columns to 1024 (768 with a fp32 residual), which one warp has without barriers.  Longer rows would take more than
    // five pairs a thread (9000 x 3074 bf16: 68 us, 57).
    const bool one_warp = sizeof(T) == 2 && cols > 2 * 256 && cols <= (sizeof(R) == 4 ? 8 * 96 : 8 * 128);
    if (cols <= 2 * 1280 && !one_warp && fits(2)) {
        if (cols <= 2 * 256) return launch<T, R, W, 2, 64, 4>(a, stream);
        if (cols <= 2 * 768) return launch<T, R, W, 2, 256, 3>(a, stream);
        return launch<T, R, W, 2, 256, 5>(a, stream);
    }
    if constexpr (std::is_same<T, float>::value)  // the longest rows in fp32 leave no room for the output buffers
        if (row_buffer(cols, 4) * (a.gate_kind == WISP_GATE_FULL ? 5 : 4) > kMostShared)
            return launch<T, R, W, 1, 1024, 16>(a, stream);
    // A row of one warp needs no barriers; above, as few warps as hold the row in two pieces a thread (us as above): 513
    // columns 43.7 with 32 x 4, 53.4 with 64 x 2 | 35.1, 40.2 | 32.6, 33.2 (771: 39.7, 39.5 | 33.0, 32.2 | 34.7, 30.3); 1025
    // 41.0 with 96 x 2, 41.3 with 128 x 2, 58.3 with 256 x 2 | 31.9, 32.1, 43.3 | 29.3, 30.3, 40.2; 1795 34.1 with 128 x 2, 35.4
    // with 64 x 4 | 30.2, 37.2 | 30.1, 35.3; 2051 40.0 with 224 x 2, 40.5 with 256 x 2, 49.2 with 320 x 2 | 33.0, 32.7, 37.3 |
    // 31.0, 32.4, 36.8; 4097 37.3 with 320 x 2, 43.1 with 416 x 2, 61.8 with 512 x 2 | 33.2, 36.3, 35.2 | 33.3, 44.3, 42.4;
    // 5121 38.7 with 416 x 2, 54.5 with 512 x 2 | 35.0, 34.5 | 43.4, 40.8; 6657 46.1 with 512 x 2, 52.0 with 1024 x 1 | 38.9,
    // 42.9 | 38.1, 38.9.
    if (cols <= 8 * 32) return launch_any<T, R, W, 32, 1>(a, stream);
    if (cols <= 8 * 64) return launch_any<T, R, W, 32, 2>(a, stream);
    if (cols <= 8 * 128) return launch_any<T, R, W, 32, 4>(a, stream);
    if (cols <= 8 * 192) return launch_any<T, R, W, 96, 2>(a, stream);
    if (cols <= 8 * 256) return launch_any<T, R, W, 128, 2>(a, stream);
    if (cols <= 8 * 448) return launch_any<T, R, W, 224, 2>(a, stream);
    if (cols <= 8 * 512) return launch_any<T, R, W, 256, 2>(a, stream);
    if (cols <= 8 * 640) return launch_any<T, R, W, 320, 2>(a, stream);
    if (cols <= 8 * 832) return launch_any<T, R, W, 416, 2>(a, stream);
    if (cols <= 8 * 1024) return launch_any<T, R, W, 512, 2>(a, stream);
    return launch_any<T, R, W, 1024, 2>(a, stream);
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
    const size_t size = dtype == WISP_FP32 ? 4 : 2, res_size = residual_dtype == WISP_FP32 ? 4 : 2,
                 w_size = weight_dtype == WISP_FP32 ? 4 : 2;
    const auto off = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; };
    if (off(y, size) || off(normed, size) || off(gate, size) || off(residual, res_size) || off(residual_out, res_size) ||
        off(pre_weight, w_size) || off(post_weight, w_size))
        return set_error("wisp_block_norm: a tensor is not aligned to its values"), WISP_ERR_INVALID;
    if (rows > 1 && (y_stride < 0 || residual_stride < 0 || gate_stride < 0))
        return set_error("wisp_block_norm: negative stride"), WISP_ERR_INVALID;
    // A row's outputs are written while other rows are still to be read.  In place is fine: a CTA reads a row before it
    // writes it, each thread its own columns.
    const auto span = [&](const void *p, int64_t stride, int64_t n, size_t of) {
        return ByteRows{reinterpret_cast<uintptr_t>(p), rows, stride * (int64_t)of, n * (int64_t)of};
    };
    const bool full = gate_kind == WISP_GATE_FULL || (gate_kind == WISP_GATE_TOKEN && cols == 1);
    const ByteRows row_inputs[] = {span(y, y_stride, cols, size), span(residual, residual_stride, cols, res_size),
                               full ? span(gate, gate_stride, cols, size) : ByteRows{0, 1, 0, 0}};
    const ByteRows others[] = {span(pre_weight, 0, cols, w_size), post_weight ? span(post_weight, 0, cols, w_size) : ByteRows{0, 1, 0, 0},
                           gate && !full ? span(gate, gate_stride, gate_kind == WISP_GATE_CHANNEL ? cols : 1, size)
                                         : ByteRows{0, 1, 0, 0}};
    const ByteRows outputs[] = {span(normed, cols, cols, size), span(residual_out, cols, cols, res_size)};
    bool clash = outputs[0].meets(outputs[1].at, rows * outputs[1].bytes);
    for (const ByteRows &o : outputs) {
        for (const ByteRows &in : row_inputs) {
            const bool in_place = in.at == o.at && in.bytes == o.bytes && (in.stride == o.stride || rows == 1);
            clash |= !in_place && in.meets(o.at, rows * o.bytes);
        }
        for (const ByteRows &in : others) clash |= in.meets(o.at, rows * o.bytes);
    }
    if (clash)
        return set_error("wisp_block_norm: an output overlaps an input (other than row by row in its place) or the other "
                         "output"),
               WISP_ERR_INVALID;
    const NormArgs a{y,    residual,        pre_weight, post_weight, gate, normed, residual_out, rows, y_stride,
                     residual_stride, gate_stride, cols,       gate_kind,   scale, eps, 0};
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == WISP_BF16) return dispatch_types<__nv_bfloat16>(a, residual_dtype, weight_dtype, s);
    if (dtype == WISP_FP16) return dispatch_types<__half>(a, residual_dtype, weight_dtype, s);
    return dispatch_types<float>(a, residual_dtype, weight_dtype, s);
}
