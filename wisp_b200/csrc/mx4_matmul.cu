// Products of MXFP4 matrices, grouped: out[r] = A[r] W[g]^T for the rows r of
// group g (offsets[g] <= r < offsets[g + 1]), on the block-scaled tensor cores
// (tcgen05.mma kind::mxf4: exact products of E2M1 values and their scales,
// fp32 accumulation in tensor memory, one rounding to bf16).
//
// A group is an expert and its rows the tokens routed to it, so the sizes are
// ragged and known to the device only: every CTA scans the offsets itself and
// walks the tiles (128 rows x 192 columns) of all groups with a fixed stride,
// row tiles fastest, so that the CTAs that run at the same time share the
// columns' weights in L2.  192 columns, because two accumulators (the epilogue
// of a tile runs while the next one accumulates) and the scales of every ring
// stage have to fit 512 columns of tensor memory; of the widths that do, a
// wider tile reads A less often.
//
// Ten warps: TMA producer (5 stages of 256 values of K: 16 KB of A, 24 KB of
// W), MMA issuer, 4 epilogue warps, 4 warps that bring the scale bytes.  These
// lie row by row in memory (the layout of the checkpoint, which paging copies
// as it is), 8 bytes of a row a stage, and go to the scale atoms of shared
// memory through registers, four stages ahead of their use; no TMA box can
// make that arrangement.
//
// Bound by HBM for few rows a group (the weights are read once), for many by
// L2: a stage brings 40 KB for 4 instructions of 96 cycles each.
#include "mx4_mma.cuh"

namespace wisp {
namespace mx4 {

namespace {

__device__ int g_status = 0;

constexpr int kTileM = 128, kTileN = 192;
constexpr int kStages = 5;
constexpr int kABytes = kTileM * 128, kBBytes = kTileN * 128;
constexpr int kSfABytes = 2 * kAtomBytes, kSfBBytes = 4 * kAtomBytes;  // [two halves of K][row atoms]
constexpr int kStageBytes = kABytes + kBBytes + kSfABytes + kSfBBytes;
constexpr int kSfCols = 24;                    // of a stage: two halves of 4 (A) + 8 (W) columns
constexpr int kSfCol0 = 2 * kTileN;            // behind the two accumulators
static_assert(kSfCol0 + kStages * kSfCols <= 512, "tensor memory");
constexpr int kTmemCols = 512;
constexpr int kThreads = 320;
constexpr int kEpiWarp = 2, kSfWarp = 6;
constexpr int kSfThreads = 128;
constexpr int kMaxGroups = 1024;

struct MatmulArgs {
    const int32_t *offsets;  // [groups + 1], or nullptr: one group of all rows
    const uint8_t *a_scales, *w_scales;
    __nv_bfloat16 *out;
    int64_t rows;
    int *status;
    int groups, N, blocks, a_align, w_align, vec_out;
};

struct Control {
    uint64_t full[kStages], sf_full[kStages], empty[kStages];
    uint64_t acc_full[2], acc_empty[2], mma_done;
    uint32_t tmem_base;
    int abort, issued, consumed;
    int scan[kThreads / 32];
    int first[kMaxGroups + 1];  // first row tile of each group
};

struct Tile {
    int row0, rows, n0, wrow0;  // first row, rows of the group from there on, first column, its row of W
};

// Rows [begin, end) of group g; offsets that are not in order, or outside the
// matrix, make an empty or a shorter group.
__device__ __forceinline__ void group_rows(const MatmulArgs &a, int g, int &begin, int &end) {
    const int rows = (int)a.rows;
    begin = a.offsets ? min(max(__ldg(a.offsets + g), 0), rows) : 0;
    end = a.offsets ? min(max(__ldg(a.offsets + g + 1), begin), rows) : rows;
}

__device__ __forceinline__ Tile tile_of(const Control &C, const MatmulArgs &a, int t, int ntiles_n) {
    // the last group whose first tile is not behind this one
    const int mt = t / ntiles_n;  // tiles of a group are consecutive: groups * column tiles keep the order
    int lo = 0, hi = a.groups - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (C.first[mid] <= mt)
            lo = mid;
        else
            hi = mid - 1;
    }
    const int mtiles = C.first[lo + 1] - C.first[lo];
    const int in = t - C.first[lo] * ntiles_n;
    const int n = in / mtiles, m = in - n * mtiles;
    Tile r;
    int begin, end;
    group_rows(a, lo, begin, end);
    r.row0 = begin + m * kTileM;
    r.rows = end - r.row0;
    r.n0 = n * kTileN;
    r.wrow0 = lo * a.N + r.n0;
    return r;
}

// Row tiles of every group.
__device__ void scan_groups(Control &C, const MatmulArgs &a) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kPer = (kMaxGroups + kThreads - 1) / kThreads;
    int count[kPer], own = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int g = tid * kPer + i;
        count[i] = 0;
        if (g < a.groups) {
            int begin, end;
            group_rows(a, g, begin, end);
            count[i] = (end - begin + kTileM - 1) / kTileM;
        }
        own += count[i];
    }
    int run = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += v;
    }
    if (lane == 31) C.scan[warp] = run;
    __syncthreads();
    int at = run - own;
    for (int w = 0; w < warp; ++w) at += C.scan[w];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int g = tid * kPer + i;
        if (g <= a.groups) C.first[g] = at;
        at += count[i];
    }
    __syncthreads();
}

__device__ void load_operands(Control &C, unsigned char *stages, const CUtensorMap *map_a, const CUtensorMap *map_w,
                              const MatmulArgs &a, int tiles, int ntiles_n, int steps) {
    volatile int *abort = &C.abort;
    int k = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
        const Tile tile = tile_of(C, a, t, ntiles_n);
        for (int kb = 0; kb < steps; ++kb, ++k) {
            const int s = k % kStages;
            if (k >= kStages && !wait_or_abort(&C.empty[s], ((k / kStages) - 1) & 1, abort, a.status)) return;
            unsigned char *st = stages + s * kStageBytes;
            mbar_expect_tx(&C.full[s], kABytes + kBBytes);
            tma_load_2d(st, map_a, kb * 128, tile.row0, &C.full[s]);
            tma_load_2d(st + kABytes, map_w, kb * 128, tile.wrow0, &C.full[s]);
            C.issued = k + 1;
        }
    }
}

__device__ void load_all_scales(Control &C, unsigned char *stages, const MatmulArgs &a, int tiles, int ntiles_n,
                                int steps) {
    constexpr int kDeep = 4;  // stages whose scale bytes are in registers
    const int tid = threadIdx.x - kSfWarp * 32;
    volatile int *abort = &C.abort;
    const int64_t wrows = (int64_t)a.groups * a.N;
    // the load side runs kDeep steps ahead
    int lt = blockIdx.x, lkb = 0;
    const uint8_t *pa = nullptr, *pw[2] = {};
    auto point = [&] {
        if (lt >= tiles) return;
        const Tile tile = tile_of(C, a, lt, ntiles_n);
        const int64_t ra = tile.row0 + tid;
        pa = ra < a.rows ? a.a_scales + ra * a.blocks : nullptr;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t rw = (int64_t)tile.wrow0 + tid + i * 128;
            pw[i] = tid + i * 128 < kTileN && rw < wrows ? a.w_scales + rw * a.blocks : nullptr;
        }
    };
    const uint2 none = make_uint2(0, 0);
    uint2 va[kDeep], vw[kDeep][2];
    auto load = [&](uint2 &x, uint2 (&y)[2]) {
        if (lt >= tiles) return;
        x = pa ? load_scales(pa, lkb, a.blocks, a.a_align) : none;
#pragma unroll
        for (int i = 0; i < 2; ++i) y[i] = pw[i] ? load_scales(pw[i], lkb, a.blocks, a.w_align) : none;
        if (++lkb == steps) {
            lkb = 0;
            lt += gridDim.x;
            point();
        }
    };
    point();
#pragma unroll
    for (int i = 0; i < kDeep; ++i) load(va[i], vw[i]);
    const int mine = blockIdx.x < tiles ? (tiles - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
    const int total = mine * steps;
    for (int k0 = 0; k0 < total; k0 += kDeep) {
#pragma unroll
        for (int i = 0; i < kDeep; ++i) {
            const int k = k0 + i;
            if (k >= total) break;
            const int s = k % kStages;
            if (k >= kStages && !wait_or_abort(&C.empty[s], ((k / kStages) - 1) & 1, abort, a.status)) return;
            unsigned char *sfa = stages + s * kStageBytes + kABytes + kBBytes, *sfw = sfa + kSfABytes;
            *reinterpret_cast<uint32_t *>(sfa + atom_at(tid)) = va[i].x;
            *reinterpret_cast<uint32_t *>(sfa + kAtomBytes + atom_at(tid)) = va[i].y;
            *reinterpret_cast<uint32_t *>(sfw + atom_at(tid)) = vw[i][0].x;
            *reinterpret_cast<uint32_t *>(sfw + 2 * kAtomBytes + atom_at(tid)) = vw[i][0].y;
            if (tid < kTileN - 128) {
                *reinterpret_cast<uint32_t *>(sfw + kAtomBytes + atom_at(tid)) = vw[i][1].x;
                *reinterpret_cast<uint32_t *>(sfw + 3 * kAtomBytes + atom_at(tid)) = vw[i][1].y;
            }
            fence_async_shared();
            __syncwarp();
            if ((tid & 31) == 0) mbar_arrive(&C.sf_full[s]);
            load(va[i], vw[i]);
        }
    }
}

__device__ void issue_products(Control &C, unsigned char *stages, const MatmulArgs &a, int tiles, int steps) {
    volatile int *abort = &C.abort;
    int k = 0, i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
        const int b = i & 1;
        if (i >= 2 && !wait_or_abort(&C.acc_empty[b], ((i / 2) - 1) & 1, abort, a.status)) break;
        tc_fence_after();
        const uint32_t acc = C.tmem_base + b * kTileN;
        bool ok = true;
        for (int kb = 0; kb < steps && ok; ++kb, ++k) {
            const int s = k % kStages;
            ok = wait_or_abort(&C.full[s], (k / kStages) & 1, abort, a.status) &&
                 wait_or_abort(&C.sf_full[s], (k / kStages) & 1, abort, a.status);
            if (!ok) break;
            tc_fence_after();
            const uint32_t a0 = s_addr(stages + s * kStageBytes), b0 = a0 + kABytes, sfa = b0 + kBBytes,
                           sfw = sfa + kSfABytes;
            const uint32_t cols = C.tmem_base + kSfCol0 + s * kSfCols;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                copy_atom(cols + h * 12, sfa + h * kAtomBytes);
                copy_atom(cols + h * 12 + 4, sfw + h * 2 * kAtomBytes);
                copy_atom(cols + h * 12 + 8, sfw + h * 2 * kAtomBytes + kAtomBytes);
            }
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 64 values = 32 bytes further along K
                umma_mxf4(acc, smem_desc_k_sw128(a0 + kk * 32), smem_desc_k_sw128(b0 + kk * 32),
                          idesc_mxf4(kTileM, kTileN, (kk & 1) * 2), cols + (kk >> 1) * 12, cols + (kk >> 1) * 12 + 4,
                          (kb | kk) != 0);
            umma_commit(&C.empty[s]);
            C.consumed = k + 1;
        }
        if (!ok) break;
        umma_commit(&C.acc_full[b]);
    }
    umma_commit(&C.mma_done);
}

__device__ void store_tiles(Control &C, const MatmulArgs &a, int tiles, int ntiles_n) {
    volatile int *abort = &C.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
    int i = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++i) {
        const Tile tile = tile_of(C, a, t, ntiles_n);
        const int b = i & 1;
        if (!wait_or_abort(&C.acc_full[b], (i / 2) & 1, abort, a.status)) return;
        tc_fence_after();
        const int r = quarter * 32 + lane;
        __nv_bfloat16 *row = a.out + ((int64_t)tile.row0 + r) * a.N + tile.n0;
        const int cols = min(kTileN, a.N - tile.n0);
#pragma unroll 1
        for (int c0 = 0; c0 < kTileN; c0 += 32) {
            uint32_t v[32];
            gemm::tmem_ld32(C.tmem_base + b * kTileN + ((uint32_t)(quarter * 32) << 16) + c0, v);
            if (r >= tile.rows || c0 >= cols) continue;
            if (a.vec_out) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (c0 + j * 8 >= cols) break;
                    float f[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(v[j * 8 + x]);
                    Vec8<__nv_bfloat16>::store(row + c0 + j * 8, f);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    if (c0 + j < cols) row[c0 + j] = __float2bfloat16_rn(__uint_as_float(v[j]));
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&C.acc_empty[b]);
    }
}

__global__ void __launch_bounds__(kThreads, 1)
    matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                  const MatmulArgs a) {
    extern __shared__ unsigned char raw[];
    unsigned char *stages = raw + ((1024u - (s_addr(raw) & 1023u)) & 1023u);
    Control &C = *reinterpret_cast<Control *>(stages + kStages * kStageBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.sf_full[s], kSfThreads / 32);
            mbar_init(&C.empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&C.acc_full[b], 1);
            mbar_init(&C.acc_empty[b], 4);
        }
        mbar_init(&C.mma_done, 1);
        C.abort = C.issued = C.consumed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) gemm::tmem_alloc(&C.tmem_base, kTmemCols);
    tc_fence_before();
    scan_groups(C, a);  // with barriers of the whole CTA
    tc_fence_after();
    const int ntiles_n = (a.N + kTileN - 1) / kTileN, tiles = C.first[a.groups] * ntiles_n;
    const int steps = (a.blocks + kStepBlocks - 1) / kStepBlocks;
    if (warp == 0) {
        if (lane == 0) load_operands(C, stages, &map_a, &map_w, a, tiles, ntiles_n, steps);
    } else if (warp == 1) {
        if (lane == 0) issue_products(C, stages, a, tiles, steps);
    } else if (warp < kSfWarp) {
        store_tiles(C, a, tiles, ntiles_n);
    } else {
        load_all_scales(C, stages, a, tiles, ntiles_n, steps);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0) {
        // after an abort: copies and products in flight end before the memory is given back
        volatile int no_abort = 0;
        for (int k = C.consumed; k < C.issued; ++k)
            gemm::mbar_wait(&C.full[k % kStages], (k / kStages) & 1, kWaitNs, &no_abort);
        gemm::mbar_wait(&C.mma_done, 0, kWaitNs, &no_abort);
    }
    __syncthreads();
    if (warp == 0) gemm::tmem_dealloc(C.tmem_base, kTmemCols);
}

int *g_words[64] = {};  // address of g_status on each device

constexpr int kSmemBytes = kStages * kStageBytes + 1024 + sizeof(Control);
static_assert(kSmemBytes <= 232448, "shared memory");

}  // namespace

int status_word(int **word) {
    int dev = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 64 && g_words[dev]) return *word = g_words[dev], WISP_OK;
    void *p = nullptr;
    WISP_CUDA_TRY(cudaGetSymbolAddress(&p, g_status));
    if (dev < 64) g_words[dev] = reinterpret_cast<int *>(p);  // the same value from every thread
    return *word = reinterpret_cast<int *>(p), WISP_OK;
}

}  // namespace mx4
}  // namespace wisp

using namespace wisp;
using namespace wisp::mx4;

extern "C" int wisp_mx4_matmul(const void *a_codes, const void *a_scales, int64_t rows, const void *w_codes,
                               const void *w_scales, int32_t groups, int32_t n, int32_t k, const int32_t *offsets,
                               void *out, void *stream) {
    if (rows < 0 || rows > (1 << 30) || groups < 1 || groups > kMaxGroups || n < 1 || n > (1 << 24) || k < kBlock ||
        k % kBlock || k > (1 << 24))
        return set_error("wisp_mx4_matmul: need 0 <= rows <= 2^30, 1 to 1024 groups, n >= 1, k a multiple of 32"),
               WISP_ERR_INVALID;
    if ((int64_t)groups * n > INT32_MAX || rows * ((n + kTileN - 1) / kTileN) > ((int64_t)1 << 36))
        return set_error("wisp_mx4_matmul: groups * n or rows * n too large"), WISP_ERR_INVALID;
    if (!offsets && groups != 1) return set_error("wisp_mx4_matmul: several groups need offsets"), WISP_ERR_INVALID;
    if (rows == 0) return WISP_OK;
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out)
        return set_error("wisp_mx4_matmul: NULL tensor"), WISP_ERR_INVALID;
    for (const void *p : {a_codes, w_codes})
        if (reinterpret_cast<uintptr_t>(p) % 16)
            return set_error("wisp_mx4_matmul: codes must be aligned to 16 bytes"), WISP_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(out) % 2) return set_error("wisp_mx4_matmul: unaligned out"), WISP_ERR_INVALID;
    CUtensorMap ma, mw;
    if (const int rc = gemm::make_byte_map(&ma, a_codes, rows, k / 2, kTileM)) return rc;
    if (const int rc = gemm::make_byte_map(&mw, w_codes, (uint64_t)groups * n, k / 2, kTileN)) return rc;
    MatmulArgs a{};
    a.offsets = offsets;
    a.a_scales = reinterpret_cast<const uint8_t *>(a_scales);
    a.w_scales = reinterpret_cast<const uint8_t *>(w_scales);
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.rows = rows, a.groups = groups, a.N = n, a.blocks = k / kBlock;
    if (const int rc = status_word(&a.status)) return rc;
    a.a_align = scale_align(a_scales, a.blocks), a.w_align = scale_align(w_scales, a.blocks);
    a.vec_out = n % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    int dev = 0, sms = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    WISP_CUDA_TRY(cudaFuncSetAttribute(matmul_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    // no more CTAs than tiles there can be (every group may end in a partial one)
    const int64_t most = (rows / kTileM + groups) * ((n + kTileN - 1) / kTileN);
    matmul_kernel<<<(unsigned)(most < sms ? most : sms), kThreads, kSmemBytes, reinterpret_cast<cudaStream_t>(stream)>>>(
        ma, mw, a);
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}

extern "C" int wisp_mx4_sync(void *stream) {
    WISP_CUDA_TRY(cudaStreamSynchronize(reinterpret_cast<cudaStream_t>(stream)));
    int status = 0;
    WISP_CUDA_TRY(cudaMemcpyFromSymbol(&status, g_status, sizeof(status)));
    if (status == WISP_OK) return WISP_OK;
    const int zero = 0;
    WISP_CUDA_TRY(cudaMemcpyToSymbol(g_status, &zero, sizeof(zero)));
    set_error("wisp_mx4: a wait inside a kernel ran out; its output is not complete");
    return status;
}
