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
// wider tile reads A less often.  Few tiles are 64 columns wide (Narrow).  The
// steps along K are the same, and so are the bits.
//
// 14 warps: TMA producer (4 stages of 256 values of K: 16 KB of A, 24 KB of
// W), MMA issuer, 4 epilogue warps, 8 warps that bring the scale bytes.  These
// lie row by row in memory (the layout of the checkpoint, which paging copies
// as it is), 8 bytes of a row a stage, and go to the scale atoms of shared
// memory through registers, ahead of their use; no TMA box can make that
// arrangement.
//
// Measured (in a graph of calls whose inputs, in turn, exceed L2): 128 experts
// x 128 rows x 1536 x 2048 (282 MB to read and write) 57 us, 4.9 TB/s, the weights
// read once (232 MB from HBM, 709 MB through L2: a ragged group has one or two
// row tiles).  8 experts x 512 rows x 28672 x 4096 (962 GFLOP) 293 us, 3.3
// PFLOP/s, 43 KB of L2 a stage and SM, 11.2 TB/s over the chip (281 on one input;
// back to back the power limit makes that up to 340).  One small product is
// latency: 16 x 4096 x 4096 takes 12.0 us (10.7 with its weights in L2), of which
// a launch and the first loads are 6.
#include <atomic>
#include <map>
#include <mutex>

#include "mx4_mma.cuh"

namespace wisp {
namespace mx4 {

namespace {

__device__ int g_status[2] = {0, WISP_MX4_DEFAULT_TRIES};  // see status_word
std::atomic<int> g_dropped{0};

constexpr int kTileM = 128;
constexpr int kEpiWarp = 2, kSfWarp = 6;
constexpr int kThreads = (kSfWarp + kScaleGroups * kScaleGroupWarps) * 32;
constexpr int kMaxGroups = 1024;
constexpr int kWindow = 2;  // stages of a window of scale bytes
constexpr int kTmemCols = 512;
constexpr int kOutBytes = 32 * 128;  // staging of an epilogue warp: 32 rows of 64 columns

// The sizes that follow from a tile's columns.
template <int N, int STAGES>
struct Shape {
    static constexpr int kTileN = N, kStages = STAGES;
    static constexpr int kABytes = kTileM * 128, kBBytes = kTileN * 128;
    static constexpr int kWAtoms = (kTileN + 127) / 128;  // row atoms of W's scales
    static constexpr int kSfABytes = 2 * kAtomBytes, kSfBBytes = 2 * kWAtoms * kAtomBytes;  // [two halves of K][row atoms]
    static constexpr int kStageBytes = kABytes + kBBytes + kSfABytes + kSfBBytes;
    static constexpr int kSfHalf = 4 + 4 * kWAtoms;  // columns of tensor memory: A's atom, W's
    static constexpr int kSfCols = 2 * kSfHalf;      // of a stage
    static constexpr int kSfCol0 = 2 * kTileN;       // behind the two accumulators
    static constexpr int kCols = 64;                 // the epilogue's piece
    static_assert(kSfCol0 + kStages * kSfCols <= kTmemCols, "tensor memory");
    static_assert(kStages > kWindow, "a parity wait has to know its phase");
    static_assert(kTileN % kCols == 0 && kTileN <= 256, "tile");
};

struct MatmulArgs {
    const int32_t *offsets;  // [groups + 1], or nullptr: one group of all rows
    const uint8_t *a_scales, *w_scales;
    __nv_bfloat16 *out;
    int64_t rows;
    int *status;
    int groups, N, blocks, align, vec_out;
    int drop;  // tests: arrivals that every stage's scale bytes wait for in vain
};

template <class S>
struct Control {
    uint64_t full[S::kStages], sf_full[S::kStages], empty[S::kStages];
    uint64_t acc_full[2], acc_empty[2], mma_done;
    uint32_t tmem_base;
    int abort, issued, consumed;
    int scan[kThreads / 32];
    int first[kMaxGroups + 1];  // first row tile of each group
};

// Rows [begin, end) of group g; offsets that are not in order, or outside the
// matrix, make an empty or a shorter group.
__device__ __forceinline__ void group_rows(const MatmulArgs &a, int g, int &begin, int &end) {
    const int rows = (int)a.rows;
    begin = a.offsets ? min(max(__ldg(a.offsets + g), 0), rows) : 0;
    end = a.offsets ? min(max(__ldg(a.offsets + g + 1), begin), rows) : rows;
}

// A CTA's walk over the tiles of all groups, gridDim.x apart; row tiles fastest
// within a group.  For a converged warp: 32 groups are looked at together.
template <class S>
struct Walk {
    int t, tiles, ntiles_n, g = 0;
    // the tile: first row, rows of the group from there on, first column, its row of W
    int row0, rows, n0, wrow0;
    __device__ __forceinline__ Walk(const Control<S> &C, const MatmulArgs &a) {
        ntiles_n = (a.N + S::kTileN - 1) / S::kTileN;
        tiles = C.first[a.groups] * ntiles_n;
        t = blockIdx.x;
    }
    // False behind the last tile.
    __device__ __forceinline__ bool at(const Control<S> &C, const MatmulArgs &a) {
        if (t >= tiles) return false;
        const int lane = threadIdx.x & 31;
        while (true) {  // groups that end before this tile
            const int i = g + 1 + lane;
            const unsigned behind = __ballot_sync(0xFFFFFFFFu, i <= a.groups && C.first[min(i, a.groups)] * ntiles_n <= t);
            g += __popc(behind);
            if (behind != 0xFFFFFFFFu) break;
        }
        const int mtiles = C.first[g + 1] - C.first[g], in = t - C.first[g] * ntiles_n;
        const int n = in / mtiles;
        int begin, end;
        group_rows(a, g, begin, end);
        row0 = begin + (in - n * mtiles) * kTileM;
        rows = end - row0;
        n0 = n * S::kTileN;
        wrow0 = g * a.N + n0;
        return true;
    }
    __device__ __forceinline__ void next() { t += gridDim.x; }
};

// Row tiles of every group.
template <class S>
__device__ void scan_groups(Control<S> &C, const MatmulArgs &a) {
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

template <class S>
__device__ void load_operands(Control<S> &C, unsigned char *stages, const CUtensorMap *map_a, const CUtensorMap *map_w,
                              const MatmulArgs &a, int steps) {
    volatile int *abort = &C.abort;
    RingPos<S::kStages> ring;
    int issued = 0;
    for (Walk<S> t(C, a); t.at(C, a); t.next())
        for (int kb = 0; kb < steps; ++kb, ring.next()) {
            if (!warp_wait(&C.empty[ring.slot], ring.turn ^ 1, abort, a.status)) return;
            if (elect_one()) {
                unsigned char *st = stages + ring.slot * S::kStageBytes;
                mbar_expect_tx(&C.full[ring.slot], S::kABytes + S::kBBytes);
                tma_load_2d(st, map_a, kb * 128, t.row0, &C.full[ring.slot]);
                tma_load_2d(st + S::kABytes, map_w, kb * 128, t.wrow0, &C.full[ring.slot]);
                C.issued = ++issued;
            }
        }
}

template <class S>
__device__ void load_all_scales(Control<S> &C, unsigned char *stages, const MatmulArgs &a, int steps) {
    const int group = (threadIdx.x >> 5) - kSfWarp >= kScaleGroupWarps;
    const int tid = threadIdx.x % (kScaleGroupWarps * 32);
    volatile int *abort = &C.abort;
    const int64_t wrows = (int64_t)a.groups * a.N;
    unsigned char *sf = stages + S::kABytes + S::kBBytes + atom_at(tid);
    RingPos<S::kStages> ring;
    // the loads run DEEP of the group's windows ahead of the stores
    Walk<S> ahead(C, a);
    bool more = ahead.at(C, a);
    int kb = 0;
    const uint8_t *pa = nullptr, *pw[2] = {};  // rows of the tile
    auto point = [&] {
        const int64_t ra = ahead.row0 + tid;
        pa = ra < a.rows ? a.a_scales + ra * a.blocks : nullptr;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int64_t rw = (int64_t)ahead.wrow0 + tid + i * 128;
            pw[i] = tid + i * 128 < S::kTileN && rw < wrows ? a.w_scales + rw * a.blocks : nullptr;
        }
    };
    auto count = [&] { return more ? min(kWindow, steps - kb) : 0; };
    // to the next window, which may be of another tile
    auto advance = [&] {
        kb += kWindow;
        if (kb < steps || !more) return false;
        kb = 0;
        ahead.next();
        more = ahead.at(C, a);
        return more;
    };
    struct Window {
        ScaleWords<kWindow> a, w[2];
        uint32_t a_shift, w_shift[2];
        int count, skip;  // stages of the window, and of the other group's window behind it
        int left;         // scale bytes of a row from here on
    } x, next;
    auto load = [&](Window &x) {
        x.count = count();
        if (!more) return;
        x.left = a.blocks - kb * kStepBlocks;
        x.a.zero(), x.w[0].zero(), x.w[1].zero();
        if (pa) x.a.load(pa + kb * kStepBlocks, x.count, x.left, a.align);
        x.a_shift = row_shift(pa);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (pw[i]) x.w[i].load(pw[i] + kb * kStepBlocks, x.count, x.left, a.align);
            x.w_shift[i] = row_shift(pw[i]);
        }
        bool moved = advance();
        x.skip = count();
        moved |= advance();
        if (moved && more) point();
    };
    if (group == 1) {
        ring.skip(count());
        advance();
    }
    if (more) point();
    x.count = x.skip = 0;
#pragma unroll 1
    while (true) {
        load(next);  // ahead of what it waits for here
#pragma unroll
        for (int j = 0; j < kWindow; ++j) {
            if (j >= x.count) break;
            if (!warp_wait(&C.empty[ring.slot], ring.turn ^ 1, abort, a.status)) return;
            unsigned char *sfa = sf + ring.slot * S::kStageBytes, *sfw = sfa + S::kSfABytes;
            uint2 v = x.a.stage(j, x.a_shift, x.left);
            *reinterpret_cast<uint32_t *>(sfa) = v.x;
            *reinterpret_cast<uint32_t *>(sfa + kAtomBytes) = v.y;
            v = x.w[0].stage(j, x.w_shift[0], x.left);
            *reinterpret_cast<uint32_t *>(sfw) = v.x;
            *reinterpret_cast<uint32_t *>(sfw + S::kWAtoms * kAtomBytes) = v.y;
            if (tid < S::kTileN - 128) {
                v = x.w[1].stage(j, x.w_shift[1], x.left);
                *reinterpret_cast<uint32_t *>(sfw + kAtomBytes) = v.x;
                *reinterpret_cast<uint32_t *>(sfw + (S::kWAtoms + 1) * kAtomBytes) = v.y;
            }
            fence_async_shared();
            __syncwarp();
            if ((tid & 31) == 0) mbar_arrive(&C.sf_full[ring.slot]);
            ring.next();
        }
        ring.skip(x.skip);
        if (!next.count) break;
        x = next;
    }
}

// The whole warp walks, one lane issues.  While the unit works off three of a
// stage's four products the warp waits for the next stage: the waits take as
// long as two products even when there is nothing to wait for.
template <class S>
__device__ void issue_products(Control<S> &C, unsigned char *stages, const MatmulArgs &a, int steps) {
    volatile int *abort = &C.abort;
    const uint32_t base = s_addr(stages), tmem = C.tmem_base;
    const uint64_t a0 = smem_desc_k_sw128(base), b0 = smem_desc_k_sw128(base + S::kABytes),
                   sf0 = smem_desc_atom(base + S::kABytes + S::kBBytes);
    RingPos<S::kStages> ring;
    RingPos<2> accs;
    int consumed = 0;
    bool ready = false;  // whether the stage at `ring` has been waited for
    auto wait_stage = [&](const RingPos<S::kStages> &at) {
        return warp_wait(&C.full[at.slot], at.turn, abort, a.status) &&
               warp_wait(&C.sf_full[at.slot], at.turn, abort, a.status);
    };
    for (Walk<S> t(C, a); t.at(C, a); t.next(), accs.next()) {
        if (!warp_wait(&C.acc_empty[accs.slot], accs.turn ^ 1, abort, a.status)) return;
        tc_fence_after();
        const uint32_t acc = tmem + accs.slot * S::kTileN;
        const bool last_tile = t.t + (int)gridDim.x >= t.tiles;
        for (int kb = 0; kb < steps; ++kb) {
            if (!ready && !wait_stage(ring)) return;
            tc_fence_after();
            const int s = ring.slot;
            // addresses are in units of 16 bytes; 64 values are 32 bytes further along K
            const uint64_t step = (uint64_t)(s * (S::kStageBytes >> 4));
            const uint64_t da = a0 + step, db = b0 + step, ds = sf0 + step;
            const uint32_t cols = tmem + S::kSfCol0 + s * S::kSfCols;
            auto product = [&](int kk) {
                umma_mxf4(acc, da + kk * 2, db + kk * 2, idesc_mxf4(kTileM, S::kTileN, (kk & 1) * 2), cols + (kk >> 1) * S::kSfHalf,
                          cols + (kk >> 1) * S::kSfHalf + 4, kb | kk);
            };
            if (elect_one()) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t to = cols + h * S::kSfHalf;
                    copy_atom(to, ds + h * (kAtomBytes >> 4));
#pragma unroll
                    for (int i = 0; i < S::kWAtoms; ++i)
                        copy_atom(to + 4 + i * 4, ds + ((S::kSfABytes + (h * S::kWAtoms + i) * kAtomBytes) >> 4));
                }
                product(0);
                product(1);
                product(2);
            }
            ring.next();
            const bool more = kb + 1 < steps || !last_tile;
            const bool ok = !more || wait_stage(ring);
            ready = more;
            if (elect_one()) {
                product(3);
                umma_commit(&C.empty[s]);
                C.consumed = ++consumed;
            }
            if (!ok) return;
        }
        if (elect_one()) umma_commit(&C.acc_full[accs.slot]);
    }
}

// Epilogue warps: 64 columns at a time through shared memory (16-byte pieces
// swizzled by the row), so that a store instruction writes 128 bytes of four
// rows and not 16 bytes of 32.
template <class S>
__device__ void store_tiles(Control<S> &C, unsigned char *staging, const MatmulArgs &a) {
    volatile int *abort = &C.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
    unsigned char *mine = staging + (warp - kEpiWarp) * kOutBytes;
    RingPos<2> accs;
    for (Walk<S> t(C, a); t.at(C, a); t.next(), accs.next()) {
        if (!warp_wait(&C.acc_full[accs.slot], accs.turn, abort, a.status)) return;
        tc_fence_after();
        const int rows = t.rows - quarter * 32, cols = min(S::kTileN, a.N - t.n0);
        __nv_bfloat16 *out = a.out + ((int64_t)t.row0 + quarter * 32) * a.N + t.n0;
        const uint32_t taddr = C.tmem_base + accs.slot * S::kTileN + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int c0 = 0; c0 < cols && rows > 0; c0 += S::kCols) {
#pragma unroll
            for (int h = 0; h < S::kCols / 32; ++h) {
                uint32_t v[32];
                gemm::tmem_ld32(taddr + c0 + h * 32, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) f[x] = __uint_as_float(v[j * 8 + x]);
                    Vec8<__nv_bfloat16>::store(
                        reinterpret_cast<__nv_bfloat16 *>(mine + lane * 128 + (((h * 4 + j) ^ (lane & 7)) << 4)), f);
                }
            }
            __syncwarp();
            const int c = c0 + (lane & 7) * 8, end = min(cols, c0 + S::kCols);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + (lane >> 3);
                const uint4 v = *reinterpret_cast<const uint4 *>(mine + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
                if (r >= rows || c >= end) continue;
                __nv_bfloat16 *at = out + (int64_t)r * a.N + c;
                if (a.vec_out) {
                    *reinterpret_cast<uint4 *>(at) = v;
                } else {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        if (c + x < end)
                            at[x] = __ushort_as_bfloat16((unsigned short)(x & 1 ? w[x / 2] >> 16 : w[x / 2]));
                }
            }
            __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&C.acc_empty[accs.slot]);
    }
}

template <class S>
__global__ void __launch_bounds__(kThreads, 1)
    matmul_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                  const MatmulArgs a) {
    extern __shared__ unsigned char raw[];
    unsigned char *stages = raw + ((1024u - (s_addr(raw) & 1023u)) & 1023u);
    unsigned char *staging = stages + S::kStages * S::kStageBytes;
    Control<S> &C = *reinterpret_cast<Control<S> *>(staging + 4 * kOutBytes);
    const int tid = threadIdx.x, warp = tid >> 5;
    if (tid == 0) {
        for (int s = 0; s < S::kStages; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.sf_full[s], kScaleGroupWarps + a.drop);
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
    const int steps = (a.blocks + kStepBlocks - 1) / kStepBlocks;
    if (warp == 0) {
        load_operands(C, stages, &map_a, &map_w, a, steps);
    } else if (warp == 1) {
        issue_products(C, stages, a, steps);
        __syncwarp();
        if (elect_one()) umma_commit(&C.mma_done);
    } else if (warp < kSfWarp) {
        store_tiles(C, staging, a);
    } else {
        load_all_scales(C, stages, a, steps);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0) {
        // after an abort: copies and products in flight end before the memory is given back
        volatile int no_abort = 0;
        for (int k = C.consumed; k < C.issued; ++k)
            wait_tries(&C.full[k % S::kStages], (k / S::kStages) & 1, &no_abort, a.status);
        wait_tries(&C.mma_done, 0, &no_abort, a.status);
    }
    __syncthreads();
    if (warp == 0) gemm::tmem_dealloc(C.tmem_base, kTmemCols);
}

int *g_words[64] = {};  // address of g_status on each device, as found

template <class S>
int launch(const CUtensorMap &ma, const void *w_codes, const MatmulArgs &a, int64_t tiles, int sms, cudaStream_t stream) {
    constexpr int kSmemBytes = S::kStages * S::kStageBytes + 4 * kOutBytes + 1024 + sizeof(Control<S>);
    static_assert(kSmemBytes <= 232448, "shared memory");
    CUtensorMap mw;
    if (const int rc = gemm::make_byte_map(&mw, w_codes, (uint64_t)a.groups * a.N, a.blocks * (kBlock / 2), S::kTileN))
        return rc;
    WISP_CUDA_TRY(cudaFuncSetAttribute(matmul_kernel<S>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    matmul_kernel<S><<<(unsigned)(tiles < sms ? tiles : sms), kThreads, kSmemBytes, stream>>>(ma, mw, a);
    WISP_CUDA_TRY(cudaGetLastError());
    return WISP_OK;
}
using Wide = Shape<192, 4>;
// Where the tiles are so few that SMs would go without: the time is then the
// latency of a tile's steps, which narrow tiles, with more stages in flight,
// shorten (us on one input, narrow against wide, 16 rows x 4096 x 4096: 11.0, 12.3; 40
// groups of 223 rows x 180 x 3200: 11.0, 12.4; 128 x 9472 x 2048: 8.8, 10.2).
// With more narrow tiles than SMs the wide ones win (512 x 4096 x 4096: 18.4,
// 13.8); 32 columns were no better anywhere (13.1 at the first size).
using Narrow = Shape<64, 7>;

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
int dropped() { return g_dropped.load(std::memory_order_relaxed); }

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
    if ((int64_t)groups * n > INT32_MAX || rows * ((n + Wide::kTileN - 1) / Wide::kTileN) > ((int64_t)1 << 36))
        return set_error("wisp_mx4_matmul: groups * n or rows * n too large"), WISP_ERR_INVALID;
    if (!offsets && groups != 1) return set_error("wisp_mx4_matmul: several groups need offsets"), WISP_ERR_INVALID;
    if (rows == 0) return WISP_OK;
    if (!a_codes || !a_scales || !w_codes || !w_scales || !out)
        return set_error("wisp_mx4_matmul: NULL tensor"), WISP_ERR_INVALID;
    for (const void *p : {a_codes, w_codes})
        if (reinterpret_cast<uintptr_t>(p) % 16)
            return set_error("wisp_mx4_matmul: codes must be aligned to 16 bytes"), WISP_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(out) % 2) return set_error("wisp_mx4_matmul: unaligned out"), WISP_ERR_INVALID;
    const int64_t wrows = (int64_t)groups * n, out_bytes = rows * n * 2;
    if (meets(a_codes, rows * (k / 2), out, out_bytes) || meets(a_scales, rows * (k / kBlock), out, out_bytes) ||
        meets(w_codes, wrows * (k / 2), out, out_bytes) || meets(w_scales, wrows * (k / kBlock), out, out_bytes) ||
        (offsets && meets(offsets, 4 * (int64_t)(groups + 1), out, out_bytes)))
        return set_error("wisp_mx4_matmul: out overlaps an input"), WISP_ERR_INVALID;
    CUtensorMap ma;
    if (const int rc = gemm::make_byte_map(&ma, a_codes, rows, k / 2, kTileM)) return rc;
    MatmulArgs a{};
    a.offsets = offsets;
    a.a_scales = reinterpret_cast<const uint8_t *>(a_scales);
    a.w_scales = reinterpret_cast<const uint8_t *>(w_scales);
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.rows = rows, a.groups = groups, a.N = n, a.blocks = k / kBlock;
    if (const int rc = status_word(&a.status)) return rc;
    a.drop = dropped() == WISP_MX4_DROP_SCALES;
    const int aa = scale_align(a_scales, a.blocks), wa = scale_align(w_scales, a.blocks);
    a.align = aa < wa ? aa : wa;
    a.vec_out = n % 8 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0;
    int dev = 0, sms = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    // no more tiles than this (every group may end in a partial one)
    const int64_t row_tiles = rows / kTileM + groups;
    auto tiles = [&](int width) { return row_tiles * ((n + width - 1) / width); };
    const auto on = reinterpret_cast<cudaStream_t>(stream);
    if (tiles(Narrow::kTileN) <= sms) return launch<Narrow>(ma, w_codes, a, tiles(Narrow::kTileN), sms, on);
    return launch<Wide>(ma, w_codes, a, tiles(Wide::kTileN), sms, on);
}

// The device's count goes up with every wait that runs out and never back, and
// each asker compares it with what it was told last, so that none takes a
// report away from another.
extern "C" int wisp_mx4_timeouts(void *stream, int64_t *count) {
    if (!count) return set_error("wisp_mx4_timeouts: NULL result"), WISP_ERR_INVALID;
    const auto s = reinterpret_cast<cudaStream_t>(stream);
    uint32_t n = 0;
    WISP_CUDA_TRY(cudaMemcpyFromSymbolAsync(&n, g_status, sizeof(n), 0, cudaMemcpyDeviceToHost, s));
    WISP_CUDA_TRY(cudaStreamSynchronize(s));
    *count = n;
    return WISP_OK;
}

extern "C" int wisp_mx4_sync(void *stream) {
    static std::mutex mu;
    static std::map<unsigned long long, int64_t> told;  // by stream id, which no later stream has
    int64_t count = 0;
    if (const int rc = wisp_mx4_timeouts(stream, &count)) return rc;
    if (count == 0) return WISP_OK;
    unsigned long long id = 0;
    WISP_CUDA_TRY(cudaStreamGetId(reinterpret_cast<cudaStream_t>(stream), &id));
    std::lock_guard<std::mutex> lock(mu);
    int64_t &last = told[id];
    if (last == count) return WISP_OK;
    last = count;
    set_error("wisp_mx4: a wait inside a kernel ran out; its output is not complete");
    return WISP_ERR_TIMEOUT;
}

extern "C" int wisp_mx4_config(int32_t key, int64_t value) {
    if (key == WISP_MX4_TRIES && value >= 1 && value <= WISP_MX4_DEFAULT_TRIES) {
        const int tries = (int)value;
        WISP_CUDA_TRY(cudaMemcpyToSymbol(g_status, &tries, sizeof(tries), sizeof(int)));
        return WISP_OK;
    }
    if (key == WISP_MX4_DROP && value >= 0 && value <= WISP_MX4_DROP_TERMS) return g_dropped = (int)value, WISP_OK;
    return set_error("wisp_mx4_config: unknown key or value"), WISP_ERR_INVALID;
}
