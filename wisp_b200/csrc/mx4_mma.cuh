// tcgen05.mma on MXFP4 operands (kind::mxf4, one E8M0 scale for 32 values).
//
// Operand tiles lie in shared memory as TMA boxes of 128 bytes (256 values) a
// row with 128-byte swizzle; one instruction takes 64 values of K, 32 bytes
// along the row.  The scales of an instruction lie in tensor memory: of 128
// rows, row 32 g + l in lane l, column c + g (all four lane quarters hold a
// copy), its four scale bytes of 128 values of K in one 32-bit cell, of which
// an instruction of K 64 uses the lower or the upper half (the scale id of
// the instruction descriptor, 0 or 2).  tcgen05.cp 32x128b.warpx4 brings such
// a block there from 512 bytes of shared memory in which row 32 g + l's word
// lies at 16 l + 4 g ("scale atom").
#pragma once
#include "gemm_sm100.cuh"
#include "mx4.cuh"

namespace wisp {
namespace mx4 {

using gemm::mbar_arrive;
using gemm::mbar_expect_tx;
using gemm::mbar_init;
using gemm::mbar_try;
using gemm::s_addr;
using gemm::smem_desc_k_sw128;
using gemm::tc_fence_after;
using gemm::tc_fence_before;
using gemm::tma_load_2d;
using gemm::umma_commit;

constexpr int kStepK = 256;                 // values of K in a stage: 128 bytes a row
constexpr int kStepBlocks = kStepK / kBlock;  // scale bytes of a row in a stage
constexpr int kAtomBytes = 512;             // scales of 128 rows x 128 values

// The current device's words of the kernels' waits (mx4_matmul.cu): [0] how many
// ran out, [1] limit of one wait in tries.
int status_word(int **word);
// What a test lets a launch wait for in vain (wisp_mx4_config).
int dropped();

// Instruction descriptor: E2M1 A and B, K-major, E8M0 scales, fp32 D, M x N;
// `sf` 0 or 2: which half of the scale words (K 64 of 128).
__host__ __device__ constexpr uint32_t idesc_mxf4(int M, int N, int sf) {
    return ((uint32_t)sf << 4)            // scale id of B
           | (1u << 7)                    // A: E2M1
           | (1u << 10)                   // B: E2M1
           | ((uint32_t)(N >> 3) << 17)   // N / 8
           | (1u << 23)                   // scales: E8M0
           | ((uint32_t)(M >> 7) << 27)   // M / 128
           | ((uint32_t)sf << 29);        // scale id of A
}
__device__ __forceinline__ void umma_mxf4(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t tmem_sfa, uint32_t tmem_sfb, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(
            tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(tmem_sfa), "r"(tmem_sfb), "r"(accumulate)
        : "memory");
}
// One lane of the (converged) warp, the same every time: the instructions of
// the tensor cores are issued by it, while the whole warp computes their
// addresses, which keeps them in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xFFFFFFFF;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
// Position in a ring of STAGES: slot, and the parity of its turn.
template <int STAGES>
struct RingPos {
    int slot = 0;
    uint32_t turn = 0;
    __device__ __forceinline__ void next() {
        if (++slot == STAGES) slot = 0, turn ^= 1;
    }
    __device__ __forceinline__ void skip(int n) {  // n <= STAGES
        slot += n;
        if (slot >= STAGES) slot -= STAGES, turn ^= 1;
    }
};
// Scale atom: 32 rows of 16 bytes, groups of 8 rows 128 bytes apart, no swizzle.
__device__ __forceinline__ uint64_t smem_desc_atom(uint32_t saddr) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)1u << 16;           // leading byte offset (one column of core matrices: not used)
    d |= (uint64_t)(128u >> 4) << 32;  // stride byte offset
    d |= (uint64_t)1u << 46;           // version
    return d;
}
// One scale atom to four columns of tensor memory, in every lane quarter.
__device__ __forceinline__ void copy_atom(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// Byte offset of row r's word in a scale atom.
__device__ __forceinline__ int atom_at(int r) { return (r & 31) * 16 + (r >> 5) * 4; }

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Whether a wait gives up after its i-th try: `abort` was set, or the limit is
// reached.  Looked at after every 256th only; the usual wait is far shorter.
__device__ __forceinline__ bool gives_up(uint32_t i, const volatile int *abort, const int *status) {
    return i % 256 == 0 && (*abort || i >= (uint32_t) reinterpret_cast<const volatile int *>(status)[1]);
}
// Waits until the barrier's phase is over.  A try suspends the thread for a
// while: the limit is seconds, where no wait here is longer than a few memory
// latencies.
__device__ __forceinline__ bool wait_tries(uint64_t *bar, uint32_t parity, const volatile int *abort,
                                           const int *status) {
    for (uint32_t i = 1; !mbar_try(bar, parity); ++i)
        if (gives_up(i, abort, status)) return false;
    return true;
}
__device__ __forceinline__ void give_up(volatile int *abort, int *status) {
    *abort = 1;
    atomicAdd(status, 1);
}
// The wait of a role; one that runs out sets the status and the CTA's abort word.
// (One copy of the loop for a kernel's many waits: roles that run at the same
// time share one instruction cache.  A kernel of 228 KB, everything inlined and
// unrolled, spent as long on fetching instructions as on memory.)
static __device__ __noinline__ bool wait_long(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    if (wait_tries(bar, parity, abort, status)) return true;
    give_up(abort, status);
    return false;
}
__device__ __forceinline__ bool wait_or_abort(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    return mbar_try(bar, parity) || wait_long(bar, parity, abort, status);
}

// For a converged warp: all lanes wait, all go on or none does.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *status) {
    return __all_sync(0xFFFFFFFFu, wait_or_abort(bar, parity, abort, status));
}

// The scale bytes come in windows of up to WINDOW stages of a tile, each taken
// by one of two groups of four warps in turn, so that one stores while the
// other loads.  The rows of a tile lie in as many lines of the cache, so a load
// instruction of 32 rows costs 32 lookups whatever it brings: 16 bytes (two
// stages) a row and instruction where the rows' alignment allows it.  What a
// new tile costs a thread (its rows' addresses) comes once in a window.  (One
// group that loaded 8 bytes a stage needed 1000 cycles a stage, twice what the
// products of a stage take.)
//
// A group passes over the other one's windows without waiting for their slots.
// A parity wait tells a phase from the one before it, not from the one before
// that, so when the group waits for stage k - STAGES to be released it has to
// know that stage k - 2 STAGES was.  Its own stage before k is k - 1 - WINDOW
// at the earliest, for which it saw k - 1 - WINDOW - STAGES released, and stages
// are released in order: STAGES > WINDOW is enough.
constexpr int kScaleGroups = 2, kScaleGroupWarps = 4;

// The first `left` of eight scale bytes; what lies behind a row's last block is
// not a scale.
__device__ __forceinline__ uint2 first_bytes(uint2 v, int left) {
    if (left < 8) {
        const uint64_t keep = (1ull << (8 * left)) - 1;
        v.x &= (uint32_t)keep, v.y &= (uint32_t)(keep >> 32);
    }
    return v;
}
// A window's scale bytes of a row as they were loaded: aligned words.
// stage() shifts them into place where they are used, so that nothing waits for
// a load where it is issued.
template <int WINDOW>
struct ScaleWords {
    uint32_t w[2 * WINDOW + 1];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i <= 2 * WINDOW; ++i) w[i] = 0;
    }
    // The eight bytes of the window's j-th stage; `shift`: bits by which the row
    // is out of its words, `left`: bytes of the row from the window's first on.
    __device__ __forceinline__ uint2 stage(int j, uint32_t shift, int left) const {
        const uint2 v = make_uint2(__funnelshift_r(w[2 * j], w[2 * j + 1], shift),
                                   __funnelshift_r(w[2 * j + 1], w[2 * j + 2], shift));
        return first_bytes(v, left - j * kStepBlocks);
    }
    // `count` stages from p on, `left` bytes of which are the row's.  `align`:
    // what p is aligned to.  Rows of any alignment are read as the 32-bit words
    // that hold a byte of theirs.  NC: through the read-only path.
    template <bool NC = true>
    __device__ __forceinline__ void load(const uint8_t *p, int count, int left, int align) {
        static_assert(WINDOW % 2 == 0, "pairs of stages");
        if (align >= 16) {
#pragma unroll
            for (int i = 0; i < WINDOW; i += 2)
                if (i < count) {
                    const uint4 r = NC ? __ldg(reinterpret_cast<const uint4 *>(p) + i / 2) : ld_cg16(p + i * kStepBlocks);
                    w[2 * i] = r.x, w[2 * i + 1] = r.y, w[2 * i + 2] = r.z, w[2 * i + 3] = r.w;
                }
        } else if (align >= 8) {
#pragma unroll
            for (int i = 0; i < WINDOW; ++i)
                if (i < count) {
                    const uint2 r = NC ? __ldg(reinterpret_cast<const uint2 *>(p) + i)
                                       : __ldcg(reinterpret_cast<const uint2 *>(p) + i);
                    w[2 * i] = r.x, w[2 * i + 1] = r.y;
                }
        } else {
            const int off = (int)(reinterpret_cast<uintptr_t>(p) & 3), bytes = min(left, count * kStepBlocks) + off;
            const uint32_t *q = reinterpret_cast<const uint32_t *>(p - off);
#pragma unroll
            for (int i = 0; i <= 2 * WINDOW; ++i)
                if (4 * i < bytes) w[i] = __ldg(q + i);
        }
    }
};
// Bits by which a row of scale bytes is out of its words.
__device__ __forceinline__ uint32_t row_shift(const uint8_t *p) {
    return (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3) * 8;
}
// What a matrix's rows of scale bytes are aligned to.
__host__ __device__ inline int scale_align(const void *scales, int blocks) {
    const uintptr_t p = reinterpret_cast<uintptr_t>(scales) | (uintptr_t)blocks;
    return p % 16 == 0 ? 16 : p % 8 == 0 ? 8 : p % 4 == 0 ? 4 : 1;
}

}  // namespace mx4
}  // namespace wisp
