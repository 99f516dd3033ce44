// A whole MoE layer for a few tokens, in one launch, from MXFP4 experts.
//
//   l = x R^T                         router (or the caller's weights and ids)
//   p = softmax over the k largest l  (over all of them when not renormalised)
//   h = W13[e] x, a = silu(h[:I]) h[I:], y = W2[e] a     for each routed e
//   out = sum over the token's experts of p_e y_e
//
// Weights are MXFP4 in checkpoint layout and go to the block-scaled tensor
// cores (tcgen05.mma kind::mxf4) as they are: nothing is unpacked on the way.
// Activations keep their precision: a block of 32 of them is written as a sum
// of eight MXFP4 terms, each the rounding of what the terms before it left.  A
// term's scale s is the smallest power of two under which the remainder's
// largest value is at most 6, so that this value m lies above 3 s.  The first
// term leaves at most 0.5 s where m <= 4.5 s, and s (1 of 5) above.  What is
// left, r <= s, has a scale of s / 8 where r <= 0.75 s, and at most that is left
// of it; else s / 4, under which it is at most 4, and half of that is left: s / 8
// again.  (From 0.5 s it is s / 16, likewise.)  So eight terms leave at most
// 8^-7 / 4.5 < 2^-23 of the block's largest value, or 2^-129, half the smallest
// code, where that is more.  A remainder is a whole number of its value's last
// places: a bf16 value that is at least 2^-15 of the largest is held exactly.
// The terms of a token are the 8 rows of a swizzle pattern of the product's
// small operand, 16 tokens a tile; weights take the 128 rows of the other side,
// a token's result is the sum of its eight accumulator columns.  (Six terms,
// with two rows unused, were 0.4 us faster at one token of the layer below, 0.8 at 16, 2 at
// 64, and lost 2e-4 of the small values in blocks with one 1000 times larger.)
// h, the SiLU and the weighted sum are fp32; out is rounded to bf16 once.
// (Unpacking to fp16 for mma.sync instead cost 110 us at 16 tokens of a
// Qwen3-30B-A3B layer, twice this kernel: it is bound by the four hundred
// instructions that 128 columns of 16 rows take.)
//
// Bound by HBM: a few tokens use every byte of a routed expert once.  A
// cooperative launch of one CTA of 16 warps per SM runs
//   R  router products (a warp per expert row and token group), x to terms
//   S  (after a grid barrier, every CTA for itself) top-k and the lists of
//      each expert's tokens in groups of at most 16
//   G  gate-up: tiles of 64 gate rows and the matching 64 up rows of a group's
//      expert; the epilogue brings g and u of a value together through shared
//      memory and writes silu(g) u as terms again
//   D  (a group's tiles once the group's tiles of G are counted; weights are on
//      their way before) down: tiles of 128 rows of the hidden size, a large
//      intermediate size in pieces; p_e y_e in fp32
//   C  (after a second barrier) the sum over a token's experts, in routing order: no
//      atomics, the same bits every run
// In G and D a warp each feeds a ring of 5 stages of 256 values of K (weights
// by TMA, the terms by bulk copies of 1 KB a token, laid out by their writers
// as the swizzle wants them) and issues the products, eight bring the scale
// bytes (mx4_mma.cuh), four read the accumulators.
//
// Measured (in a graph of calls whose inputs, in turn, exceed L2), 128 experts
// of 2048 x 768, top-8: 21.5 us for one token (21 MB; three phases that wait for
// one another, 2 to 3 us each, and the launch), 53 for 16 (207 MB, 3.9 TB/s), 95
// for 64.  8 experts of 4096 x 14336, top-2, 8 tokens: 127 us (675 MB, 5.3 TB/s).
// With many tokens an expert the terms, 8 rows each, are as many bytes from L2
// as the weights (64 tokens there: 293).  Writing the terms of two or four
// blocks together in G, for their chains of roundings (six then) to overlap, was
// 1 to 6 us slower everywhere.
#include <cooperative_groups.h>

#include <algorithm>

#include "mx4_mma.cuh"

namespace wisp {
namespace mx4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kEpiWarp = 2, kSfWarp = 6;       // four warps and two groups of four; 0: copies, 1: products
constexpr int kWarps = 16;                     // two of them in R, S and C only
static_assert(kSfWarp + kScaleGroups * kScaleGroupWarps <= kWarps, "roles");
constexpr int kThreads = kWarps * 32;
constexpr int kTerms = 8;                      // terms of an activation
constexpr int kRows = kTerms;                  // rows of a token in the small operand, those of a swizzle pattern
constexpr int kGroup = 16;                     // tokens of a tile
constexpr int kStages = 5;
constexpr int kTermBytes = kRows * 128;        // terms of a token in a stage
constexpr int kABytes = 128 * 128, kBBytes = kGroup * kTermBytes;
constexpr int kStageBytes = kABytes + kBBytes + 4 * kAtomBytes;
constexpr int kAccCols = kGroup * kRows;       // of an accumulator; two of them
constexpr int kSfCol0 = 2 * kAccCols, kSfCols = 16;
constexpr int kTmemCols = 512;
static_assert(kSfCol0 + kStages * kSfCols <= kTmemCols, "tensor memory");
constexpr int kWindow = 4;                     // stages of a window of scale bytes
static_assert(kStages > kWindow, "a parity wait has to know its phase");
constexpr int kMaxTokens = 64;
constexpr int kMaxTopK = 16;
constexpr int kMaxPairs = kMaxTokens * kMaxTopK;
constexpr int kMaxExperts = 1024;
constexpr int kMaxGroups = kMaxPairs;          // no group is empty
constexpr int kMaxSplit = 16;                  // pieces of the intermediate size in D

struct MoeArgs {
    const __nv_bfloat16 *x;
    int64_t x_stride;
    const __nv_bfloat16 *router;  // [E][H], or nullptr: ids and weights are given
    const void *ids;
    const float *weights;
    const int32_t *expert_map;    // [E] slot of each expert, or nullptr: slot = expert
    const uint8_t *s13, *s2;
    int w13_rows, s13_rows, w2_rows, s2_rows;  // rows from slot to slot: codes, scale bytes
    __nv_bfloat16 *out;
    float *logits;                // [T][E]
    uint8_t *xq, *xs;             // terms of x: [T][steps][kTermBytes], scales [T][kRows][steps * 8]
    uint8_t *aq, *as;             // terms of silu(g) u: the same for each pair
    float *y;                     // [split][T * k][H]
    uint32_t *done;               // [groups] tiles of G that are finished
    int *status;
    int T, E, k, H, I, slots, ids64, renormalize, s13_align, s2_align;
    uint32_t inv_k;               // p / k = p * inv_k >> 16 for every pair p
    int drop;                     // tests: what is waited for in vain
};

// What the lists are built from; lies where the ring will be.
struct Scratch {
    int ids[kMaxPairs];              // expert of pair t * k + j, -1: none
    uint32_t tokens[kMaxExperts][2];  // the tokens routed to an expert, a bit each
    int begin[kMaxExperts];          // where its pairs begin, -1: no slot
    int scan[2][kWarps];
};
struct Lists {
    float w[kMaxPairs];                // routing weight of a pair
    unsigned short pair[kMaxPairs];    // pairs by group
    unsigned short off[kMaxGroups + 1];  // where a group's pairs begin
    int slots[kMaxGroups];             // its expert's slot
    unsigned char has[kMaxPairs];      // whether the pair is in a group
    int n;                             // groups
};

// ---- phase R ------------------------------------------------------------------
// 8 x 8 transpose of nibbles over 8 lanes: lane r's nibble c goes to lane c's
// nibble r.
__device__ __forceinline__ uint32_t transpose_nibbles(uint32_t w, int r) {
    uint32_t o = __shfl_xor_sync(0xFFFFFFFFu, w, 4);
    w = r & 4 ? (w & 0xFFFF0000u) | (o >> 16) : (w & 0x0000FFFFu) | (o << 16);
    o = __shfl_xor_sync(0xFFFFFFFFu, w, 2);
    w = r & 2 ? (w & 0xFF00FF00u) | ((o >> 8) & 0x00FF00FFu) : (w & 0x00FF00FFu) | ((o & 0x00FF00FFu) << 8);
    o = __shfl_xor_sync(0xFFFFFFFFu, w, 1);
    return r & 1 ? (w & 0xF0F0F0F0u) | ((o >> 4) & 0x0F0F0F0Fu) : (w & 0x0F0F0F0Fu) | ((o & 0x0F0F0F0Fu) << 4);
}

// One block of 32 values, one a lane, as terms: codes to `codes` (16 bytes of
// row 0, rows 128 bytes apart, 16-byte pieces swizzled by the row) and scale
// bytes to `scales` (rows `stride` apart).  A term needs the one before it, so
// only that chain is in the loop: a lane collects its eight codes in a word and
// the words are transposed together.
__device__ __forceinline__ void write_terms(float v, uint8_t *codes, uint8_t *scales, int stride, int piece, int lane) {
    uint32_t word = 0, my_byte = 0;
#pragma unroll
    for (int q = 0; q < kTerms; ++q) {
        const uint32_t m = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v) & 0x7FFFFFFFu);
        const int e = (int)(m >> 23);
        // the smallest scale under which the largest value is at most 6
        int byte = e - 2 + ((m & 0x7FFFFFu) > 0x400000u);
        byte = e == 255 ? 255 : max(byte, 0);
        const float inv = byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23);
        uint32_t c;
        asm("{\n .reg .b8 b;\n cvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n cvt.u32.u8 %0, b;\n}"
            : "=r"(c)
            : "f"(v * inv), "f"(0.f));
        const uint32_t h = e2m1x2_to_f16x2(c);
        v = fmaf(-__low2float(*reinterpret_cast<const __half2 *>(&h)), scale_value(byte), v);
        word |= c << (4 * q);
        my_byte = lane == q ? (uint32_t)byte : my_byte;
    }
    const int q = lane & 7;
    word = transpose_nibbles(word, q);
    *reinterpret_cast<uint32_t *>(codes + q * 128 + ((piece ^ q) << 4) + (lane >> 3) * 4) = word;
    if (lane < kTerms) scales[lane * stride] = (uint8_t)my_byte;
}

__device__ void convert_tokens(const MoeArgs &a, int gw, int nw, int lane) {
    const int blocks = a.H / kBlock, steps = (blocks + kStepBlocks - 1) / kStepBlocks;
    for (int u = gw; u < a.T * blocks; u += nw) {
        const int t = u / blocks, b = u - t * blocks, kb = b / kStepBlocks, piece = b % kStepBlocks;
        const float v = __bfloat162float(a.x[t * a.x_stride + b * kBlock + lane]);
        const int stride = steps * kStepBlocks;
        write_terms(v, a.xq + ((size_t)t * steps + kb) * kTermBytes, a.xs + (size_t)t * kRows * stride + b, stride, piece,
                    lane);
    }
}

constexpr int kAhead = 8;  // 16-byte loads of a lane in flight

// One expert's row times TOKENS tokens.
template <int TOKENS>
__device__ void route_products(const MoeArgs &a, int gw, int nw, int lane) {
    constexpr int kDeep = TOKENS == 1 ? kAhead : 2;
    const int groups = (a.T + TOKENS - 1) / TOKENS;
    for (int u = gw; u < a.E * groups; u += nw) {
        const int e = u % a.E, t0 = u / a.E * TOKENS;
        const __nv_bfloat16 *row = a.router + (size_t)e * a.H;
        float acc[TOKENS] = {};
        for (int h0 = lane * 8; h0 < a.H; h0 += 256 * kDeep) {
            uint4 w[kDeep], x[kDeep][TOKENS];
#pragma unroll
            for (int i = 0; i < kDeep; ++i) {
                const bool in = h0 + i * 256 < a.H;
                w[i] = in ? ld_cached16(row + h0 + i * 256) : make_uint4(0, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < TOKENS; ++j)
                    x[i][j] = in ? ld_cached16(a.x + min(t0 + j, a.T - 1) * a.x_stride + h0 + i * 256)
                                 : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kDeep; ++i)
#pragma unroll
                for (int j = 0; j < TOKENS; ++j) acc[j] = dot8(w[i], x[i][j], acc[j]);
        }
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) {
            const float s = warp_sum(acc[j]);
            if (lane == 0 && t0 + j < a.T) a.logits[(size_t)(t0 + j) * a.E + e] = s;
        }
    }
}

// ---- phase S ------------------------------------------------------------------
// Order-preserving key of a logit; a NaN lies below every number.
__device__ __forceinline__ uint32_t key_of(float v) {
    if (isnan(v)) return 1;
    const uint32_t b = __float_as_uint(v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float logit_of(uint32_t key) {
    return key == 1 ? NAN : __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// The weights of a token whose lane j holds its j-th logit's key and expert.
__device__ void finish_token(const MoeArgs &a, Lists &L, Scratch &S, int t, int lane, uint32_t mine, int my_id) {
    const float l = logit_of(mine), mx = __shfl_sync(0xFFFFFFFFu, l, 0);
    float p = 0.f, all = 0.f;
    if (lane < a.k) p = all = expf(l - mx);
    if (!a.renormalize) {
        all = 0.f;
#pragma unroll 1
        for (int e = lane; e < a.E; e += 32) all += expf(__ldcg(a.logits + (size_t)t * a.E + e) - mx);
    }
    const float sum = warp_sum(all);
    if (lane < a.k) {
        S.ids[t * a.k + lane] = my_id;
        L.w[t * a.k + lane] = p / sum;
    }
}

// Top-k of tokens t, t + kWarps, .. (N of them, those behind the last are
// left out) by (logit descending, id ascending), softmax weights.  Every CTA
// does this for itself, so its latency counts: a round is two reductions of
// the warp (the largest key, the lowest id that has it) without a branch, and
// a warp's tokens go through their rounds together.
template <int PER_LANE, int N>
__device__ void route_tokens(const MoeArgs &a, Lists &L, Scratch &S, int t0, int lane) {
    uint32_t key[N][PER_LANE], mine[N] = {};
    int my_id[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const float *logits = a.logits + (size_t)min(t0 + n * kWarps, a.T - 1) * a.E;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i) {
            const int e = i * 32 + lane;
            key[n][i] = e < a.E ? key_of(__ldcg(logits + e)) : 0;
        }
    }
    for (int j = 0; j < a.k; ++j) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            uint32_t best = 0;
            int id = 0;
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i)
                if (key[n][i] > best) best = key[n][i], id = i * 32 + lane;
            const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
            id = (int)__reduce_min_sync(0xFFFFFFFFu, best == top ? (uint32_t)id : 0x7FFFFFFFu);
#pragma unroll
            for (int i = 0; i < PER_LANE; ++i) key[n][i] = i * 32 + lane == id ? 0 : key[n][i];
            mine[n] = lane == j ? top : mine[n];
            my_id[n] = lane == j ? id : my_id[n];
        }
    }
#pragma unroll 1
    for (int n = 0; n < N; ++n) {
        const int t = t0 + n * kWarps;
        if (t >= a.T) break;
        finish_token(a, L, S, t, lane, n ? mine[N - 1] : mine[0], n ? my_id[N - 1] : my_id[0]);
    }
}
// The same for more experts than a lane has registers for: `keys` [E] in
// shared memory, this warp's own.
__device__ void route_token_shared(const MoeArgs &a, Lists &L, Scratch &S, uint32_t *keys, int t, int lane) {
    const float *logits = a.logits + (size_t)t * a.E;
    uint32_t mine = 0;
    int my_id = 0;
#pragma unroll 4
    for (int e = lane; e < a.E; e += 32) keys[e] = key_of(__ldcg(logits + e));
    for (int j = 0; j < a.k; ++j) {
        uint32_t best = 0;
        int id = 0;
#pragma unroll 4
        for (int e = lane; e < a.E; e += 32)
            if (keys[e] > best) best = keys[e], id = e;
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        id = (int)__reduce_min_sync(0xFFFFFFFFu, best == top ? (uint32_t)id : 0x7FFFFFFFu);
        if ((id & 31) == lane) keys[id] = 0;
        mine = lane == j ? top : mine;
        my_id = lane == j ? id : my_id;
    }
    finish_token(a, L, S, t, lane, mine, my_id);
}

// The caller's routing of token t; an expert named twice is taken once, with
// the sum of its weights.
__device__ void given_token(const MoeArgs &a, Lists &L, Scratch &S, int t) {
    for (int j = 0; j < a.k; ++j) {
        const int p = t * a.k + j;
        const long long e = load_id64(a.ids, a.ids64, p);
        int id = e < 0 || e >= a.E ? -1 : (int)e;
        for (int i = 0; i < j && id >= 0; ++i)
            if (S.ids[t * a.k + i] == id) {
                L.w[t * a.k + i] += a.weights[p];
                id = -1;
            }
        S.ids[p] = id;
        L.w[p] = a.weights[p];
    }
}

// Pairs by expert, the experts with a slot in ascending order, in groups of at
// most kGroup.  Every CTA has to come to the same groups, so an expert's pairs
// lie in the order of their tokens (a token names an expert at most once): the
// expert's set of tokens, a bit each, gives count and rank whatever the order
// in which the bits were set.
__device__ void build_lists(const MoeArgs &a, Lists &L, Scratch &S) {
    const int P = a.T * a.k, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int p = tid; p < P; p += kThreads) {
        const int e = S.ids[p], t = (int)(p * a.inv_k >> 16);
        if (e >= 0) atomicOr(&S.tokens[e][t >> 5], 1u << (t & 31));
    }
    __syncthreads();
    int total = 0;  // of the rounds so far: pairs in the low half, groups in the high half
    for (int e0 = 0, round = 0; e0 < a.E; e0 += kThreads, ++round) {
        const int e = e0 + tid;
        int slot = 0, count = e < a.E ? __popc(S.tokens[e][0]) + __popc(S.tokens[e][1]) : 0;
        if (count) {
            slot = a.expert_map ? a.expert_map[e] : e;
            if (slot < 0 || slot >= a.slots) count = 0;
        }
        const int own = count + ((count + kGroup - 1) / kGroup << 16);
        int run = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xFFFFFFFFu, run, o);
            if (lane >= o) run += v;
        }
        if (lane == 31) S.scan[round & 1][warp] = run;
        __syncthreads();
        const int sum = lane < kWarps ? S.scan[round & 1][lane] : 0;
        const int at = total + run - own + __reduce_add_sync(0xFFFFFFFFu, lane < warp ? sum : 0);
        total += __reduce_add_sync(0xFFFFFFFFu, sum);
        if (e < a.E) S.begin[e] = count ? at & 0xFFFF : -1;
        for (int done = 0, g = at >> 16; done < count; done += kGroup, ++g) {
            L.slots[g] = slot;
            L.off[g] = (unsigned short)((at & 0xFFFF) + done);
        }
    }
    if (tid == 0) {
        L.n = total >> 16;
        L.off[total >> 16] = (unsigned short)(total & 0xFFFF);
    }
    __syncthreads();
    for (int p = tid; p < P; p += kThreads) {
        const int e = S.ids[p], at = e >= 0 ? S.begin[e] : -1, t = (int)(p * a.inv_k >> 16);
        L.has[p] = at >= 0;
        if (at < 0) continue;
        const uint32_t before = (1u << (t & 31)) - 1;
        const int rank = t < 32 ? __popc(S.tokens[e][0] & before)
                                : __popc(S.tokens[e][0]) + __popc(S.tokens[e][1] & before);
        L.pair[at + rank] = (unsigned short)p;
    }
    __syncthreads();
}

// ---- phases G and D ---------------------------------------------------------------
// The tiles of a phase, in the order group, piece of K, rows; a CTA takes every
// gridDim.x-th.  An expert's matrix has `rows` rows; slots lie slot_rows rows
// of codes and scale_slot_rows rows of scale bytes apart.  The first 64 rows
// of a tile are m0 .., the second 64 lie `second` rows further on.  K: `blocks`
// scale bytes a row, `steps` steps of 256 values, in `split` pieces.
struct Phase {
    const CUtensorMap *map;
    const uint8_t *w_scales, *b_codes, *b_scales;
    const uint32_t *done;  // where the terms are made by tiles of this launch: how many of a group's are finished
    uint32_t done_tiles;   // and how many there are
    int groups, m_tiles, split, rows_m, rows, slot_rows, scale_slot_rows, second, blocks, steps, align, term_align;
    uint32_t inv_div;  // pair * inv_div >> 16: which terms are the pair's
};
struct Control {
    uint64_t full[kStages], sf_full[kStages], empty[kStages];
    uint64_t acc_full[2], acc_empty[2], mma_done;
    uint32_t tmem_base;
    int abort, issued, consumed;
    Phase phase[2];  // G, D
    int cut[kMaxSplit + 1];  // K steps at which the pieces of D begin
};
// A CTA's walk over the tiles.  (Roles that are one thread or warp feel every
// instruction: no divisions here, nor remainders in the ring's positions.)
struct Walk {
    int per_group, dg, din;  // gridDim.x in groups and tiles
    int g, in;
    // the tile
    int m0 = 0, kb0 = 0, kb1 = 0, off = 0, n = 0, piece = 0;
    int row = 0, slot = 0;  // row of the weight matrix, slot
    __device__ __forceinline__ Walk(const Phase &ph) {
        per_group = ph.m_tiles * ph.split;
        dg = gridDim.x / per_group, din = gridDim.x - dg * per_group;
        g = blockIdx.x / per_group, in = blockIdx.x - g * per_group;
    }
    // False behind the last tile.
    __device__ __forceinline__ bool at(const Phase &ph, const Lists &L, const Control &C) {
        if (g >= ph.groups) return false;
        int m = in;
        piece = 0, kb0 = 0, kb1 = ph.steps;
        if (ph.split > 1) {
            for (; m >= ph.m_tiles; m -= ph.m_tiles) ++piece;
            kb0 = C.cut[piece], kb1 = C.cut[piece + 1];
        }
        m0 = m * ph.rows_m;
        off = L.off[g];
        n = L.off[g + 1] - off;
        slot = L.slots[g];
        row = slot * ph.slot_rows + m0;
        return true;
    }
    __device__ __forceinline__ void next() {
        g += dg, in += din;
        if (in >= per_group) in -= per_group, ++g;
    }
};

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     s_addr(dst)),
                 "l"(src), "r"(bytes), "r"(s_addr(bar))
                 : "memory");
}

// Waits (a converged warp, bounded) until the terms of a group are in memory,
// and makes them visible to this thread's loads and copies.
__device__ __forceinline__ bool wait_terms(const Phase &ph, int group, volatile int *abort, int *status) {
    if (!ph.done) return true;
    uint32_t n;
    bool ok = false;
#pragma unroll 1
    for (uint32_t i = 1;; ++i) {
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(n) : "l"(ph.done + group) : "memory");
        ok = n >= ph.done_tiles;
        if (ok || gives_up(i, abort, status)) break;
    }
    asm volatile("fence.proxy.async;" ::: "memory");
    if (!ok) give_up(abort, status);
    return __all_sync(0xFFFFFFFFu, ok);
}

// What of a role lives on from phase to phase.
struct Cursor {
    RingPos<kStages> ring;
    RingPos<2> acc;
    int first = 0;  // the scale group whose turn the next window is
};

__device__ __forceinline__ void load_weights(unsigned char *st, const Phase &ph, const Walk &t, int kb, uint64_t *bar) {
    tma_load_2d(st, ph.map, kb * 128, t.row, bar);
    tma_load_2d(st + kABytes / 2, ph.map, kb * 128, t.row + ph.second, bar);
}

// Copies of a phase's steps: the first lane brings the weights (those of the
// first `early` steps are on their way already), lane i token i's terms.
__device__ void run_copies(Control &C, unsigned char *stages, const Phase &ph, const Lists &L, Cursor &cur, int early,
                           int *status) {
    volatile int *abort = &C.abort;
    const int lane = threadIdx.x & 31;
    int issued = C.issued;
    for (Walk t(ph); t.at(ph, L, C); t.next()) {
        // The weights of the first `early` steps are on their way (copy_early), announced together with the terms.
        // Where a wait for terms gives up, what lies in their place is copied for these steps all the same, so that
        // their barriers complete: the copies have to be over before the CTA ends.
        const bool ok = wait_terms(ph, t.g, abort, status);
        if (!ok && early == 0) return;
        const uint8_t *terms =
            lane < t.n ? ph.b_codes + ((size_t)(L.pair[t.off + lane] * ph.inv_div >> 16) * ph.steps + t.kb0) * kTermBytes
                       : nullptr;
        const uint32_t bytes = kABytes + t.n * kTermBytes;
        for (int kb = t.kb0; kb < t.kb1; ++kb, cur.ring.next()) {
            unsigned char *st = stages + cur.ring.slot * kStageBytes;
            uint64_t *full = &C.full[cur.ring.slot];
            if (early > 0) {
                --early;
            } else {
                if (!ok || !warp_wait(&C.empty[cur.ring.slot], cur.ring.turn ^ 1, abort, status)) return;
                if (lane == 0) {
                    mbar_expect_tx(full, bytes);
                    load_weights(st, ph, t, kb, full);
                }
                __syncwarp();  // the bytes are announced before any of them can arrive
            }
            if (terms) {
                bulk_load(st + kABytes + lane * kTermBytes, terms, kTermBytes, full);
                terms += kTermBytes;
            }
            if (lane == 0) C.issued = ++issued;
        }
    }
}
// The weights of the phase's first steps, as many as the ring holds; returns
// how many.
__device__ int copy_early(Control &C, unsigned char *stages, const Phase &ph, const Lists &L, RingPos<kStages> ring,
                          int *status) {
    volatile int *abort = &C.abort;
    const int lane = threadIdx.x & 31;
    int early = 0;
    for (Walk t(ph); t.at(ph, L, C); t.next())
        for (int kb = t.kb0; kb < t.kb1; ++kb, ring.next()) {
            if (early == kStages || !warp_wait(&C.empty[ring.slot], ring.turn ^ 1, abort, status)) return early;
            if (lane == 0) {
                mbar_expect_tx(&C.full[ring.slot], kABytes + t.n * kTermBytes);
                load_weights(stages + ring.slot * kStageBytes, ph, t, kb, &C.full[ring.slot]);
            }
            ++early;
        }
    return early;
}

__device__ void run_scales(Control &C, unsigned char *stages, const Phase &ph, const Lists &L, Cursor &cur, int *status) {
    const int group = (threadIdx.x >> 5) - kSfWarp >= kScaleGroupWarps;
    const int tid = threadIdx.x - (kSfWarp + group * kScaleGroupWarps) * 32;
    volatile int *abort = &C.abort;
    unsigned char *sf = stages + kABytes + kBBytes + atom_at(tid);
    // a window is loaded as soon as the one before it is stored; the other group's comes between them
    Walk ahead(ph);
    bool more = ahead.at(ph, L, C);
    int kb = ahead.kb0;
    const uint8_t *pw = nullptr, *pb = nullptr;  // rows of the tile
    const int my_row = tid < 64 ? tid : ph.second + tid - 64;
    const int term_stride = ph.steps * kStepBlocks;
    auto point = [&] {
        if (!wait_terms(ph, ahead.g, abort, status)) {
            more = false;
            return;
        }
        const int row = ahead.m0 + my_row;
        pw = row < ph.rows ? ph.w_scales + ((int64_t)ahead.slot * ph.scale_slot_rows + row) * ph.blocks : nullptr;
        const int i = tid / kRows, q = tid % kRows;
        pb = i < ahead.n
                 ? ph.b_scales + (size_t)((L.pair[ahead.off + i] * ph.inv_div >> 16) * kRows + q) * term_stride
                 : nullptr;
    };
    auto count = [&] { return more ? min(kWindow, ahead.kb1 - kb) : 0; };
    // to the next window, which may be of another tile
    auto advance = [&] {
        kb += kWindow;
        if (!more || kb < ahead.kb1) return false;
        ahead.next();
        more = ahead.at(ph, L, C);
        kb = ahead.kb0;
        return more;
    };
    struct Window {
        ScaleWords<kWindow> w, b;
        uint32_t w_shift;
        int count, skip;  // stages of the window, and of the other group's window behind it
        int left;         // scale bytes of a row from here on
    } x;
    auto load = [&] {
        x.count = count();
        if (!more) return;
        x.left = ph.blocks - kb * kStepBlocks;
        x.w.zero(), x.b.zero();
        if (pw) x.w.load(pw + kb * kStepBlocks, x.count, x.left, ph.align);
        x.w_shift = row_shift(pw);
        if (pb) x.b.load<false>(pb + kb * kStepBlocks, x.count, x.left, ph.term_align);  // written by this kernel
        bool moved = advance();
        x.skip = count();
        moved |= advance();
        if (moved && more) point();
    };
    RingPos<kStages> ring = cur.ring;
    int last = -1;  // the group that had the last window
    if (group != cur.first && more) {
        last = 1 - group;
        ring.skip(count());
        advance();
    }
    if (more) point();
#pragma unroll 1
    while (true) {
        load();
        if (!x.count) break;
        last = x.skip ? 1 - group : group;
#pragma unroll
        for (int j = 0; j < kWindow; ++j) {
            if (j >= x.count) break;
            if (!warp_wait(&C.empty[ring.slot], ring.turn ^ 1, abort, status)) return;
            unsigned char *at = sf + ring.slot * kStageBytes;
            const uint2 scales = x.w.stage(j, x.w_shift, x.left), terms = x.b.stage(j, 0, x.left);
            *reinterpret_cast<uint32_t *>(at) = scales.x;
            *reinterpret_cast<uint32_t *>(at + kAtomBytes) = scales.y;
            *reinterpret_cast<uint32_t *>(at + 2 * kAtomBytes) = terms.x;
            *reinterpret_cast<uint32_t *>(at + 3 * kAtomBytes) = terms.y;
            fence_async_shared();
            __syncwarp();
            if ((tid & 31) == 0) mbar_arrive(&C.sf_full[ring.slot]);
            ring.next();
        }
        ring.skip(x.skip);
    }
    // both groups have come past the phase's last stage, and go on in turn
    cur.ring = ring;
    if (last >= 0) cur.first = 1 - last;
}

// The whole warp walks, one lane issues.
__device__ void run_products(Control &C, unsigned char *stages, const Phase &ph, const Lists &L, Cursor &cur, int *status) {
    volatile int *abort = &C.abort;
    const uint32_t base = s_addr(stages);
    const uint64_t a0 = smem_desc_k_sw128(base), b0 = smem_desc_k_sw128(base + kABytes),
                   sf0 = smem_desc_atom(base + kABytes + kBBytes);
    const uint32_t tmem = C.tmem_base;
    int consumed = C.consumed;
    for (Walk t(ph); t.at(ph, L, C); t.next(), cur.acc.next()) {
        if (!warp_wait(&C.acc_empty[cur.acc.slot], cur.acc.turn ^ 1, abort, status)) return;
        tc_fence_after();
        const uint32_t acc = tmem + cur.acc.slot * kAccCols;
        const uint32_t id0 = idesc_mxf4(128, (t.n * kRows + 15) / 16 * 16, 0), id1 = id0 | (2u << 4) | (2u << 29);
        uint32_t more = 0;
        for (int kb = t.kb0; kb < t.kb1; ++kb, cur.ring.next()) {
            const int s = cur.ring.slot;
            if (!warp_wait(&C.full[s], cur.ring.turn, abort, status) ||
                !warp_wait(&C.sf_full[s], cur.ring.turn, abort, status))
                return;
            tc_fence_after();
            // addresses are in units of 16 bytes; 64 values are 32 bytes further along K
            const uint64_t step = (uint64_t)(s * (kStageBytes >> 4));
            const uint64_t da = a0 + step, db = b0 + step, ds = sf0 + step;
            const uint32_t cols = tmem + kSfCol0 + s * kSfCols;
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < 4; ++i) copy_atom(cols + i * 4, ds + i * (kAtomBytes >> 4));
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                    umma_mxf4(acc, da + kk * 2, db + kk * 2, kk & 1 ? id1 : id0, cols + (kk >> 1) * 4,
                              cols + 8 + (kk >> 1) * 4, more | kk);
                umma_commit(&C.empty[s]);
                C.consumed = ++consumed;
            }
            more = 1;
        }
        if (elect_one()) umma_commit(&C.acc_full[cur.acc.slot]);
    }
}

// Four tokens' columns of this thread's row.
__device__ __forceinline__ void read_rows(uint32_t taddr, float (&v)[4]) {
    uint32_t r[32];
    gemm::tmem_ld32(taddr, r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = 0.f;
#pragma unroll
        for (int q = 0; q < kTerms; ++q) v[i] += __uint_as_float(r[i * kRows + q]);
    }
}
__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

__device__ void run_gate_up(Control &C, const Phase &ph, const Lists &L, Cursor &cur, const MoeArgs &a, float *ex,
                            int steps_out) {
    volatile int *abort = &C.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
    for (Walk tile(ph); tile.at(ph, L, C); tile.next(), cur.acc.next()) {
        const int b = cur.acc.slot;
        const bool ok = warp_wait(&C.acc_full[b], cur.acc.turn, abort, a.status);
        if (ok) {
            tc_fence_after();
            for (int i = 0; i < tile.n; i += 4) {
                float v[4];
                read_rows(C.tmem_base + b * kAccCols + ((uint32_t)(quarter * 32) << 16) + i * kRows, v);
#pragma unroll
                for (int j = 0; j < 4; ++j) ex[(i + j) * 128 + quarter * 32 + lane] = v[j];
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&C.acc_empty[b]);
        }
        epilogue_barrier();
        // warp: one block of 32 intermediate values, every other token
        const int j0 = tile.m0 + (quarter & 1) * 32;
        if (ok && j0 < a.I)
            for (int i = quarter >> 1; i < tile.n; i += 2) {
                const float g = ex[i * 128 + (quarter & 1) * 32 + lane], u = ex[i * 128 + 64 + (quarter & 1) * 32 + lane];
                const int p = L.pair[tile.off + i], kb = j0 / kStepK, piece = j0 / kBlock % kStepBlocks;
                const int stride = steps_out * kStepBlocks;
                write_terms(g / (1.f + __expf(-g)) * u, a.aq + ((size_t)p * steps_out + kb) * kTermBytes,
                            a.as + (size_t)p * kRows * stride + j0 / kBlock, stride, piece, lane);
            }
        // the terms are read by copies and loads of other CTAs once the group's count says so; the barrier puts
        // every warp's stores before the release, which costs one thread and not all of them a fence of the GPU
        asm volatile("fence.proxy.async.global;" ::: "memory");
        epilogue_barrier();
        if (quarter == 0 && lane == 0)
            asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.done + tile.g) : "memory");
    }
}

__device__ void run_down(Control &C, const Phase &ph, const Lists &L, Cursor &cur, const MoeArgs &a) {
    volatile int *abort = &C.abort;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quarter = warp & 3;
    for (Walk tile(ph); tile.at(ph, L, C); tile.next(), cur.acc.next()) {
        const int b = cur.acc.slot;
        if (!warp_wait(&C.acc_full[b], cur.acc.turn, abort, a.status)) return;
        tc_fence_after();
        const int h = tile.m0 + quarter * 32 + lane;
        for (int i = 0; i < tile.n; i += 4) {
            float v[4];
            read_rows(C.tmem_base + b * kAccCols + ((uint32_t)(quarter * 32) << 16) + i * kRows, v);
            if (h >= a.H) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (i + j >= tile.n) break;
                const int p = L.pair[tile.off + i + j];
                a.y[((size_t)tile.piece * a.T * a.k + p) * a.H + h] = v[j] * L.w[p];
            }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&C.acc_empty[b]);
    }
}

// Pieces of the intermediate size in D.  They let a few experts' tiles fill the
// SMs evenly (two experts of 4096 x 14336 are 64 tiles of 1 MB), and depend on
// the sizes alone, so that a token's bits do not depend on the tokens beside it.
__host__ __device__ constexpr int pieces_of(int steps) { return (steps + 15) / 16; }
static_assert(pieces_of(65536 / kStepK) <= kMaxSplit, "largest intermediate size");

__global__ void __launch_bounds__(kThreads, 1)
    moe_kernel(const __grid_constant__ CUtensorMap map13, const __grid_constant__ CUtensorMap map2, const MoeArgs a) {
    extern __shared__ unsigned char raw[];
    unsigned char *stages = raw + ((1024u - (s_addr(raw) & 1023u)) & 1023u);
    float *ex = reinterpret_cast<float *>(stages + kStages * kStageBytes);  // [kGroup][128]
    Control &C = *reinterpret_cast<Control *>(ex + kGroup * 128);
    Lists &L = *reinterpret_cast<Lists *>(&C + 1);
    Scratch &S = *reinterpret_cast<Scratch *>(stages);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nw = gridDim.x * kWarps;

    if (tid == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&C.full[s], 1);
            mbar_init(&C.sf_full[s], kScaleGroupWarps + (a.drop == WISP_MX4_DROP_SCALES));
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

    // R: warps in turn over the SMs, so that few units spread
    const int gw = warp * gridDim.x + blockIdx.x;
    if (a.router) {
        if (a.E * a.T <= nw)
            route_products<1>(a, gw, nw, lane);
        else
            route_products<4>(a, gw, nw, lane);
    }
    convert_tokens(a, nw - 1 - gw, nw, lane);
    for (int i = tid; i < 2 * a.E; i += kThreads) (&S.tokens[0][0])[i] = 0;
    for (int i = blockIdx.x * kThreads + tid; i < a.T * a.k; i += gridDim.x * kThreads) a.done[i] = 0;  // groups <= pairs
    asm volatile("fence.proxy.async;" ::: "memory");  // the terms are read by bulk copies
    cg::this_grid().sync();
    tc_fence_after();

    // S
    if (a.router) {
        if (a.E <= 128 && a.T <= kWarps) {
            if (warp < a.T) route_tokens<4, 1>(a, L, S, warp, lane);
        } else if (a.E <= 128)
            for (int t = warp; t < a.T; t += 2 * kWarps) route_tokens<4, 2>(a, L, S, t, lane);
        else
            for (int t = warp; t < a.T; t += kWarps)
                route_token_shared(a, L, S, reinterpret_cast<uint32_t *>(&S + 1) + warp * a.E, t, lane);
    } else if (tid < a.T) {
        given_token(a, L, S, tid);
    }
    __syncthreads();
    build_lists(a, L, S);
    // the ring's memory was written as plain memory, the copies come next
    asm volatile("fence.proxy.async;" ::: "memory");
    __syncthreads();

    if (tid == 0) {
        Phase &up = C.phase[0], &down = C.phase[1];
        up.map = &map13, up.w_scales = a.s13, up.b_codes = a.xq, up.b_scales = a.xs;
        up.blocks = a.H / kBlock, up.steps = (up.blocks + kStepBlocks - 1) / kStepBlocks, up.align = a.s13_align;
        up.groups = L.n, up.m_tiles = (a.I + 63) / 64, up.split = 1, up.rows_m = 64;
        up.rows = 2 * a.I, up.slot_rows = a.w13_rows, up.scale_slot_rows = a.s13_rows, up.second = a.I;
        up.inv_div = a.inv_k, up.done = nullptr;
        down.map = &map2, down.w_scales = a.s2, down.b_codes = a.aq, down.b_scales = a.as;
        down.blocks = a.I / kBlock, down.steps = (down.blocks + kStepBlocks - 1) / kStepBlocks, down.align = a.s2_align;
        down.groups = L.n, down.m_tiles = (a.H + 127) / 128, down.rows_m = 128;
        down.split = pieces_of(down.steps);
        down.rows = a.H, down.slot_rows = a.w2_rows, down.scale_slot_rows = a.s2_rows, down.second = 64;
        down.inv_div = 65536, down.done = a.done, down.done_tiles = up.m_tiles + (a.drop == WISP_MX4_DROP_TERMS);
        // (pieces of D begin at whole 16-byte loads of scale bytes)
        up.term_align = up.steps % 2 ? 8 : 16, down.term_align = down.steps % 2 ? 8 : 16;
        const int unit = down.align >= 16 || down.term_align >= 16 ? 2 : 1;
        for (int i = 0; i <= down.split; ++i) C.cut[i] = i * down.steps / down.split / unit * unit;
    }
    __syncthreads();

    // G and D, by the same code and without a barrier between them: a tile of D waits for its group's tiles of G
    Cursor cur;
    int early = 0;
#pragma unroll 1
    for (int phase = 0; phase < 2; ++phase) {
        const Phase ph = C.phase[phase];
        if (warp == 0) {
            run_copies(C, stages, ph, L, cur, early, a.status);
            if (phase == 0) early = copy_early(C, stages, C.phase[1], L, cur.ring, a.status);
        } else if (warp == 1) {
            run_products(C, stages, ph, L, cur, a.status);
            __syncwarp();
            if (phase == 1 && elect_one()) umma_commit(&C.mma_done);
        } else if (warp < kSfWarp) {
            if (phase == 0)
                run_gate_up(C, ph, L, cur, a, ex, C.phase[1].steps);
            else
                run_down(C, ph, L, cur, a);
        } else if (warp < kSfWarp + kScaleGroups * kScaleGroupWarps) {
            run_scales(C, stages, ph, L, cur, a.status);
        }
        __syncwarp();
    }
    tc_fence_before();
    cg::this_grid().sync();
    tc_fence_after();

    // C
    const int P = a.T * a.k, split = C.phase[1].split;
    for (int i = blockIdx.x * kThreads + tid; i < a.T * (a.H / 4); i += gridDim.x * kThreads) {
        const int t = i / (a.H / 4), h = (i - t * (a.H / 4)) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < split; ++s) {
            const float *y = a.y + ((size_t)s * P + t * a.k) * a.H + h;
            for (int j0 = 0; j0 < a.k; j0 += 8) {  // eight loads in flight
                float4 v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    v[j] = j0 + j < a.k && L.has[t * a.k + j0 + j]
                               ? __ldcg(reinterpret_cast<const float4 *>(y + (size_t)(j0 + j) * a.H))
                               : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int j = 0; j < 8; ++j) sum.x += v[j].x, sum.y += v[j].y, sum.z += v[j].z, sum.w += v[j].w;
            }
        }
        __nv_bfloat162 o[2] = {__floats2bfloat162_rn(sum.x, sum.y), __floats2bfloat162_rn(sum.z, sum.w)};
        memcpy(a.out + (size_t)t * a.H + h, o, 8);
    }
    if (tid == 0) {
        // after an abort: copies and products in flight end before the memory is given back
        volatile int no_abort = 0;
        for (int k = C.consumed; k < C.issued; ++k)
            wait_tries(&C.full[k % kStages], (k / kStages) & 1, &no_abort, a.status);
        wait_tries(&C.mma_done, 0, &no_abort, a.status);
    }
    __syncthreads();
    if (warp == 0) gemm::tmem_dealloc(C.tmem_base, kTmemCols);
}

struct Workspace {
    size_t logits, xq, xs, aq, as, y, done, bytes;
    Workspace(int T, int E, int k, int H, int I) {
        size_t at = 0;
        const auto take = [&](size_t n) { const size_t here = at; at += (n + 255) / 256 * 256; return here; };
        const size_t up = (H + kStepK - 1) / kStepK, down = (I + kStepK - 1) / kStepK, P = (size_t)T * k;
        logits = take((size_t)T * E * 4);
        xq = take(T * up * kTermBytes);
        xs = take(T * up * kRows * kStepBlocks);
        aq = take(P * down * kTermBytes);
        as = take(P * down * kRows * kStepBlocks);
        y = take((size_t)pieces_of((int)down) * P * H * 4);
        done = take(P * 4);
        bytes = at;
    }
};
constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kGroup * 128 * 4 + sizeof(Control) + sizeof(Lists);
static_assert(kSmemBytes <= 232448, "shared memory");
static_assert(sizeof(Scratch) + kWarps * kMaxExperts * 4 <= kStages * kStageBytes, "the lists' scratch lies in the ring");

int check_shape(int32_t T, int32_t E, int32_t k, int32_t H, int32_t I, int32_t slots) {
    if (T < 0 || T > kMaxTokens || E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E || slots < 1)
        return set_error("wisp_mx4_moe: need at most 64 tokens, 1024 experts, 1 <= top_k <= min(16, experts)"),
               WISP_ERR_INVALID;
    if (H < 32 || H % 32 || H > 32768 || I < 32 || I % 32 || I > 65536)
        return set_error("wisp_mx4_moe: hidden and intermediate sizes are multiples of 32, at most 32768 and 65536"),
               WISP_ERR_INVALID;
    return WISP_OK;
}

// Rows of `row_bytes` from slot to slot, from a stride in bytes.
int slot_rows(int64_t stride, int64_t row_bytes, int64_t rows, int32_t slots, int *out) {
    if (stride % row_bytes || stride / row_bytes < rows || stride / row_bytes * slots > INT32_MAX)
        return set_error("wisp_mx4_moe: slots must be whole rows apart and not overlap, with at most 2^31 rows in all"),
               WISP_ERR_INVALID;
    *out = (int)(stride / row_bytes);
    return WISP_OK;
}

}  // namespace
}  // namespace mx4
}  // namespace wisp

using namespace wisp;
using namespace wisp::mx4;

extern "C" int wisp_mx4_moe_workspace(int32_t num_tokens, int32_t num_experts, int32_t top_k, int32_t hidden,
                                      int32_t inter, int64_t *bytes) {
    if (const int rc = check_shape(num_tokens, num_experts, top_k, hidden, inter, 1)) return rc;
    if (!bytes) return set_error("wisp_mx4_moe_workspace: NULL result"), WISP_ERR_INVALID;
    *bytes = (int64_t)Workspace(num_tokens, num_experts, top_k, hidden, inter).bytes;
    return WISP_OK;
}

extern "C" int wisp_mx4_moe(const void *x, int64_t x_stride, const void *router, const void *topk_ids,
                            int32_t ids_int64, const float *topk_weights, const int32_t *expert_map,
                            const void *w13_codes, const void *w13_scales, const void *w2_codes, const void *w2_scales,
                            const int64_t *slot_strides, int32_t num_slots, int32_t num_tokens, int32_t num_experts,
                            int32_t top_k, int32_t hidden, int32_t inter, int32_t renormalize, void *workspace,
                            int64_t workspace_bytes, void *out, void *stream) {
    if (const int rc = check_shape(num_tokens, num_experts, top_k, hidden, inter, num_slots)) return rc;
    if (num_tokens == 0) return WISP_OK;
    if (!x || !w13_codes || !w13_scales || !w2_codes || !w2_scales || !workspace || !out)
        return set_error("wisp_mx4_moe: NULL tensor"), WISP_ERR_INVALID;
    if (router ? topk_ids || topk_weights : !topk_ids || !topk_weights)
        return set_error("wisp_mx4_moe: give either the router's weights or ids and weights"), WISP_ERR_INVALID;
    if (!expert_map && num_slots < num_experts)
        return set_error("wisp_mx4_moe: fewer slots than experts, and no expert map"), WISP_ERR_INVALID;
    for (const void *p : {x, router, w13_codes, w2_codes, (const void *)workspace, (const void *)out})
        if (reinterpret_cast<uintptr_t>(p) % 16)
            return set_error("wisp_mx4_moe: x, router, codes, workspace and out must be aligned to 16 bytes"),
                   WISP_ERR_INVALID;
    if (num_tokens > 1 && (x_stride < hidden || x_stride % 8))
        return set_error("wisp_mx4_moe: rows of x must not overlap and must start on 16-byte boundaries"),
               WISP_ERR_INVALID;
    const Workspace w(num_tokens, num_experts, top_k, hidden, inter);
    if (workspace_bytes < (int64_t)w.bytes)
        return set_error("wisp_mx4_moe: workspace too small (wisp_mx4_moe_workspace)"), WISP_ERR_INVALID;
    unsigned char *ws = reinterpret_cast<unsigned char *>(workspace);
    MoeArgs a{};
    a.x = reinterpret_cast<const __nv_bfloat16 *>(x);
    a.x_stride = x_stride;
    a.router = reinterpret_cast<const __nv_bfloat16 *>(router);
    a.ids = topk_ids;
    a.weights = topk_weights;
    a.expert_map = expert_map;
    a.s13 = reinterpret_cast<const uint8_t *>(w13_scales);
    a.s2 = reinterpret_cast<const uint8_t *>(w2_scales);
    a.s13_align = scale_align(w13_scales, hidden / kBlock), a.s2_align = scale_align(w2_scales, inter / kBlock);
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.logits = reinterpret_cast<float *>(ws + w.logits);
    a.xq = ws + w.xq, a.xs = ws + w.xs, a.aq = ws + w.aq, a.as = ws + w.as;
    a.y = reinterpret_cast<float *>(ws + w.y);
    a.done = reinterpret_cast<uint32_t *>(ws + w.done);
    const int64_t hb = hidden / 2, ib = inter / 2;
    const int64_t packed[4] = {2 * inter * hb, 2 * inter * (hb / 16), hidden * ib, hidden * (ib / 16)};
    const int64_t *st = slot_strides ? slot_strides : packed;
    int rc = slot_rows(st[0], hb, 2 * inter, num_slots, &a.w13_rows);
    if (!rc) rc = slot_rows(st[1], hb / 16, 2 * inter, num_slots, &a.s13_rows);
    if (!rc) rc = slot_rows(st[2], ib, hidden, num_slots, &a.w2_rows);
    if (!rc) rc = slot_rows(st[3], ib / 16, hidden, num_slots, &a.s2_rows);
    if (!rc) rc = status_word(&a.status);
    CUtensorMap m13, m2;  // they end with the last slot's last row
    if (!rc) rc = gemm::make_byte_map(&m13, w13_codes, (uint64_t)a.w13_rows * (num_slots - 1) + 2 * inter, hb, 64);
    if (!rc) rc = gemm::make_byte_map(&m2, w2_codes, (uint64_t)a.w2_rows * (num_slots - 1) + hidden, ib, 64);
    if (rc) return rc;
    // a slot's scale bytes are aligned like the first slot's only where the stride keeps that
    a.s13_align = std::min(a.s13_align, scale_align(nullptr, (int)(st[1] & 15)));
    a.s2_align = std::min(a.s2_align, scale_align(nullptr, (int)(st[3] & 15)));
    a.T = num_tokens, a.E = num_experts, a.k = top_k, a.H = hidden, a.I = inter, a.slots = num_slots;
    a.ids64 = ids_int64, a.renormalize = renormalize, a.inv_k = 65536 / top_k + 1;
    a.drop = dropped();
    int dev = 0, sms = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    WISP_CUDA_TRY(cudaFuncSetAttribute(moe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
    void *params[] = {&m13, &m2, &a};
    WISP_CUDA_TRY(cudaLaunchCooperativeKernel(reinterpret_cast<const void *>(moe_kernel), dim3(sms), dim3(kThreads),
                                              params, kSmemBytes, reinterpret_cast<cudaStream_t>(stream)));
    return WISP_OK;
}
