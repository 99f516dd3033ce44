// A whole MoE layer for a few tokens, in one launch, from MXFP4 experts.
//
//   l = x R^T                         router (or the caller's weights and ids)
//   p = softmax over the k largest l  (over all of them when not renormalised)
//   h = W13[e] x, a = silu(h[:I]) h[I:], y = W2[e] a     for each routed e
//   out = sum over the token's experts of p_e y_e
//
// Weights are MXFP4 in checkpoint layout, activations 16-bit floats: a product
// multiplies the E2M1 value (exact in fp16) with the activation (fp16, scaled
// by a power of two of its own row so that the largest lies in [2^14, 2^15):
// exact for bf16 activations down to 2^-29 of the row's largest), sums 32 of
// them in fp32 on the tensor cores, and adds the block's sum times the block's
// scale to the fp32 accumulator.  h, the SiLU and the weighted sum are fp32; a
// is rounded to fp16 once (half a step of 2^-11; groups of 8 share a power of
// two, which the down product brings to one for the pair) and out to bf16 once.
//
// Bound by HBM: a few tokens use every byte of a routed expert once.  A
// cooperative launch of one 512-thread CTA per SM runs
//   R  router products (a warp per expert row and four tokens), x to fp16
//   S  (after a grid barrier, every CTA for itself) top-k and the lists of
//      each expert's tokens
//   G  gate-up: a warp takes 8 gate rows and the matching 8 up rows of an
//      expert as the 16 rows of mma.m16n8k16, so g and u of a value meet in
//      one thread; tokens are the 8 columns (1, 2, 4 or 8 column tiles)
//   D  (after a second grid barrier) down: a CTA takes 16 rows of the hidden
//      size, its warps the experts (and pieces of I, when there are few), so
//      that a token's sum over its experts ends in one CTA: no partial sums in
//      memory, no atomics, the same bits every run.
// A warp streams its rows through a ring of its own in shared memory: 16 rows
// x 128 columns (1 KB of codes and 64 scale bytes) a stage, cp.async of 16
// bytes a lane, 7 stages ahead across its units; the 16-byte pieces of a row
// are swizzled so that reading one word a lane is free of conflicts.  With 8
// token columns the tensor core work is far from its limit; what counts is the
// number of instructions a weight costs (about 1.6 a value and lane: 4
// conversions, 2 matrix instructions and 4 multiply-adds per 16 values).
#include <cooperative_groups.h>

#include "mx4.cuh"

namespace wisp {
namespace mx4 {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;
constexpr int kChunk = 512;                    // columns of a stage
constexpr int kSub = 128;                      // columns a thread's registers hold at a time
constexpr int kRowBytes = kChunk / 2;          // codes of a row in a stage
constexpr int kRowBlocks = kChunk / kBlock;    // 16-byte pieces of a row, and its scale bytes
constexpr int kCodeBytes = 16 * kRowBytes;
constexpr int kStageBytes = kCodeBytes + 16 * kRowBlocks;
constexpr int kMaxTokens = 64;
constexpr int kMaxTopK = 16;
constexpr int kMaxPairs = kMaxTokens * kMaxTopK;
constexpr int kMaxExperts = 1024;

struct MoeArgs {
    const __nv_bfloat16 *x;
    int64_t x_stride;
    const __nv_bfloat16 *router;  // [E][H], or nullptr: ids and weights are given
    const void *ids;
    const float *weights;
    const int32_t *expert_map;    // [E] slot of each expert, or nullptr: slot = expert
    const uint8_t *w13, *s13, *w2, *s2;
    __nv_bfloat16 *out;
    float *logits;                // [T][E]
    __half *xs;                   // [T][H]
    float *x_scale;               // [T]: x = xs * x_scale
    __half *act;                  // [T * k][I]: silu(g) u = act * 2^(its group's exponent - 141)
    uint8_t *act_exp;             // [T * k][exp_stride]: exponent of each group of 8 (exp_at)
    uint32_t *act_max;            // [T * k]: the pair's largest exponent
    int T, E, k, H, I, slots, ids64, renormalize, exp_stride;
};

struct Lists {
    int ids[kMaxPairs];             // expert of pair t * k + j, -1: none
    float w[kMaxPairs];             // its weight
    unsigned short pair[kMaxPairs];  // pairs by expert
    unsigned short rank[kMaxPairs];
    int count[kMaxExperts];
    int uslot[kMaxExperts];         // slots of the experts that have pairs
    unsigned short uoff[kMaxExperts + 1];
    int scan[kWarps];
    int n;                          // how many
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_async_ca(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1, const float (&c)[4]) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, "
        "%12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Power of two that brings values whose largest has the fp32 exponent field
// `e` into fp16, the largest in [2^14, 2^15), and its reciprocal.  e is held
// to [15, 254].
__device__ __forceinline__ int half_exponent(uint32_t e) { return min(max((int)e, 15), 254); }
__device__ __forceinline__ float half_back(int e) { return __uint_as_float((uint32_t)(e - 14) << 23); }  // 2^(e - 141)
__device__ __forceinline__ void half_scale(uint32_t field, float &to_half, float &back) {
    const int e = half_exponent(field);
    to_half = __uint_as_float((uint32_t)(268 - e) << 23);  // 2^(141 - e)
    back = half_back(e);
}
// Where the exponent of the group of 8 intermediate values 8 g .. lies in its
// pair's row: the four of a thread's columns in a stage of 128 are one word.
__device__ __forceinline__ int exp_at(int g) { return (g & ~15) | ((g & 3) << 2) | ((g >> 2) & 3); }
__device__ __forceinline__ uint32_t bf16x2_to_f16x2(uint32_t v, float s) {
    const __half2 h = __floats2half2_rn(bf16lo(v) * s, bf16hi(v) * s);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// ---- phase R ------------------------------------------------------------------
constexpr int kAhead = 8;  // 16-byte loads of a lane in flight

__device__ void convert_token(const MoeArgs &a, int t, int lane) {
    const __nv_bfloat16 *row = a.x + t * a.x_stride;
    uint32_t m = 0;
    for (int h0 = lane * 8; h0 < a.H; h0 += 256 * kAhead) {
        uint4 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            v[i] = h0 + i * 256 < a.H ? ld_cached16(row + h0 + i * 256) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) m = max(m, max((w[j] << 16) & 0x7FFFFFFFu, w[j] & 0x7FFF0000u));
        }
    }
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    float s, back;
    half_scale(m >> 23, s, back);
    for (int h = lane * 8; h < a.H; h += 256) {
        uint4 v = ld_cached16(row + h);
        v.x = bf16x2_to_f16x2(v.x, s), v.y = bf16x2_to_f16x2(v.y, s);
        v.z = bf16x2_to_f16x2(v.z, s), v.w = bf16x2_to_f16x2(v.w, s);
        *reinterpret_cast<uint4 *>(a.xs + (size_t)t * a.H + h) = v;
    }
    if (lane == 0) a.x_scale[t] = back;
}

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

// Top-k of token t by (logit descending, id ascending), softmax weights.
template <int PER_LANE>
__device__ void route_token(const MoeArgs &a, Lists &L, int t, int lane) {
    uint32_t key[PER_LANE];
#pragma unroll
    for (int i = 0; i < PER_LANE; ++i) {
        const int e = i * 32 + lane;
        key[i] = e < a.E ? key_of(__ldcg(a.logits + (size_t)t * a.E + e)) : 0;
    }
    float mx = 0.f, all = 0.f, mine = 0.f;
    int my_id = -1;
    for (int j = 0; j < a.k; ++j) {
        uint32_t best = 0;
        int id = 0;
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (key[i] > best) best = key[i], id = i * 32 + lane;
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        const unsigned who = __ballot_sync(0xFFFFFFFFu, best == top);
        if (who & (who - 1))  // equal logits: the lowest id
            id = (int)__reduce_min_sync(0xFFFFFFFFu, best == top ? (uint32_t)id : 0x7FFFFFFFu);
        else
            id = __shfl_sync(0xFFFFFFFFu, id, __ffs(who) - 1);
        if (j == 0) {
            mx = logit_of(top);
            if (!a.renormalize) {
#pragma unroll
                for (int i = 0; i < PER_LANE; ++i)
                    if (key[i]) all += expf(logit_of(key[i]) - mx);
            }
        }
#pragma unroll
        for (int i = 0; i < PER_LANE; ++i)
            if (i * 32 + lane == id) key[i] = 0;
        if (lane == j) mine = logit_of(top), my_id = id;
    }
    const float p = lane < a.k ? expf(mine - mx) : 0.f;
    const float sum = warp_sum(a.renormalize ? p : all);
    if (lane < a.k) {
        L.ids[t * a.k + lane] = my_id;
        L.w[t * a.k + lane] = p / sum;
    }
}

// The caller's routing of token t; an expert named twice is taken once, with
// the sum of its weights.
__device__ void given_token(const MoeArgs &a, Lists &L, int t) {
    for (int j = 0; j < a.k; ++j) {
        const int p = t * a.k + j;
        const long long e = load_id64(a.ids, a.ids64, p);
        int id = e < 0 || e >= a.E ? -1 : (int)e;
        for (int i = 0; i < j && id >= 0; ++i)
            if (L.ids[t * a.k + i] == id) {
                L.w[t * a.k + i] += a.weights[p];
                id = -1;
            }
        L.ids[p] = id;
        L.w[p] = a.weights[p];
    }
}

// Pairs by expert, experts with a slot in ascending order.  (The order of an
// expert's pairs is not fixed: each is a column of its own.)
__device__ void build_lists(const MoeArgs &a, Lists &L) {
    const int P = a.T * a.k, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    for (int p = tid; p < P; p += kThreads) {
        const int e = L.ids[p];
        L.rank[p] = (unsigned short)(e >= 0 ? atomicAdd(&L.count[e], 1) : 0);
    }
    __syncthreads();
    int count[2], slot[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = tid * 2 + i;
        count[i] = e < a.E ? L.count[e] : 0;
        if (!count[i]) continue;
        slot[i] = a.expert_map ? a.expert_map[e] : e;
        if (slot[i] < 0 || slot[i] >= a.slots) count[i] = 0;
    }
    // pairs in the low half, experts in the high half
    const int own = count[0] + count[1] + (((count[0] > 0) + (count[1] > 0)) << 16);
    int run = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, run, o);
        if (lane >= o) run += v;
    }
    if (lane == 31) L.scan[warp] = run;
    __syncthreads();
    int before = run - own, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        const int v = L.scan[w];
        if (w < warp) before += v;
        total += v;
    }
    int pos = before & 0xFFFF, u = before >> 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int e = tid * 2 + i;
        if (e < a.E) L.count[e] = count[i] ? pos : -1;  // from here on: where the expert's pairs begin
        if (!count[i]) continue;
        L.uslot[u] = slot[i];
        L.uoff[u++] = (unsigned short)pos;
        pos += count[i];
    }
    if (tid == 0) {
        L.n = total >> 16;
        L.uoff[total >> 16] = (unsigned short)(total & 0xFFFF);
    }
    __syncthreads();
    for (int p = tid; p < P; p += kThreads) {
        const int e = L.ids[p], at = e >= 0 ? L.count[e] : -1;
        if (at >= 0) L.pair[at + L.rank[p]] = (unsigned short)p;
    }
    __syncthreads();
}

// ---- the weight stream of a warp ------------------------------------------------
// 16 rows: 8 from `a` on and 8 from `b` on, row_bytes apart; their scale bytes
// from `sa` and `sb` on, blocks apart.
struct Source {
    const uint8_t *a, *b, *sa, *sb;
};
// 16-byte piece (row r of 16, block b of the stage): swizzled, so that the
// words that 8 rows' lanes read together lie in different banks.
__device__ __forceinline__ uint32_t piece_at(int r, int b) {
    return (uint32_t)(r * kRowBytes + (((b ^ r) & 7) << 4) + (b & ~7) * 16);
}

__device__ __forceinline__ void issue_chunk(uint32_t slot, const Source &src, int c, int blocks, int lane) {
    constexpr int kPerPass = 32 / kRowBlocks;  // rows of one instruction
    const int b = lane % kRowBlocks, r0 = lane / kRowBlocks;
    const bool valid = c * kRowBlocks + b < blocks;
    const int64_t row_bytes = blocks * 16;
    const uint8_t *pa = src.a + r0 * row_bytes + (valid ? c * kRowBytes + b * 16 : 0);
    const uint8_t *pb = src.b + r0 * row_bytes + (valid ? c * kRowBytes + b * 16 : 0);
#pragma unroll
    for (int i = 0; i < 8 / kPerPass; ++i) {
        cp_async16(slot + piece_at(r0 + i * kPerPass, b), pa + i * kPerPass * row_bytes, valid);
        cp_async16(slot + piece_at(8 + r0 + i * kPerPass, b), pb + i * kPerPass * row_bytes, valid);
    }
    if (lane < 16) {
        const uint32_t at = slot + kCodeBytes + lane * kRowBlocks;
        const uint8_t *s = (lane < 8 ? src.sa : src.sb) + (lane & 7) * blocks + c * kRowBlocks;
        if (blocks % kRowBlocks == 0) {
            cp_async_ca<kRowBlocks>(at, s);
        } else {  // the rows' scale bytes are not aligned, or end within the stage
#pragma unroll
            for (int w = 0; w < kRowBlocks / 4; ++w) {
                uint32_t v = 0;
                for (int i = 0; i < 4; ++i)
                    if (c * kRowBlocks + w * 4 + i < blocks) v |= (uint32_t)s[w * 4 + i] << (8 * i);
                asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + w * 4), "r"(v) : "memory");
            }
        }
    }
}

// Byte i of w as an exponent field: 2^(byte - 127), 0 for byte 0 (a block of
// zeros).  Two instructions; the special values of scale_value() cost as much
// as the rest of a block's arithmetic (246 cycles a stage against 132), so a
// NaN (255) is looked for once a word instead (nan_bytes).
template <int I>
__device__ __forceinline__ float scale_bits(uint32_t w) {
    return __uint_as_float((I < 3 ? w << (23 - 8 * I) : w >> 1) & 0x7F800000u);
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return (~w - 0x01010101u) & w & 0x80808080u; }

// acc[nt] += rows of the stage times the columns of token tile nt, 128 columns
// from 128 h on.  `take(nt, b)`: eight fp16 activations of this lane's token,
// columns 32 b + 8 (lane % 4) of them on.
template <int NT, class TakeB>
__device__ __forceinline__ void chunk_mma(uint32_t slot, int h, int lane, float (&acc)[NT][4], uint32_t (&nan)[2], TakeB take) {
    const int r = lane >> 2, t = lane & 3;
    const uint32_t sc = slot + kCodeBytes + r * kRowBlocks + h * 4;
    const uint32_t sa = lds32(sc), sb = lds32(sc + 8 * kRowBlocks);
    nan[0] |= nan_bytes(sa), nan[1] |= nan_bytes(sb);
    uint32_t wa[4], wb[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const uint32_t at = slot + piece_at(r, h * 4 + b) + t * 4;
        wa[b] = lds32(at), wb[b] = lds32(at + 8 * kRowBytes);
    }
    const float fa[4] = {scale_bits<0>(sa), scale_bits<1>(sa), scale_bits<2>(sa), scale_bits<3>(sa)};
    const float fb[4] = {scale_bits<0>(sb), scale_bits<1>(sb), scale_bits<2>(sb), scale_bits<3>(sb)};
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        uint32_t ha[4], hb[4];
        e2m1x8_to_f16(wa[b], ha);
        e2m1x8_to_f16(wb[b], hb);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint4 x = take(nt, b);
            const float zero[4] = {};
            float d[4];
            mma_f16(d, ha[0], hb[0], ha[1], hb[1], x.x, x.y, zero);
            mma_f16(d, ha[2], hb[2], ha[3], hb[3], x.z, x.w, d);
            acc[nt][0] = fmaf(fa[b], d[0], acc[nt][0]), acc[nt][1] = fmaf(fa[b], d[1], acc[nt][1]);
            acc[nt][2] = fmaf(fb[b], d[2], acc[nt][2]), acc[nt][3] = fmaf(fb[b], d[3], acc[nt][3]);
        }
    }
}
// Rows that met a NaN scale.
template <int NT>
__device__ __forceinline__ void mark_nan(float (&acc)[NT][4], const uint32_t (&nan)[2]) {
    if (!(nan[0] | nan[1])) return;
    // a row's four lanes read the same scale bytes
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (nan[i >> 1]) acc[nt][i] = NAN;
}

// Eight fp16 activations of the c-th 128 columns, or zeros behind the last column.
__device__ __forceinline__ uint4 load_b(const __half *row, int c, int b, int blocks) {
    return c * 4 + b < blocks ? *reinterpret_cast<const uint4 *>(row + c * kSub + b * 32)
                              : make_uint4(0, 0, 0, 0);
}

// Ring of a warp: stage i of the stream lies in slot i % kStages.
struct Ring {
    uint32_t base;
    int issued, taken;
    __device__ __forceinline__ uint32_t slot(int i) const { return base + (uint32_t)(i % kStages) * kStageBytes; }
};

__global__ void __launch_bounds__(kThreads, 1) moe_kernel(const MoeArgs a) {
    extern __shared__ __align__(16) unsigned char smem[];
    Lists &L = *reinterpret_cast<Lists *>(smem);
    unsigned char *rings = smem + (sizeof(Lists) + 15) / 16 * 16;
    float *sums = reinterpret_cast<float *>(rings + kWarps * kStages * kStageBytes);  // [kWarps][T][16]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int nw = gridDim.x * kWarps, gw = blockIdx.x * kWarps + warp;
    const int P = a.T * a.k;

    // R
    for (int i = blockIdx.x * kThreads + tid; i < P; i += gridDim.x * kThreads) a.act_max[i] = 0;
    for (int t = nw - 1 - gw; t < a.T; t += nw) convert_token(a, t, lane);
    if (a.router) {
        if (a.E * a.T <= nw)  // a warp for each product
            route_products<1>(a, gw, nw, lane);
        else
            route_products<4>(a, gw, nw, lane);
    }
    for (int e = tid; e < a.E; e += kThreads) L.count[e] = 0;
    cg::this_grid().sync();

    // S
    if (a.router) {
        for (int t = warp; t < a.T; t += kWarps) {
            if (a.E <= 128)
                route_token<4>(a, L, t, lane);
            else if (a.E <= 256)
                route_token<8>(a, L, t, lane);
            else
                route_token<32>(a, L, t, lane);
        }
    } else if (tid < a.T) {
        given_token(a, L, tid);
    }
    __syncthreads();
    build_lists(a, L);
    const int U = L.n;

    Ring ring{(uint32_t)__cvta_generic_to_shared(rings) + warp * kStages * kStageBytes, 0, 0};
    const int r = lane >> 2, tcol = lane & 3;

    // G: unit u = (expert u / JT, intermediate values 8 (u % JT) ..)
    {
        const int JT = a.I / 8, chunks = (a.H + kChunk - 1) / kChunk, blocks = a.H / kBlock;
        const int64_t N = (int64_t)U * JT;
        const int lo = (int)(N * blockIdx.x / gridDim.x), hi = (int)(N * (blockIdx.x + 1) / gridDim.x);
        const int64_t row_bytes = a.H / 2;
        int pu = lo + warp, pc = 0;  // next chunk to issue
        Source src{};
        auto issue = [&] {
            if (pu < hi) {
                if (pc == 0) {
                    const int ue = pu / JT, j = (pu - ue * JT) * 8;
                    const int64_t base = (int64_t)L.uslot[ue] * 2 * a.I;
                    src.a = a.w13 + (base + j) * row_bytes;
                    src.b = src.a + a.I * row_bytes;
                    src.sa = a.s13 + (base + j) * blocks;
                    src.sb = src.sa + (int64_t)a.I * blocks;
                }
                issue_chunk(ring.slot(ring.issued), src, pc, blocks, lane);
                if (++pc == chunks) pc = 0, pu += kWarps;
            }
            ++ring.issued;
            cp_async_commit();
        };
        for (int i = 0; i < kStages - 1; ++i) issue();
        // the first token tile's activations are loaded a stage ahead, across units
        auto token_row = [&](int ue, int nt) {
            const int off = L.uoff[ue], n = L.uoff[ue + 1] - off;
            return (uint32_t)(L.pair[off + min(nt * 8 + r, n - 1)] / a.k) * a.H + tcol * 8;
        };
        uint4 ahead[4];
        if (lo + warp < hi) {
            const uint32_t row = token_row((lo + warp) / JT, 0);
#pragma unroll
            for (int b = 0; b < 4; ++b) ahead[b] = load_b(a.xs + row, 0, b, blocks);
        }
        auto unit = [&](auto tiles, int ue, int j0, int next_ue) {
            constexpr int NT = decltype(tiles)::value;
            const int off = L.uoff[ue], n = L.uoff[ue + 1] - off;
            float acc[NT][4] = {};
            uint32_t nan[2] = {};
            uint32_t xrow[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) xrow[nt] = token_row(ue, nt);
            const uint32_t next_row = token_row(next_ue, 0);
            for (int c = 0; c < chunks; ++c) {
                cp_async_wait<kStages - 2>();
                __syncwarp();
                issue();
                const uint32_t slot = ring.slot(ring.taken++);
#pragma unroll 1
                for (int h = 0; h < kChunk / kSub; ++h) {
                    const int k = c * (kChunk / kSub) + h;
                    const bool last = (k + 1) * 4 >= blocks;
                    const uint32_t ahead_row = last ? next_row : xrow[0];
                    const int ahead_k = last ? 0 : k + 1;
                    chunk_mma<NT>(slot, h, lane, acc, nan, [&](int nt, int b) {
                        if (nt) return load_b(a.xs + xrow[nt], k, b, blocks);
                        const uint4 v = ahead[b];
                        ahead[b] = load_b(a.xs + ahead_row, ahead_k, b, blocks);
                        return v;
                    });
                    if (last) break;
                }
            }
            mark_nan<NT>(acc, nan);
            const int j = j0 + r;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int q = nt * 8 + tcol * 2 + i;
                    const int p = L.pair[off + min(q, n - 1)];
                    const float xs = a.x_scale[p / a.k];
                    const float g = acc[nt][i] * xs, u = acc[nt][2 + i] * xs;
                    const float v = g / (1.f + __expf(-g)) * u;
                    // the 8 lanes that share lane % 4 hold 8 intermediate values of the pair
                    uint32_t m = __float_as_uint(v) & 0x7FFFFFFFu;
                    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 4));
                    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 8));
                    m = max(m, __shfl_xor_sync(0xFFFFFFFFu, m, 16));
                    if (q >= n) continue;
                    float to_half, back;
                    half_scale(m >> 23, to_half, back);
                    a.act[(size_t)p * a.I + j] = __float2half_rn(v * to_half);
                    if (r == 0) {
                        const int e = half_exponent(m >> 23);
                        a.act_exp[(size_t)p * a.exp_stride + exp_at(j0 >> 3)] = (uint8_t)e;
                        atomicMax(a.act_max + p, (uint32_t)e);
                    }
                }
        };
        for (int u = lo + warp; u < hi; u += kWarps) {
            const int ue = u / JT, j0 = (u - ue * JT) * 8, n = L.uoff[ue + 1] - L.uoff[ue];
            const int next = u + kWarps < hi ? (u + kWarps) / JT : ue;
            if (n <= 8)
                unit(std::integral_constant<int, 1>(), ue, j0, next);
            else if (n <= 16)
                unit(std::integral_constant<int, 2>(), ue, j0, next);
            else if (n <= 32)
                unit(std::integral_constant<int, 4>(), ue, j0, next);
            else
                unit(std::integral_constant<int, 8>(), ue, j0, next);
        }
        cp_async_wait<0>();
        __syncwarp();
    }

    // D: tile = 16 rows of the hidden size; unit v = (expert v / segs, piece v % segs of I)
    {
        const int tiles = a.H / 16, chunks = (a.I + kChunk - 1) / kChunk, blocks = a.I / kBlock;
        // at least four units a warp, where I has the chunks for it
        const int segs = U ? max(1, min(chunks, (2 * kWarps + U - 1) / U)) : 1;
        const int V = U * segs;
        const int64_t row_bytes = a.I / 2;
        float *mine = sums + warp * a.T * 16;
        for (int i = lane; i < a.T * 16; i += 32) mine[i] = 0.f;
        ring.issued = ring.taken = 0;
        int ptile = blockIdx.x, pv = warp, pc = 0, pend = 0;
        if (pv >= V) ptile = tiles;
        Source src{};
        bool fresh = true;
        auto issue = [&] {
            if (ptile < tiles) {
                if (fresh) {
                    const int ue = pv / segs, seg = pv - ue * segs;
                    pc = seg * chunks / segs, pend = (seg + 1) * chunks / segs;
                    const int64_t row = (int64_t)L.uslot[ue] * a.H + ptile * 16;
                    src.a = a.w2 + row * row_bytes;
                    src.b = src.a + 8 * row_bytes;
                    src.sa = a.s2 + row * blocks;
                    src.sb = src.sa + 8 * blocks;
                    fresh = false;
                }
                issue_chunk(ring.slot(ring.issued), src, pc, blocks, lane);
                if (++pc == pend) {
                    fresh = true;
                    pv += kWarps;
                    if (pv >= V) pv = warp, ptile += gridDim.x;
                }
            }
            ++ring.issued;
            cp_async_commit();
        };
        for (int i = 0; i < kStages - 1; ++i) issue();
        cg::this_grid().sync();
        // the first token tile's activations are loaded a stage ahead, across units
        auto pair_of = [&](int ue, int nt) {
            const int off = L.uoff[ue], n = L.uoff[ue + 1] - off;
            return (int)L.pair[off + min(nt * 8 + r, n - 1)];
        };
        auto load_exp = [&](int p, int c) {
            return *reinterpret_cast<const uint32_t *>(a.act_exp + (size_t)p * a.exp_stride + c * 16 + tcol * 4);
        };
        // to the pair's common scale: groups 2^24 below the largest vanish
        auto common = [&](uint4 v, uint32_t exps, int b, int top) {
            const float f = __uint_as_float((uint32_t)max(127 - max(top - (int)((exps >> (8 * b)) & 255), 0), 0) << 23);
            const __half2 s = __floats2half2_rn(f, f);
            __half2 h[4];
            memcpy(h, &v, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = __hmul2(h[i], s);
            memcpy(&v, h, 16);
            return v;
        };
        uint4 ahead[4];
        uint32_t ahead_exp = 0;
        if (V > warp && blockIdx.x < tiles) {
            const int ue = warp / segs, p = pair_of(ue, 0);
            const int c = (warp - ue * segs) * chunks / segs * (kChunk / kSub);
            ahead_exp = load_exp(p, c);
#pragma unroll
            for (int b = 0; b < 4; ++b) ahead[b] = load_b(a.act + (uint32_t)p * a.I + tcol * 8, c, b, blocks);
        }
        auto unit = [&](auto tiles_, int ue, int seg, int next_ue, int next_c) {
            constexpr int NT = decltype(tiles_)::value;
            const int off = L.uoff[ue], n = L.uoff[ue + 1] - off;
            float acc[NT][4] = {};
            uint32_t nan[2] = {};
            int pr[NT], top[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                pr[nt] = pair_of(ue, nt);
                top[nt] = (int)a.act_max[pr[nt]];
            }
            const int next_p = pair_of(next_ue, 0);
            const int end = (seg + 1) * chunks / segs;
            for (int c = seg * chunks / segs; c < end; ++c) {
                cp_async_wait<kStages - 2>();
                __syncwarp();
                issue();
                const uint32_t slot = ring.slot(ring.taken++);
#pragma unroll 1
                for (int h = 0; h < kChunk / kSub; ++h) {
                    const int k = c * (kChunk / kSub) + h;
                    const bool done = (k + 1) * 4 >= blocks, last = done || (h + 1 == kChunk / kSub && c + 1 == end);
                    const int ahead_p = last ? next_p : pr[0], ahead_k = last ? next_c * (kChunk / kSub) : k + 1;
                    uint32_t exps[NT];
                    exps[0] = ahead_exp;
                    ahead_exp = load_exp(ahead_p, ahead_k);
#pragma unroll
                    for (int nt = 1; nt < NT; ++nt) exps[nt] = load_exp(pr[nt], k);
                    chunk_mma<NT>(slot, h, lane, acc, nan, [&](int nt, int b) {
                        if (nt)
                            return common(load_b(a.act + (uint32_t)pr[nt] * a.I + tcol * 8, k, b, blocks), exps[nt], b,
                                          top[nt]);
                        const uint4 v = common(ahead[b], exps[0], b, top[0]);
                        ahead[b] = load_b(a.act + (uint32_t)ahead_p * a.I + tcol * 8, ahead_k, b, blocks);
                        return v;
                    });
                    if (done) break;
                }
            }
            mark_nan<NT>(acc, nan);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int q = nt * 8 + tcol * 2 + i;
                    if (q >= n) continue;
                    const int p = L.pair[off + q];
                    const float back = half_back((int)a.act_max[p]) * L.w[p];
                    float *at = mine + (p / a.k) * 16 + r;
                    at[0] = fmaf(acc[nt][i], back, at[0]);
                    at[8] = fmaf(acc[nt][2 + i], back, at[8]);
                }
            __syncwarp();
        };
        for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            for (int v = warp; v < V; v += kWarps) {
                const int ue = v / segs, seg = v - ue * segs, n = L.uoff[ue + 1] - L.uoff[ue];
                const int nv = v + kWarps < V ? v + kWarps : warp;  // the next tile's units are the same
                const int next = nv / segs, next_c = (nv - next * segs) * chunks / segs;
                if (n <= 8)
                    unit(std::integral_constant<int, 1>(), ue, seg, next, next_c);
                else if (n <= 16)
                    unit(std::integral_constant<int, 2>(), ue, seg, next, next_c);
                else if (n <= 32)
                    unit(std::integral_constant<int, 4>(), ue, seg, next, next_c);
                else
                    unit(std::integral_constant<int, 8>(), ue, seg, next, next_c);
            }
            __syncthreads();
            for (int i = tid; i < a.T * 16; i += kThreads) {
                float s = 0.f;
                for (int w = 0; w < kWarps; ++w) {
                    s += sums[w * a.T * 16 + i];
                    sums[w * a.T * 16 + i] = 0.f;
                }
                a.out[(size_t)(i >> 4) * a.H + tile * 16 + (i & 15)] = __float2bfloat16_rn(s);
            }
            __syncthreads();
        }
        cp_async_wait<0>();
    }
}

size_t align16(size_t v) { return (v + 15) / 16 * 16; }
constexpr int exp_stride(int I) { return (I + kSub - 1) / kSub * 16; }
struct Workspace {
    size_t logits, xs, x_scale, act, act_exp, act_max, bytes;
    Workspace(int T, int E, int k, int H, int I) {
        size_t at = 0;
        const auto take = [&](size_t n) { const size_t here = at; at += (n + 255) / 256 * 256; return here; };
        logits = take((size_t)T * E * 4);
        xs = take((size_t)T * H * 2);
        x_scale = take((size_t)T * 4);
        act = take((size_t)T * k * I * 2);
        act_exp = take((size_t)T * k * exp_stride(I));
        act_max = take((size_t)T * k * 4);
        bytes = at;
    }
};
size_t smem_bytes(int T) {
    return align16(sizeof(Lists)) + (size_t)kWarps * kStages * kStageBytes + (size_t)kWarps * T * 16 * sizeof(float);
}

int check_shape(int32_t T, int32_t E, int32_t k, int32_t H, int32_t I, int32_t slots) {
    if (T < 0 || T > kMaxTokens || E < 1 || E > kMaxExperts || k < 1 || k > kMaxTopK || k > E || slots < 1)
        return set_error("wisp_mx4_moe: need at most 64 tokens, 1024 experts, 1 <= top_k <= min(16, experts)"),
               WISP_ERR_INVALID;
    if (H < 32 || H % 32 || H > 32768 || I < 32 || I % 32 || I > 65536)
        return set_error("wisp_mx4_moe: hidden and intermediate sizes are multiples of 32, at most 32768 and 65536"),
               WISP_ERR_INVALID;
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
                            int32_t num_slots, int32_t num_tokens, int32_t num_experts, int32_t top_k, int32_t hidden,
                            int32_t inter, int32_t renormalize, void *workspace, int64_t workspace_bytes, void *out,
                            void *stream) {
    if (const int rc = check_shape(num_tokens, num_experts, top_k, hidden, inter, num_slots)) return rc;
    if (num_tokens == 0) return WISP_OK;
    if (!x || !w13_codes || !w13_scales || !w2_codes || !w2_scales || !workspace || !out)
        return set_error("wisp_mx4_moe: NULL tensor"), WISP_ERR_INVALID;
    if (router ? topk_ids || topk_weights : !topk_ids || !topk_weights)
        return set_error("wisp_mx4_moe: give either the router's weights or ids and weights"), WISP_ERR_INVALID;
    if (!expert_map && num_slots < num_experts)
        return set_error("wisp_mx4_moe: fewer slots than experts, and no expert map"), WISP_ERR_INVALID;
    for (const void *p : {x, router, w13_codes, w2_codes, (const void *)workspace})
        if (reinterpret_cast<uintptr_t>(p) % 16)
            return set_error("wisp_mx4_moe: x, router, codes and workspace must be aligned to 16 bytes"),
                   WISP_ERR_INVALID;
    for (const void *p : {w13_scales, w2_scales})
        if (reinterpret_cast<uintptr_t>(p) % 4)
            return set_error("wisp_mx4_moe: scales must be aligned to 4 bytes"), WISP_ERR_INVALID;
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
    a.w13 = reinterpret_cast<const uint8_t *>(w13_codes);
    a.s13 = reinterpret_cast<const uint8_t *>(w13_scales);
    a.w2 = reinterpret_cast<const uint8_t *>(w2_codes);
    a.s2 = reinterpret_cast<const uint8_t *>(w2_scales);
    a.out = reinterpret_cast<__nv_bfloat16 *>(out);
    a.logits = reinterpret_cast<float *>(ws + w.logits);
    a.xs = reinterpret_cast<__half *>(ws + w.xs);
    a.x_scale = reinterpret_cast<float *>(ws + w.x_scale);
    a.act = reinterpret_cast<__half *>(ws + w.act);
    a.act_exp = ws + w.act_exp;
    a.exp_stride = exp_stride(inter);
    a.act_max = reinterpret_cast<uint32_t *>(ws + w.act_max);
    a.T = num_tokens, a.E = num_experts, a.k = top_k, a.H = hidden, a.I = inter, a.slots = num_slots;
    a.ids64 = ids_int64, a.renormalize = renormalize;
    int dev = 0, sms = 0;
    WISP_CUDA_TRY(cudaGetDevice(&dev));
    WISP_CUDA_TRY(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    const size_t smem = smem_bytes(num_tokens);
    WISP_CUDA_TRY(cudaFuncSetAttribute(moe_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       (int)smem_bytes(kMaxTokens)));
    void *params[] = {&a};
    WISP_CUDA_TRY(cudaLaunchCooperativeKernel(reinterpret_cast<const void *>(moe_kernel), dim3(sms), dim3(kThreads),
                                              params, smem, reinterpret_cast<cudaStream_t>(stream)));
    return WISP_OK;
}
