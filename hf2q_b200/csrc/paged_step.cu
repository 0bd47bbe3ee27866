// Attention over a paged cache for few rows of a sequence at a time: single tokens, drafted tokens.
//
// Bound by memory: keys and values of a position are read once for all query heads of their KV head and for a tile of up to 16 rows
// (rows of a sequence times heads of the group), and there are 4 flops a byte and row.  A CTA takes a tile, a KV head and a part of the
// positions, and each of its warps 16 positions at a time, straight from global memory to registers: pages of 16 and more mean that
// one page number serves the step.  Scores and weighted values run on m16n8k16 with N = 8 rows of the tile, transposed:
//
//   scores   S^T = K Q^T, M = 16 positions.  The order of the contraction over a head's elements is free, so that a lane takes whole
//            16-byte units of a key and reads the query's elements in the order that this gives;
//   values   O^T = V^T P^T, M = 16 elements of the head: the same element of two neighbouring positions, picked from two 16-byte units with
//            byte permutations.  P^T is S^T's accumulator, rounded to 16 bits and transposed by movmatrix.
//
// (With the rows as M half of every product is empty for 8 rows and fewer, and each accumulator pair is moved into a group of four.)
// Codes of keys enter as f16 subnormals, (code + 128) 2^-24, and 128 times the sum of q is taken off again; codes of values as f16 whole
// numbers.  Their weights are p * v_scale * 256 / U with U a power of two above all value scales of the warp's steps so far, which
// keeps them inside the f16 range whatever the scales are; below its normal numbers p * v_scale is off by at most 2^-32 of the largest
// value scale.  Loads of the next step are under way while this step's products run: the
// next keys once the scores are done, the next values once the values are.
//
// Roundings.  The matrix instructions take 16-bit operands, so queries in f32 and the weights above the fraction are rounded to the type of their
// product: f16 beside codes, bf16 beside bf16 pages (2^-11 and 2^-8 of each number at most).  The weights' sum below it, maxima and outputs
// stay in f32.  Against 64 bits, root of the mean square over that of the result: bf16 pages and result 0.0021 to 0.0023, where the result's own rounding
// makes 0.0017; codes and f16 result 0.0003, of which 0.0002; codes and bf16 result 0.0017, all of it.  Weights in two 16-bit halves would double the
// products with the values to take off that last third.
//
// Measured (32 query heads of 8 KV heads, dim 128): one token behind 131071 positions of codes 57 us, 4.8 TB/s, of bf16 90 us, 5.9 TB/s; one token of each of 32
// sequences of up to 8192 positions of codes 81 us, 3.9 TB/s, of bf16 126 us, 4.8 TB/s (the parts are as long as the longest sequence wants them, the
// others end early); with the rows as M codes were 95 and 122 us.  One token behind 200 positions 6.2 us, of which the launch and the chain page
// number - key - score - value are nearly all.
#include <math_constants.h>

#include <type_traits>

#include "paged_bits.cuh"
#include "paged_common.cuh"
#include "tc_common.cuh"

namespace hf2q {
using namespace paged;
namespace {

constexpr uint32_t WARPS = 8, STEP_LOG = 4, STEP = 16;
constexpr float ROOM = 7.0f, UNITS = 256.0f;       // weights in f16 stay below 2^7 * 256 = 2^15

__device__ __forceinline__ uint4 load16(const void* p) { return __ldcg(static_cast<const uint4*>(p)); }

template <bool CODES>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (CODES)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// rows and columns of an 8 x 8 matrix of 16-bit numbers exchanged: lane 4 r + t holds columns 2 t, 2 t + 1 of row r
__device__ __forceinline__ uint32_t transposed(uint32_t a) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ float2 half_pair(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

template <int DIM, bool CODES, bool TALL>
constexpr uint32_t step_smem() { return WARPS * (TALL ? 16 : 8) * (DIM + 4) * 4; }

// TALL: tiles of 16 rows, else of 8.  The tile's rows are u = token * group + head of the sequence's new tokens and the KV head's query heads.
template <int DIM, bool CODES, bool TALL, typename Q, typename OUT>
__global__ void __launch_bounds__(WARPS * 32, step_ctas(DIM, CODES, TALL))
attend_step_kernel(Pool c, Batch b, Look look, uint32_t heads, uint32_t group, const Q* q, uint32_t ldq, bool wide_q, OUT* out, uint32_t ldo, uint32_t chunk_steps, uint32_t chunks,
                   bool shrink, float* part, float* part_ml, uint32_t* status) {
    constexpr int R = TALL ? 16 : 8, KS = DIM / 16;                       // rows, contraction steps of a score
    constexpr int UE = CODES ? 16 : 8;                                    // elements of a 16-byte unit
    constexpr int KU = DIM / UE / 4;                                      // units of a key row in a lane
    constexpr int VE = CODES && DIM == 64 ? 8 : UE, VU = DIM / 8 / VE;    // elements of a value unit; units of a value row in a lane
    constexpr int VW = VE * (CODES ? 1 : 2) / 4;                          // words of a value unit
    constexpr uint32_t ROW = DIM * (CODES ? 1 : 2);                       // bytes of a key
    extern __shared__ __align__(16) float red[];                          // [WARPS][R][DIM + 4]
    __shared__ float red_m[WARPS][R], red_l[WARPS][R];
    pdl_trigger();
    pdl_wait();
    const uint32_t s = blockIdx.z, kvh = blockIdx.x % c.kv_heads, tile = blockIdx.x / c.kv_heads, chunk = blockIdx.y;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, t = lane & 3;
    const Span span = span_of(b, c.shift, s);
    const uint32_t part_steps = part_units(b, STEP_LOG, chunk_steps, chunks, 8, shrink);
    if (span.bad && threadIdx.x == 0 && blockIdx.x == 0 && chunk == 0) atomicOr(status, STATUS_BAD_PAGE);
    const uint32_t u0 = tile * R, units = span.rows * group;
    if (u0 >= units) return;
    const uint32_t tok0 = u0 / group, tok1 = (min(u0 + R, units) - 1) / group;
    const uint32_t lost = span.rows > span.length ? span.rows - span.length : 0;      // rows in front of position 0: they see nothing
    const uint32_t before = span.length - span.rows;                      // position of token 0 (wraps where rows are lost)
    const bool any = tok1 >= lost;
    const uint32_t first = any ? before + max(tok0, lost) : 0, last = any ? before + tok1 : 0;
    const Blocks blocks = blocks_of(look, first, last, STEP_LOG);
    const uint32_t lo = static_cast<uint32_t>(min(static_cast<uint64_t>(chunk) * part_steps, static_cast<uint64_t>(blocks.count)));
    const uint32_t hi = any ? min(lo + part_steps, blocks.count) : lo;
    if (chunks > 1 && lo >= hi) {                                         // nothing for this part: its sums count for nothing
        for (uint32_t u = u0 + threadIdx.x; u < min(u0 + R, units); u += WARPS * 32)
            *reinterpret_cast<float2*>(part_ml + 2 * (((static_cast<size_t>(span.row0) + u / group) * heads + kvh * group + u % group) * chunks + chunk)) = make_float2(-CUDART_INF_F, 0.f);
        return;
    }
    // rows of this lane in scores and output: 2 t, 2 t + 1 (and 8 more)
    constexpr int NT = TALL ? 2 : 1, LR = 2 * NT;
    uint32_t at[LR];
    bool held[LR];
#pragma unroll
    for (int i = 0; i < LR; ++i) {
        const uint32_t tok = min(u0 + 2 * t + (i & 1) + 8 * (i >> 1), units - 1) / group;
        held[i] = tok >= lost;
        at[i] = before + max(tok, lost);
    }
    float mx[LR], l[LR];
    float o[NT][DIM / 16][4];                                             // elements e(gid, 2 m), e(gid, 2 m + 1) of rows 2 t, 2 t + 1: [0], [1]; [2], [3]
#pragma unroll
    for (int i = 0; i < LR; ++i) { mx[i] = -CUDART_INF_F; l[i] = 0.f; }
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int m = 0; m < DIM / 16; ++m)
#pragma unroll
            for (int x = 0; x < 4; ++x) o[i][m][x] = 0.f;
    bool bad = false, clipped = false;
    float unit = 0x1p-100f, per_unit = 0.f;                               // U, UNITS / U
    // steps that start at full0 .. full0 + full_reach are seen whole by every row (those of the first positions beside a window are not counted here)
    const uint32_t from = look.window && last >= look.window ? last - look.window + 1 : 0;
    const bool some = tok0 >= lost && first >= from + (STEP - 1);
    const uint32_t full0 = some ? from : 1u << 31, full_reach = some ? first - (STEP - 1) - from : 0;

    if (lo + warp < hi) {
        // keys and values first: their page and they themselves are two trips to memory, q one
        uint4 kr[2][KU];
        uint32_t vr[4][VU][VW];
        float ks[2], vs[2];                                               // of positions gid, gid + 8
        const uint8_t *k_at = static_cast<const uint8_t*>(c.k) + gid * ROW + 16 * t, *v_at = static_cast<const uint8_t*>(c.v) + 2 * t * ROW + gid * (VW * 4);
        const float *ks_at = CODES ? c.k_scale + gid : nullptr, *vs_at = CODES ? c.v_scale + gid : nullptr;
        auto place = [&](uint32_t step) {                                 // where the step's positions lie in this head, in sixteens of rows
            const uint32_t p = blocks.at(step) << STEP_LOG;
            return ((page_of(c, b, s, p, bad) * c.kv_heads + kvh) << (c.shift - STEP_LOG)) + ((p & (c.size() - 1)) >> STEP_LOG);
        };
        auto load_k = [&](uint32_t at16) {
            const uint8_t* rows = k_at + static_cast<uint64_t>(at16) * (STEP * ROW);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < KU; ++i) kr[n][i] = load16(rows + 8 * n * ROW + 64 * i);
            if constexpr (CODES) {
                const float* sc = ks_at + static_cast<uint64_t>(at16) * STEP;
                ks[0] = __ldcg(sc);
                ks[1] = __ldcg(sc + 8);
            }
        };
        auto load_v = [&](uint32_t at16) {
            const uint8_t* from = v_at + static_cast<uint64_t>(at16) * (STEP * ROW);
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < VU; ++i) {
                    const uint8_t* here = from + ((x & 1) + 8 * (x >> 1)) * ROW + 8 * i * (VW * 4);
                    if constexpr (VW == 4) { const uint4 w = load16(here); vr[x][i][0] = w.x; vr[x][i][1] = w.y; vr[x][i][2] = w.z; vr[x][i][3] = w.w; }
                    else { const uint2 w = __ldcg(reinterpret_cast<const uint2*>(here)); vr[x][i][0] = w.x; vr[x][i][1] = w.y; }
                }
            if constexpr (CODES) {
                const float* sc = vs_at + static_cast<uint64_t>(at16) * STEP;
                vs[0] = __ldcg(sc);
                vs[1] = __ldcg(sc + 8);
            }
        };
        uint32_t step = lo + warp, here = place(step), next = step + WARPS < hi ? place(step + WARPS) : here;
        load_k(here);
        load_v(here);
        uint32_t qa[NT][KS][2];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const uint32_t u = u0 + gid + 8 * i;
            const Q* row = q + static_cast<size_t>(span.row0 + (u < units ? u / group : 0)) * ldq + (static_cast<size_t>(kvh) * group + (u < units ? u % group : 0)) * DIM;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const uint32_t e0 = CODES ? (4 * (j / 4) + t) * 16 + 4 * (j % 4) : (4 * (j / 2) + t) * 8 + 4 * (j % 2);
                float e[4] = {0.f, 0.f, 0.f, 0.f};
                if (u < units) {
                    if constexpr (std::is_same_v<Q, float>) {
                        if (wide_q) { const float4 f = *reinterpret_cast<const float4*>(row + e0); e[0] = f.x; e[1] = f.y; e[2] = f.z; e[3] = f.w; }
                        else for (int x = 0; x < 4; ++x) e[x] = row[e0 + x];
                    } else {
                        if (wide_q) {
                            const uint2 f = *reinterpret_cast<const uint2*>(row + e0);
                            e[0] = __uint_as_float(f.x << 16); e[1] = __uint_as_float(f.x & 0xffff0000u); e[2] = __uint_as_float(f.y << 16); e[3] = __uint_as_float(f.y & 0xffff0000u);
                        } else for (int x = 0; x < 4; ++x) e[x] = __bfloat162float(row[e0 + x]);
                    }
                    if constexpr (CODES)
                        for (int x = 0; x < 4; ++x) { clipped |= fabsf(e[x]) > 65504.0f; e[x] = fabsf(e[x]) > 65504.0f ? copysignf(65504.0f, e[x]) : e[x]; }
                }
                qa[i][j][0] = pack2<CODES>(e[0], e[1]);
                qa[i][j][1] = pack2<CODES>(e[2], e[3]);
            }
        }
        float q128[LR];                                                   // 128 times what a row of q adds up to: codes enter as code + 128
        if constexpr (CODES) {
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const float2 x = half_pair(qa[i][j][0]), y = half_pair(qa[i][j][1]);
                    sum += (x.x + x.y) + (y.x + y.y);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                for (int x = 0; x < 2; ++x) q128[2 * i + x] = 128.0f * __shfl_sync(0xffffffffu, sum, 4 * (2 * t + x));
            }
        }
#pragma unroll 1
        for (; step < hi; step += WARPS) {
            const uint32_t p0 = blocks.at(step) << STEP_LOG;
            const bool more = step + WARPS < hi, full = p0 - full0 <= full_reach;
            const uint32_t later = step + 2 * WARPS < hi ? place(step + 2 * WARPS) : next;
            // ---- scores: sc[i][2 n + x] of position p0 + gid + 8 n and row 2 t + x + 8 i
            float sc[NT][4];
#pragma unroll
            for (int i = 0; i < NT; ++i) sc[i][0] = sc[i][1] = sc[i][2] = sc[i][3] = 0.f;
#pragma unroll
            for (int i = 0; i < KU; ++i) {
                const uint32_t a[4] = {kr[0][i].x, kr[0][i].y, kr[0][i].z, kr[0][i].w}, e[4] = {kr[1][i].x, kr[1][i].y, kr[1][i].z, kr[1][i].w};
#pragma unroll
                for (int x = 0; x < (CODES ? 4 : 2); ++x) {
                    uint32_t f[4];
                    if constexpr (CODES) {                                // code + 128 in every byte: with a byte of zeros above an f16 of 2^-24 times that
                        const uint32_t y = a[x] ^ 0x80808080u, z = e[x] ^ 0x80808080u;
                        f[0] = __byte_perm(y, 0u, 0x4140u); f[1] = __byte_perm(z, 0u, 0x4140u);
                        f[2] = __byte_perm(y, 0u, 0x4342u); f[3] = __byte_perm(z, 0u, 0x4342u);
                    } else {
                        f[0] = a[(2 * x) & 3]; f[1] = e[(2 * x) & 3]; f[2] = a[(2 * x + 1) & 3]; f[3] = e[(2 * x + 1) & 3];
                    }
#pragma unroll
                    for (int r = 0; r < NT; ++r) mma<CODES>(sc[r], f[0], f[1], f[2], f[3], qa[r][(CODES ? 4 : 2) * i + x][0], qa[r][(CODES ? 4 : 2) * i + x][1]);
                }
            }
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if constexpr (CODES) sc[i][x] = fmaf(sc[i][x], 0x1p24f, -q128[2 * i + (x & 1)]) * (look.scale * ks[x >> 1]);
                    else sc[i][x] *= look.scale;
                }
            if (more) load_k(next);
            // ---- what the rows do not see
            uint32_t seen = 0xffu;                                        // bit 4 i + x, as in sc
            if (!full) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const bool yes = held[2 * i + (x & 1)] && look.sees(at[2 * i + (x & 1)], p0 + gid + 8 * (x >> 1));
                        seen |= static_cast<uint32_t>(yes) << (4 * i + x);
                        if (!yes) sc[i][x] = -CUDART_INF_F;
                    }
            }
            // ---- softmax against the maximum of earlier steps, as long as no score passes it by more than 2^ROOM, and no value scale passes U
            bool change = false;
#pragma unroll
            for (int i = 0; i < LR; ++i) change |= fmaxf(sc[i >> 1][i & 1], sc[i >> 1][2 + (i & 1)]) > mx[i] + ROOM;
            if constexpr (CODES) change |= fmaxf(fabsf(vs[0]), fabsf(vs[1])) >= unit;
            if (__any_sync(0xffffffffu, change)) {
                float corr[LR];
#pragma unroll
                for (int i = 0; i < LR; ++i) {
                    float top = fmaxf(sc[i >> 1][i & 1], sc[i >> 1][2 + (i & 1)]);
                    for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    const float to = fmaxf(mx[i], top);
                    corr[i] = tc::ex2(mx[i] - (to == -CUDART_INF_F ? 0.f : to));
                    mx[i] = to;
                    l[i] *= corr[i];
                }
                if constexpr (CODES) {
                    float large = 0.f;
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        const float a = fabsf(vs[n]);
                        if (a < CUDART_INF_F && (full || some_see(look, first, last, p0 + gid + 8 * n))) large = fmaxf(large, a);
                    }
                    for (int d = 4; d < 32; d <<= 1) large = fmaxf(large, __shfl_xor_sync(0xffffffffu, large, d));
                    const float above = fmaxf(unit, unit_above(large));
#pragma unroll
                    for (int i = 0; i < LR; ++i) corr[i] *= unit / above;
                    unit = above;
                    per_unit = UNITS / above;
                }
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int m = 0; m < DIM / 16; ++m)
#pragma unroll
                        for (int x = 0; x < 4; ++x) o[i][m][x] *= corr[2 * i + (x & 1)];
            }
            float w[NT][4];
            const float v0 = vs[0] * per_unit, v1 = vs[1] * per_unit;
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float top = mx[2 * i + (x & 1)], e = tc::ex2(sc[i][x] - (top == -CUDART_INF_F ? 0.f : top));
                    l[2 * i + (x & 1)] += e;                              // (of this lane's positions; the lanes of a row are added at the end)
                    w[i][x] = CODES ? ((seen >> (4 * i + x)) & 1 ? e * (x >> 1 ? v1 : v0) : 0.f) : e;
                }
            // ---- values
            bool odd = false;                                             // infinities or NaN among values that some of the rows do not see
            if constexpr (!CODES) {
                if (!full) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const bool yes = some_see(look, first, last, p0 + 2 * t + (x & 1) + 8 * (x >> 1));
#pragma unroll
                        for (int i = 0; i < VU; ++i)
#pragma unroll
                            for (int y = 0; y < VW; ++y) {
                                if (!yes) vr[x][i][y] = 0u;
                                odd |= holds_nonfinite(vr[x][i][y]);
                            }
                    }
                    odd = __any_sync(0xffffffffu, odd) && first != last;
                }
            }
            if (!odd) {
                uint32_t b0[NT], b1[NT];
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    b0[i] = transposed(pack2<CODES>(w[i][0], w[i][1]));
                    b1[i] = transposed(pack2<CODES>(w[i][2], w[i][3]));
                }
                auto add = [&](int m, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
#pragma unroll
                    for (int i = 0; i < NT; ++i) mma<CODES>(o[i][m], a0, a1, a2, a3, b0[i], b1[i]);
                };
#pragma unroll
                for (int i = 0; i < VU; ++i)
#pragma unroll
                    for (int y = 0; y < VW; ++y) {
                        const uint32_t va = vr[0][i][y], vb = vr[1][i][y], vc = vr[2][i][y], vd = vr[3][i][y];
                        if constexpr (CODES) {
                            // bytes of the row pairs side by side, then f16 whole numbers of either two
                            const __half2 bias = __float2half2_rn(1152.0f);
                            const uint32_t lo01 = __byte_perm(va, vb, 0x5140u) ^ 0x80808080u, hi01 = __byte_perm(va, vb, 0x7362u) ^ 0x80808080u;
                            const uint32_t lo89 = __byte_perm(vc, vd, 0x5140u) ^ 0x80808080u, hi89 = __byte_perm(vc, vd, 0x7362u) ^ 0x80808080u;
                            const int m = (i * VE + 4 * y) / 2;
                            add(m, tc::h2_bits(tc::codes01(lo01, bias)), tc::h2_bits(tc::codes23(lo01, bias)), tc::h2_bits(tc::codes01(lo89, bias)), tc::h2_bits(tc::codes23(lo89, bias)));
                            add(m + 1, tc::h2_bits(tc::codes01(hi01, bias)), tc::h2_bits(tc::codes23(hi01, bias)), tc::h2_bits(tc::codes01(hi89, bias)), tc::h2_bits(tc::codes23(hi89, bias)));
                        } else {
                            add((i * VE + 2 * y) / 2, __byte_perm(va, vb, 0x5410u), __byte_perm(va, vb, 0x7632u), __byte_perm(vc, vd, 0x5410u), __byte_perm(vc, vd, 0x7632u));
                        }
                    }
            } else if constexpr (!CODES) {
                // 0 times infinity is not 0: each row adds up the positions that it sees, one by one
                const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(c.v) + static_cast<uint64_t>(here) * (STEP * DIM);
#pragma unroll 1
                for (uint32_t p = 0; p < STEP; ++p) {
#pragma unroll
                    for (int i = 0; i < LR; ++i) {
                        const float weight = __shfl_sync(0xffffffffu, p < 8 ? w[i >> 1][i & 1] : w[i >> 1][2 + (i & 1)], 4 * (p & 7) + t);
                        if (held[i] && look.sees(at[i], p0 + p)) {
#pragma unroll
                            for (int e = 0; e < DIM / 8; ++e) {
                                float& to = o[i >> 1][e / 2][2 * (e & 1) + (i & 1)];
                                to = fmaf(weight, __bfloat162float(v[p * DIM + (gid + 8 * (e / VE)) * VE + e % VE]), to);
                            }
                        }
                    }
                }
                __syncwarp();
            }
            if (more) {
                load_v(next);
                here = next;
                next = later;
            }
        }
    }
    // ---- the warps' rows meet in shared memory
    const float back = CODES ? unit * (1.0f / UNITS) : 1.0f;
#pragma unroll
    for (int i = 0; i < LR; ++i) {
        const uint32_t r = 2 * t + (i & 1) + 8 * (i >> 1);
        for (int d = 4; d < 32; d <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], d);
        if (gid == 0) { red_m[warp][r] = mx[i]; red_l[warp][r] = l[i]; }
        float* row = red + (warp * R + r) * (DIM + 4);
#pragma unroll
        for (int e = 0; e < DIM / 8; e += 4) {
            const float (*x)[4] = o[i >> 1] + e / 2;
            *reinterpret_cast<float4*>(row + (gid + 8 * (e / VE)) * VE + e % VE) =
                make_float4(x[0][i & 1] * back, x[0][2 + (i & 1)] * back, x[1][i & 1] * back, x[1][2 + (i & 1)] * back);
        }
    }
    __syncthreads();
    constexpr int LANES = DIM / 4;                                        // threads of a row, four elements each
    for (uint32_t i = threadIdx.x; i < R * LANES; i += WARPS * 32) {
        const uint32_t r = i / LANES, d = 4 * (i % LANES), u = u0 + r;
        if (u >= units) break;
        float m_all = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < static_cast<int>(WARPS); ++w) m_all = fmaxf(m_all, red_m[w][r]);
        float sum = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < static_cast<int>(WARPS); ++w) {
            const float f = part_factor(red_m[w][r], red_l[w][r], m_all);
            if (f == 0.f) continue;
            const float4 v = *reinterpret_cast<const float4*>(red + (w * R + r) * (DIM + 4) + d);
            sum += red_l[w][r] * f;
            a.x += v.x * f; a.y += v.y * f; a.z += v.z * f; a.w += v.w * f;
        }
        const uint32_t tok = u / group, h = kvh * group + u % group;
        const size_t row = span.row0 + tok;
        if (chunks > 1) {
            const size_t at_part = (row * heads + h) * chunks + chunk;
            *reinterpret_cast<float4*>(part + at_part * DIM + d) = a;
            if (d == 0) *reinterpret_cast<float2*>(part_ml + 2 * at_part) = make_float2(m_all, sum);
        } else {
            const float inv = sum == 0.f ? 0.f : 1.0f / sum;
            OUT* to = out + row * ldo + static_cast<size_t>(h) * DIM + d;
            const float v[4] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv};
            __align__(16) OUT e[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) e[x] = out_value<OUT>(v[x], clipped);
            if (reinterpret_cast<uintptr_t>(to) % (4 * sizeof(OUT)) == 0) {
                if constexpr (sizeof(OUT) == 4) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(e);
                else *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(e);
            } else {
                for (int x = 0; x < 4; ++x) to[x] = e[x];
            }
        }
    }
    if (clipped) atomicOr(status, STATUS_X_CLIPPED);
    if (bad) atomicOr(status, STATUS_BAD_PAGE);
}

template <int DIM, bool CODES, bool TALL, typename Q, typename OUT>
cudaError_t launch(const AttendCall& a) {
    constexpr uint32_t smem = step_smem<DIM, CODES, TALL>();
    static PerDeviceFlag flag;
    const auto kern = attend_step_kernel<DIM, CODES, TALL, Q, OUT>;
    if (smem > 48 * 1024)
        if (const cudaError_t e = ensure_max_dynamic_smem(kern, smem, flag); e != cudaSuccess) return e;
    const uint32_t group = a.heads / a.c.kv_heads, R = TALL ? 16 : 8, tiles = static_cast<uint32_t>((static_cast<uint64_t>(a.b.max_new) * group + R - 1) / R);
    const bool wide = reinterpret_cast<uintptr_t>(a.q) % (4 * sizeof(Q)) == 0 && a.ldq % 4 == 0;
    return launch_pdl(kern, dim3(tiles * a.c.kv_heads, a.chunks, a.b.seqs), dim3(WARPS * 32), smem, a.st, a.c, a.b, a.look, a.heads, group, static_cast<const Q*>(a.q), a.ldq, wide,
                      static_cast<OUT*>(a.out), a.ldo, a.chunk >> STEP_LOG, a.chunks, a.shrink, a.part, a.part_ml, a.status);
}
template <int DIM, bool CODES, bool TALL, typename Q>
cudaError_t launch_out(const AttendCall& a) {
    return a.out_dtype == HF2Q_DT_F32 ? launch<DIM, CODES, TALL, Q, float>(a) : a.out_dtype == HF2Q_DT_F16 ? launch<DIM, CODES, TALL, Q, __half>(a) : launch<DIM, CODES, TALL, Q, __nv_bfloat16>(a);
}
template <int DIM, bool CODES>
cudaError_t launch_tall(const AttendCall& a) {
    const bool tall = static_cast<uint64_t>(a.b.max_new) * (a.heads / a.c.kv_heads) > 8;
    if (a.q_dtype == HF2Q_DT_F32) return tall ? launch_out<DIM, CODES, true, float>(a) : launch_out<DIM, CODES, false, float>(a);
    return tall ? launch_out<DIM, CODES, true, __nv_bfloat16>(a) : launch_out<DIM, CODES, false, __nv_bfloat16>(a);
}

}  // namespace

cudaError_t paged::launch_attend_step(const AttendCall& a, uint32_t dim, bool codes) {
    return dim == 128 ? (codes ? launch_tall<128, true>(a) : launch_tall<128, false>(a)) : (codes ? launch_tall<64, true>(a) : launch_tall<64, false>(a));
}

}  // namespace hf2q
