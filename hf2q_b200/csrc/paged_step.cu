// Attention over a paged cache for few rows of a sequence at a time: single tokens, drafted tokens.
//
// Bound by memory: keys and values of a position are read once for all query heads of their KV head and for a tile of up to 16 rows
// (rows of a sequence times heads of the group), and there are 4 flops a byte and row.  A CTA takes a tile, a KV head and a part of the
// positions, and each of its warps 16 positions at a time, straight from global memory to registers: pages of 16 and more mean that
// one page number serves the step.  Scores and weighted values run on m16n8k16 with M = the rows of the tile:
//
//   scores   the order of the contraction over a head's elements is free, so that a lane takes whole 16-byte units of a key
//            and reads the query's elements in the order that this gives;
//   values   the weights go from accumulators to the A operand as they lie; B takes the same element of two neighbouring
//            positions, picked from two 16-byte units with byte permutations.
//
// Codes enter as f16 whole numbers.  Their weights are p * v_scale * 2^12 / U with U a power of two above all value scales of the warp's
// steps so far, which keeps them inside the f16 range whatever the scales are.  Loads of the next step are under way while this
// step's products run: the next keys once the scores are done, the next values once the values are.
#include <math_constants.h>

#include <type_traits>

#include "paged_common.cuh"
#include "tc_common.cuh"

namespace hf2q {
using namespace paged;
namespace {

constexpr uint32_t WARPS = 8, STEP_LOG = 4, STEP = 16;

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
template <bool CODES> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (CODES) return tc::pack_h2(a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ bool holds_nonfinite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }

// a power of two above |v| (v finite), within what 2^12 / U can be
__device__ __forceinline__ float unit_above(float v) {
    const uint32_t e = (__float_as_uint(v) & 0x7f800000u) + 0x00800000u;
    return fminf(fmaxf(__uint_as_float(e), 0x1p-100f), 0x1p100f);
}

template <int DIM, bool CODES, bool TALL>
constexpr uint32_t step_smem() { return WARPS * (TALL ? 16 : 8) * (DIM + 4) * 4; }

// TALL: tiles of 16 rows, else of 8.  The tile's rows are u = token * group + head of the sequence's new tokens and the KV head's query heads.
template <int DIM, bool CODES, bool TALL, typename Q, typename OUT>
__global__ void __launch_bounds__(WARPS * 32, DIM == 64 || (CODES && !TALL) ? 2 : 1)
attend_step_kernel(Pool c, Batch b, Look look, uint32_t heads, uint32_t group, const Q* q, uint32_t ldq, bool wide_q, OUT* out, uint32_t ldo, uint32_t chunk_steps, uint32_t chunks,
                   float* part, float* part_ml, uint32_t* status) {
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
    if (span.bad && threadIdx.x == 0 && blockIdx.x == 0 && chunk == 0) atomicOr(status, STATUS_BAD_PAGE);
    const uint32_t u0 = tile * R, units = span.rows * group;
    if (u0 >= units) return;
    const uint32_t tok0 = u0 / group, tok1 = (min(u0 + R, units) - 1) / group;
    const uint32_t lost = span.rows > span.length ? span.rows - span.length : 0;      // rows in front of position 0: they see nothing
    const uint32_t before = span.length - span.rows;                      // position of token 0 (wraps where rows are lost)
    const bool any = tok1 >= lost;
    const uint32_t first = any ? before + max(tok0, lost) : 0, last = any ? before + tok1 : 0;
    const Blocks blocks = blocks_of(look, first, last, STEP_LOG);
    const uint32_t lo = static_cast<uint32_t>(min(static_cast<uint64_t>(chunk) * chunk_steps, static_cast<uint64_t>(blocks.count)));
    const uint32_t hi = any ? min(lo + chunk_steps, blocks.count) : lo;
    if (chunks > 1 && lo >= hi) {                                         // nothing for this part: its sums count for nothing
        for (uint32_t u = u0 + threadIdx.x; u < min(u0 + R, units); u += WARPS * 32)
            *reinterpret_cast<float2*>(part_ml + 2 * (((static_cast<size_t>(span.row0) + u / group) * heads + kvh * group + u % group) * chunks + chunk)) = make_float2(-CUDART_INF_F, 0.f);
        return;
    }
    // rows of this lane: gid and gid + 8
    uint32_t at[2];
    bool held[2];
#pragma unroll
    for (int i = 0; i < (TALL ? 2 : 1); ++i) {
        const uint32_t tok = min(u0 + gid + 8 * i, units - 1) / group;
        held[i] = tok >= lost;
        at[i] = before + max(tok, lost);
    }
    float mx[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
    float o[DIM / 8][TALL ? 4 : 2];
#pragma unroll
    for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
        for (int i = 0; i < (TALL ? 4 : 2); ++i) o[n][i] = 0.f;
    bool bad = false, clipped = false;
    float unit = 0x1p-100f;

    if (lo + warp < hi) {
        uint32_t qa[KS][TALL ? 4 : 2];
#pragma unroll
        for (int i = 0; i < (TALL ? 2 : 1); ++i) {
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
                qa[j][i] = pack2<CODES>(e[0], e[1]);
                qa[j][(TALL ? 2 : 1) + i] = pack2<CODES>(e[2], e[3]);
            }
        }
        uint4 kr[2][KU];
        uint32_t vr[4][VU][VW];
        float ks[4], vs[4];
        auto base_of = [&](uint32_t step) {                               // first row of the step's positions in this head
            const uint32_t p = blocks.at(step) << STEP_LOG;
            return c.row(page_of(c, b, s, p, bad), kvh, p & (c.size() - 1));
        };
        auto load_k = [&](size_t base) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < KU; ++i) kr[n][i] = load16(static_cast<const uint8_t*>(c.k) + (base + 8 * n + gid) * ROW + (4 * i + t) * 16);
            if constexpr (CODES) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float2 a = __ldcg(reinterpret_cast<const float2*>(c.k_scale + base + 8 * n) + t);
                    ks[2 * n] = a.x; ks[2 * n + 1] = a.y;
                }
            }
        };
        auto load_v = [&](size_t base) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < VU; ++i) {
                    const uint8_t* from = static_cast<const uint8_t*>(c.v) + (base + 2 * t + (x & 1) + 8 * (x >> 1)) * ROW + (gid + 8 * i) * (VW * 4);
                    if constexpr (VW == 4) { const uint4 w = load16(from); vr[x][i][0] = w.x; vr[x][i][1] = w.y; vr[x][i][2] = w.z; vr[x][i][3] = w.w; }
                    else { const uint2 w = __ldcg(reinterpret_cast<const uint2*>(from)); vr[x][i][0] = w.x; vr[x][i][1] = w.y; }
                }
            if constexpr (CODES) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float2 a = __ldcg(reinterpret_cast<const float2*>(c.v_scale + base + 8 * n) + t);
                    vs[2 * n] = a.x; vs[2 * n + 1] = a.y;
                }
            }
        };
        uint32_t step = lo + warp;
        size_t base = base_of(step), next = step + WARPS < hi ? base_of(step + WARPS) : base;
        load_k(base);
        load_v(base);
        for (; step < hi; step += WARPS) {
            const uint32_t p0 = blocks.at(step) << STEP_LOG;
            const bool more = step + WARPS < hi;
            // ---- scores: n-tile n holds positions p0 + 8 n + 2 t, + 1 of rows gid (and gid + 8)
            float sc[2][4];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < KU; ++i) {
                    const uint32_t w[4] = {kr[n][i].x, kr[n][i].y, kr[n][i].z, kr[n][i].w};
                    if constexpr (CODES) {
                        const __half2 bias = __float2half2_rn(1152.0f);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const uint32_t y = w[x] ^ 0x80808080u;
                            const uint32_t(&f)[TALL ? 4 : 2] = qa[4 * i + x];
                            mma<true>(a, f[0], TALL ? f[1] : 0u, f[TALL ? 2 : 1], TALL ? f[TALL ? 3 : 0] : 0u, tc::h2_bits(tc::codes01(y, bias)), tc::h2_bits(tc::codes23(y, bias)));
                        }
                    } else {
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const uint32_t(&f)[TALL ? 4 : 2] = qa[2 * i + x];
                            mma<false>(a, f[0], TALL ? f[1] : 0u, f[TALL ? 2 : 1], TALL ? f[TALL ? 3 : 0] : 0u, w[2 * x], w[2 * x + 1]);
                        }
                    }
                }
                float f0 = look.scale, f1 = look.scale;
                if constexpr (CODES) { f0 *= ks[2 * n]; f1 *= ks[2 * n + 1]; }
                sc[n][0] = a[0] * f0; sc[n][1] = a[1] * f1; sc[n][2] = a[2] * f0; sc[n][3] = a[3] * f1;
            }
            if (more) load_k(next);
            // ---- what the rows do not see
            const bool full = all_see(look, first, last, p0, STEP) && tok0 >= lost;
            uint32_t seen = 0xffu;                                        // bit 4 i + 2 n + x: row i, position p0 + 8 n + 2 t + x
            if (!full) {
                seen = 0;
#pragma unroll
                for (int i = 0; i < (TALL ? 2 : 1); ++i)
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const bool yes = held[i] && look.sees(at[i], p0 + 8 * n + 2 * t + x);
                            seen |= static_cast<uint32_t>(yes) << (4 * i + 2 * n + x);
                            if (!yes) sc[n][2 * i + x] = -CUDART_INF_F;
                        }
            }
            // ---- softmax: maximum and sum so far of each row
            float w[2][4], corr[2] = {1.f, 1.f};
#pragma unroll
            for (int i = 0; i < (TALL ? 2 : 1); ++i) {
                float top = fmaxf(fmaxf(sc[0][2 * i], sc[0][2 * i + 1]), fmaxf(sc[1][2 * i], sc[1][2 * i + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float to = fmaxf(mx[i], top), zero = to == -CUDART_INF_F ? 0.f : to;
                corr[i] = tc::ex2(mx[i] - zero);
                mx[i] = to;
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        w[n][2 * i + x] = tc::ex2(sc[n][2 * i + x] - zero);
                        sum += w[n][2 * i + x];
                    }
                l[i] = l[i] * corr[i] + sum;                              // (of this lane's positions; the lanes of a row are added at the end)
            }
            if constexpr (CODES) {
                float top = 0.f;
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float a = fabsf(vs[2 * n + x]);
                        if (a < CUDART_INF_F && (full || some_see(look, first, last, p0 + 8 * n + 2 * t + x))) top = fmaxf(top, a);
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float above = fmaxf(unit, unit_above(top)), f = 4096.0f / above;
                if (above != unit) { corr[0] *= unit / above; corr[1] *= unit / above; unit = above; }
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int x = 0; x < (TALL ? 4 : 2); ++x) w[n][x] = (seen >> (4 * (x >> 1) + 2 * n + (x & 1))) & 1 ? w[n][x] * (vs[2 * n + (x & 1)] * f) : 0.f;
            }
            const bool rescale = corr[0] != 1.f || (TALL && corr[1] != 1.f);
            if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll
                for (int n = 0; n < DIM / 8; ++n) {
                    o[n][0] *= corr[0]; o[n][1] *= corr[0];
                    if constexpr (TALL) { o[n][2] *= corr[1]; o[n][3] *= corr[1]; }
                }
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
                const uint32_t a0 = pack2<CODES>(w[0][0], w[0][1]), a2 = pack2<CODES>(w[1][0], w[1][1]);
                const uint32_t a1 = TALL ? pack2<CODES>(w[0][2], w[0][3]) : 0u, a3 = TALL ? pack2<CODES>(w[1][2], w[1][3]) : 0u;
                auto add = [&](int n, uint32_t b0, uint32_t b1) {
                    float d[4] = {o[n][0], o[n][1], TALL ? o[n][TALL ? 2 : 0] : 0.f, TALL ? o[n][TALL ? 3 : 0] : 0.f};
                    mma<CODES>(d, a0, a1, a2, a3, b0, b1);
#pragma unroll
                    for (int x = 0; x < (TALL ? 4 : 2); ++x) o[n][x] = d[x];
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
                            const int n = i * VE + 4 * y;
                            add(n, tc::h2_bits(tc::codes01(lo01, bias)), tc::h2_bits(tc::codes01(lo89, bias)));
                            add(n + 1, tc::h2_bits(tc::codes23(lo01, bias)), tc::h2_bits(tc::codes23(lo89, bias)));
                            add(n + 2, tc::h2_bits(tc::codes01(hi01, bias)), tc::h2_bits(tc::codes01(hi89, bias)));
                            add(n + 3, tc::h2_bits(tc::codes23(hi01, bias)), tc::h2_bits(tc::codes23(hi89, bias)));
                        } else {
                            const int n = i * VE + 2 * y;
                            add(n, __byte_perm(va, vb, 0x5410u), __byte_perm(vc, vd, 0x5410u));
                            add(n + 1, __byte_perm(va, vb, 0x7632u), __byte_perm(vc, vd, 0x7632u));
                        }
                    }
            } else if constexpr (!CODES) {
                // 0 times infinity is not 0: each row adds up the positions that it sees, one by one
                const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(c.v) + base * DIM;
#pragma unroll 1
                for (uint32_t p = 0; p < STEP; ++p) {
                    const uint32_t from = (lane & ~3u) | ((p & 7) >> 1);
#pragma unroll
                    for (int i = 0; i < (TALL ? 2 : 1); ++i) {
                        const float a = p & 1 ? (p < 8 ? w[0][2 * i + 1] : w[1][2 * i + 1]) : (p < 8 ? w[0][2 * i] : w[1][2 * i]);
                        const float weight = __shfl_sync(0xffffffffu, a, from);
                        if (held[i] && look.sees(at[i], p0 + p)) {
#pragma unroll
                            for (int n = 0; n < DIM / 8; ++n)
#pragma unroll
                                for (int x = 0; x < 2; ++x)
                                    o[n][2 * i + x] = fmaf(weight, __bfloat162float(v[p * DIM + (2 * t + x + 8 * (n / VE)) * VE + n % VE]), o[n][2 * i + x]);
                        }
                    }
                }
            }
            if (more) {
                load_v(next);
                base = next;
                if (step + 2 * WARPS < hi) next = base_of(step + 2 * WARPS);
            }
        }
    }
    // ---- the warps' rows meet in shared memory
    const float back = CODES ? unit * (1.0f / 4096.0f) : 1.0f;
#pragma unroll
    for (int i = 0; i < (TALL ? 2 : 1); ++i) {
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        if (t == 0) { red_m[warp][gid + 8 * i] = mx[i]; red_l[warp][gid + 8 * i] = l[i]; }
        float* mine = red + (warp * R + gid + 8 * i) * (DIM + 4);
#pragma unroll
        for (int n = 0; n < DIM / 8; n += 4)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                *reinterpret_cast<float4*>(mine + (2 * t + x + 8 * (n / VE)) * VE + n % VE) =
                    make_float4(o[n][2 * i + x] * back, o[n + 1][2 * i + x] * back, o[n + 2][2 * i + x] * back, o[n + 3][2 * i + x] * back);
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
                      static_cast<OUT*>(a.out), a.ldo, a.chunk >> STEP_LOG, a.chunks, a.part, a.part_ml, a.status);
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
