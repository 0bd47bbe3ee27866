// Attention over a paged cache for many rows of a sequence: portions of prompts, on the 5th-generation tensor cores.
//
// One CTA owns two tiles of 128 rows = TOK tokens x the group of query heads of one KV head (TOK = 128 / group), and walks the positions
// that they see in blocks of 128:
//
//   warps 8-11  loaders.  Bring the block's keys and values from its pages to shared memory as 16-bit operands with the 128-byte swizzle,
//               once for both tiles.  Codes pass through registers and become exact f16 whole numbers, the next block's loads already
//               under way; bf16 is copied asynchronously.  K is [position][dim], the K-major B operand of the scores; V has the same
//               layout, read MN-major as the B operand of the output.
//   warp 12     one lane issues the products, S = Q K^T and O += P V, of the two tiles in turn: one tile's softmax runs under the other
//               tile's products.
//   warps 0-3   softmax of the first tile, a thread to a row: scores from tensor memory, exponentials in f32, P back as the 16-bit A
//   warps 4-7   operand in the place of S.  The same for the second tile.  The output row is rescaled only when the running
//               maximum grew by more than 2^ROOM.
//
// Tensor memory: S 2 x 128 columns, O 2 x dim.  Codes: the scale of K multiplies the f32 score; the weight is p * v_scale * 2^12 / U in f16, U
// a power of two above all value scales of the blocks so far, which the loaders keep: it grows seldom, and the output is rescaled
// with the maximum's correction.  What a row does not see gets weight 0 by selection, whatever its scales and scores are.  bf16 values
// that are infinite or NaN in blocks that only some rows see would turn a weight of 0 into NaN: the loaders find them, hand zeros to the
// product, and the rows that see them add them up one by one.
#include <math_constants.h>

#include <type_traits>

#include "paged_common.cuh"
#include "tc_common.cuh"

namespace hf2q {
using namespace paged;
using namespace tc;
namespace {

constexpr uint32_t ROWS = 128, BP_LOG = 7, BP = 1 << BP_LOG, SLOTS = 4, PANEL = BP * 128;
constexpr uint32_t SOFTMAX_WARPS = 8, LOAD_WARPS = 4, THREADS = (SOFTMAX_WARPS + LOAD_WARPS + 1) * 32, COLS = 512;
template <int DIM> constexpr uint32_t tiles_smem() { return 2 * ROWS * DIM * 2 + 4 * BP * DIM * 2 + 1024; }

__device__ __forceinline__ uint32_t claim_columns(uint32_t* slot) {       // by one warp; every other CTA of the SM gives its own back by itself
    tmem_alloc(slot, COLS);
    tmem_relinquish();
    return 0;
}
__device__ __forceinline__ bool elected() {                               // one lane of a whole warp
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// The bounded wait with its loop out of line: what every role goes through stays small (the instruction cache of a scheduler serves four roles).
__device__ __noinline__ bool wait_on(uint64_t* bar, uint32_t parity, uint32_t* status) { return mbar_wait_slow<0>(bar, parity, status); }
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t* status) { return mbar_try_wait(bar, parity) || wait_on(bar, parity, status); }
// all loader warps have come here for the n-th time (false: the wait ran out)
__device__ __forceinline__ bool loaders_meet(uint64_t* bar, uint32_t n, uint32_t lane, uint32_t* status) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    return __all_sync(0xffffffffu, wait(bar, n & 1, status));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {       // zeros past `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ bool holds_nonfinite(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
__device__ __forceinline__ float unit_above(float v) {                    // a power of two above |v| (v finite), within what 2^12 / U can be
    return fminf(fmaxf(__uint_as_float((__float_as_uint(v) & 0x7f800000u) + 0x00800000u), 0x1p-100f), 0x1p100f);
}
template <bool CODES> __device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (CODES) return pack_h2(a, b);
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool CODES> __device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (CODES) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// byte of 16-byte chunk `chunk` of row `row` in a swizzled operand of rows of 64 elements a panel
__device__ __forceinline__ uint32_t chunk_at(uint32_t row, uint32_t chunk, uint32_t panel) { return (chunk >> 3) * panel + row * 128 + (((chunk & 7) ^ (row & 7)) << 4); }

// sixteen signed bytes -> f16 whole numbers; odd panels store their chunks in the other order (a quarter-warp then meets all banks)
__device__ __forceinline__ void store_codes(uint8_t* block, uint32_t row, uint32_t c16, const uint4& q) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    uint32_t h[8];
    const __half2 bias = __float2half2_rn(1152.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = w[i] ^ 0x80808080u;                            // code + 128; 0x6400 | b is 1024 + b
        h[2 * i] = h2_bits(codes01(x, bias));
        h[2 * i + 1] = h2_bits(codes23(x, bias));
    }
    const uint32_t flip = (c16 >> 2) & 1;
    const uint4 lo = make_uint4(h[0], h[1], h[2], h[3]), hi = make_uint4(h[4], h[5], h[6], h[7]);
    *reinterpret_cast<uint4*>(block + chunk_at(row, 2 * c16 + flip, PANEL)) = flip ? hi : lo;
    *reinterpret_cast<uint4*>(block + chunk_at(row, 2 * c16 + 1 - flip, PANEL)) = flip ? lo : hi;
}

template <typename Q> __device__ __forceinline__ void load8(const Q* p, bool wide, float (&e)[8]) {
    if constexpr (std::is_same_v<Q, float>) {
        if (wide) {
            const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
            e[0] = a.x; e[1] = a.y; e[2] = a.z; e[3] = a.w; e[4] = b.x; e[5] = b.y; e[6] = b.z; e[7] = b.w;
        } else for (int i = 0; i < 8; ++i) e[i] = p[i];
    } else {
        if (wide) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
            for (int i = 0; i < 4; ++i) { e[2 * i] = __uint_as_float(w[i] << 16); e[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
        } else for (int i = 0; i < 8; ++i) e[i] = __bfloat162float(p[i]);
    }
}

struct Shape {
    uint32_t heads, group, tokens;           // tokens of a tile
    uint32_t ldq, ldo, chunk_blocks, chunks;
    bool wide_q;
};

// The sequence and the first token of CTA tile `index` (tiles of 2 * tokens tokens, the sequences one after the other); false: there is none.
__device__ __forceinline__ bool find_tile(const Batch& b, uint32_t shift, uint32_t per, uint32_t index, uint32_t& seq, uint32_t& tok) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t s0 = 0; s0 < b.seqs; s0 += 32) {
        const uint32_t mine = s0 + lane < b.seqs ? (span_of(b, shift, s0 + lane).rows + per - 1) / per : 0u;
        uint32_t upto = mine;
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= static_cast<uint32_t>(o)) upto += x;
        }
        const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
        if (index < all) {
            const uint32_t at = __popc(__ballot_sync(0xffffffffu, upto <= index));
            seq = s0 + at;
            tok = (index - __shfl_sync(0xffffffffu, upto - mine, at)) * per;
            return true;
        }
        index -= all;
    }
    return false;
}

template <int DIM, bool CODES, typename Q, typename OUT>
__global__ void __launch_bounds__(THREADS, 1) attend_tiles_kernel(Pool c, Batch b, Look look, Shape sh, const Q* q, OUT* out, float* part, float* part_ml, uint32_t* status) {
    constexpr uint32_t Q_PANEL = ROWS * 128, Q_BYTES = ROWS * DIM * 2, KV_BYTES = BP * DIM * 2, COL_O = 2 * BP;
    constexpr float ROOM = CODES ? 3.0f : 8.0f;
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t *qs = smem, *ks = smem + 2 * Q_BYTES, *vs = ks + 2 * KV_BYTES;
    // Scales of a block have a barrier per slot.  Slot j % 4 is written next for block j + 4, after K(j + 2) left its place, that is after S(j + 2)
    // of both tiles, which follows P(j + 1) of every softmax warp.
    __shared__ __align__(16) float s_ks[SLOTS][BP], s_vs[SLOTS][BP];
    __shared__ float s_unit[SLOTS];
    __shared__ uint32_t s_odd[2];
    __shared__ uint64_t k_full[2], v_full[2], k_free[2], v_free[2], sc_full[SLOTS], s_full[2], p_full[2], o_done[2], meet;
    __shared__ uint32_t tmem_slot;
    const uint32_t kvh = blockIdx.x % c.kv_heads, chunk = blockIdx.y, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t seq = 0, tok0 = 0;
    if (!find_tile(b, c.shift, 2 * sh.tokens, (gridDim.x - 1 - blockIdx.x) / c.kv_heads, seq, tok0)) return;      // (the tiles with the most positions first)
    const Span span = span_of(b, c.shift, seq);
    if (span.bad && threadIdx.x == 0) atomicOr(status, STATUS_BAD_PAGE);
    const uint32_t end_tok = min(tok0 + 2 * sh.tokens, span.rows), tiles = end_tok - tok0 > sh.tokens ? 2 : 1;
    const uint32_t lost = span.rows > span.length ? span.rows - span.length : 0;      // rows in front of position 0: they see nothing
    const uint32_t before = span.length - span.rows;                      // position of token 0 (wraps where rows are lost)
    const bool any = end_tok > lost;
    const uint32_t first = any ? before + max(tok0, lost) : 0, last = any ? before + end_tok - 1 : 0;
    const Blocks blocks = blocks_of(look, first, last, BP_LOG);
    const uint32_t lo = static_cast<uint32_t>(min(static_cast<uint64_t>(chunk) * sh.chunk_blocks, static_cast<uint64_t>(blocks.count)));
    const uint32_t nb = any ? min(sh.chunk_blocks, blocks.count - lo) : 0;
    if (nb == 0) {
        // nothing to see here: a part that counts for nothing, or zeros
        const uint32_t units = (end_tok - tok0) * sh.group;
        if (sh.chunks > 1) {
            for (uint32_t u = threadIdx.x; u < units; u += THREADS)
                *reinterpret_cast<float2*>(part_ml + 2 * (((static_cast<size_t>(span.row0) + tok0 + u / sh.group) * sh.heads + kvh * sh.group + u % sh.group) * sh.chunks + chunk)) =
                    make_float2(-CUDART_INF_F, 0.f);
        } else {
            bool no = false;
            for (uint32_t i = threadIdx.x; i < units * DIM; i += THREADS) {
                const uint32_t u = i / DIM;
                out[(static_cast<size_t>(span.row0) + tok0 + u / sh.group) * sh.ldo + (kvh * sh.group + u % sh.group) * DIM + i % DIM] = out_value<OUT>(0.f, no);
            }
        }
        return;
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], LOAD_WARPS);
            mbar_init(&v_full[i], LOAD_WARPS);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&o_done[i], 1);
            s_odd[i] = 0;
        }
        for (uint32_t i = 0; i < SLOTS; ++i) mbar_init(&sc_full[i], LOAD_WARPS);
        mbar_init(&meet, LOAD_WARPS);
        mbar_fence_init();
    }
    if (warp == SOFTMAX_WARPS + LOAD_WARPS) claim_columns(&tmem_slot);
    // Q: two tiles of 128 rows in 16 bits; a negative scale is taken over by q, so that the largest product is the largest score
    bool clipped = false;
    for (uint32_t i = threadIdx.x; i < 2 * ROWS * (DIM / 8); i += THREADS) {
        const uint32_t ch = i % (DIM / 8), r = i / (DIM / 8), tile = r >> 7, rr = r & 127, in_tile = rr / sh.group, tok = tok0 + tile * sh.tokens + in_tile;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (in_tile < sh.tokens && tok < end_tok) {
            float e[8];
            load8(q + static_cast<size_t>(span.row0 + tok) * sh.ldq + static_cast<size_t>(kvh * sh.group + rr % sh.group) * DIM + 8 * ch, sh.wide_q, e);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                if (look.scale < 0.f) e[x] = -e[x];
                if constexpr (CODES) { clipped |= fabsf(e[x]) > 65504.0f; e[x] = fabsf(e[x]) > 65504.0f ? copysignf(65504.0f, e[x]) : e[x]; }
            }
            w = make_uint4(pack2<CODES>(e[0], e[1]), pack2<CODES>(e[2], e[3]), pack2<CODES>(e[4], e[5]), pack2<CODES>(e[6], e[7]));
        }
        *reinterpret_cast<uint4*>(qs + tile * Q_BYTES + chunk_at(rr, ch, Q_PANEL)) = w;
    }
    proxy_fence();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const float scale = fabsf(look.scale);

    if (warp >= SOFTMAX_WARPS && warp < SOFTMAX_WARPS + LOAD_WARPS) {
        constexpr uint32_t CH = CODES ? DIM / 16 : DIM / 8, RP = LOAD_WARPS * 32 / CH, NP = BP / RP;      // 16-byte chunks of a row; rows of a pass; passes
        constexpr uint32_t ROW = DIM * (CODES ? 1 : 2);
        const uint32_t tid = threadIdx.x - SOFTMAX_WARPS * 32, ch = tid % CH, row0 = tid / CH, last16 = last & ~15u;
        bool bad = false, ok = true;
        // lane g holds where positions 16 g .. 16 g + 15 of a block lie, in sixteens of rows; positions past the last one repeat the last sixteen
        auto places = [&](uint32_t j) {
            const uint32_t p = min((blocks.at(lo + j) << BP_LOG) + 16 * (lane & 7), last16);
            return static_cast<uint32_t>(c.row(page_of(c, b, seq, p, bad), kvh, p & (c.size() - 1)) >> 4);
        };
        auto group = [&](uint32_t i) { return RP <= 16 ? RP * i >> 4 : (RP * i + row0) >> 4; };
        auto place = [&](const void* array, uint32_t at16, uint32_t i, uint32_t row_bytes) {      // this thread's chunk of pass i
            return static_cast<const uint8_t*>(array) + static_cast<uint64_t>(__shfl_sync(0xffffffffu, at16, group(i))) * (16 * row_bytes) + ((RP * i + row0) & 15) * row_bytes + 16 * ch;
        };
        uint32_t here = places(0), there = nb > 1 ? places(1) : here;
        if constexpr (CODES) {
            uint4 kq[NP], vq[NP];
            // every warp holds the scales of the whole block, four positions a lane, for the largest of V's; a quarter of the lanes stores
            float4 k4, v4;
            float unit = 0x1p-100f;
            auto scales = [&](uint32_t at16) {
                const uint64_t r = static_cast<uint64_t>(__shfl_sync(0xffffffffu, at16, lane >> 2)) * 16 + (4 * lane & 15);
                k4 = __ldcg(reinterpret_cast<const float4*>(c.k_scale + r));
                v4 = __ldcg(reinterpret_cast<const float4*>(c.v_scale + r));
            };
            auto load = [&](const void* from, uint32_t at16, uint4 (&x)[NP]) {
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) x[i] = __ldcg(reinterpret_cast<const uint4*>(place(from, at16, i, ROW)));
            };
            uint32_t p0 = blocks.at(lo) << BP_LOG;
            load(c.k, here, kq);
            scales(here);
            load(c.v, here, vq);
            for (uint32_t j = 0; j < nb; ++j) {
                const uint32_t st = j & 1, par = ((j >> 1) - 1) & 1, slot = j % SLOTS;
                const uint32_t p1 = j + 1 < nb ? blocks.at(lo + j + 1) << BP_LOG : 0;
                if (j >= 2) ok = wait(&k_free[st], par, status);
                if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) store_codes(ks + st * KV_BYTES, RP * i + row0, ch, kq[i]);
                const float vv[4] = {fabsf(v4.x), fabsf(v4.y), fabsf(v4.z), fabsf(v4.w)};
                float top = 0.f;
#pragma unroll
                for (uint32_t x = 0; x < 4; ++x)
                    if (vv[x] < CUDART_INF_F && some_see(look, first, last, p0 + 4 * lane + x)) top = fmaxf(top, vv[x]);
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                unit = fmaxf(unit, unit_above(top));
                if (lane >> 3 == (warp & 3)) {
                    const float f = 4096.0f / unit;
                    *reinterpret_cast<float4*>(&s_ks[slot][4 * lane]) = make_float4(k4.x * scale, k4.y * scale, k4.z * scale, k4.w * scale);
                    *reinterpret_cast<float4*>(&s_vs[slot][4 * lane]) = make_float4(v4.x * f, v4.y * f, v4.z * f, v4.w * f);
                }
                if (tid == 0) s_unit[slot] = unit;
                proxy_fence();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sc_full[slot]);
                    mbar_arrive(&k_full[st]);
                }
                if (j + 1 < nb) {
                    load(c.k, there, kq);
                    scales(there);
                }
                if (j >= 2) ok = wait(&v_free[st], par, status);
                if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) store_codes(vs + st * KV_BYTES, RP * i + row0, ch, vq[i]);
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (j + 1 < nb) {
                    load(c.v, there, vq);
                    p0 = p1;
                    if (j + 2 < nb) there = places(j + 2);
                }
            }
        } else {
            const uint32_t to0 = chunk_at(row0, ch, PANEL);                  // (a pass is 8 rows or a multiple: the swizzle of a thread's chunk stays)
            auto copy = [&](const void* from, uint8_t* to, uint32_t at16, uint32_t p0, bool zeros) {
                const uint32_t dst = smem_u32(to) + to0;
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) {
                    const bool take = !zeros || some_see(look, first, last, p0 + RP * i + row0);      // (values that nobody sees are zeros)
                    copy16(dst + RP * i * 128, place(from, at16, i, ROW), take ? 16 : 0);
                }
                copies_close();
            };
            uint32_t p0 = blocks.at(lo) << BP_LOG;
            copy(c.k, ks, here, p0, false);
            copy(c.v, vs, here, p0, !all_see(look, first, last, p0, BP));
            uint32_t met = 0;
            for (uint32_t j = 0; j < nb; ++j) {
                const uint32_t st = j & 1, other = st ^ 1, par = ((j + 1) >> 1) - 1 & 1;
                const bool more = j + 1 < nb;
                const uint32_t p1 = more ? blocks.at(lo + j + 1) << BP_LOG : 0;
                if (more) {
                    if (j >= 1) ok = wait(&k_free[other], par, status);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    copy(c.k, ks + other * KV_BYTES, there, p1, false);
                    copies_wait<2>();
                } else copies_wait<1>();
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                if (more) copies_wait<1>(); else copies_wait<0>();
                if (!all_see(look, first, last, p0, BP) && (first != last)) {
                    bool odd = false;
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) {
                        const uint4 w = *reinterpret_cast<const uint4*>(vs + st * KV_BYTES + chunk_at(RP * i + row0, ch, PANEL));
                        odd |= holds_nonfinite(w.x) || holds_nonfinite(w.y) || holds_nonfinite(w.z) || holds_nonfinite(w.w);
                    }
                    // (s_odd of block j - 2 has been read: its V left this place.)  The loaders agree, and then none keeps its part.
                    if (tid == 0) s_odd[st] = 0;
                    ok = loaders_meet(&meet, met++, lane, status);
                    if (odd) s_odd[st] = 1;
                    ok = ok && loaders_meet(&meet, met++, lane, status);
                    if (!ok) break;
                    if (*static_cast<volatile uint32_t*>(&s_odd[st]))
#pragma unroll
                        for (uint32_t i = 0; i < NP; ++i) *reinterpret_cast<uint4*>(vs + st * KV_BYTES + chunk_at(RP * i + row0, ch, PANEL)) = make_uint4(0u, 0u, 0u, 0u);
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (more) {
                    if (j >= 1) ok = wait(&v_free[other], par, status);
                    if (!__all_sync(0xffffffffu, ok)) break;
                    copy(c.v, vs + other * KV_BYTES, there, p1, !all_see(look, first, last, p1, BP));
                    p0 = p1;
                    if (j + 2 < nb) there = places(j + 2);
                }
            }
            copies_wait<0>();
        }
        if (bad) atomicOr(status, STATUS_BAD_PAGE);
    } else if (warp >= SOFTMAX_WARPS + LOAD_WARPS) {
        if (warp == SOFTMAX_WARPS + LOAD_WARPS) {
            // D f32; A and B f16 or bf16; M = 128; S: both K-major, N = 128; O: B MN-major, N = dim.  The whole warp goes through the waits, so that
            // addresses and descriptors stay in uniform registers; one lane issues.
            constexpr uint32_t ID = (1u << 4) | (CODES ? 0u : (1u << 7) | (1u << 10)) | ((ROWS >> 4) << 24), ID_S = ID | ((BP >> 3) << 17), ID_O = ID | (1u << 16) | ((DIM >> 3) << 17);
            const uint32_t n = __shfl_sync(0xffffffffu, nb, 0), nt = __shfl_sync(0xffffffffu, tiles, 0), base = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t q_desc = smem_desc_sw128(smem_u32(qs)), k_desc = smem_desc_sw128(smem_u32(ks)), v_desc = smem_desc_mn_sw128(smem_u32(vs), PANEL);
            bool ok = true;
            // (one place in the code for each product: S(j) of a tile behind its O += P(j - 1) V)
            for (uint32_t j = 0; j <= n && ok; ++j) {
                const uint32_t st = j & 1, was = st ^ 1;
                for (uint32_t t = 0; t < nt && ok; ++t) {
                    if (j) {
                        if (t == 0) ok = wait(&v_full[was], ((j - 1) >> 1) & 1, status);
                        if (ok) ok = wait(&p_full[t], (j - 1) & 1, status);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        tc_fence_after();
                        if (elected()) {
                            const uint64_t vd = v_desc + was * (KV_BYTES >> 4);
#pragma unroll
                            for (uint32_t kk = 0; kk < BP / 16; ++kk) umma_ts(base + COL_O + t * DIM, base + t * BP + 8 * kk, vd + kk * (16 * 128 >> 4), ID_O, 1u);
                            tc_commit(&o_done[t]);
                            if (t + 1 == nt) tc_commit(&v_free[was]);
                        }
                        __syncwarp();
                    }
                    if (j == n) continue;
                    if (t == 0) ok = wait(&k_full[st], (j >> 1) & 1, status);
                    if (ok && j) ok = wait(&o_done[t], (j - 1) & 1, status);                  // P(j - 1) is read: S(j) takes its place
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    tc_fence_after();
                    if (elected()) {
                        const uint64_t qd = q_desc + t * (Q_BYTES >> 4), kd = k_desc + st * (KV_BYTES >> 4);
#pragma unroll
                        for (uint32_t kk = 0; kk < DIM / 16; ++kk)
                            umma_ss(base + t * BP, qd + (kk >> 2) * (Q_PANEL >> 4) + 2 * (kk & 3), kd + (kk >> 2) * (PANEL >> 4) + 2 * (kk & 3), ID_S, kk ? 1u : 0u);
                        tc_commit(&s_full[t]);
                        if (t + 1 == nt) tc_commit(&k_free[st]);
                    }
                    __syncwarp();
                }
            }
        }
    } else {
        const uint32_t tile = warp / 4, row = threadIdx.x & 127, at = tmem + (((warp & 3) * 32u) << 16), at_s = at + tile * BP, at_o = at + COL_O + tile * DIM;
        const uint32_t in_tile = row / sh.group, tile_tok = tok0 + tile * sh.tokens, tile_end = min(tile_tok + sh.tokens, end_tok), tok = tile_tok + in_tile;
        const bool live = in_tile < sh.tokens && tok < end_tok, held = live && tok >= lost;
        const uint32_t seen = before + max(min(tok, tile_end - 1), lost);          // (rows that are not there compute on zeros and are not stored)
        const uint32_t t_first = before + max(tile_tok, lost), t_last = before + max(tile_end - 1, lost);
        // the row sees positions from `low` on, `reach` more, and those below `firsts`
        const uint32_t low = !held ? 1u << 31 : look.window && seen >= look.window ? seen - look.window + 1 : 0, reach = held ? seen - low : 0;
        const uint32_t firsts = held && look.window ? min(look.sinks, seen + 1) : 0;
        float mx = -CUDART_INF_F, unit = 0x1p-100f;
        f2 sum = 0;
        bool ok = true;
        {
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
#pragma unroll
            for (uint32_t col = 0; col < DIM; col += 32) tmem_st32(at_o + col, zero);
        }
        if (tile < tiles) {
        for (uint32_t j = 0; j < nb; ++j) {
            const uint32_t slot = j % SLOTS, st = j & 1, p0 = blocks.at(lo + j) << BP_LOG;
            ok = wait(&s_full[tile], j & 1, status);
            if constexpr (CODES) { if (ok) ok = wait(&sc_full[slot], (j / SLOTS) & 1, status); }
            const bool full = all_see(look, t_first, t_last, p0, BP) && tile_tok >= lost;
            bool odd = false;
            if constexpr (!CODES) {
                if (!all_see(look, first, last, p0, BP) && first != last) {
                    if (ok) ok = wait(&v_full[st], (j >> 1) & 1, status);
                    odd = *static_cast<volatile uint32_t*>(&s_odd[st]) != 0;
                }
            }
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const ulonglong2 *k2 = reinterpret_cast<const ulonglong2*>(s_ks[slot]), *v2 = reinterpret_cast<const ulonglong2*>(s_vs[slot]);
            const auto sees = [&](uint32_t p) { return p - low <= reach || p < firsts; };
            auto block = [&](auto masked) {
                constexpr bool MASKED = decltype(masked)::value;
                // twice over the scores, 32 columns at a time: the maximum, then the exponentials
                float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll 1
                for (uint32_t x = 0; x < BP / 32; ++x) {
                    uint32_t r[32];
                    tmem_ld32(at_s + 32 * x, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float2 v = make_float2(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1]));
                        if constexpr (CODES) { const ulonglong2 k = k2[8 * x + i / 2]; v = f2_parts(f2_mul(f2_of(v.x, v.y), i & 1 ? k.y : k.x)); }
                        if constexpr (MASKED) {
                            if (!sees(p0 + 32 * x + 2 * i)) v.x = -CUDART_INF_F;
                            if (!sees(p0 + 32 * x + 2 * i + 1)) v.y = -CUDART_INF_F;
                        }
                        top[i & 3] = fmaxf(fmaxf(top[i & 3], v.x), v.y);
                    }
                }
                float bm = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                if constexpr (!CODES) bm = bm == -CUDART_INF_F ? bm : bm * scale;
                // the output is in units of `unit` times exp2 of the maximum
                const float above = CODES ? s_unit[slot] : unit;
                const bool grew = bm > mx + ROOM || (mx == -CUDART_INF_F && bm > mx);
                if (__any_sync(0xffffffffu, grew || above != unit)) {
                    const float to = grew ? bm : mx;
                    float corr = grew ? ex2(mx - to) : 1.0f;
                    sum = f2_mul(sum, f2_both(corr));
                    mx = to;
                    corr *= unit / above;
                    unit = above;
                    if (j) {                                              // (S(j) followed the output of block j - 1)
#pragma unroll 1
                        for (uint32_t col = 0; col < DIM; col += 16) {
                            uint32_t o[16];
                            tmem_ld16(at_o + col, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                            tmem_st16(at_o + col, o);
                        }
                    }
                }
                const f2 nm = f2_both(mx == -CUDART_INF_F ? 0.f : -mx), sc2 = f2_both(scale);
#pragma unroll 1
                for (uint32_t x = 0; x < BP / 32; ++x) {
                    uint32_t r[32], p[16];
                    tmem_ld32(at_s + 32 * x, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        f2 k = sc2;
                        if constexpr (CODES) { const ulonglong2 kk = k2[8 * x + i / 2]; k = i & 1 ? kk.y : kk.x; }
                        float2 d = f2_parts(f2_fma(f2_of(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), k, nm));
                        bool s0 = true, s1 = true;
                        if constexpr (MASKED) {
                            s0 = sees(p0 + 32 * x + 2 * i);
                            s1 = sees(p0 + 32 * x + 2 * i + 1);
                            if (!s0) d.x = -CUDART_INF_F;
                            if (!s1) d.y = -CUDART_INF_F;
                        }
                        const f2 e = f2_of(ex2(d.x), ex2(d.y));
                        sum = f2_add(sum, e);
                        float2 w = f2_parts(e);
                        if constexpr (CODES) {
                            const ulonglong2 v = v2[8 * x + i / 2];
                            w = f2_parts(f2_mul(e, i & 1 ? v.y : v.x));
                            if constexpr (MASKED) {                       // (also where the scale of V is infinite or NaN)
                                if (!s0) w.x = 0.f;
                                if (!s1) w.y = 0.f;
                            }
                        }
                        p[i] = pack2<CODES>(w.x, w.y);
                    }
                    tmem_st16(at_s + 16 * x, p);                          // over scores that have been read
                }
            };
            if (full) block(std::false_type{}); else block(std::true_type{});
            if constexpr (!CODES) {
                if (odd) {
                    tmem_wait_st();
#pragma unroll 1
                    for (uint32_t p16 = 0; p16 < BP / 16; ++p16) {
                        uint32_t w[16];
                        tmem_ld16(at_s + 8 * (p16 & ~1u), w);             // (two sixteens at a time)
                        tmem_wait_ld();
                        const uint32_t p = min(p0 + 16 * p16, last & ~15u);
                        bool bad = false;
                        const __nv_bfloat16* v = static_cast<const __nv_bfloat16*>(c.v) + c.row(page_of(c, b, seq, p, bad), kvh, p & (c.size() - 1)) * DIM;
#pragma unroll 1
                        for (uint32_t col = 0; col < DIM; col += 16) {
                            uint32_t o[16];
                            tmem_ld16(at_o + col, o);
                            tmem_wait_ld();
#pragma unroll
                            for (uint32_t i = 0; i < 16; ++i) {
                                const float2 x = unpack2<false>(p16 & 1 ? w[8 + i / 2] : w[i / 2]);
                                if (sees(p0 + 16 * p16 + i))
#pragma unroll
                                    for (int d = 0; d < 16; ++d) o[d] = __float_as_uint(fmaf(i & 1 ? x.y : x.x, __bfloat162float(v[i * DIM + col + d]), __uint_as_float(o[d])));
                            }
                            __syncwarp();
                            tmem_st16(at_o + col, o);
                            tmem_wait_st();
                        }
                    }
                }
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[tile]);
        }
        if (ok) ok = __all_sync(0xffffffffu, wait(&o_done[tile], (nb - 1) & 1, status));
        if (ok) {
            tc_fence_after();
            const float l = f2_sum(sum), back = CODES ? unit * (1.0f / 4096.0f) : 1.0f, inv = sh.chunks > 1 ? back : l == 0.f ? 0.f : back / l;
            const size_t orow = static_cast<size_t>(span.row0) + (live ? tok : tok0), head = static_cast<size_t>(kvh) * sh.group + (live ? row % sh.group : 0);
            OUT* dst = out + orow * sh.ldo + head * DIM;
            const size_t at_part = (orow * sh.heads + head) * sh.chunks + chunk;
            const bool wide = reinterpret_cast<uintptr_t>(dst) % 16 == 0;
            if (sh.chunks > 1 && live) *reinterpret_cast<float2*>(part_ml + 2 * at_part) = make_float2(mx, l);
#pragma unroll 1
            for (uint32_t col = 0; col < DIM; col += 32) {
                uint32_t o[32];
                tmem_ld32(at_o + col, o);
                tmem_wait_ld();
                if (live && sh.chunks > 1) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        reinterpret_cast<float4*>(part + at_part * DIM + col)[i] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                                                                               __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                } else if (live) {
                    __align__(16) OUT h[32];
#pragma unroll
                    for (int i = 0; i < 32; ++i) h[i] = out_value<OUT>(l == 0.f ? 0.f : __uint_as_float(o[i]) * inv, clipped);
                    if (wide) {
#pragma unroll
                        for (int i = 0; i < static_cast<int>(2 * sizeof(OUT)); ++i) reinterpret_cast<uint4*>(dst + col)[i] = reinterpret_cast<const uint4*>(h)[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) dst[col + i] = h[i];
                    }
                }
                __syncwarp();                                             // the next load from tensor memory is the whole warp's
            }
        }
        }
        tc_fence_before();
    }
    if (clipped) atomicOr(status, STATUS_X_CLIPPED);
    __syncthreads();
    if (warp == SOFTMAX_WARPS + LOAD_WARPS) { tc_fence_after(); tmem_dealloc(tmem, COLS); }
}

template <int DIM, bool CODES, typename Q, typename OUT>
cudaError_t launch(const AttendCall& a) {
    constexpr uint32_t smem = tiles_smem<DIM>();
    static PerDeviceFlag flag;
    const auto kern = attend_tiles_kernel<DIM, CODES, Q, OUT>;
    if (const cudaError_t e = ensure_max_dynamic_smem(kern, smem, flag); e != cudaSuccess) return e;
    const uint32_t group = a.heads / a.c.kv_heads, tokens = ROWS / group;
    const uint64_t tiles = a.b.rows / (2 * tokens) + std::min(a.b.seqs, a.b.rows);      // at most: each sequence's last tile may be a part
    if (tiles * a.c.kv_heads > 0x7fffffffull) return cudaErrorInvalidValue;
    const bool wide = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.ldq % (16 / sizeof(Q)) == 0;
    const Shape sh{a.heads, group, tokens, a.ldq, a.ldo, a.chunk >> BP_LOG, a.chunks, wide};
    kern<<<dim3(static_cast<uint32_t>(tiles) * a.c.kv_heads, a.chunks), THREADS, smem, a.st>>>(a.c, a.b, a.look, sh, static_cast<const Q*>(a.q), static_cast<OUT*>(a.out), a.part, a.part_ml,
                                                                                              a.status);
    return cudaGetLastError();
}
template <int DIM, bool CODES, typename Q>
cudaError_t launch_out(const AttendCall& a) {
    return a.out_dtype == HF2Q_DT_F32 ? launch<DIM, CODES, Q, float>(a) : a.out_dtype == HF2Q_DT_F16 ? launch<DIM, CODES, Q, __half>(a) : launch<DIM, CODES, Q, __nv_bfloat16>(a);
}
template <int DIM, bool CODES>
cudaError_t launch_q(const AttendCall& a) {
    return a.q_dtype == HF2Q_DT_F32 ? launch_out<DIM, CODES, float>(a) : launch_out<DIM, CODES, __nv_bfloat16>(a);
}

}  // namespace

cudaError_t paged::launch_attend_tiles(const AttendCall& a, uint32_t dim, bool codes) {
    return dim == 128 ? (codes ? launch_q<128, true>(a) : launch_q<128, false>(a)) : (codes ? launch_q<64, true>(a) : launch_q<64, false>(a));
}

}  // namespace hf2q
