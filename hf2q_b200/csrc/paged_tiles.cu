// Attention over a paged cache for many rows of a sequence: portions of prompts, drafts of several heads, on the 5th-generation tensor cores.
//
// One CTA owns two tiles of 128 rows = TOK tokens x the group of query heads of one KV head (TOK = 128 / group), and walks the positions
// that they see in blocks of 64:
//
//   warps 8-11   loaders of the keys, warps 12-15 of the values, each block once for both tiles, as 16-bit operands with the 128-byte swizzle in four
//                places.  Codes pass through registers and become exact f16 whole numbers, the next two blocks' loads already under way; bf16
//                is copied asynchronously, three blocks ahead.  K is [position][dim], the K-major B operand of the scores; V has the same layout,
//                read MN-major as the B operand of the output.
//   warps 16, 17 issue the products of a tile each, S = Q K^T and O += P V; the scores of the next block are ready when the softmax of this one ends.
//                (One warp for both tiles was the chain that everything waited for: a wait, a vote and a commit are 100 to 200 cycles.)  The second
//                tile starts half a round behind the first, so that one takes exponentials while the other loads, stores and waits.
//   warps 0-3    softmax of the first tile, a thread to a row: scores from tensor memory, exponentials in f32, P back as the 16-bit A
//   warps 4-7    operand in the place of S.  The same for the second tile.  One pass: weights are taken against the maximum of earlier blocks, and only
//                when a row's weights of a block add up to more than MOST is the maximum taken anew and the output row rescaled.
//
// Tensor memory: S 2 x 2 x 64 columns, O 2 x dim.  Codes: the scale of K multiplies the f32 score; the weight is p * v_scale * UNITS / U in f16, U
// a power of two above all value scales of the blocks so far, which the loaders keep: it grows seldom, and the output is rescaled
// with it; below the f16 normal numbers p * v_scale is off by at most 2^-28 of the largest value scale.  What a row does not see gets weight 0 by selection, whatever its scales and scores are.  bf16 values
// that are infinite or NaN in blocks that only some rows see would turn a weight of 0 into NaN: the loaders find them, hand zeros to the
// product, and the rows that see them add them up one by one.
//
// Queries and weights are rounded to the 16 bits that the products take, maxima, sums and outputs are f32, as in paged_step.cu; the errors
// against 64 bits are the same there and here.
//
// Measured (32 query heads of 8 KV heads, dim 128): 4096 rows behind 12288 positions of codes 1.37 ms, 700 TFLOP/s or 0.42 of the matrix rate, of bf16 1.16 ms,
// 830 TFLOP/s; six sequences of up to 701 rows, window 2048, bf16 188 us, 530 TFLOP/s; 64 rows behind 32768 positions of codes 75 us.  A block takes a CTA 1.7 us with codes and 1.4
// with bf16, where its products alone are 0.6.  What the rest is, from copies with parts left out: shared memory (Q is read again for 64 columns, scales
// are read by every warp; half of a round), and the chain from scores to weights to output of a tile, which two tiles hide only in part.  Blocks of
// 128 positions read Q half as often but leave one S a tile: long prompts 3 % faster, windows and short parts 10 % slower.  Short calls
// are bound by their ends: 12 us for launch, page numbers, Q, the first block and the output.
#include <math_constants.h>

#include <type_traits>

#include "paged_bits.cuh"
#include "paged_common.cuh"
#include "tc_common.cuh"

namespace hf2q {
using namespace paged;
using namespace tc;
namespace {

constexpr uint32_t ROWS = 128, BP_LOG = 6, BP = 1 << BP_LOG, STAGES = 4, SLOTS = 8, PANEL = BP * 128;
constexpr uint32_t SOFTMAX_WARPS = 8, LOAD_WARPS = 4, ISSUE_WARP = SOFTMAX_WARPS + 2 * LOAD_WARPS, THREADS = (ISSUE_WARP + 4) * 32, COLS = 512;
// Registers of a thread: 96 at launch; the softmax threads take 48 more, which the loaders and the issuing group of four warps give up (2 x 144 + 2 x 72
// + 48 = 5 x 96).
constexpr int SOFTMAX_REGS = 144, LOAD_REGS = 72, ISSUE_REGS = 48;
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr uint32_t APART = 8;
template <int DIM> constexpr uint32_t tiles_smem() { return 2 * ROWS * DIM * 2 + 2 * STAGES * BP * DIM * 2 + 1024; }

__device__ __forceinline__ void claim_columns(uint32_t* slot) {           // by one warp; every other CTA of the SM gives its own back by itself
    tmem_alloc(slot, COLS);
    tmem_relinquish();
}
__device__ __forceinline__ bool elected() {                               // one lane of a whole warp
    uint32_t yes;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
    return yes != 0;
}
// The bounded wait (about a second) in few instructions: the instruction cache of a scheduler serves all roles.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
    if (mbar_try_wait(bar, parity)) return true;
    const long long t0 = clock64();
    while (!mbar_try_wait_parked(bar, parity, 2000u)) {
        if (clock64() - t0 > (1ll << 31)) {
            atomicOr(status, STATUS_WAIT_TIMEOUT);
            return false;
        }
    }
    return true;
}
// all warps that count on `bar` have come here for the n-th time (false: the wait ran out)
__device__ __forceinline__ bool warps_meet(uint64_t* bar, uint32_t n, uint32_t lane, uint32_t* status) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
    return __all_sync(0xffffffffu, wait(bar, n & 1, status));
}
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {       // zeros past `bytes`
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
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
    uint32_t heads, group, inv_group, tokens;           // inv_group: r * inv_group >> 16 = r / group for r < 128; tokens of a tile
    uint32_t ldq, ldo, chunk_blocks, chunks;
    bool wide_q, shrink;
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
    constexpr uint32_t Q_PANEL = ROWS * 128, Q_BYTES = ROWS * DIM * 2, KV_BYTES = BP * DIM * 2, COL_O = 4 * BP;
    constexpr float MOST = 0x1p11f, UNITS = 16.0f;      // what a block's weights may add up to; a weight is p * v_scale * UNITS / U
    extern __shared__ uint8_t raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~static_cast<uintptr_t>(1023));
    uint8_t *qs = smem, *ks = smem + 2 * Q_BYTES, *vs = ks + STAGES * KV_BYTES;
    // Scales of a block have a slot and a barrier each.  Slot j % 8 is written next for block j + 8, after K(j + 4) left its place, that is after
    // S(j + 4), which follows the output of block j + 2 and so every softmax warp's reading of block j.
    __shared__ __align__(16) float s_ks[SLOTS][BP], s_vs[SLOTS][BP];
    __shared__ float s_unit[SLOTS];
    __shared__ uint32_t s_odd[STAGES];
    __shared__ uint64_t k_full[STAGES], v_full[STAGES], k_free[STAGES], v_free[STAGES], sc_full[SLOTS], s_full[4], p_full[4], o_done[2], o_all[2], meet, apart;      // s, p: tile * 2 + (block & 1)
    __shared__ uint32_t tmem_slot;
    const uint32_t kvh = blockIdx.x % c.kv_heads, chunk = blockIdx.y, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint32_t seq = 0, tok0 = 0;
    pdl_wait();
    if (blockIdx.x == 0 && chunk == 0)                                    // (a sequence that does not fit may have no tile to say so)
        for (uint32_t s = threadIdx.x; s < b.seqs; s += THREADS)
            if (span_of(b, c.shift, s).bad) atomicOr(status, STATUS_BAD_PAGE);
    if (!find_tile(b, c.shift, 2 * sh.tokens, (gridDim.x - 1 - blockIdx.x) / c.kv_heads, seq, tok0)) return;      // (the tiles with the most positions first)
    const Span span = span_of(b, c.shift, seq);
    const uint32_t end_tok = min(tok0 + 2 * sh.tokens, span.rows), tiles = end_tok - tok0 > sh.tokens ? 2 : 1;
    const uint32_t lost = span.rows > span.length ? span.rows - span.length : 0;      // rows in front of position 0: they see nothing
    const uint32_t before = span.length - span.rows;                      // position of token 0 (wraps where rows are lost)
    const bool any = end_tok > lost;
    const uint32_t first = any ? before + max(tok0, lost) : 0, last = any ? before + end_tok - 1 : 0;
    const Blocks blocks = blocks_of(look, first, last, BP_LOG);
    const uint32_t part_blocks = part_units(b, BP_LOG, sh.chunk_blocks, sh.chunks, 4, sh.shrink);
    const uint32_t lo = static_cast<uint32_t>(min(static_cast<uint64_t>(chunk) * part_blocks, static_cast<uint64_t>(blocks.count)));
    const uint32_t nb = any ? min(part_blocks, blocks.count - lo) : 0;
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
        for (uint32_t i = 0; i < STAGES; ++i) {
            mbar_init(&k_full[i], LOAD_WARPS);
            mbar_init(&v_full[i], LOAD_WARPS);
            mbar_init(&k_free[i], tiles);
            mbar_init(&v_free[i], tiles);
            s_odd[i] = 0;
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&o_done[i], 1);
            mbar_init(&o_all[i], 1);
        }
        for (uint32_t i = 0; i < SLOTS; ++i) mbar_init(&sc_full[i], 2 * LOAD_WARPS);
        mbar_init(&meet, LOAD_WARPS);
        mbar_init(&apart, 1);
        mbar_fence_init();
    }
    if (warp == ISSUE_WARP) claim_columns(&tmem_slot);
    // Q: two tiles of 128 rows in 16 bits; a negative scale is taken over by q, so that the largest product is the largest score
    bool clipped = false;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < tiles * ROWS * (DIM / 8); i += THREADS) {
        const uint32_t ch = i % (DIM / 8), r = i / (DIM / 8), tile = r >> 7, rr = r & 127, in_tile = rr * sh.inv_group >> 16, tok = tok0 + tile * sh.tokens + in_tile;
        uint4 w = make_uint4(0u, 0u, 0u, 0u);
        if (in_tile < sh.tokens && tok < end_tok) {
            float e[8];
            load8(q + static_cast<size_t>(span.row0 + tok) * sh.ldq + static_cast<size_t>(kvh * sh.group + rr - in_tile * sh.group) * DIM + 8 * ch, sh.wide_q, e);
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
    pdl_trigger();                                                        // (not before the columns are held: a launch behind may take them and then wait for this one)
    const uint32_t tmem = tmem_slot;
    const float scale = fabsf(look.scale);

    if (warp >= SOFTMAX_WARPS && warp < ISSUE_WARP) {
        // Four warps for the keys, four for the values.
        fewer_registers<LOAD_REGS>();
        constexpr uint32_t CH = CODES ? DIM / 16 : DIM / 8, RP = LOAD_WARPS * 32 / CH, NP = BP / RP;      // 16-byte chunks of a row; rows of a pass; passes
        constexpr uint32_t ROW = DIM * (CODES ? 1 : 2), G = BP / 16;
        const bool keys = warp < SOFTMAX_WARPS + LOAD_WARPS;
        const uint32_t tid = threadIdx.x & 127, ch = tid % CH, row0 = tid / CH, last16 = last & ~15u;
        uint8_t* stages = keys ? ks : vs;
        uint64_t *full_bars = keys ? k_full : v_full, *free_bars = keys ? k_free : v_free;
        bool bad = false, ok = true;
        // Where eight blocks lie: lane 4 i + g has positions 16 g .. 16 g + 15 of block 8 m + i, in sixteens of rows (the last sixteen again past
        // the last position).  The eight blocks behind are asked for as these come into use.
        auto places = [&](uint32_t m) {
            const uint32_t j = m * (32 / G) + lane / G, p = min((blocks.at(lo + min(j, nb - 1)) << BP_LOG) + 16 * (lane % G), last16);
            return static_cast<uint32_t>(c.row(page_of(c, b, seq, p, bad), kvh, p & (c.size() - 1)) >> 4);
        };
        uint32_t here = places(0), there = places(1);
        auto reach_block = [&](uint32_t j) {                              // (blocks are taken in order)
            if (j % (32 / G) == 0 && j) { here = there; there = places(j / (32 / G) + 1); }
        };
        const uint8_t* mine = static_cast<const uint8_t*>(keys ? c.k : c.v) + (row0 & 15) * ROW + 16 * ch;
        auto place = [&](uint32_t j, uint32_t i) {                        // this thread's chunk of pass i of block j
            const uint32_t at16 = __shfl_sync(0xffffffffu, here, (j * G & 31) + (RP <= 16 ? RP * i >> 4 : (RP * i + row0) >> 4));
            return mine + static_cast<uint64_t>(at16) * (16 * ROW) + (RP * i & 15) * ROW;
        };
        if constexpr (CODES) {
            // Two blocks ahead, a set of registers for even and one for odd blocks.  Every warp holds the scales of the whole block, two positions a
            // lane, for the largest of V's; a quarter of the lanes stores.
            const float* scales = keys ? c.k_scale : c.v_scale;
            uint4 x[2][NP];
            float2 sc[2];
            float unit = 0x1p-100f;
            auto load = [&](uint32_t j, uint32_t u) {
#pragma unroll
                for (uint32_t i = 0; i < NP; ++i) x[u][i] = __ldcg(reinterpret_cast<const uint4*>(place(j, i)));
                sc[u] = __ldcg(reinterpret_cast<const float2*>(scales + (static_cast<uint64_t>(__shfl_sync(0xffffffffu, here, (j * G & 31) + (lane >> 3))) * 16 + (2 * lane & 15))));
            };
            load(0, 0);
            if (nb > 1) load(1, 1);
#pragma unroll 1
            for (uint32_t j0 = 0; j0 < nb && ok; j0 += 2) {
#pragma unroll
                for (uint32_t u = 0; u < 2; ++u) {
                    const uint32_t j = j0 + u, st = j % STAGES, slot = j % SLOTS;
                    if (j >= nb || !ok) break;
                    if (j >= STAGES) ok = wait(&free_bars[st], (j / STAGES - 1) & 1, status);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) store_codes(stages + st * KV_BYTES, RP * i + row0, ch, x[u][i]);
                    const float2 s = sc[u];
                    if (j + 2 < nb) {
                        reach_block(j + 2);
                        load(j + 2, u);
                    }
                    float f = scale;
                    if (!keys) {
                        const uint32_t p0 = blocks.at(lo + j) << BP_LOG;
                        const bool all = all_see(look, first, last, p0, BP);
                        float top = 0.f;
                        if (fabsf(s.x) < CUDART_INF_F && (all || some_see(look, first, last, p0 + 2 * lane))) top = fabsf(s.x);
                        if (fabsf(s.y) < CUDART_INF_F && (all || some_see(look, first, last, p0 + 2 * lane + 1))) top = fmaxf(top, fabsf(s.y));
                        unit = fmaxf(unit, unit_above(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)))));       // (of numbers >= 0 the order is that of their bits)
                        f = __uint_as_float((258u << 23) - __float_as_uint(unit));          // UNITS / unit, of powers of two
                        if (tid == 0) s_unit[slot] = unit;
                    }
                    if (lane >> 3 == (warp & 3)) *reinterpret_cast<float2*>(&(keys ? s_ks : s_vs)[slot][2 * lane]) = make_float2(s.x * f, s.y * f);
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sc_full[slot]);
                        mbar_arrive(&full_bars[st]);
                    }
                }
            }
        } else {
            const uint32_t to0 = smem_u32(stages) + chunk_at(row0, ch, PANEL);       // (a pass is 8 rows or a multiple: the swizzle of a thread's chunk stays)
            uint32_t met = 0;
            constexpr int AHEAD = 3;                                      // blocks on their way: the next is asked for when the first was handed over
            auto bring = [&](uint32_t j) {                                // block j, as a group of copies
                const uint32_t st = j % STAGES, p0 = blocks.at(lo + j) << BP_LOG, to = to0 + st * KV_BYTES;
                reach_block(j);
                if (j >= STAGES) ok = wait(&free_bars[st], (j / STAGES - 1) & 1, status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) return;
                if (keys || all_see(look, first, last, p0, BP)) {
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) copy16(to + RP * i * 128, place(j, i), 16);
                } else {                                                  // (values that nobody sees are zeros)
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) copy16(to + RP * i * 128, place(j, i), some_see(look, first, last, p0 + RP * i + row0) ? 16 : 0);
                }
                copies_close();
            };
            for (uint32_t j = 0; j < AHEAD; ++j) {
                if (j < nb) bring(j); else copies_close();
            }
#pragma unroll 1
            for (uint32_t j = 0; j < nb && ok; ++j) {
                const uint32_t st = j % STAGES, p0 = blocks.at(lo + j) << BP_LOG;
                copies_wait<AHEAD - 1>();
                if (!keys && !all_see(look, first, last, p0, BP) && first != last) {
                    uint8_t* to = stages + st * KV_BYTES + chunk_at(row0, ch, PANEL);
                    bool odd = false;
#pragma unroll
                    for (uint32_t i = 0; i < NP; ++i) {
                        const uint4 w = *reinterpret_cast<const uint4*>(to + RP * i * 128);
                        odd |= holds_nonfinite(w.x) || holds_nonfinite(w.y) || holds_nonfinite(w.z) || holds_nonfinite(w.w);
                    }
                    // (s_odd of the block before in this place has been read: its V left.)  The loaders agree, and then none keeps its part.
                    if (tid == 0) s_odd[st] = 0;
                    ok = warps_meet(&meet, met++, lane, status);
                    if (odd) s_odd[st] = 1;
                    ok = ok && warps_meet(&meet, met++, lane, status);
                    if (!ok) break;
                    if (*static_cast<volatile uint32_t*>(&s_odd[st]))
#pragma unroll
                        for (uint32_t i = 0; i < NP; ++i) *reinterpret_cast<uint4*>(to + RP * i * 128) = make_uint4(0u, 0u, 0u, 0u);
                }
                proxy_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(&full_bars[st]);
                if (j + AHEAD < nb) bring(j + AHEAD); else copies_close();
            }
            copies_wait<0>();
        }
        if (bad) atomicOr(status, STATUS_BAD_PAGE);
    } else if (warp >= ISSUE_WARP) {
        fewer_registers<ISSUE_REGS>();
        // A warp for each tile.  D f32; A and B f16 or bf16; M = 128; S: both K-major, N = 64; O: B MN-major, N = dim.  The whole warp goes through the
        // waits, so that addresses and descriptors stay in uniform registers; one lane issues.
        constexpr uint32_t ID = (1u << 4) | (CODES ? 0u : (1u << 7) | (1u << 10)) | ((ROWS >> 4) << 24), ID_S = ID | ((BP >> 3) << 17), ID_O = ID | (1u << 16) | ((DIM >> 3) << 17);
        const uint32_t t = warp - ISSUE_WARP, n = t < __shfl_sync(0xffffffffu, tiles, 0) ? __shfl_sync(0xffffffffu, nb, 0) : 0, base = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_desc = smem_desc_sw128(smem_u32(qs)) + t * (Q_BYTES >> 4), k_desc = smem_desc_sw128(smem_u32(ks)), v_desc = smem_desc_mn_sw128(smem_u32(vs), PANEL);
        const bool leader = elected();
        bool ok = true;
        // The second tile starts when the first has its first weights: half a round later, so that one takes exponentials while the other loads, stores
        // and waits.  (Few blocks end sooner side by side.)
        if (t == 1 && n >= APART) ok = wait(&apart, 0, status);
        // S(j), then O += P(j - 1) V: the next scores are ready when the softmax of this block ends
#pragma unroll 1
        for (uint32_t j = 0; n && j <= n; ++j) {
            const uint32_t st = j % STAGES, was = (j - 1) % STAGES;
            if (j < n) {
                if (j >= 2) {                                             // P(j - 2) is read: S(j) takes its place; and the values' place is free
                    ok = wait(&o_done[t], j & 1, status);
                    if (leader && ok) mbar_arrive(&v_free[(j - 2) % STAGES]);         // (the loader may want it before it says that K(j) is there)
                }
                if (ok) ok = wait(&k_full[st], (j / STAGES) & 1, status);
                if (!__all_sync(0xffffffffu, ok)) break;
                tc_fence_after();
                if (leader) {
                    const uint64_t kd = k_desc + st * (KV_BYTES >> 4);
                    const uint32_t d = base + (2 * t + (j & 1)) * BP;
#pragma unroll
                    for (uint32_t kk = 0; kk < DIM / 16; ++kk)
                        umma_ss(d, q_desc + (kk >> 2) * (Q_PANEL >> 4) + 2 * (kk & 3), kd + (kk >> 2) * (PANEL >> 4) + 2 * (kk & 3), ID_S, kk ? 1u : 0u);
                    tc_commit(&s_full[2 * t + (j & 1)]);
                }
                __syncwarp();
            }
            if (j == 0) continue;
            ok = wait(&v_full[was], ((j - 1) / STAGES) & 1, status);
            if (ok) ok = wait(&p_full[2 * t + ((j - 1) & 1)], ((j - 1) >> 1) & 1, status);
            if (!__all_sync(0xffffffffu, ok)) break;
            tc_fence_after();
            if (leader) {
                const uint64_t vd = v_desc + was * (KV_BYTES >> 4);
                const uint32_t p = base + (2 * t + ((j - 1) & 1)) * BP;
#pragma unroll
                for (uint32_t kk = 0; kk < BP / 16; ++kk) umma_ts(base + COL_O + t * DIM, p + 8 * kk, vd + kk * (16 * 128 >> 4), ID_O, 1u);
                tc_commit(j == n ? &o_all[t] : &o_done[t]);               // (the last output has a barrier to itself: who waits for it may come late)
            }
            __syncwarp();
        }
    } else {
        more_registers<SOFTMAX_REGS>();
        const uint32_t tile = warp / 4, row = threadIdx.x & 127, at = tmem + (((warp & 3) * 32u) << 16), at_o = at + COL_O + tile * DIM;
        const uint32_t in_tile = row * sh.inv_group >> 16, tile_tok = tok0 + tile * sh.tokens, tile_end = min(tile_tok + sh.tokens, end_tok), tok = tile_tok + in_tile;
        const bool live = in_tile < sh.tokens && tok < end_tok, held = live && tok >= lost;
        const uint32_t seen = before + max(min(tok, tile_end - 1), lost);          // (rows that are not there compute on zeros and are not stored)
        const uint32_t t_first = before + max(tile_tok, lost), t_last = before + max(tile_end - 1, lost);
        // the row sees positions from `low` on, `reach` more, and those below `firsts`
        const uint32_t low = !held ? 1u << 31 : look.window && seen >= look.window ? seen - look.window + 1 : 0, reach = held ? seen - low : 0;
        const uint32_t firsts = held && look.window ? min(look.sinks, seen + 1) : 0;
        const auto sees = [&](uint32_t p) { return static_cast<bool>((p - low <= reach) | (p < firsts)); };
        // blocks that start at full0 .. full0 + full_reach are seen whole by every row of the tile (blocks of the first positions beside a window are not
        // counted here)
        const uint32_t from = look.window && t_last >= look.window ? t_last - look.window + 1 : 0;
        const bool some = tile_tok >= lost && t_first >= from + (BP - 1);
        const uint32_t full0 = some ? from : 1u << 31, full_reach = some ? t_first - (BP - 1) - from : 0;
        float mx = held ? -CUDART_INF_F : 0.f, unit = 0x1p-100f;          // (a row that sees nothing needs no maximum)
        f2 sum = 0;
        bool ok = true;
        const uint32_t n = tile < tiles ? nb : 0;
        const f2 sc2 = f2_both(scale);
        auto scale_output = [&](uint32_t j, float corr) {                 // what blocks before j gave
            ok = ok && __all_sync(0xffffffffu, wait(&o_done[tile], (j - 1) & 1, status));
            if (!ok) return;
            tc_fence_after();
#pragma unroll 1
            for (uint32_t col = 0; col < DIM; col += 16) {
                uint32_t o[16];
                tmem_ld16(at_o + col, o);
                tmem_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
                tmem_st16(at_o + col, o);
            }
            tmem_wait_st();
        };
        {
            uint32_t zero[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) zero[i] = 0u;
#pragma unroll
            for (uint32_t col = 0; col < DIM; col += 32) tmem_st32(at_o + col, zero);
        }
#pragma unroll 1
        for (uint32_t j = 0; j < n; ++j) {
            const uint32_t slot = j % SLOTS, st = j % STAGES, p0 = blocks.at(lo + j) << BP_LOG, at_s = at + (2 * tile + (j & 1)) * BP;
            const bool full = p0 - full0 <= full_reach;
            ok = wait(&s_full[2 * tile + (j & 1)], (j >> 1) & 1, status);
            if constexpr (CODES) { if (ok) ok = wait(&sc_full[slot], (j / SLOTS) & 1, status); }
            bool odd = false;
            if constexpr (!CODES) {
                if (!all_see(look, first, last, p0, BP) && first != last) {
                    if (ok) ok = wait(&v_full[st], (j / STAGES) & 1, status);
                    odd = *static_cast<volatile uint32_t*>(&s_odd[st]) != 0;
                }
            }
            if (ok && row == 0) mbar_arrive(&k_free[st]);                 // the scores are there: the keys' place is free
            ok = __all_sync(0xffffffffu, ok);                             // (and the warp is together again, as accesses to tensor memory want it)
            if (!ok) break;
            tc_fence_after();
            const ulonglong2 *k2 = reinterpret_cast<const ulonglong2*>(s_ks[slot]), *v2 = reinterpret_cast<const ulonglong2*>(s_vs[slot]);
            if constexpr (CODES) {
                const float above = s_unit[slot];
                if (above != unit) {
                    if (j) scale_output(j, unit / above);
                    unit = above;
                }
            }
            // weights of 32 columns -> tensor memory, over scores that have been read
            auto store = [&](uint32_t x, const f2* e, auto masked) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float2 w = f2_parts(e[i]);
                    if constexpr (CODES) {
                        const ulonglong2 v = v2[8 * x + i / 2];
                        w = f2_parts(f2_mul(e[i], i & 1 ? v.y : v.x));
                        if constexpr (decltype(masked)::value) {          // (also where the scale of V is infinite or NaN)
                            if (!sees(p0 + 32 * x + 2 * i)) w.x = 0.f;
                            if (!sees(p0 + 32 * x + 2 * i + 1)) w.y = 0.f;
                        }
                    }
                    p[i] = pack2<CODES>(w.x, w.y);
                }
                if constexpr (decltype(masked)::value) __syncwarp();
                tmem_st16(at_s + 16 * x, p);
            };
            auto factor = [&](uint32_t x, int i) {
                if constexpr (!CODES) return sc2;
                const ulonglong2 k = k2[8 * x + i / 2];
                return static_cast<f2>(i & 1 ? k.y : k.x);
            };
            if (full && !__any_sync(0xffffffffu, mx == -CUDART_INF_F)) {
                // All rows have a maximum of earlier blocks: weights are taken against that, in one pass, and as long as they add up to no more
                // than MOST it stays (what they add up to is at least the largest of them).
                f2 e[BP / 2], part;
                for (bool again = false;; again = true) {
                    uint32_t r[2][32];
                    tmem_ld32(at_s, r[0]);
                    tmem_ld32(at_s + 32, r[1]);
                    tmem_wait_ld();
                    const f2 nm = f2_both(-mx);
                    f2 s0 = 0, s1 = 0;
#pragma unroll
                    for (int i = 0; i < static_cast<int>(BP / 2); ++i) {
                        const float2 d = f2_parts(f2_fma(f2_of(__uint_as_float(r[i / 16][2 * (i % 16)]), __uint_as_float(r[i / 16][2 * (i % 16) + 1])), factor(i / 16, i % 16), nm));
                        e[i] = f2_of(ex2(d.x), ex2(d.y));
                        if (i & 1) s1 = f2_add(s1, e[i]); else s0 = f2_add(s0, e[i]);
                    }
                    part = f2_add(s0, s1);
                    if (again || !__any_sync(0xffffffffu, f2_sum(part) > MOST)) break;
                    // a new maximum: output and sums so far follow
                    float top = 0.f;
#pragma unroll 1
                    for (uint32_t x = 0; x < BP / 32; ++x) {
                        tmem_ld32(at_s + 32 * x, r[0]);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 d = f2_parts(f2_fma(f2_of(__uint_as_float(r[0][2 * i]), __uint_as_float(r[0][2 * i + 1])), factor(x, i), nm));
                            top = fmaxf(top, fmaxf(d.x, d.y));
                        }
                    }
                    const float corr = ex2(-top);
                    mx += top;
                    sum = f2_mul(sum, f2_both(corr));
                    scale_output(j, corr);                                // (there is a block before: it gave the maximum)
                }
                sum = f2_add(sum, part);
                store(0, e, std::false_type{});
                store(1, e + 16, std::false_type{});
            } else {
                // masks, or the first block that a row sees: twice over the scores
                float top = -CUDART_INF_F;
                auto score = [&](uint32_t x, int i, const uint32_t (&r)[32]) {
                    float2 v = f2_parts(f2_mul(f2_of(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), factor(x, i)));
                    if (!sees(p0 + 32 * x + 2 * i)) v.x = -CUDART_INF_F;
                    if (!sees(p0 + 32 * x + 2 * i + 1)) v.y = -CUDART_INF_F;
                    return v;
                };
#pragma unroll 1
                for (uint32_t x = 0; x < BP / 32; ++x) {
                    uint32_t r[32];
                    tmem_ld32(at_s + 32 * x, r);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) { const float2 v = score(x, i, r); top = fmaxf(top, fmaxf(v.x, v.y)); }
                    __syncwarp();
                }
                const bool grew = top > mx;
                if (__any_sync(0xffffffffu, grew)) {
                    const float to = grew ? top : mx, corr = grew ? ex2(mx - to) : 1.0f;
                    sum = f2_mul(sum, f2_both(corr));
                    mx = to;
                    if (j) scale_output(j, corr);
                }
                const float zero = mx == -CUDART_INF_F ? 0.f : mx;
#pragma unroll 1
                for (uint32_t x = 0; x < BP / 32; ++x) {
                    uint32_t r[32];
                    tmem_ld32(at_s + 32 * x, r);
                    tmem_wait_ld();
                    f2 e[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float2 v = score(x, i, r);
                        e[i] = f2_of(ex2(v.x - zero), ex2(v.y - zero));
                        sum = f2_add(sum, e[i]);
                    }
                    store(x, e, std::true_type{});
                }
            }
            tmem_wait_st();
            if constexpr (!CODES) {
                if (odd) {
                    // What blocks before gave has to be there before it is read and written back (S(j), which this warp has seen, says nothing about it).
                    if (j) ok = __all_sync(0xffffffffu, ok && wait(&o_done[tile], (j - 1) & 1, status));
                    if (!ok) break;
                    tc_fence_after();
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
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[2 * tile + (j & 1)]);
            if (threadIdx.x == 0 && j == 0) mbar_arrive(&apart);
        }
        if (ok && n) ok = wait(&o_all[tile], 0, status);
        ok = __all_sync(0xffffffffu, ok && n);
        if (ok) {
            tc_fence_after();
            const float l = f2_sum(sum), back = CODES ? unit * (1.0f / UNITS) : 1.0f, inv = sh.chunks > 1 ? back : l == 0.f ? 0.f : back / l;
            const size_t orow = static_cast<size_t>(span.row0) + (live ? tok : tok0), head = static_cast<size_t>(kvh) * sh.group + (live ? row % sh.group : 0);
            OUT* dst = out + orow * sh.ldo + head * DIM;
            const size_t at_part = (orow * sh.heads + head) * sh.chunks + chunk;
            const bool wide = reinterpret_cast<uintptr_t>(dst) % 16 == 0;
            if (sh.chunks > 1) {
                // A thread has a row of numbers; parts are written by half-warps, half the columns at a time through what Q has left (a row by each thread
                // would be 32 lines a store).
                if (live) *reinterpret_cast<float2*>(part_ml + 2 * at_part) = make_float2(mx, l);
                const uint32_t rows_live = __ballot_sync(0xffffffffu, live);
                constexpr uint32_t HALF = DIM / 2, CH = HALF / 4;
                float4* stage = reinterpret_cast<float4*>(qs + tile * Q_BYTES + (warp & 3) * (Q_BYTES / 4));
#pragma unroll 1
                for (uint32_t half = 0; rows_live && half < 2; ++half) {
#pragma unroll 1
                    for (uint32_t c4 = 0; c4 < CH; c4 += 4) {
                        uint32_t o[16];
                        tmem_ld16(at_o + half * HALF + 4 * c4, o);
                        tmem_wait_ld();
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            stage[lane * CH + ((c4 + i) ^ (lane % CH))] = make_float4(__uint_as_float(o[4 * i]) * inv, __uint_as_float(o[4 * i + 1]) * inv,
                                                                                     __uint_as_float(o[4 * i + 2]) * inv, __uint_as_float(o[4 * i + 3]) * inv);
                    }
                    __syncwarp();
#pragma unroll 4
                    for (uint32_t r0 = 0; r0 < 32; r0 += 32 / CH) {
                        const uint32_t r = r0 + lane / CH, ch = lane % CH;
                        float* to = part + __shfl_sync(0xffffffffu, static_cast<unsigned long long>(at_part), r) * DIM + half * HALF + 4 * ch;
                        if (rows_live >> r & 1) *reinterpret_cast<float4*>(to) = stage[r * CH + (ch ^ (r % CH))];
                    }
                    __syncwarp();
                }
            } else {
#pragma unroll 1
                for (uint32_t col = 0; col < DIM; col += 16) {
                    uint32_t o[16];
                    tmem_ld16(at_o + col, o);
                    tmem_wait_ld();
                    if (live) {
                        __align__(16) OUT h[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) h[i] = out_value<OUT>(l == 0.f ? 0.f : __uint_as_float(o[i]) * inv, clipped);
                        if (wide) {
#pragma unroll
                            for (int i = 0; i < static_cast<int>(sizeof(OUT)); ++i) reinterpret_cast<uint4*>(dst + col)[i] = reinterpret_cast<const uint4*>(h)[i];
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; ++i) dst[col + i] = h[i];
                        }
                    }
                    __syncwarp();                                         // the next load from tensor memory is the whole warp's
                }
            }
        }
        tc_fence_before();
    }
    if (clipped) atomicOr(status, STATUS_X_CLIPPED);
    __syncthreads();
    if (warp == ISSUE_WARP) { tc_fence_after(); tmem_dealloc(tmem, COLS); }
}

template <int DIM, bool CODES, typename Q, typename OUT>
cudaError_t launch(const AttendCall& a) {
    constexpr uint32_t smem = tiles_smem<DIM>();
    static PerDeviceFlag flag;
    const auto kern = attend_tiles_kernel<DIM, CODES, Q, OUT>;
    if (const cudaError_t e = ensure_max_dynamic_smem(kern, smem, flag); e != cudaSuccess) return e;
    const uint32_t group = a.heads / a.c.kv_heads, tokens = ROWS / group;
    // at most: each sequence's last tile may be a part
    const uint64_t per = 2 * tokens, seqs = std::min(a.b.seqs, a.b.rows), tiles = std::min(a.b.rows / per + seqs, seqs * ((a.b.max_new + per - 1) / per));
    if (tiles * a.c.kv_heads > 0x7fffffffull) return cudaErrorInvalidValue;
    const bool wide = reinterpret_cast<uintptr_t>(a.q) % 16 == 0 && a.ldq % (16 / sizeof(Q)) == 0;
    const Shape sh{a.heads, group, 65536 / group + 1, tokens, a.ldq, a.ldo, a.chunk >> BP_LOG, a.chunks, wide, a.shrink};
    return launch_pdl(kern, dim3(static_cast<uint32_t>(tiles) * a.c.kv_heads, a.chunks), dim3(THREADS), smem, a.st, a.c, a.b, a.look, sh, static_cast<const Q*>(a.q),
                      static_cast<OUT*>(a.out), a.part, a.part_ml, a.status);
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
