// What writes and moves the pages of a paged key-value cache: rotary turn and append, copies of pages and of single rows.
//
// Append.  A pair (a, b) at position p with frequency f becomes (a cos pf - b sin pf, a sin pf + b cos pf).  The angle of a far position
// does not fit 32 bits (at position 10^6 half a unit in the last place of f32 is 0.03 rad), so that product, sine and cosine are
// taken in 64 bits, once per pair and CTA (a CTA a token; few tokens share their heads among several), and rounded to f32 together; the turn
// itself is f32, each product and sum rounded by itself.
// Bytes: scale = amax / 127 over the head, code = the nearest whole number of value * (127 / amax).
// Bound by bytes where there are many rows.  Measured (32 query heads of 8 KV heads, dim 128): three prompts of up to 2048 rows to codes 49 us, 4.5 TB/s (47.5 without
// a turn), to bf16 47.5 us; one token of 16 sequences 2.8 us, a launch.
//
// Copies.  Bound by bytes: 12 pages of 16 rows in 32 layers of codes, 26 MB, 4.4 us; 8192 rows in four layers of bf16, 269 MB, 45 us, 6.0 TB/s.
#include <math_constants.h>

#include "paged_common.cuh"
#include "seq_common.cuh"

namespace hf2q {
using namespace paged;
namespace {

struct Turn {
    const float* freq;
    const uint32_t* pos;
    uint32_t rot, halves;
    float factor;
};
struct AppendShape {
    uint32_t heads, ldx, ldq;
    bool wide_x, wide_q;                     // rows of x / q_out on 16-byte boundaries (8 for their 16-bit forms)
};

// The sequence that owns row t: the last one that starts at or before it.  All lanes of the warp get the same answer; b.seqs: none.
__device__ __forceinline__ uint32_t sequence_of(const Batch& b, uint32_t t) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t at = 0;
    for (uint32_t s0 = 0; s0 <= b.seqs; s0 += 32) {
        const bool before = s0 + lane <= b.seqs && b.start[s0 + lane] <= t;
        const uint32_t n = __popc(__ballot_sync(0xffffffffu, before));
        at += n;
        if (n < 32) break;
    }
    return at == 0 || at > b.seqs ? b.seqs : at - 1;
}

// V consecutive elements of a row (V 2 or 4)
template <int V> __device__ __forceinline__ void load_some(const float* p, bool wide, float (&e)[V]) {
    if (wide) {
        if constexpr (V == 4) { const float4 f = *reinterpret_cast<const float4*>(p); e[0] = f.x; e[1] = f.y; e[2] = f.z; e[3] = f.w; }
        else { const float2 f = *reinterpret_cast<const float2*>(p); e[0] = f.x; e[1] = f.y; }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = p[j];
    }
}
template <int V> __device__ __forceinline__ void load_some(const __nv_bfloat16* p, bool wide, float (&e)[V]) {
    if (wide) {
        uint32_t w[V / 2];
        if constexpr (V == 4) { const uint2 u = *reinterpret_cast<const uint2*>(p); w[0] = u.x; w[1] = u.y; }
        else w[0] = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
        for (int j = 0; j < V / 2; ++j) { e[2 * j] = seq::bf_lo(w[j]); e[2 * j + 1] = seq::bf_hi(w[j]); }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = __bfloat162float(p[j]);
    }
}
template <int V> __device__ __forceinline__ void store_some(float* p, bool wide, const float (&e)[V]) {
    if (wide) {
        if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(e[0], e[1], e[2], e[3]);
        else *reinterpret_cast<float2*>(p) = make_float2(e[0], e[1]);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = e[j];
    }
}
template <int V> __device__ __forceinline__ void store_some(__nv_bfloat16* p, bool wide, const float (&e)[V]) {
    __align__(8) __nv_bfloat16 h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = __float2bfloat16_rn(e[j]);
    if (wide) {
        if constexpr (V == 4) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(h);
        else *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(h);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) p[j] = h[j];
    }
}

// A CTA per row of the batch, or a share of its heads where the rows alone would leave SMs idle; a warp per head, dim / 32 elements a
// lane, the next head's load under way.
constexpr uint32_t AP_WARPS = 8;
template <int DIM, typename X, typename Q, bool CODES>
__global__ void __launch_bounds__(AP_WARPS * 32) append_kernel(Pool c, Batch b, Turn turn, AppendShape sh, const X* x, Q* q_out, uint32_t* status) {
    constexpr int V = DIM / 32;
    __shared__ float2 cs[DIM / 2];                                       // cosine, sine
    __shared__ __align__(16) float head[AP_WARPS][DIM];
    pdl_trigger();
    pdl_wait();
    const uint32_t t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, all = sh.heads + 2 * c.kv_heads;
    const uint32_t s = sequence_of(b, t);
    if (s == b.seqs) return;                                             // in front of the first sequence or behind the last
    const Span span = span_of(b, c.shift, s);
    const bool held = t - span.row0 < span.rows && span.length + (t - span.row0) >= span.rows;       // it has a position (padding in front has none)
    const uint32_t pos = held ? span.length - span.rows + (t - span.row0) : 0;
    bool bad = span.bad;
    const uint32_t page = held ? page_of(c, b, s, pos, bad) : 0;
    if (bad && threadIdx.x == 0) atomicOr(status, STATUS_BAD_PAGE);
    if (bad || !held) return;
    const uint32_t half = turn.rot / 2;
    const X* row = x + static_cast<size_t>(t) * sh.ldx;
    const uint32_t h0 = warp + blockIdx.y * AP_WARPS, step = gridDim.y * AP_WARPS;
    float e[V], later[V];                                                // a head, and the next one on its way
    if (h0 < all) load_some<V>(row + static_cast<size_t>(h0) * DIM + V * lane, sh.wide_x, later);
    if (threadIdx.x < half) {
        double sn, co;
        sincos(static_cast<double>(turn.pos ? turn.pos[t] : pos) * static_cast<double>(turn.freq[threadIdx.x]), &sn, &co);
        cs[threadIdx.x] = make_float2(static_cast<float>(co) * turn.factor, static_cast<float>(sn) * turn.factor);
    }
    __syncthreads();
    // cosine and sine of this lane's elements, the same for all heads; the sine with the sign that it has there
    float co[V], si[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const uint32_t i = V * lane + j;
        const bool second = turn.halves ? i >= half : (i & 1);
        const float2 w = i < turn.rot ? cs[turn.halves ? (second ? i - half : i) : i >> 1] : make_float2(1.f, 0.f);
        co[j] = w.x;
        si[j] = second ? w.y : -w.y;
    }
    // halves: the partner is the same element of another lane, or (halves that end inside a lane's elements) comes through shared memory
    const bool by_lane = half % V == 0;
    const uint32_t partner = V * lane < half ? lane + half / V : lane - half / V;
    const uint32_t in_page = pos & (c.size() - 1);
    for (uint32_t h = h0; h < all; h += step) {
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = later[j];
        if (h + step < all) load_some<V>(row + static_cast<size_t>(h + step) * DIM + V * lane, sh.wide_x, later);
        if (half && h < sh.heads + c.kv_heads) {
            float other[V];
            if (!turn.halves) {
#pragma unroll
                for (int j = 0; j < V; ++j) other[j] = e[j ^ 1];
            } else if (by_lane) {
#pragma unroll
                for (int j = 0; j < V; ++j) other[j] = __shfl_sync(0xffffffffu, e[j], partner & 31);
            } else {
                float* mine = head[warp];
                store_some<V>(mine + V * lane, true, e);
                __syncwarp();
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const uint32_t i = V * lane + j;
                    other[j] = i < turn.rot ? mine[i >= half ? i - half : i + half] : 0.f;
                }
                __syncwarp();
            }
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (V * lane + j < turn.rot) e[j] = __fadd_rn(__fmul_rn(e[j], co[j]), __fmul_rn(other[j], si[j]));
        }
        if (h < sh.heads) {
            store_some<V>(q_out + static_cast<size_t>(t) * sh.ldq + static_cast<size_t>(h) * DIM + V * lane, sh.wide_q, e);
            continue;
        }
        const bool is_k = h < sh.heads + c.kv_heads;
        const size_t at = c.row(page, h - sh.heads - (is_k ? 0 : c.kv_heads), in_page);
        if constexpr (CODES) {
            float top = 0.f;
            bool number = true;
#pragma unroll
            for (int j = 0; j < V; ++j) { top = fmaxf(top, fabsf(e[j])); number &= e[j] == e[j]; }
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (!__all_sync(0xffffffffu, number)) top = CUDART_NAN_F;     // (a maximum leaves NaN out: the scale has to say it, codes cannot)
            const float up = top < 0x1p-100f ? 0x1p100f : 1.0f;           // (127 / top would pass the range below 2^-121)
            const float inv = top > 0.f ? 127.0f / (top * up) : 0.f;
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < V; ++j) w |= (static_cast<uint32_t>(__float2int_rn(e[j] * up * inv)) & 0xffu) << (8 * j);
            int8_t* codes = static_cast<int8_t*>(is_k ? c.k : c.v) + at * DIM + V * lane;
            if constexpr (V == 4) *reinterpret_cast<uint32_t*>(codes) = w;
            else *reinterpret_cast<uint16_t*>(codes) = static_cast<uint16_t>(w);
            if (lane == 0) (is_k ? c.k_scale : c.v_scale)[at] = top / 127.0f;
        } else {
            store_some<V>(static_cast<__nv_bfloat16*>(is_k ? c.k : c.v) + at * DIM + V * lane, true, e);
        }
    }
}

template <int DIM, typename X, typename Q>
cudaError_t launch_append(const Pool& c, bool codes, const Batch& b, const Turn& t, const AppendShape& sh, const void* x, void* q, uint32_t* status, int sms, cudaStream_t st) {
    const uint32_t all = (sh.heads + 2 * c.kv_heads + AP_WARPS - 1) / AP_WARPS, room = 2u * static_cast<uint32_t>(sms) / b.rows;
    const dim3 grid(b.rows, room < 1 ? 1 : all < room ? all : room);
    return codes ? launch_pdl(append_kernel<DIM, X, Q, true>, grid, dim3(AP_WARPS * 32), 0, st, c, b, t, sh, static_cast<const X*>(x), static_cast<Q*>(q), status)
                 : launch_pdl(append_kernel<DIM, X, Q, false>, grid, dim3(AP_WARPS * 32), 0, st, c, b, t, sh, static_cast<const X*>(x), static_cast<Q*>(q), status);
}
template <int DIM>
cudaError_t launch_append_types(const Pool& c, bool codes, const Batch& b, const Turn& t, const AppendShape& sh, const void* x, bool x16, void* q, bool q16,
                                uint32_t* status, int sms, cudaStream_t st) {
    using h = __nv_bfloat16;
    return x16 ? (q16 ? launch_append<DIM, h, h>(c, codes, b, t, sh, x, q, status, sms, st) : launch_append<DIM, h, float>(c, codes, b, t, sh, x, q, status, sms, st))
               : (q16 ? launch_append<DIM, float, h>(c, codes, b, t, sh, x, q, status, sms, st) : launch_append<DIM, float, float>(c, codes, b, t, sh, x, q, status, sms, st));
}

// ---- moves.  Bound by memory: every byte is read once and written once.
struct Arrays {
    uint8_t *k, *v, *ks, *vs;                // scales: NULL without codes
    size_t layer, layer_scale;               // bytes of a layer's keys (values), scales
};

// Whole pages: a page's keys (values) are one run of bytes.  A CTA moves COPY_PART bytes of the keys and as many of the values of one
// page in one layer, four 16-byte loads of each under way in every thread, and its part of the scales.
constexpr uint32_t COPY_THREADS = 256, COPY_PART = COPY_THREADS * 16 * 4;
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(Arrays a, uint32_t pages, uint32_t page_bytes, uint32_t scale_bytes, const uint32_t* src, const uint32_t* dst,
                                                                  uint32_t* status) {
    pdl_trigger();
    pdl_wait();
    const uint32_t from = src[blockIdx.x], to = dst[blockIdx.x];
    if (from >= pages || to >= pages) {
        if (threadIdx.x == 0) atomicOr(status, STATUS_BAD_PAGE);
        return;
    }
    const size_t base = blockIdx.y * a.layer, f = base + static_cast<size_t>(from) * page_bytes, t = base + static_cast<size_t>(to) * page_bytes;
    uint4 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t at = blockIdx.z * COPY_PART + (i * COPY_THREADS + threadIdx.x) * 16;
        if (at < page_bytes) {
            k[i] = *reinterpret_cast<const uint4*>(a.k + f + at);
            v[i] = *reinterpret_cast<const uint4*>(a.v + f + at);
        }
    }
    const uint32_t s = (blockIdx.z * COPY_THREADS + threadIdx.x) * 16;
    const size_t sb = blockIdx.y * a.layer_scale, sf = sb + static_cast<size_t>(from) * scale_bytes + s, sto = sb + static_cast<size_t>(to) * scale_bytes + s;
    if (a.ks && s < scale_bytes) {           // (a page has fewer bytes of scales than of codes, so that the parts cover them)
        *reinterpret_cast<uint4*>(a.ks + sto) = *reinterpret_cast<const uint4*>(a.ks + sf);
        *reinterpret_cast<uint4*>(a.vs + sto) = *reinterpret_cast<const uint4*>(a.vs + sf);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t at = blockIdx.z * COPY_PART + (i * COPY_THREADS + threadIdx.x) * 16;
        if (at < page_bytes) {
            *reinterpret_cast<uint4*>(a.k + t + at) = k[i];
            *reinterpret_cast<uint4*>(a.v + t + at) = v[i];
        }
    }
}

// Single rows: 64 to 256 bytes of each head.  Consecutive threads take the 16-byte units of a row, then the next row of the list in the
// same head: rows that follow one another in a page are then neighbours in memory on the side where they are packed.
constexpr uint32_t ROW_THREADS = 256, ROW_EACH = 4;
__global__ void __launch_bounds__(ROW_THREADS) copy_rows_kernel(Arrays a, uint32_t pages, uint32_t shift, uint32_t kv_heads, uint32_t unit_log, const uint32_t* src,
                                                                const uint32_t* dst, uint32_t n, uint32_t* status) {
    pdl_trigger();
    pdl_wait();
    const uint32_t head = blockIdx.y, mask = (1u << shift) - 1;
    const uint64_t rows = static_cast<uint64_t>(pages) << shift;
    const uint8_t *kf[ROW_EACH], *vf[ROW_EACH];
    uint8_t *kt[ROW_EACH], *vt[ROW_EACH];
    uint4 k[ROW_EACH], v[ROW_EACH];
    float ks[ROW_EACH], vs[ROW_EACH];
    size_t st[ROW_EACH];
    bool live[ROW_EACH], first[ROW_EACH];
    bool bad = false;
#pragma unroll
    for (uint32_t i = 0; i < ROW_EACH; ++i) {
        const uint64_t at = (static_cast<uint64_t>(blockIdx.x) * ROW_EACH + i) * ROW_THREADS + threadIdx.x, r = at >> unit_log;
        const uint32_t u = static_cast<uint32_t>(at) & ((1u << unit_log) - 1);
        live[i] = r < n;
        uint32_t f = 0, t = 0;
        if (live[i]) { f = src[r]; t = dst[r]; }
        if (f >= rows || t >= rows) { bad = true; live[i] = false; f = t = 0; }
        const size_t fr = ((static_cast<size_t>(f >> shift) * kv_heads + head) << shift) + (f & mask), tr = ((static_cast<size_t>(t >> shift) * kv_heads + head) << shift) + (t & mask);
        const size_t base = blockIdx.z * a.layer, sbase = blockIdx.z * a.layer_scale;
        kf[i] = a.k + base + (((fr << unit_log) + u) << 4); kt[i] = a.k + base + (((tr << unit_log) + u) << 4);
        vf[i] = a.v + base + (((fr << unit_log) + u) << 4); vt[i] = a.v + base + (((tr << unit_log) + u) << 4);
        first[i] = live[i] && u == 0 && a.ks;
        st[i] = sbase + 4 * tr;
        if (live[i]) { k[i] = *reinterpret_cast<const uint4*>(kf[i]); v[i] = *reinterpret_cast<const uint4*>(vf[i]); }
        if (first[i]) { ks[i] = *reinterpret_cast<const float*>(a.ks + sbase + 4 * fr); vs[i] = *reinterpret_cast<const float*>(a.vs + sbase + 4 * fr); }
    }
#pragma unroll
    for (uint32_t i = 0; i < ROW_EACH; ++i) {
        if (live[i]) { *reinterpret_cast<uint4*>(kt[i]) = k[i]; *reinterpret_cast<uint4*>(vt[i]) = v[i]; }
        if (first[i]) { *reinterpret_cast<float*>(a.ks + st[i]) = ks[i]; *reinterpret_cast<float*>(a.vs + st[i]) = vs[i]; }
    }
    if (bad) atomicOr(status, STATUS_BAD_PAGE);
}

Arrays arrays_of(const hf2q_pages* c) {
    const size_t rows = static_cast<size_t>(c->pages) * c->kv_heads * c->page;
    const bool codes = c->dtype == HF2Q_DT_I8;
    return Arrays{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), codes ? reinterpret_cast<uint8_t*>(c->k_scale) : nullptr,
                  codes ? reinterpret_cast<uint8_t*>(c->v_scale) : nullptr, rows * c->dim * (codes ? 1 : 2), rows * 4};
}


}  // namespace
}  // namespace hf2q

using namespace hf2q;

extern "C" {

HF2Q_API int32_t hf2q_cuda_pages_append(hf2q_ctx* ctx, void* stream, const hf2q_pages* c, const hf2q_page_batch* b, const hf2q_rotary* rotary, const void* x,
                                        uint32_t x_dtype, uint32_t ldx, uint32_t heads, void* q_out, uint32_t q_dtype, uint32_t ldq) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    const char* who = "pages_append";
    if (const char* e = pages_error(c)) return refuse(ctx, who, e);
    if (const char* e = batch_error(b)) return refuse(ctx, who, e);
    if (b->rows && (!x || (heads && !q_out))) return refuse(ctx, who, "null pointer");       // (arrays without elements have no address)
    if ((x_dtype != HF2Q_DT_F32 && x_dtype != HF2Q_DT_BF16) || (heads && q_dtype != HF2Q_DT_F32 && q_dtype != HF2Q_DT_BF16)) return refuse(ctx, who, "rows are F32 or BF16");
    if (heads > 65535) return refuse(ctx, who, "at most 65535 query heads");
    if (ldx < static_cast<uint64_t>(heads + 2 * c->kv_heads) * c->dim || (heads && ldq < static_cast<uint64_t>(heads) * c->dim)) return refuse(ctx, who, "rows overlap (ldx or ldq is too small)");
    const size_t xs = x_dtype == HF2Q_DT_F32 ? 4 : 2, qs = q_dtype == HF2Q_DT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(x) % xs || (heads && reinterpret_cast<uintptr_t>(q_out) % qs)) return refuse(ctx, who, "rows start between two elements");
    if (rotary && (rotary->rot_dim % 2 || rotary->rot_dim > c->dim || (rotary->rot_dim && !rotary->freq))) return refuse(ctx, who, "rot_dim is even and at most dim, with a frequency for each pair");
    if (b->rows == 0) return HF2Q_OK;
    const Turn turn = rotary ? Turn{rotary->freq, rotary->pos, rotary->rot_dim, rotary->halves, rotary->factor} : Turn{nullptr, nullptr, 0, 0, 1.0f};
    const size_t v = c->dim / 32;
    const auto wide = [&](const void* p, uint32_t ld, size_t size) { return reinterpret_cast<uintptr_t>(p) % (v * size) == 0 && ld % v == 0; };
    const AppendShape sh{heads, ldx, ldq, wide(x, ldx, xs), wide(q_out, ldq, qs)};
    const OnDevice on(ctx_device(ctx));
    const auto launch = c->dim == 128 ? launch_append_types<128> : launch_append_types<64>;
    return ctx_cuda_result(ctx, launch(pool_of(c), c->dtype == HF2Q_DT_I8, batch_of(b), turn, sh, x, xs == 2, q_out, heads && qs == 2, ctx_status_word(ctx), ctx_sm_count(ctx),
                                       static_cast<cudaStream_t>(stream)), who, 1);
}

HF2Q_API int32_t hf2q_cuda_pages_copy(hf2q_ctx* ctx, void* stream, const hf2q_pages* c, uint32_t layers, const uint32_t* src, const uint32_t* dst, uint32_t n) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    if (const char* e = pages_error(c)) return refuse(ctx, "pages_copy", e);
    if (layers == 0 || layers > 65535) return refuse(ctx, "pages_copy", "1 to 65535 layers");
    if (n == 0) return HF2Q_OK;
    if (!src || !dst) return refuse(ctx, "pages_copy", "null pointer");
    if (n > 0x7fffffffu) return refuse(ctx, "pages_copy", "too many pages");
    const uint64_t bytes = static_cast<uint64_t>(c->kv_heads) * c->page * c->dim * (c->dtype == HF2Q_DT_I8 ? 1 : 2);
    if (bytes >= 1u << 30) return refuse(ctx, "pages_copy", "a page's keys take less than 2^30 bytes");
    const OnDevice on(ctx_device(ctx));
    const dim3 grid(n, layers, static_cast<uint32_t>((bytes + COPY_PART - 1) / COPY_PART));
    return ctx_cuda_result(ctx, launch_pdl(copy_pages_kernel, grid, dim3(COPY_THREADS), 0, static_cast<cudaStream_t>(stream), arrays_of(c), c->pages, static_cast<uint32_t>(bytes),
                                           c->kv_heads * c->page * 4, src, dst, ctx_status_word(ctx)), "pages_copy", 1);
}

HF2Q_API int32_t hf2q_cuda_pages_copy_rows(hf2q_ctx* ctx, void* stream, const hf2q_pages* c, uint32_t layers, const uint32_t* src, const uint32_t* dst, uint32_t n) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    if (const char* e = pages_error(c)) return refuse(ctx, "pages_copy_rows", e);
    if (layers == 0 || layers > 65535) return refuse(ctx, "pages_copy_rows", "1 to 65535 layers");
    if (n == 0) return HF2Q_OK;
    if (!src || !dst) return refuse(ctx, "pages_copy_rows", "null pointer");
    const uint32_t unit_log = static_cast<uint32_t>(__builtin_ctz(c->dim * (c->dtype == HF2Q_DT_I8 ? 1 : 2) / 16));
    const uint64_t ctas = ((static_cast<uint64_t>(n) << unit_log) + ROW_THREADS * ROW_EACH - 1) / (ROW_THREADS * ROW_EACH);
    if (ctas > 0x7fffffffu) return refuse(ctx, "pages_copy_rows", "too many rows");
    const OnDevice on(ctx_device(ctx));
    const dim3 grid(static_cast<uint32_t>(ctas), c->kv_heads, layers);
    return ctx_cuda_result(ctx, launch_pdl(copy_rows_kernel, grid, dim3(ROW_THREADS), 0, static_cast<cudaStream_t>(stream), arrays_of(c), c->pages,
                                           static_cast<uint32_t>(__builtin_ctz(c->page)), c->kv_heads, unit_log, src, dst, n, ctx_status_word(ctx)), "pages_copy_rows", 1);
}

}  // extern "C"
