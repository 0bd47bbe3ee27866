// Attention of a batch's rows over a paged key-value cache:
//
//   out[i] = sum_j p[i, j] v[j] / sum_j p[i, j],   p[i, j] = exp(scale q[i] . k[j] - max_j(..)) over the positions j that row i sees:
//   j <= i and, with a window, i - j < window or j < sinks.
//
// Two kernels: paged_step.cu for few rows of a sequence (warp-level products, bound by memory), paged_tiles.cu for many (tcgen05).  Here are
// the choice between them, how positions are split, and the sum of the parts.
#include <math_constants.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged_common.cuh"

namespace hf2q {
using namespace paged;
namespace {

// out[row][head] = sum of the parts, each weighted by exp2(its maximum - the largest), over the same sum of their weights.  Bound by the parts'
// bytes, so a warp asks for eight parts before it adds the first, in the order of the parts.  Up to JOIN_FEW parts a warp per row and head; more are
// shared by four warps, whose sums are added in the order of the warps.
constexpr uint32_t JOIN_WARPS = 4, JOIN_FEW = 16;
template <int DIM, typename OUT, uint32_t SHARE>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_kernel(Batch b, uint32_t heads, uint32_t chunks, const float* part, const float* part_ml, OUT* out, uint32_t ldo, uint32_t* status) {
    constexpr int V = DIM / 32, DEEP = 8;
    using Vec = std::conditional_t<V == 4, float4, float2>;
    __shared__ float others[SHARE][DIM + 1];
    pdl_trigger();
    pdl_wait();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % SHARE;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * (JOIN_WARPS / SHARE) + warp / SHARE;
    const uint32_t end = min(b.start[b.seqs], b.rows), begin = b.start[0];
    if (unit >= static_cast<uint64_t>(end) * heads || unit / heads < begin) return;       // (all warps that share a row and head)
    const float2* ml = reinterpret_cast<const float2*>(part_ml) + unit * chunks;
    float m_all = -CUDART_INF_F;
    for (uint32_t i = lane; i < chunks; i += 32) m_all = fmaxf(m_all, ml[i].x);
    for (int o = 16; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
    const uint32_t mine = (chunks + SHARE - 1) / SHARE, from = min(share * mine, chunks), upto = min(from + mine, chunks);
    const float* at = part + unit * chunks * DIM + V * lane;
    float acc[V] = {}, sum = 0.f;
#pragma unroll 1
    for (uint32_t i0 = from; i0 < upto; i0 += DEEP) {
        float f[DEEP], l[DEEP];
        Vec p[DEEP];
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            const float2 x = i0 + u < upto ? ml[i0 + u] : make_float2(0.f, 0.f);
            f[u] = part_factor(x.x, x.y, m_all);
            l[u] = x.y;
        }
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {                                  // (a part that counts for nothing was not written)
            p[u] = Vec{};
            if (f[u] != 0.f) p[u] = *reinterpret_cast<const Vec*>(at + static_cast<uint64_t>(i0 + u) * DIM);
        }
#pragma unroll
        for (int u = 0; u < DEEP; ++u) {
            if (f[u] == 0.f) continue;
            sum += l[u] * f[u];
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += reinterpret_cast<const float*>(&p[u])[e] * f[u];
        }
    }
    if constexpr (SHARE > 1) {
#pragma unroll
        for (int e = 0; e < V; ++e) others[share][V * lane + e] = acc[e];
        if (lane == 0) others[share][DIM] = sum;
        __syncthreads();
        if (share) return;
#pragma unroll
        for (uint32_t w = 1; w < SHARE; ++w) {
            sum += others[w][DIM];
#pragma unroll
            for (int e = 0; e < V; ++e) acc[e] += others[w][V * lane + e];
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    bool clipped = false;
    OUT* to = out + unit / heads * ldo + unit % heads * DIM + V * lane;
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = out_value<OUT>(acc[e] * inv, clipped);
    if (clipped) atomicOr(status, STATUS_X_CLIPPED);
}
template <int DIM, typename OUT>
cudaError_t launch_join_out(const AttendCall& a) {
    const uint64_t units = static_cast<uint64_t>(a.b.rows) * a.heads;
    const bool few = a.chunks <= JOIN_FEW;
    const uint64_t ctas = few ? (units + JOIN_WARPS - 1) / JOIN_WARPS : units;
    if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
    return launch_pdl(few ? join_kernel<DIM, OUT, 1> : join_kernel<DIM, OUT, JOIN_WARPS>, dim3(static_cast<uint32_t>(ctas)), dim3(JOIN_WARPS * 32), 0, a.st, a.b, a.heads, a.chunks,
                      static_cast<const float*>(a.part), static_cast<const float*>(a.part_ml), static_cast<OUT*>(a.out), a.ldo, a.status);
}
template <int DIM>
cudaError_t launch_join(const AttendCall& a) {
    return a.out_dtype == HF2Q_DT_F32 ? launch_join_out<DIM, float>(a) : a.out_dtype == HF2Q_DT_F16 ? launch_join_out<DIM, __half>(a) : launch_join_out<DIM, __nv_bfloat16>(a);
}

// How a call is laid out, from the bounds that the host knows.
// Rows of a sequence (tokens times heads of a group) that the step kernel takes: one tile of 16, with codes two, whatever the context; and up to four as
// long as all its tiles together go through few positions, since the other kernel takes longer to begin and end but its tiles of 128 rows read
// them once (us, step / tiles, 8 KV heads.  Codes: 32 rows of 8000 positions 18.1 / 24.8, of 16 sequences of 3000 80 / 85; 64 rows of 300 10.3 / 16.1, of 8000
// 23.8 / 25.8, of 32768 68 / 54, of 16 sequences of 3000 116 / 89.  bf16: 64 rows of 1000 12.2 / 15.2, 32 rows of 32768 49 / 41; 4 KV heads, 35 rows of 8 sequences
// of up to 3001 30 / 22).
constexpr uint64_t STEP_UNITS = 16, STEP_UNITS_CODES = 32, STEP_UNITS_MOST = 64, STEP_WORK = 1 << 17, STEP_WORK_CODES = 1 << 18;
struct Plan {
    bool step, shrink;
    uint32_t chunk, chunks;
    uint64_t scratch;
};
Plan plan_of(const hf2q_pages& c, const hf2q_page_batch& b, uint32_t heads, uint32_t window, uint32_t sinks, int sms) {
    Plan p{};
    const uint64_t group = heads / c.kv_heads, units = b.max_new * group;
    const bool codes = c.dtype == HF2Q_DT_I8;
    const uint64_t most = window ? std::min<uint64_t>(b.max_length, static_cast<uint64_t>(window) + b.max_new + sinks) : b.max_length;
    const uint64_t work = most * c.kv_heads * std::min(b.seqs, b.rows) * ((units + 15) / 16);
    p.step = units <= (codes ? STEP_UNITS_CODES : STEP_UNITS) || (units <= STEP_UNITS_MOST && work <= (codes ? STEP_WORK_CODES : STEP_WORK));
    const uint64_t rows = units <= 8 ? 8 : p.step ? 16 : 2 * (128 / group) * group;
    // most positions that a tile goes through, and tiles as if every sequence that can have rows had the most
    const uint64_t ceil128 = (std::max(1u, b.max_length) + 127ull) / 128 * 128, seqs = std::min(b.seqs, b.rows);
    uint64_t seen = ceil128;
    if (window) seen = std::min<uint64_t>(seen, (static_cast<uint64_t>(window) + b.max_new + sinks + (p.step ? 32 : 256) + 127) / 128 * 128);
    const uint64_t tiles = static_cast<uint64_t>(c.kv_heads) * seqs * ((units + rows - 1) / rows);
    uint64_t chunk = seen;
    if (p.step) {
        // A CTA takes about 4 us to begin and end; 64 positions take 1 us where two CTAs share an SM (half of it with heads of 64), 0.7 where one has it, and
        // 0.8 of that while the SMs are not full; joining parts takes 3 us.  One sequence: whole rounds of equal parts.  Several, of several lengths: one round as long as there is one;
        // else what they hold together, 0.65 of the most (all of it in a window), shared evenly, and half of one part for the end.  (Codes, 4 sequences of
        // up to 30000: 10 parts 47 us, 17 parts 56, 4 parts 89.  32 sequences of up to 8191: 1 part 97, 4 parts 79, 10 parts 88.  16 sequences of up to 2000 in
        // bf16: 1 part 25, 2 parts 31.  24 sequences with a window of 1024 in 64 elements: whole 12, parts of 512 18.)
        const uint32_t on_sm = step_ctas(c.dim, c.dtype == HF2Q_DT_I8, units > 8);
        const double places = static_cast<double>(sms) * on_sm, block = c.dim == 64 ? 0.5 : on_sm > 1 ? 1.0 : 0.7, held = seqs == 1 || seen < ceil128 ? 1.0 : 0.65;
        double best = 0.0;
        for (uint64_t parts = 1; parts <= 256 && (parts == 1 || seen / parts >= 128); ++parts) {
            const uint64_t size = ((seen + parts - 1) / parts + 127) / 128 * 128;
            const double one = 4.0 + block * size / 64.0, all = tiles * held * (4.0 * parts + block * seen / 64.0), join = parts > 1 ? 3.0 : 0.0;
            const double cost = seqs == 1 ? std::ceil(tiles * parts / places) * one : tiles * parts <= places ? 4.0 + 0.8 * block * size / 64.0 : std::max(one, all / places + 0.5 * one);
            if (parts == 1 || cost + join < best) { best = cost + join; chunk = size; }
        }
    } else {
        // In units of 64 positions of a CTA (1.7 us): it takes 8 of them to begin and end, there is one CTA on an SM, and joining takes 2 and reads and
        // writes every part (2.5 MB a us).  Whole rounds, as if all sequences were of the largest length: a few CTAs too many cost a round, some SMs
        // left over little.  (The last part is the shortest, so that one may follow another on an SM.)  A prompt that is long against what is before
        // it has tiles of all lengths: what they take together, and half of one part for the end.  (64 rows of 8 heads after 32768 positions: 19 parts
        // 71 us, 18 75, 20 120, 8 132.  640 rows after 8192: 1 part 246, 3 parts 185, 7 parts 217.  Eight sequences, 5 rows of 4 heads after 3001: 4 parts 23,
        // 5 parts 33; 22 both where they are of 1500 to 3001.)
        const bool even = seen < ceil128 || 4ull * b.max_new <= seen;
        const double places = sms, held = (b.max_length - b.max_new / 2) / static_cast<double>(std::max(1u, b.max_length));
        const double bytes = static_cast<double>(b.rows) * heads * c.dim * 8.0;
        double best = 0.0;
        for (uint64_t parts = 1; parts <= 256 && (parts == 1 || seen / parts >= 256); ++parts) {
            const uint64_t size = ((seen + parts - 1) / parts + 127) / 128 * 128, count = (seen + size - 1) / size, ctas = tiles * count, full = tiles * (count - 1);
            const double one = 8.0 + size / 64.0, end = 8.0 + (seen - (count - 1) * size) / 64.0, join = count > 1 ? 2.0 + count * bytes / 4.2e6 : 0.0;
            double cost = std::ceil(ctas / places) * one;
            if (full < static_cast<uint64_t>(sms) && ctas > static_cast<uint64_t>(sms) && ctas - sms <= sms - full) cost = std::max(one, 2.0 * end);
            if (!even) cost = std::max(one, ctas / places * held * one + 0.5 * one);
            if (parts == 1 || cost + join < best) { best = cost + join; chunk = size; }
        }
    }
    p.chunks = static_cast<uint32_t>((seen + chunk - 1) / chunk);
    p.chunk = static_cast<uint32_t>(chunk);
    p.shrink = p.chunks > 1 && b.seqs <= 32 && tiles * p.chunks <= static_cast<uint64_t>(sms) * (p.step ? step_ctas(c.dim, codes, units > 8) : 1);
    p.scratch = p.chunks > 1 && b.rows ? (static_cast<uint64_t>(b.rows) * heads * p.chunks * (c.dim + 2) * 4 + 255) / 256 * 256 : 256;
    return p;
}

const char* heads_error(const hf2q_pages* c, uint32_t heads) {
    return heads == 0 || heads > 65535 || heads % c->kv_heads || heads / c->kv_heads > 128 ? "query heads are a multiple of the KV heads, up to 128 to one" : nullptr;
}

}  // namespace
}  // namespace hf2q

using namespace hf2q;

extern "C" {

HF2Q_API int32_t hf2q_cuda_pages_attend_scratch_bytes(hf2q_ctx* ctx, const hf2q_pages* c, const hf2q_page_batch* b, uint32_t heads, uint32_t window, uint32_t sinks, uint64_t* out) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    const char* who = "pages_attend_scratch_bytes";
    if (const char* e = pages_error(c)) return refuse(ctx, who, e);
    if (const char* e = batch_error(b)) return refuse(ctx, who, e);
    if (const char* e = heads_error(c, heads)) return refuse(ctx, who, e);
    if (!out) return refuse(ctx, who, "null pointer");
    *out = plan_of(*c, *b, heads, window, sinks, ctx_sm_count(ctx)).scratch;
    return HF2Q_OK;
}

HF2Q_API int32_t hf2q_cuda_pages_attend(hf2q_ctx* ctx, void* stream, const hf2q_pages* c, const hf2q_page_batch* b, const void* q, uint32_t q_dtype, uint32_t ldq, uint32_t heads,
                                        float scale, uint32_t window, uint32_t sinks, void* out, uint32_t out_dtype, uint32_t ldo, void* scratch, uint64_t scratch_bytes) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    const char* who = "pages_attend";
    if (const char* e = pages_error(c)) return refuse(ctx, who, e);
    if (const char* e = batch_error(b)) return refuse(ctx, who, e);
    if (const char* e = heads_error(c, heads)) return refuse(ctx, who, e);
    const bool none = b->rows == 0 || b->max_new == 0;                    // (arrays without elements have no address)
    if (!none && (!q || !out)) return refuse(ctx, who, "null pointer");
    if (q_dtype != HF2Q_DT_F32 && q_dtype != HF2Q_DT_BF16) return refuse(ctx, who, "q is F32 or BF16");
    if (out_dtype != HF2Q_DT_F32 && out_dtype != HF2Q_DT_BF16 && out_dtype != HF2Q_DT_F16) return refuse(ctx, who, "out is F32, BF16 or F16");
    const uint64_t width = static_cast<uint64_t>(heads) * c->dim;
    if (ldq < width || ldo < width) return refuse(ctx, who, "rows overlap (ldq or ldo is too small)");
    if (reinterpret_cast<uintptr_t>(q) % (q_dtype == HF2Q_DT_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(out) % (out_dtype == HF2Q_DT_F32 ? 4 : 2)) return refuse(ctx, who, "rows start between two elements");
    if (none) return HF2Q_OK;
    const Plan p = plan_of(*c, *b, heads, window, sinks, ctx_sm_count(ctx));
    if (!scratch || scratch_bytes < p.scratch) return ctx_fail(ctx, HF2Q_ERR_WORKSPACE, "pages_attend: scratch missing or too small (ask hf2q_cuda_pages_attend_scratch_bytes)");
    if (reinterpret_cast<uintptr_t>(scratch) % 256) return refuse(ctx, who, "scratch is 256-byte aligned");
    const OnDevice on(ctx_device(ctx));
    float* part = static_cast<float*>(scratch);
    const AttendCall a{pool_of(c), batch_of(b), Look{window, sinks, scale * 1.4426950408889634f}, heads, q, q_dtype, ldq, out, out_dtype, ldo, p.chunk, p.chunks, p.shrink,
                       part, part + static_cast<size_t>(b->rows) * heads * p.chunks * c->dim, ctx_status_word(ctx), static_cast<cudaStream_t>(stream)};
    cudaError_t e = (p.step ? launch_attend_step : launch_attend_tiles)(a, c->dim, c->dtype == HF2Q_DT_I8);
    if (e == cudaSuccess && p.chunks > 1) e = c->dim == 128 ? launch_join<128>(a) : launch_join<64>(a);
    return ctx_cuda_result(ctx, e, who, p.chunks > 1 ? 2 : 1);
}

}  // extern "C"
