// Attention of a batch's rows over a paged key-value cache:
//
//   out[i] = sum_j p[i, j] v[j] / sum_j p[i, j],   p[i, j] = exp(scale q[i] . k[j] - max_j(..)) over the positions j that row i sees:
//   j <= i and, with a window, i - j < window or j < sinks.
//
// attend_kernel: a warp per row and query head, 32 positions at a time with a running maximum and sum, all in f32.
#include <math_constants.h>

#include <type_traits>

#include "paged_common.cuh"
#include "seq_common.cuh"

namespace hf2q {
using namespace paged;
namespace {

struct Look {                                // what a row sees, and the scale of its scores in units of log2
    uint32_t window, sinks;
    float scale;
    __device__ bool sees(uint32_t i, uint32_t j) const { return j <= i && (window == 0 || i - j < window || j < sinks); }
};

template <typename OUT> __device__ __forceinline__ OUT out_value(float v, bool& clipped) {
    if constexpr (std::is_same_v<OUT, float>) return v;
    else if constexpr (std::is_same_v<OUT, __half>) return panel_f16(v, clipped);
    else return __float2bfloat16_rn(v);
}

constexpr uint32_t ROW_WARPS = 4;
template <int DIM, bool CODES, typename Q, typename OUT>
__global__ void __launch_bounds__(ROW_WARPS * 32) attend_kernel(Pool c, Batch b, Look look, uint32_t heads, const Q* q, uint32_t ldq, OUT* out, uint32_t ldo, uint32_t* status) {
    __shared__ float qs[ROW_WARPS][DIM];
    constexpr int V = DIM / 32;
    const uint32_t s = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Span span = span_of(b, c.shift, s);
    if (span.bad && threadIdx.x == 0 && blockIdx.x == 0) atomicOr(status, STATUS_BAD_PAGE);
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * ROW_WARPS + warp;
    if (unit >= static_cast<uint64_t>(span.rows) * heads) return;
    const uint32_t r = static_cast<uint32_t>(unit / heads), h = static_cast<uint32_t>(unit % heads), kvh = h / (heads / c.kv_heads);
    const size_t row = span.row0 + r;
    for (uint32_t d = lane; d < DIM; d += 32) qs[warp][d] = seq::to_f32(q[row * ldq + static_cast<size_t>(h) * DIM + d]) * look.scale;
    __syncwarp();
    const bool any = span.length + r >= span.rows;
    const uint32_t i = any ? span.length - span.rows + r : 0;
    float mx = -CUDART_INF_F, l = 0.f, acc[V] = {};
    bool bad = false;
    for (uint32_t j0 = 0; any && j0 <= i; j0 += 32) {
        const uint32_t j = j0 + lane;
        const bool seen = look.sees(i, j);
        if (!__any_sync(0xffffffffu, seen)) continue;
        float x = -CUDART_INF_F, vsc = 0.f;
        size_t at = 0;
        if (seen) {
            at = c.row(page_of(c, b, s, j, bad), kvh, j & (c.size() - 1));
            x = 0.f;
            if constexpr (CODES) {
                const int8_t* k = static_cast<const int8_t*>(c.k) + at * DIM;
                for (int d = 0; d < DIM; ++d) x = fmaf(qs[warp][d], static_cast<float>(k[d]), x);
                x *= c.k_scale[at];
                vsc = c.v_scale[at];
            } else {
                const __nv_bfloat16* k = static_cast<const __nv_bfloat16*>(c.k) + at * DIM;
                for (int d = 0; d < DIM; ++d) x = fmaf(qs[warp][d], __bfloat162float(k[d]), x);
                vsc = 1.f;
            }
        }
        float top = x;
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float to = fmaxf(mx, top), base = to == -CUDART_INF_F ? 0.f : to, corr = exp2f(mx - base), p = seen ? exp2f(x - base) : 0.f;
        mx = to;
        l = l * corr + p;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] *= corr;
        for (uint32_t o = 0; o < 32; ++o) {
            const size_t there = __shfl_sync(0xffffffffu, at, o);
            const float w = __shfl_sync(0xffffffffu, p * vsc, o);
            if (!__shfl_sync(0xffffffffu, seen, o)) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const size_t d = there * DIM + V * lane + e;
                acc[e] = fmaf(w, CODES ? static_cast<float>(static_cast<const int8_t*>(c.v)[d]) : __bfloat162float(static_cast<const __nv_bfloat16*>(c.v)[d]), acc[e]);
            }
        }
    }
    l = seq::warp_sum(l);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    bool clipped = false;
    for (int e = 0; e < V; ++e) out[row * ldo + static_cast<size_t>(h) * DIM + V * lane + e] = out_value<OUT>(l == 0.f ? 0.f : acc[e] * inv, clipped);
    if (clipped) atomicOr(status, STATUS_X_CLIPPED);
    if (bad) atomicOr(status, STATUS_BAD_PAGE);
}

struct Call {
    Pool c;
    Batch b;
    Look look;
    uint32_t heads;
    const void* q;
    uint32_t ldq;
    void* out;
    uint32_t ldo;
    uint32_t* status;
    cudaStream_t st;
};
template <int DIM, bool CODES, typename Q, typename OUT>
cudaError_t launch(const Call& a) {
    const uint64_t units = static_cast<uint64_t>(a.b.max_new) * a.heads;
    attend_kernel<DIM, CODES, Q, OUT><<<dim3(static_cast<uint32_t>((units + ROW_WARPS - 1) / ROW_WARPS), a.b.seqs), ROW_WARPS * 32, 0, a.st>>>(
        a.c, a.b, a.look, a.heads, static_cast<const Q*>(a.q), a.ldq, static_cast<OUT*>(a.out), a.ldo, a.status);
    return cudaGetLastError();
}
template <int DIM, bool CODES, typename Q>
cudaError_t launch_out(const Call& a, uint32_t out_dtype) {
    return out_dtype == HF2Q_DT_F32 ? launch<DIM, CODES, Q, float>(a) : out_dtype == HF2Q_DT_F16 ? launch<DIM, CODES, Q, __half>(a) : launch<DIM, CODES, Q, __nv_bfloat16>(a);
}
template <int DIM, bool CODES>
cudaError_t launch_q(const Call& a, uint32_t q_dtype, uint32_t out_dtype) {
    return q_dtype == HF2Q_DT_F32 ? launch_out<DIM, CODES, float>(a, out_dtype) : launch_out<DIM, CODES, __nv_bfloat16>(a, out_dtype);
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
    *out = 256;
    return HF2Q_OK;
}

HF2Q_API int32_t hf2q_cuda_pages_attend(hf2q_ctx* ctx, void* stream, const hf2q_pages* c, const hf2q_page_batch* b, const void* q, uint32_t q_dtype, uint32_t ldq, uint32_t heads,
                                        float scale, uint32_t window, uint32_t sinks, void* out, uint32_t out_dtype, uint32_t ldo, void* scratch, uint64_t scratch_bytes) {
    if (!ctx) return HF2Q_ERR_INVALID_ARGUMENT;
    const char* who = "pages_attend";
    if (const char* e = pages_error(c)) return refuse(ctx, who, e);
    if (const char* e = batch_error(b)) return refuse(ctx, who, e);
    if (const char* e = heads_error(c, heads)) return refuse(ctx, who, e);
    if (!q || !out) return refuse(ctx, who, "null pointer");
    if (q_dtype != HF2Q_DT_F32 && q_dtype != HF2Q_DT_BF16) return refuse(ctx, who, "q is F32 or BF16");
    if (out_dtype != HF2Q_DT_F32 && out_dtype != HF2Q_DT_BF16 && out_dtype != HF2Q_DT_F16) return refuse(ctx, who, "out is F32, BF16 or F16");
    const uint64_t width = static_cast<uint64_t>(heads) * c->dim;
    if (ldq < width || ldo < width) return refuse(ctx, who, "rows overlap (ldq or ldo is too small)");
    if (reinterpret_cast<uintptr_t>(q) % (q_dtype == HF2Q_DT_F32 ? 4 : 2) || reinterpret_cast<uintptr_t>(out) % (out_dtype == HF2Q_DT_F32 ? 4 : 2)) return refuse(ctx, who, "rows start between two elements");
    if (b->rows == 0 || b->max_new == 0) return HF2Q_OK;
    uint64_t need = 0;
    if (const int32_t rc = hf2q_cuda_pages_attend_scratch_bytes(ctx, c, b, heads, window, sinks, &need)) return rc;
    if (!scratch || scratch_bytes < need) return ctx_fail(ctx, HF2Q_ERR_WORKSPACE, "pages_attend: scratch missing or too small (ask hf2q_cuda_pages_attend_scratch_bytes)");
    if (reinterpret_cast<uintptr_t>(scratch) % 256) return refuse(ctx, who, "scratch is 256-byte aligned");
    const OnDevice on(ctx_device(ctx));
    const Call a{pool_of(c), batch_of(b), Look{window, sinks, scale * 1.4426950408889634f}, heads, q, ldq, out, ldo, ctx_status_word(ctx), static_cast<cudaStream_t>(stream)};
    const bool codes = c->dtype == HF2Q_DT_I8;
    const auto go = c->dim == 128 ? (codes ? launch_q<128, true> : launch_q<128, false>) : (codes ? launch_q<64, true> : launch_q<64, false>);
    return ctx_cuda_result(ctx, go(a, q_dtype, out_dtype), who, 1);
}

}  // extern "C"
