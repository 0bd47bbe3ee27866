// What the kernels of the paged cache share: the views that a launch gets by value, and how a sequence's rows and positions are found
// on the device.  Every number that comes from device memory is checked before it becomes an address.
#pragma once
#include <cstdio>

#include "common.cuh"
#include "kernels.h"

namespace hf2q {
namespace paged {

// one layer's pool
struct Pool {
    void *k, *v;
    float *k_scale, *v_scale;
    uint32_t pages, shift, kv_heads;         // page size 1 << shift
    __host__ __device__ uint32_t size() const { return 1u << shift; }
    // first row of head `head` in page `page`, in rows
    __host__ __device__ size_t row(uint32_t page, uint32_t head, uint32_t in_page) const { return ((static_cast<size_t>(page) * kv_heads + head) << shift) + in_page; }
};

struct Batch {
    const uint32_t *start, *length, *table;
    uint32_t seqs, rows, table_ld, max_new, max_length;
};

// The new rows of a sequence and the positions it holds; what does not fit is cut to what is safe and `bad` says so.
struct Span {
    uint32_t row0, rows, length;
    bool bad;
};
__host__ __device__ __forceinline__ Span span_of(const Batch& b, uint32_t shift, uint32_t s) {
    Span o;
    const uint32_t r0 = b.start[s], r1 = b.start[s + 1], len = b.length[s];
    const uint64_t held = static_cast<uint64_t>(b.table_ld) << shift;
    const uint32_t room = held < b.max_length ? static_cast<uint32_t>(held) : b.max_length;
    o.row0 = r0 < b.rows ? r0 : b.rows;
    const uint32_t end = r1 < b.rows ? r1 : b.rows, n = end > o.row0 ? end - o.row0 : 0u;
    o.rows = n < b.max_new ? n : b.max_new;
    o.length = len < room ? len : room;
    o.bad = r1 < r0 || r1 > b.rows || r1 - r0 > b.max_new || len > room;
    return o;
}

// page that holds position p of sequence s (p below the span's length); a number out of range counts as page 0
__host__ __device__ __forceinline__ uint32_t page_of(const Pool& c, const Batch& b, uint32_t s, uint32_t p, bool& bad) {
    const uint32_t page = b.table[static_cast<size_t>(s) * b.table_ld + (p >> c.shift)];
    if (page < c.pages) return page;
    bad = true;
    return 0;
}

// What a row sees, and the scale of its scores in units of log2.
struct Look {
    uint32_t window, sinks;
    float scale;
    __host__ __device__ bool sees(uint32_t i, uint32_t j) const { return j <= i && (window == 0 || i - j < window || j < sinks); }
};

// The blocks of `unit` positions (unit = 1 << log) that rows at positions first .. last see, numbered without a gap: those of the first
// positions, then those from the window's lower end of the first row to the last row.
struct Blocks {
    uint32_t sinks, from, count;             // blocks of the first positions; first block of the window; all
    __host__ __device__ uint32_t at(uint32_t t) const { return t < sinks ? t : t - sinks + from; }
};
__host__ __device__ __forceinline__ Blocks blocks_of(const Look& k, uint32_t first, uint32_t last, uint32_t log) {
    Blocks o;
    o.from = (k.window && first >= k.window ? first - k.window + 1 : 0) >> log;
    const uint64_t s = k.window ? (static_cast<uint64_t>(k.sinks) + (1u << log) - 1) >> log : 0;
    o.sinks = s < o.from ? static_cast<uint32_t>(s) : o.from;
    o.count = o.sinks + (last >> log) + 1 - o.from;
    return o;
}
// every row at first .. last sees all of positions p .. p + n - 1; some row sees position p
__host__ __device__ __forceinline__ bool all_see(const Look& k, uint32_t first, uint32_t last, uint32_t p, uint32_t n) {
    return p + n - 1 <= first && (k.window == 0 || last - p < k.window || p + n <= k.sinks);
}
__host__ __device__ __forceinline__ bool some_see(const Look& k, uint32_t first, uint32_t last, uint32_t p) {
    return p <= last && (k.window == 0 || p >= first || first - p < k.window || p < k.sinks);
}

// One attention call as the launchers take it.  With chunks > 1 a sequence's positions are split: part `chunk` of row and head leaves its
// sum of weighted values (f32 [dim]) and (maximum, sum of weights) in scratch, and join_kernel adds the parts up in order.
struct AttendCall {
    Pool c;
    Batch b;
    Look look;
    uint32_t heads;
    const void* q;
    uint32_t q_dtype, ldq;
    void* out;
    uint32_t out_dtype, ldo;
    uint32_t chunk, chunks;                  // positions of a part, a multiple of 128
    bool shrink;                             // parts follow the lengths
    float *part, *part_ml;                   // [rows][heads][chunks][dim], [rows][heads][chunks][2]
    uint32_t* status;
    cudaStream_t st;
};
cudaError_t launch_attend_step(const AttendCall& a, uint32_t dim, bool codes);       // paged_step.cu
cudaError_t launch_attend_tiles(const AttendCall& a, uint32_t dim, bool codes);      // paged_tiles.cu

// what the sums of a part count for beside others: a part that saw nothing has none (its sum is 0), one of NaN scores alone has no maximum
__device__ __forceinline__ float part_factor(float m, float l, float m_all) { return l == 0.f ? 0.f : m == -INFINITY ? 1.0f : exp2f(m - m_all); }

// How many units of 2^log positions a part has.  A call is laid out for max_length; where up to 32 sequences are all much shorter now, their
// parts are as much shorter, down to `least`, so that as many CTAs work.  (Whole warps come here.  Either number of units covers all: there
// are `parts` times as many as the longest sequence has.)  Only where all CTAs run at once (`shrink`): else more, shorter rounds take the place
// of few.  (Codes, 8 KV heads, one token of each sequence, us with and without: 4 sequences of 2000 laid out for 32768 13 / 27, 1 of 2000 12 / 16, 8 of 1000 laid
// out for 8000 12 / 19; more than one round: 32 of 2000 laid out for 32768 75 / 49, 16 of 1000 laid out for 8000 32 / 23, 8 of 10000 laid out for 32768 61 / 56.
// 64 rows of each of 4 sequences of 4000 laid out for 16000 54 / 143.)
__device__ __forceinline__ uint32_t part_units(const Batch& b, uint32_t log, uint32_t planned, uint32_t parts, uint32_t least, bool shrink) {
    if (!shrink) return planned;
    const uint32_t lane = threadIdx.x & 31, longest = __reduce_max_sync(0xffffffffu, lane < b.seqs ? min(b.length[lane], b.max_length) : 0u);
    if (4ull * longest > 3ull * b.max_length) return planned;
    return min(planned, max(least, ((longest + (1u << log) - 1 >> log) + parts - 1) / parts));
}

// CTAs of the few-rows kernel that share an SM (tall: tiles of 16 rows)
constexpr uint32_t step_ctas(uint32_t dim, bool codes, bool tall) { return dim == 64 || (codes && !tall) ? 2 : 1; }

template <typename OUT> __device__ __forceinline__ OUT out_value(float v, bool& clipped);
template <> __device__ __forceinline__ float out_value<float>(float v, bool&) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 out_value<__nv_bfloat16>(float v, bool&) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half out_value<__half>(float v, bool& clipped) {      // (the panel of a product that follows)
    const __half h = panel_f16(v, clipped);
    return v == v ? h : __float2half_rn(v);                               // (clipping alone would turn NaN into the lowest number)
}

// the checks that all entries share; 0 or the text of what is wrong
inline const char* pages_error(const hf2q_pages* c) {
    if (!c || !c->k || !c->v) return "null cache pointer";
    if (c->dtype != HF2Q_DT_I8 && c->dtype != HF2Q_DT_BF16) return "the cache is of signed bytes (I8) or BF16";
    if (c->dtype == HF2Q_DT_I8 && (!c->k_scale || !c->v_scale)) return "a cache of bytes needs its scales";
    if (c->page < 16 || c->page > 256 || (c->page & (c->page - 1))) return "a page holds 16, 32, 64, 128 or 256 positions";
    if (c->dim != 64 && c->dim != 128) return "heads are of 64 or 128 elements";
    if (c->pages == 0 || c->kv_heads == 0 || c->kv_heads > 65535) return "a pool has 1 page or more and 1 to 65535 heads";
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) % 16)
        return "the cache's arrays start on 16-byte boundaries";
    return nullptr;
}
inline const char* batch_error(const hf2q_page_batch* b) {
    if (!b || !b->start || !b->length || !b->table) return "null batch pointer";
    if (b->seqs == 0 || b->seqs > 65535 || b->table_ld == 0) return "a batch has 1 to 65535 sequences and a table";
    if (b->max_new > b->rows || b->max_length < b->max_new || b->max_length > 1u << 30) return "max_new is at most rows and max_length, max_length at most 2^30";
    if (b->rows > 1u << 28) return "a batch has at most 2^28 rows";
    return nullptr;
}
inline int32_t refuse(hf2q_ctx* ctx, const char* who, const char* what) {
    char text[256];
    snprintf(text, sizeof text, "%s: %s", who, what);
    return ctx_fail(ctx, HF2Q_ERR_INVALID_ARGUMENT, text);
}
inline Pool pool_of(const hf2q_pages* c) {
    return Pool{c->k, c->v, c->k_scale, c->v_scale, c->pages, static_cast<uint32_t>(__builtin_ctz(c->page)), c->kv_heads};
}
inline Batch batch_of(const hf2q_page_batch* b) { return Batch{b->start, b->length, b->table, b->seqs, b->rows, b->table_ld, b->max_new, b->max_length}; }

struct OnDevice {                            // the context's device for the length of a call
    int prev = -1;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess || prev == dev) prev = -1;
        else cudaSetDevice(dev);
    }
    ~OnDevice() { if (prev >= 0) cudaSetDevice(prev); }
};

}  // namespace paged
}  // namespace hf2q
