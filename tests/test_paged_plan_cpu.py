"""How an attention call over pages is laid out on the host, compiled with stand-ins for the context and the launches: bounds of every size, none
among them."""
import subprocess
from pathlib import Path

from hf2q_b200 import build

CSRC = Path(__file__).resolve().parent.parent / "hf2q_b200" / "csrc"
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include "paged_attn.cu"
struct hf2q_ctx { int launches = 0; };
namespace hf2q {
int32_t ctx_fail(hf2q_ctx*, int32_t code, const char*) { return code; }
int32_t ctx_cuda_result(hf2q_ctx* c, cudaError_t, const char*, uint64_t n) { c->launches += n; return HF2Q_OK; }
int ctx_sm_count(const hf2q_ctx*) { return 148; }
int ctx_device(const hf2q_ctx*) { return 0; }
uint32_t* ctx_status_word(hf2q_ctx*) { return nullptr; }
namespace paged {
static AttendCall last;
cudaError_t launch_attend_step(const AttendCall& a, uint32_t, bool) { last = a; return cudaErrorUnknown; }
cudaError_t launch_attend_tiles(const AttendCall& a, uint32_t, bool) { last = a; return cudaErrorUnknown; }
}
}
static uint32_t some(uint32_t most) { return rand() % 3 == 0 ? 0 : rand() % 2 ? rand() % (most + 1) : rand() % ((most >> (rand() % 12)) + 1); }
int main() {
    hf2q_ctx ctx;
    alignas(256) static uint32_t place[64];
    for (int it = 0; it < 100000; ++it) {
        const uint32_t rows = some(5000), max_new = some(rows), max_length = max_new + some(200000), kv = 1 + rand() % 8, group = 1 + some(127), dim = rand() % 2 ? 64 : 128;
        const uint32_t seqs = 1 + some(rand() % 2 ? 10 : 60000), window = some(5000), sinks = some(200);
        const hf2q_pages c{place, place, (float*)place, (float*)place, 100, 16u << (rand() % 5), kv, dim, rand() % 2 ? HF2Q_DT_I8 : HF2Q_DT_BF16};
        const hf2q_page_batch b{place, place, place, seqs, rows, 10, max_new, max_length};
        uint64_t bytes = 7;
        if (hf2q_cuda_pages_attend_scratch_bytes(&ctx, &c, &b, kv * group, window, sinks, &bytes) != HF2Q_OK) return printf("refused\n"), 1;
        if (bytes < 256 || bytes % 256) return printf("bytes %llu\n", (unsigned long long)bytes), 1;
        ctx.launches = 0;
        void* rows_at = max_new ? place : nullptr;                        // (arrays without rows have no address)
        const int32_t rc = hf2q_cuda_pages_attend(&ctx, nullptr, &c, &b, rows_at, HF2Q_DT_F32, 1u << 30, kv * group, 1.0f, window, sinks, rows_at, HF2Q_DT_F32, 1u << 30, place, bytes);
        if (rc != HF2Q_OK || (ctx.launches == 0) != (max_new == 0)) return printf("call %d %d\n", rc, ctx.launches), 1;
        if (max_new == 0) continue;
        // the parts cover the most positions that a call can go through, in steps of every kernel, and the scratch holds them
        const paged::AttendCall& a = paged::last;
        const uint64_t seen = window ? std::min<uint64_t>(max_length, (uint64_t)window + max_new + sinks) : max_length;
        if (a.chunk == 0 || a.chunk % 128 || a.chunks == 0 || a.chunks > 256 || (uint64_t)a.chunk * a.chunks < seen) return printf("parts %u of %u\n", a.chunks, a.chunk), 1;
        // parts follow the lengths only where all CTAs run at once (two on an SM at most)
        if (a.shrink && (seqs > 32 || a.chunks == 1 || (uint64_t)a.chunks * kv * std::min(seqs, rows) > 2 * 148)) return printf("shrink\n"), 1;
        if (a.chunks > 1 && bytes < (uint64_t)rows * kv * group * a.chunks * (dim + 2) * 4) return printf("scratch\n"), 1;
    }
    printf("right\n");
    return 0;
}
"""


def test_every_bound_has_a_layout(tmp_path):
    (tmp_path / "t.cu").write_text(PROGRAM)
    r = subprocess.run([build._nvcc(), "-std=c++17", "-O1", "-ccbin", "g++", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(CSRC), str(tmp_path / "t.cu"), "-o",
                        str(tmp_path / "t")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=300)
    assert r.stdout.strip() == "right", (r.returncode, r.stdout, r.stderr)
