"""Host side of the paged cache on the CPU: what the classes refuse, the device code's index arithmetic (compiled for the host), and the
pool's books."""
import random
import subprocess
from pathlib import Path

import pytest
import torch

from hf2q_b200 import Hf2qError, build, paged

CSRC = Path(__file__).resolve().parent.parent / "hf2q_b200" / "csrc"
PROGRAM = r"""
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "paged_common.cuh"
using namespace hf2q;
using namespace hf2q::paged;
namespace hf2q {
int32_t ctx_fail(hf2q_ctx*, int32_t code, const char*) { return code; }
}
static uint32_t rnd() { return (uint32_t)rand() << 16 ^ (uint32_t)rand(); }
static uint32_t wild(uint32_t m) { return rand() % 4 ? rnd() % (m + 1) : rnd(); }
int main() {
    // spans of numbers that mean nothing stay inside the arrays
    for (int it = 0; it < 300000; ++it) {
        uint32_t start[2] = {wild(50), wild(50)}, length = wild(400);
        const uint32_t ld = 1 + rnd() % 9, shift = 4 + rnd() % 5, rows = rnd() % 50, pages = 1 + rnd() % 30, heads = 1 + rnd() % 5;
        std::vector<uint32_t> table(ld);
        for (auto& t : table) t = wild(40);
        const Batch b{start, &length, table.data(), 1, rows, ld, rnd() % (rows + 1), 1 + rnd() % 500};
        const Span s = span_of(b, shift, 0);
        if (s.row0 + (uint64_t)s.rows > rows || s.rows > b.max_new || s.length > b.max_length || s.length > ((uint64_t)ld << shift)) return printf("span\n"), 1;
        const bool fits = start[0] <= start[1] && start[1] <= rows && start[1] - start[0] <= b.max_new && length <= b.max_length && length <= ((uint64_t)ld << shift);
        if (s.bad == fits) return printf("bad\n"), 1;
        if (fits && (s.row0 != start[0] || s.rows != start[1] - start[0] || s.length != length)) return printf("cut\n"), 1;
        const Pool c{nullptr, nullptr, nullptr, nullptr, pages, shift, heads};
        for (uint32_t p = 0; p < s.length; p += 7) {
            bool bad = false;
            const uint32_t page = page_of(c, b, 0, p, bad);
            if (page >= pages || bad != (table[p >> shift] >= pages)) return printf("page\n"), 1;
            if (c.row(page, heads - 1, p & (c.size() - 1)) >= ((size_t)pages * heads << shift)) return printf("row\n"), 1;
        }
    }
    // blocks cover every position that a row sees, each once, in order; the tests of whole blocks and of single positions agree with the rows
    for (int it = 0; it < 30000; ++it) {
        const uint32_t log = 4 + rnd() % 4, unit = 1u << log, first = rnd() % 700, last = first + rnd() % 90;
        const Look k{rnd() % 3 ? 1 + rnd() % 300 : 0, rnd() % 2 ? rnd() % 200 : 0, 1.0f};
        const Blocks o = blocks_of(k, first, last, log);
        std::vector<int> in(last + 1 + unit, 0);
        uint32_t before = 0;
        for (uint32_t t = 0; t < o.count; ++t) {
            const uint32_t at = o.at(t);
            if (t && at <= before) return printf("order\n"), 1;
            before = at;
            if ((uint64_t)at << log > last) return printf("past\n"), 1;
            for (uint32_t x = 0; x < unit; ++x) if ((at << log) + x < in.size()) in[(at << log) + x]++;
            bool all = true;
            for (uint32_t i = first; i <= last; ++i) for (uint32_t x = 0; x < unit; ++x) all = all && k.sees(i, (at << log) + x);
            if (all_see(k, first, last, at << log, unit) && !all) return printf("all\n"), 1;
        }
        for (uint32_t j = 0; j <= last; ++j) {
            bool some = false;
            for (uint32_t i = first; i <= last; ++i) some = some || k.sees(i, j);
            if (some != some_see(k, first, last, j)) return printf("some %u %u %u %u %u\n", first, last, j, k.window, k.sinks), 1;
            if (some && in[j] != 1) return printf("missed\n"), 1;
            if (in[j] > 1) return printf("twice\n"), 1;
        }
    }
    printf("right\n");
    return 0;
}
"""


def test_index_arithmetic_of_the_device_code(tmp_path):
    (tmp_path / "t.cu").write_text(PROGRAM)
    r = subprocess.run([build._nvcc(), "-std=c++17", "-O1", "-ccbin", "g++", "-gencode", "arch=compute_100a,code=sm_100a", "-I", str(CSRC), str(tmp_path / "t.cu"), "-o",
                        str(tmp_path / "t")], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, timeout=120)
    assert r.stdout.strip() == "right", r.stdout


class Context:
    """What the checks ask of a context, without a device behind it."""
    device, _h, _lib = 0, None, type("lib", (), {"__getattr__": lambda self, name: None})()


@pytest.mark.parametrize("make", [
    lambda c: paged.PagedCache(c, torch.zeros((1, 2, 1, 16, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 1, 16, 64), dtype=torch.bfloat16)),
    lambda c: paged.PagedCache(c, torch.zeros((1, 2, 1, 16, 64)), torch.zeros((1, 2, 1, 16, 64))),
    lambda c: paged.PagedBatch(c, torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32), rows=1, max_new=1, max_length=1),
    lambda c: paged.PagedBatch(c, torch.zeros(2), torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32), rows=1, max_new=1, max_length=1),
    lambda c: paged.Rope(torch.zeros(32)),
])
def test_tensors_of_the_wrong_kind_or_place_are_refused(make):
    with pytest.raises(Hf2qError):
        make(Context())


def test_matrices_are_checked_before_a_call():
    with pytest.raises(Hf2qError, match="cuda:0"):
        paged._rows(torch.zeros((4, 128)), "x", (torch.float32,), 4, 128, Context())
    with pytest.raises(Hf2qError, match="dtype"):
        paged._rows(torch.zeros((4, 128), dtype=torch.int8), "x", (torch.float32,), 4, 128, Context())


def test_null_contexts_are_refused():
    build.build()
    from hf2q_b200 import _lib
    lib = _lib.load()
    assert lib.hf2q_cuda_pages_attend(None, None, None, None, None, 0, 0, 0, 1.0, 0, 0, None, 0, 0, None, 0) == _lib.ERR_INVALID_ARGUMENT
    assert lib.hf2q_cuda_pages_append(None, None, None, None, None, None, 0, 0, 0, None, 0, 0) == _lib.ERR_INVALID_ARGUMENT
    assert lib.hf2q_cuda_pages_copy(None, None, None, 1, None, None, 0) == _lib.ERR_INVALID_ARGUMENT
    assert lib.hf2q_cuda_pages_copy_rows(None, None, None, 1, None, None, 0) == _lib.ERR_INVALID_ARGUMENT


class Contents:
    """Stands in for a cache: one number a row, on the CPU."""

    def __init__(self, pages, page):
        self.pages, self.page, self.k = pages, page, torch.zeros(())
        self.rows = [-1] * (pages * page)

    def copy_rows(self, src, dst):
        src, dst = src.tolist(), dst.tolist()
        assert len(set(dst)) == len(dst) and not set(src) & set(dst)
        for a, b in zip(src, dst):
            self.rows[b] = self.rows[a]

    def copy_pages(self, src, dst):
        at = lambda t: (t[:, None] * self.page + torch.arange(self.page)).view(-1)
        self.copy_rows(at(src), at(dst))


def write(cache, pool, seq, values):
    pool.reserve(seq, len(values))
    pages, at = pool.pages_of(seq), pool.length_of(seq)
    for i, v in enumerate(values, at):
        cache.rows[pages[i // cache.page] * cache.page + i % cache.page] = v
    pool.advance(seq, len(values))


def same(cache, pool, want):
    used = set()
    for seq in range(pool.seqs):
        row = pool.table[seq].tolist()
        if seq not in want:
            assert row == [-1] * len(row) and int(pool.length[seq]) == 0
            continue
        pages = pool.pages_of(seq)
        used |= set(pages)
        assert len(set(pages)) == len(pages) and row == pages + [-1] * (len(row) - len(pages))
        assert int(pool.length[seq]) == pool.length_of(seq) == len(want[seq])
        assert [cache.rows[pages[i // cache.page] * cache.page + i % cache.page] for i in range(len(want[seq]))] == want[seq]
    assert pool.n_free_pages == cache.pages - len(used)


@pytest.mark.parametrize("seed", range(6))
def test_the_pool_keeps_every_sequence_through_branches_packing_and_want_of_pages(seed):
    rnd = random.Random(seed)
    cache = Contents(rnd.choice([5, 12, 40]), rnd.choice([1, 4, 16]))
    pool = paged.PagePool(cache, 4, 6 * cache.page + 1)
    want, mark, refused = {}, 0, 0
    for _ in range(400):
        what, seq = rnd.choice(["open", "write", "write", "write", "fork", "compact", "pack", "close"]), rnd.choice(list(want) or [None])
        if seq is None:
            what = "open"
        try:
            if what == "open":
                want[pool.open()] = []
            elif what == "write":
                n = rnd.randrange(0, 2 * cache.page + 2)
                if len(want[seq]) + n > pool.max_length:
                    with pytest.raises(Hf2qError):
                        pool.reserve(seq, n)
                    continue
                write(cache, pool, seq, list(range(mark, mark + n)))
                want[seq], mark = want[seq] + list(range(mark, mark + n)), mark + n
            elif what == "fork":
                want[pool.fork(seq)] = list(want[seq])
            elif what == "compact":
                keep = [i for i in range(len(want[seq])) if i < cache.page * rnd.randrange(3) or rnd.random() < 0.6]
                pool.compact(seq, keep)
                want[seq] = [want[seq][i] for i in keep]
            elif what == "pack":
                assert pool.pack() == cache.pages - pool.n_free_pages
                assert all(p < cache.pages - pool.n_free_pages for s in want for p in pool.pages_of(s))
            else:
                pool.close(seq)
                del want[seq]
        except RuntimeError as e:                          # nothing has changed then
            assert "no free" in str(e)
            refused += 1
        same(cache, pool, want)
    assert refused


def test_the_pool_refuses_what_its_books_do_not_allow():
    pool = paged.PagePool(Contents(4, 4), 2, 16)
    with pytest.raises(Hf2qError):
        paged.PagePool(Contents(4, 4), 0, 16)
    with pytest.raises(RuntimeError, match="not in use"):
        pool.reserve(0, 1)
    a = pool.open()
    for call in (lambda: pool.reserve(a, 17), lambda: pool.reserve(a, -1), lambda: pool.advance(a, 1), lambda: pool.compact(a, [0])):
        with pytest.raises(Hf2qError):
            call()
    pool.reserve(a, 6)
    with pytest.raises(Hf2qError):
        pool.advance(a, 9)
    pool.advance(a, 6)
    for keep in ([1, 0], [0, 0], [-1], [6]):
        with pytest.raises(Hf2qError):
            pool.compact(a, keep)
    b = pool.fork(a)
    with pytest.raises(RuntimeError, match="slot"):
        pool.open()
    pool.close(a)
    with pytest.raises(RuntimeError, match="not in use"):
        pool.close(a)
    assert pool.length_of(b) == 6 and pool.n_free_pages == 2


def test_frequencies():
    f = paged.rope_frequencies(8, 10000.0)
    assert torch.equal(f, torch.tensor([1.0, 0.1, 0.01, 0.001]))
    assert torch.equal(paged.rope_frequencies(8, 10000.0, linear=4.0), torch.tensor([0.25, 0.025, 0.0025, 0.00025]))
    # wavelengths 6.3, 63, 628 and 6283 against a trained context of 600: more than 4 turns kept, fewer than 1 divided, 600 / 628 = 0.95 of one too
    g = paged.rope_frequencies(8, 10000.0, bands={"factor": 8.0, "low": 1.0, "high": 4.0, "trained": 600})
    assert torch.equal(g, torch.tensor([1.0, 0.1, 0.01 / 8, 0.001 / 8]))
    # 1257 positions: 2 turns at 0.01, a third of the way between low and high
    g = paged.rope_frequencies(8, 10000.0, bands={"factor": 8.0, "low": 1.0, "high": 4.0, "trained": 400 * 3.141592653589793})
    torch.testing.assert_close(g[2], torch.tensor(0.01 * (1 / 3 + 2 / 3 / 8)), rtol=2 ** -23, atol=0)


def test_the_tile_kernel_lets_the_next_launch_start_when_its_columns_are_held():
    """The next launch may take tensor memory and then wait for this one, whose allocation waits without a limit."""
    text = (CSRC / "paged_tiles.cu").read_text()
    body = text[text.index("attend_tiles_kernel("):text.index("cudaError_t launch(")]
    assert body.count("pdl_trigger()") == 1 and body.count("pdl_wait()") == 1 and body.count("claim_columns(") == 1
    claim = body.index("claim_columns(")
    assert body.index("pdl_wait()") < claim < body.index("__syncthreads()", claim) < body.index("pdl_trigger()")
