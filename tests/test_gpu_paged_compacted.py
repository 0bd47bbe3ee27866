"""The decoder after a compaction with holes: against the scalar forward in which the new tokens do not see what was forgotten and every token keeps
its position."""
import numpy as np
import pytest
import torch

from hf2q_b200.decoder_paged import PagedLlamaDecoder
from hf2q_b200.engine import Engine
from oracle import llama_forward
from tests.test_gpu_decoder import CFG, LOGIT_GATE, build_model
from tests.util import rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights(gpu_ctx):
    return build_model(gpu_ctx, CFG)


def tokens(seed, n):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, CFG.vocab, size=n).astype(np.int32))


@pytest.mark.parametrize("keep", [[*range(4), *range(110, 150)], [*range(0, 150, 3)], [*range(64), *range(100, 130)]], ids=["first-and-last", "every-third", "a-gap-and-no-end"])
def test_tokens_behind_a_compaction(gpu_ctx, weights, keep):
    """A portion through the panels, single tokens, and the captured step; a branch goes on as well; then the same once more."""
    dec = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=32, n_slots=2, pages=12)
    ids, more = tokens(1, 150), tokens(2, 44)
    s = dec.open_slot()
    dec.extend(s, ids, [])
    dec.pages.compact(s, keep)
    n = keep[-1] + 1                                       # the position that the sequence goes on at
    ids = torch.cat([ids[:n], more])
    hidden = np.zeros((len(ids), len(ids)), dtype=bool)
    hidden[n:, [p for p in range(n) if p not in keep]] = True
    got = [dec.extend(s, more[:40], [0, 20, 39]), dec.extend(s, more[40:43], [2]), dec.extend(s, more[43:], [0])]
    gpu_ctx.check_status()
    want = llama_forward.forward(ids.numpy(), weights[1], CFG, hidden)
    assert rel_l2(torch.cat(got).cpu().numpy(), want[[n, n + 20, n + 39, n + 42, n + 43]]) < LOGIT_GATE
    branch = dec.fork(s)
    for slot in (s, branch):
        dec.bind(slot)
        tok = int(dec.tok[0])
        dec.generate(1)
        wider = np.pad(hidden, ((0, 1), (0, 1)))
        wider[-1] = np.append(hidden[-1], False)
        want = llama_forward.forward(np.append(ids.numpy(), np.int32(tok)), weights[1], CFG, wider)[-1]
        assert rel_l2(dec.logits.cpu().numpy()[0], want) < LOGIT_GATE
    # once more: of what is left every second place, and the last one
    left = [*keep, *range(n, n + 45)]
    places = sorted({*range(0, len(left), 2), len(left) - 1})
    dec.pages.compact(branch, places)
    ids = torch.cat([ids, torch.tensor([tok], dtype=torch.int32), tokens(3, 2)])
    gone = [p for p in range(n + 45) if p not in {left[i] for i in places}]
    wider = np.pad(hidden, ((0, 3), (0, 3)))
    wider[n + 44, :] = np.append(hidden[-1], [False] * 3)
    wider[n + 45:, gone] = True
    got = dec.extend(branch, ids[-2:], [0, 1])
    gpu_ctx.check_status()
    assert rel_l2(got.cpu().numpy(), llama_forward.forward(ids.numpy(), weights[1], CFG, wider)[-2:]) < LOGIT_GATE


@pytest.mark.parametrize("through", ["decoder", "pool"])
def test_compaction_and_packing_wait_for_the_call_before(gpu_ctx, weights, through):
    """On a stream of their own, directly behind a portion on another one."""
    ids, keep = tokens(4, 400), [*range(4), *range(200, 400, 3)]

    def run(streams):
        dec = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=400, n_slots=2, pages=20)
        out = []
        for _ in range(3):
            a, b = dec.open_slot(), dec.open_slot()
            calls = dec if through == "decoder" else dec.pages
            with torch.cuda.stream(streams[0]):
                dec.extend(a, tokens(5, 130), [])
                dec.extend(b, ids, [])
            with torch.cuda.stream(streams[1]):
                calls.compact(b, keep)
            with torch.cuda.stream(streams[2]):
                dec.close_slot(a)
                assert calls.pack() == 2
            with torch.cuda.stream(streams[0]):
                out.append(dec.extend(b, tokens(6, 9), [8]))
            with torch.cuda.stream(streams[1]):
                out.append(dec.generate(4))
            torch.cuda.synchronize()
            dec.close_slot(b)
        gpu_ctx.check_status()
        return out

    here = torch.cuda.current_stream()
    want = run([here, here, here])
    got = run([torch.cuda.Stream() for _ in range(3)])
    assert all(torch.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("keep", [range(1, 192), range(0, 192, 4), [*range(70), *range(75, 192)]], ids=["all-but-one", "every-fourth", "a-gap"])
@pytest.mark.parametrize("more", [0, 1])
def test_a_full_pool_gives_what_a_large_one_gives(gpu_ctx, weights, more, keep):
    """Packed in the sequence's own pages (and through a free one), in all layers."""
    got = []
    for pages in (20, 3 + more):
        dec = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=192, n_slots=1, pages=pages)
        s = dec.open_slot()
        dec.extend(s, tokens(7, 192), [])
        dec.compact(s, keep)
        own = torch.tensor(dec.pages.pages_of(s), device="cuda")
        at = torch.arange(len(keep), device="cuda")
        rows = lambda t: t[:, own[at // 64], :, at % 64]
        got.append([rows(t).clone() for t in (dec.cache.k, dec.cache.v, dec.cache.k_scale, dec.cache.v_scale)] + [dec.extend(s, tokens(8, 1), [0])])
        gpu_ctx.check_status()
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_prompts_one_after_another_where_the_pool_holds_one(gpu_ctx, weights):
    prompts = [tokens(9 + i, n).tolist() for i, n in enumerate((100, 70, 120))]
    got = []
    for slots, pages in ((3, 12), (2, 3)):
        dec = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=128, n_slots=slots, pages=pages)
        got.append(Engine(dec).generate(prompts, 8))
        assert dec.pages.n_free_pages == pages
    gpu_ctx.check_status()
    assert got[0] == got[1]


def test_buffers_of_a_portion_stay_while_its_stream_works(gpu_ctx, weights):
    """Made on one stream, used on a second one that is held up, replaced on a third one: what the first one allocates then is other memory."""
    ids = tokens(20, 12 + 24 + 12 + 150)

    def run(streams, hold):
        dec = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=256, n_slots=1, pages=8)
        s, out, at = dec.open_slot(), [], 0
        for i, n in enumerate((24, 12, 150)):
            with torch.cuda.stream(streams[i]):
                if hold and i == 1:
                    torch.cuda._sleep(200_000_000)         # (a tenth of a second)
                out.append(dec.extend(s, ids[at:at + n].cuda(), [n - 1]))
            at += n
        with torch.cuda.stream(streams[0]):
            junk = [torch.full((rows, cols), float("nan"), device="cuda") for rows in (24,) for cols in (CFG.hidden, dec.qkv_cols, CFG.hidden // 2, CFG.q_rows // 2, CFG.ffn // 2) for _ in "ab"]
        torch.cuda.synchronize()
        gpu_ctx.check_status()
        del junk
        return out

    here = torch.cuda.current_stream()
    want = run([here] * 3, False)
    assert all(torch.equal(a, b) for a, b in zip(run([torch.cuda.Stream() for _ in range(3)], True), want))
