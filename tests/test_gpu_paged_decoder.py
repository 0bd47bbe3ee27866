"""The quantized decoder over pages: against the scalar forward, sequences in turn against each alone, branches, and what it refuses."""
import json

import numpy as np
import pytest
import torch

from hf2q_b200 import Hf2qError, registry
from hf2q_b200.decoder_paged import PagedLlamaDecoder
from hf2q_b200.engine import Engine, Entry
from oracle import llama_forward
from tests.test_gpu_decoder import CFG, LOGIT_GATE, build_model
from tests.util import make_quant_weight, rel_l2

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def weights(gpu_ctx):
    return build_model(gpu_ctx, CFG)


@pytest.fixture()
def dec(gpu_ctx, weights):
    return PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=32, n_slots=3, pages=12)


def tokens(seed, n):
    return torch.from_numpy(np.random.default_rng(seed).integers(0, CFG.vocab, size=n).astype(np.int32))


def alone(gpu_ctx, weights, portions, n):
    """Logits after each portion and the continuation of a sequence that has a decoder for itself."""
    d = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=32, n_slots=1, pages=8)
    s = d.open_slot()
    logits = [d.extend(s, p, [len(p) - 1]) for p in portions]
    first = int(d.tok[0])
    return logits, [first] + d.generate(n).tolist()


def test_prompt_and_steps_match_the_scalar_forward(dec, weights):
    """Portions of 32, 32 and 11 rows (the products' panels), one of 5 (without them) and single tokens."""
    ids = tokens(1, 86)
    s = dec.open_slot()
    got = [dec.extend(s, ids[:75], [0, 40, 74]), dec.extend(s, ids[75:80], [4])]
    got += [dec.extend(s, ids[i:i + 1], [0]) for i in range(80, 86)]
    dec.ctx.check_status()
    want = llama_forward.forward(ids.numpy(), weights[1], CFG)
    assert rel_l2(torch.cat(got).cpu().numpy(), want[[0, 40, 74, 79, *range(80, 86)]]) < LOGIT_GATE
    assert int(dec.pos[0]) == 86 and dec.pages.length_of(s) == 86
    assert rel_l2(dec.logits.cpu().numpy()[0], want[-1]) < LOGIT_GATE
    # a step of the captured graph, the logits of its token
    tok = int(dec.tok[0])
    dec.generate(1)
    want = llama_forward.forward(np.append(ids.numpy(), np.int32(tok)), weights[1], CFG)[-1]
    assert rel_l2(dec.logits.cpu().numpy()[0], want) < LOGIT_GATE
    dec.ctx.check_status()


def test_sequences_in_turn_are_what_each_is_alone(gpu_ctx, weights, dec):
    a, b = [tokens(2, 70), tokens(3, 9)], [tokens(4, 58)]
    want_a, want_b = alone(gpu_ctx, weights, a, 9), alone(gpu_ctx, weights, b, 12)
    x, y = dec.open_slot(), dec.open_slot()
    la = [dec.extend(x, a[0], [69])]
    lb = [dec.extend(y, b[0], [57])]
    la.append(dec.extend(x, a[1], [8]))
    for got, want in ((la, want_a[0]), (lb, want_b[0])):
        assert all(torch.equal(g, w) for g, w in zip(got, want))
    out = {x: [], y: []}
    for s in (x, y):
        dec.bind(s)
        out[s].append(int(dec.tok[0]))
    for s, n in ((y, 4), (x, 5), (y, 8), (x, 4)):              # (the second takes a new page at 64, on the way)
        dec.bind(s)
        out[s] += dec.generate(n, use_graph=n != 4).tolist()
    dec.ctx.check_status()
    assert out[x] == want_a[1] and out[y] == want_b[1]


def test_branches_share_and_then_part(gpu_ctx, weights, dec):
    ids, more = tokens(5, 70), tokens(6, 20)
    plain = alone(gpu_ctx, weights, [ids], 12)[1]
    other = alone(gpu_ctx, weights, [ids, more], 3)
    x = dec.open_slot()
    dec.extend(x, ids, [])
    y = dec.fork(x)
    assert dec.pages.pages_of(x) == dec.pages.pages_of(y)
    z = dec.fork(y)
    got = dec.extend(y, more, [19])                            # into a page of its own
    assert dec.pages.pages_of(x)[0] == dec.pages.pages_of(y)[0] and dec.pages.pages_of(x)[1] != dec.pages.pages_of(y)[1]
    assert torch.equal(got, other[0][1])
    assert [int(dec.tok[0])] + dec.generate(3).tolist() == other[1]
    dec.close_slot(y)
    for s in (x, z):                                           # the branch that nothing was added to, and the stem
        dec.bind(s)
        assert [int(dec.tok[0])] + dec.generate(12).tolist() == plain
    dec.ctx.check_status()


def test_packed_pages_keep_the_sequences(gpu_ctx, weights, dec):
    ids = tokens(7, 100)
    want = alone(gpu_ctx, weights, [ids], 6)[1]
    x, y = dec.open_slot(), dec.open_slot()
    dec.extend(x, tokens(8, 150), [])
    dec.extend(y, ids, [])
    dec.close_slot(x)
    assert dec.pages.pack() == 2 and sorted(dec.pages.pages_of(y)) == [0, 1]
    dec.bind(y)
    assert [int(dec.tok[0])] + dec.generate(6).tolist() == want
    dec.ctx.check_status()


def test_compacted_sequences_go_on_where_they_end(gpu_ctx, weights, dec):
    """Back to a prefix of 70 tokens: what follows is what follows that prefix."""
    ids, more = tokens(16, 70), tokens(17, 3)
    d = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=32, n_slots=1, pages=8)
    s = d.open_slot()
    d.extend(s, ids, [])
    want_first = d.tok.clone()
    want = d.generate(4).tolist()
    x = dec.open_slot()
    dec.extend(x, ids, [])
    assert torch.equal(dec.tok, want_first)
    y = dec.fork(x)
    dec.extend(y, more, [])
    dec.generate(2)
    dec.pages.compact(y, range(70))
    dec.tok.copy_(want_first)
    assert dec.generate(4).tolist() == want
    assert int(dec.pos[0]) == 74 == dec.pages.length_of(y)
    dec.bind(x)
    assert dec.generate(4).tolist() == want
    dec.ctx.check_status()


def test_calls_on_several_streams_follow_one_another(gpu_ctx, weights, dec):
    ids = tokens(9, 90)
    want = alone(gpu_ctx, weights, [ids[:60], ids[60:]], 5)
    s, streams = dec.open_slot(), [torch.cuda.Stream() for _ in range(3)]
    with torch.cuda.stream(streams[0]):
        dec.extend(s, ids[:60], [])
    with torch.cuda.stream(streams[1]):
        got = dec.extend(s, ids[60:], [29])
        first = int(dec.tok[0])
    with torch.cuda.stream(streams[2]):
        more = dec.generate(5).tolist()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0][1]) and [first] + more == want[1]
    dec.ctx.check_status()


def test_refusals_leave_the_sequences_as_they_were(gpu_ctx, weights):
    d = PagedLlamaDecoder(gpu_ctx, CFG, weights[0], prefill_chunk=32, n_slots=2, pages=3)
    with pytest.raises(RuntimeError, match="no sequence is bound"):
        d.generate(2)
    with pytest.raises(RuntimeError, match="not in use"):
        d.extend(0, tokens(0, 4), [])
    with pytest.raises(Hf2qError):
        d.prefill(tokens(0, 4))
    ids = tokens(10, 66)
    want = alone(gpu_ctx, weights, [ids], 4)[1]
    x, y = d.open_slot(), d.open_slot()
    with pytest.raises(RuntimeError, match="slot"):
        d.open_slot()
    d.extend(x, ids, [])
    with pytest.raises(RuntimeError, match="no free page"):
        d.extend(y, tokens(11, 65), [])
    with pytest.raises(Hf2qError, match="max_seq"):
        d.extend(x, tokens(0, CFG.max_seq), [])
    with pytest.raises(Hf2qError):
        d.extend(x, tokens(0, 0), [])
    d.bind(x)
    with pytest.raises(Hf2qError):
        d.prefill(tokens(0, 4))                                # not where the sequence ends
    with pytest.raises(RuntimeError, match="no free page"):
        d.generate(200)
    assert d.generate(0).tolist() == []
    assert [int(d.tok[0])] + d.generate(4).tolist() == want
    d.close_slot(x)
    with pytest.raises(RuntimeError, match="no sequence is bound"):
        d.generate(1)
    d.extend(y, tokens(11, 65), [])
    d.ctx.check_status()


def file(path, **more):
    from hf2q_b200 import gguf
    hidden, n_q, n_kv, hd, ffn, vocab = 2048, 16, 4, 128, 6144, 512
    g = gguf.GgufWriter()
    g.add_kv("general.architecture", gguf.T_STRING, "llama")
    for k, v in {"block_count": 1, "embedding_length": hidden, "attention.head_count": n_q, "attention.head_count_kv": n_kv, "feed_forward_length": ffn}.items():
        g.add_kv("llama." + k, gguf.T_U32, v)
    g.add_kv("llama.attention.layer_norm_rms_epsilon", gguf.T_F32, 1e-5)
    g.add_kv("llama.rope.freq_base", gguf.T_F32, 10000.0)
    if "linear" in more:
        g.add_kv("llama.rope.scaling.type", gguf.T_STRING, "linear")
        g.add_kv("llama.rope.scaling.factor", gguf.T_F32, more["linear"])
    if "factors" in more:
        g.add_tensor("rope_freqs.weight", (hd // 2,), 0, np.full(hd // 2, more["factors"], np.float32))
    rng = np.random.default_rng(0)
    for name, n, k, t in (("token_embd", vocab, hidden, 12), ("output", vocab, hidden, 14), ("blk.0.attn_q", n_q * hd, hidden, 12), ("blk.0.attn_k", n_kv * hd, hidden, 12),
                          ("blk.0.attn_v", n_kv * hd, hidden, 14), ("blk.0.attn_output", hidden, n_q * hd, 12), ("blk.0.ffn_gate", ffn, hidden, 12),
                          ("blk.0.ffn_up", ffn, hidden, 12), ("blk.0.ffn_down", hidden, ffn, 14)):
        g.add_tensor(name + ".weight", (n, k), t, make_quant_weight(t, n, k, seed=len(name) + n))
    for name in ("blk.0.attn_norm.weight", "blk.0.ffn_norm.weight", "output_norm.weight"):
        g.add_tensor(name, (hidden,), 0, (1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32))
    g.write(path)
    return path


def test_a_file_through_the_registry_the_engine_and_the_command(gpu_ctx, tmp_path, capsys):
    from hf2q_b200.__main__ import main
    path = file(tmp_path / "m.gguf")
    m = registry.load_model(gpu_ctx, path, max_seq=256, n_slots=2, pages=6)
    ids = [tokens(i, n).remainder(512).tolist() for i, n in ((12, 80), (13, 41), (14, 7))]
    want = registry.load_model(gpu_ctx, path, max_seq=256)
    e, plain = Engine(m), Engine(want)
    a = [e.step([Entry("a", ids[0][:40], [10, 39]), Entry("b", ids[1], [40])]), e.step([Entry("a", ids[0][40:], [39])], end=["a", "b"])]
    w = torch.cat([plain.step([Entry("a", ids[0], [10, 39, 79])], end=["a"]), plain.step([Entry("b", ids[1], [40])], end=["b"])])
    # each is within LOGIT_GATE of the scalar forward
    assert rel_l2(torch.cat([a[0][:2], a[1], a[0][2:]]).cpu().numpy(), w.cpu().numpy()) < 2 * LOGIT_GATE
    got = Engine(m).generate(ids, 5)
    assert [len(g) for g in got] == [5, 5, 5] and m.pages.n_free_pages == 6
    capsys.readouterr()
    assert main(["generate", "--model", str(path), "--new", "5", "--max-seq", "256", "--slots", "2", "--pages", "6"] +
                [x for p in ids for x in ("--prompt", ",".join(map(str, p)))]) == 0
    assert [json.loads(line) for line in capsys.readouterr().out.splitlines() if line.startswith("[")] == got
    gpu_ctx.check_status()


def test_a_file_that_scales_its_turns(gpu_ctx, tmp_path):
    """Linear scaling by 4 is a divisor of 4 for each pair, and it does something."""
    ids = tokens(15, 60).remainder(512)
    got = []
    for i, more in enumerate(({}, {"linear": 4.0}, {"factors": 4.0})):
        m = PagedLlamaDecoder.from_gguf(gpu_ctx, file(tmp_path / f"{i}.gguf", **more), max_seq=128, n_slots=1)
        got.append(m.extend(m.open_slot(), ids, list(range(60))))
    gpu_ctx.check_status()
    assert torch.equal(got[1], got[2]) and not torch.equal(got[0], got[1])


def test_designs_without_pages_say_so(tmp_path):
    from hf2q_b200 import registry as r
    for name in r.ARCHITECTURES:
        if name != "llama":
            with pytest.raises(Hf2qError, match="pages"):
                r.ARCHITECTURES[name](None, tmp_path, torch.bfloat16, 64, 1, 64, 4)
