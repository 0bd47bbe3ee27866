"""What a GGUF file says of its rotary turns: read, refused where it is not served, and not passed over in silence."""
import warnings

import numpy as np
import pytest

from hf2q_b200 import Hf2qError, gguf
from hf2q_b200.decoder import LlamaDecoder, rotary_scaling
from hf2q_b200.decoder_paged import PagedLlamaDecoder


def file(tmp_path, factors=None, **keys):
    g = gguf.GgufWriter()
    g.add_kv("general.architecture", gguf.T_STRING, "llama")
    for k, v in keys.items():
        g.add_kv("llama.rope." + k.replace("__", "."), gguf.T_STRING if isinstance(v, str) else gguf.T_F32, v)
    if factors is not None:
        g.add_tensor("rope_freqs.weight", (len(factors),), 0, np.array(factors, np.float32))
    g.add_tensor("output_norm.weight", (4,), 0, np.ones(4, np.float32))
    g.write(tmp_path / "m.gguf")
    return tmp_path / "m.gguf"


PLAIN = [{}, {"scaling__type": "none"}, {"scaling__type": "none", "scaling__factor": 4.0}, {"scale_linear": 1.0}]
SCALED = [({"scaling__type": "linear", "scaling__factor": 4.0}, 4.0), ({"scale_linear": 2.0}, 2.0)]
OTHERS = [{"scaling__type": "yarn", "scaling__factor": 4.0}, {"scaling__type": "longrope"}]


def what(path):
    with gguf.GgufFile(path) as g:
        return rotary_scaling(g)


def test_scalings_are_read(tmp_path):
    for keys in PLAIN:
        assert what(file(tmp_path, **keys)) == ("none", 1.0, None)
    for keys, by in SCALED:
        assert what(file(tmp_path, **keys)) == ("linear", by, None)
    kind, by, factors = what(file(tmp_path, factors=[1.0, 2.0, 8.0]))
    assert (kind, by, factors.tolist()) == ("none", 1.0, [1.0, 2.0, 8.0])


@pytest.mark.parametrize("keys", OTHERS)
def test_other_scalings_are_refused_with_pages(tmp_path, keys):
    with pytest.raises(Hf2qError, match=keys["scaling__type"]):
        PagedLlamaDecoder.from_gguf(None, file(tmp_path, **keys))


def test_a_cache_that_does_not_scale_says_so(tmp_path):
    """(The files have no weights: loading goes on behind the warning, and ends there.)"""
    for keys in [k for k, _ in SCALED] + OTHERS + [{"factors": [1.0, 2.0]}]:
        with pytest.warns(UserWarning, match="scales its rotary turns") as seen, pytest.raises(TypeError):
            LlamaDecoder.from_gguf(None, file(tmp_path, **keys))
        assert seen[0].filename == __file__
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        for keys in PLAIN + [{"scaling__type": "linear", "scaling__factor": 1.0}]:
            with pytest.raises(TypeError):
                LlamaDecoder.from_gguf(None, file(tmp_path, **keys))
