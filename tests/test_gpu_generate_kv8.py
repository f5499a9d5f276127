"""Greedy decode with the 8-bit cache and with selected blocks (TorchEngine.generate).

A generated token is checked against the logits of a bf16 prefill over the same tokens: it may
lie below the best one by what its cache costs.  With every block selected that is bf16
rounding of a handful of layers (0.1 of the row's standard deviation); an 8-bit cache moves
K and V by 0.3 % (int8: half a step of a block's largest value, about 3.5 sigma, over 127) to 3 %
(e4m3: half a step of 2^-3) of their size, and with them the attention output of each of the
few layers, so 0.5 of the logits' standard deviation is far beyond it.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from helpers import scenario  # noqa: E402
from test_gpu_engine import engine_for  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


MODES = [(torch.int8, None), (torch.float8_e4m3fn, None), (None, 100), (torch.int8, 100), (torch.float8_e4m3fn, 6),
         (None, 3)]


def run(eng, tokens, n, kv, top):
    return eng.generate(eng.prefill(tokens), max_tokens=n, kv_dtype=kv, top_blocks=top)


@pytest.mark.parametrize("name", ["tiny_fp32", "tiny7_fp32"])
@pytest.mark.parametrize("kv,top", MODES)
def test_graph_replay_equals_eager_steps(name, kv, top):
    s = scenario(name)
    eng = engine_for(s)
    eng.eos = set()
    tokens = s.tokens[:75]
    replayed = run(eng, tokens, 24, kv, top)
    with ops.LaunchTimer() as t:  # a timer keeps generate from capturing a graph
        eager = run(eng, tokens, 24, kv, top)
    assert len(replayed) == 24 and replayed == eager
    called = t.summary()
    want = {(False, False): "ckv_attention", (True, False): "ckv_attention_kv8", (False, True): "ckv_attention_sparse",
            (True, True): "ckv_attention_sparse_kv8"}[(kv is not None, top is not None)]
    assert called[want]["launches"] == 24 * s.shape.n_layers


@pytest.mark.parametrize("name", ["tiny_fp32", "tiny7_fp32"])
@pytest.mark.parametrize("kv,top", [m for m in MODES if m[1] in (None, 100)])
def test_tokens_are_near_the_best_of_a_full_prefill(name, kv, top):
    s = scenario(name)
    eng = engine_for(s)
    eng.eos = set()
    tokens = list(s.tokens[:90])
    out = run(eng, tokens, 20, kv, top)
    rows = eng.prefill(tokens + out, logits_from=len(tokens) - 1).logits[:-1].float()
    gap = rows.amax(-1) - rows.gather(1, torch.tensor(out, device=rows.device)[:, None])[:, 0]
    bar = (0.1 if kv is None else 0.5) * rows.std(-1)
    assert bool((gap <= bar).all()), (gap / rows.std(-1)).tolist()


def test_generate_refuses_what_it_does_not_have():
    s = scenario("tiny_fp32")
    eng = engine_for(s)
    res = eng.prefill(s.tokens[:20])
    with pytest.raises(NotImplementedError, match="kv_dtype"):
        eng.generate(res, 2, kv_dtype=torch.float16)
    with pytest.raises(ValueError, match="top_blocks"):
        eng.generate(res, 2, top_blocks=1)
    assert len(eng.generate(res, 1, kv_dtype=torch.int8)) == 1 and eng.generate(res, 0, top_blocks=4) == []
