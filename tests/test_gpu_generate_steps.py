"""Every attention call of a greedy decode with the 8-bit cache or with selected blocks, against its
definition: the rows that have been written so far, no more and no fewer, each quantised as
its block stands.  Tolerances as in tests/test_gpu_kv8.py (tests/test_gpu_generate_kv8.py bounds
only what the options cost the logits)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from helpers import scenario  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402
from test_gpu_engine import engine_for  # noqa: E402
from test_gpu_kv8 import check_attention  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


class Watch:
    """Stands in front of the ops that a decode step calls and checks what they leave."""

    def __init__(self, monkeypatch, K0, V0):
        self.rows = [[k.clone(), v.clone()] for k, v in zip(K0, V0)]  # per layer, the bf16 rows so far
        self.caches, self.calls = {}, 0
        self.real = {n: getattr(ops, n) for n in ("kv8_write", "attention_kv8", "attention_sparse_kv8", "attention_sparse")}
        for n in self.real:
            monkeypatch.setattr(ops, n, getattr(self, n))

    def kv8_write(self, cache, k, v, start, m=None, by_position=False):
        self.real["kv8_write"](cache, k, v, start, m, by_position)
        if not by_position:  # the prefill's rows
            self.caches[id(cache)] = len(self.caches)
            return cache
        li, pos = self.caches[id(cache)], int(start)
        for side, x in zip((0, 1), (k, v)):
            assert self.rows[li][side].shape[1] == pos
            self.rows[li][side] = torch.cat([self.rows[li][side], x[:, pos:pos + 1]], 1)
        return cache

    def held(self, cache, n):
        """The cache's values of the first n tokens, after it has been found to be their quantisation."""
        out = []
        for x, codes, scale in zip(self.rows[self.caches[id(cache)]], (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
            assert x.shape[1] == n
            rc, rs = ref.quantize(x, cache.dtype)
            nb = rs.shape[1]
            assert torch.equal(codes[:, :nb * 16].float().double(), rc) and torch.equal(scale[:, :nb].double(), rs)
            out.append(ref.values(rc, rs)[:, :n])
        return out

    def attention_kv8(self, q, cache, positions, out):
        self.real["attention_kv8"](q, cache, positions, out=out)
        k, v = self.held(cache, int(positions) + 1)
        x = q.view(1, -1, cache.head_dim)
        check_attention(out, x, k, v, positions)
        self.calls += 1

    def selected(self, q, k_rows, positions, top, blocks):
        want = ref.select(q, *ref.digest(k_rows), positions, top)
        assert torch.equal(blocks.cpu().long(), want)

    def attention_sparse_kv8(self, q, cache, positions, top, out, blocks):
        self.real["attention_sparse_kv8"](q, cache, positions, top, out=out, blocks=blocks)
        k, v = self.held(cache, int(positions) + 1)
        x = q.view(1, -1, cache.head_dim)
        self.selected(x, self.rows[self.caches[id(cache)]][0], positions, top, blocks)
        check_attention(out, x, k, v, positions, blocks)
        self.calls += 1

    def attention_sparse(self, q, k_cache, v_cache, positions, top, digest, out, blocks):
        self.real["attention_sparse"](q, k_cache, v_cache, positions, top, digest=digest, out=out, blocks=blocks)
        n, x = int(positions) + 1, q.view(1, -1, k_cache.shape[2])
        li = self.calls % len(self.rows)
        first = self.rows[li][0].shape[1]
        assert torch.equal(k_cache[:, :first], self.rows[li][0]) and torch.equal(v_cache[:, :first], self.rows[li][1])
        assert bool(k_cache[:, first:n].any(-1).all()) and not k_cache[:, n:].any()
        self.selected(x, k_cache[:, :n], positions, top, blocks)
        check_attention(out, x, k_cache[:, :n], v_cache[:, :n], positions, blocks)
        self.calls += 1


@pytest.mark.parametrize("name,n", [("tiny_fp32", 75), ("tiny7_fp32", 78), ("tiny_fp32", 16), ("tiny7_fp32", 1)])
@pytest.mark.parametrize("kv,top", [(torch.int8, None), (torch.float8_e4m3fn, None), (torch.int8, 3), (torch.float8_e4m3fn, 100),
                                    (None, 3), (None, 100)])
def test_every_step_attends_to_the_rows_so_far(name, n, kv, top, monkeypatch):
    s = scenario(name)
    eng = engine_for(s)
    eng.eos = set()
    res = eng.prefill(s.tokens[:n])
    steps = 20
    plain = eng.generate(res, steps, kv_dtype=kv, top_blocks=top)
    watch = Watch(monkeypatch, *res.cache)
    with ops.LaunchTimer():  # keeps generate from capturing a graph
        watched = eng.generate(res, steps, kv_dtype=kv, top_blocks=top)
    assert watched == plain and watch.calls == steps * s.shape.n_layers
