"""Block selection at the sizes of its larger kernels, and sparse calls that run at the same time."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402
from test_gpu_kv8 import DEV, queries  # noqa: E402
from test_gpu_sparse import KINDS, caches, context, digest_of, spread_rows  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


# more than 32 pairs of token and KV head: keys in the workspace, a group of threads per pair, by
# the number of blocks (up to 512, 1024, 4096, 8192, 32768), at and around each limit
@pytest.mark.parametrize("Hq,H,D,n,m,top", [
    (8, 2, 64, 8192, 20, 40), (8, 2, 64, 8193, 20, 40), (28, 4, 128, 16384, 11, 64), (28, 4, 128, 16385, 40, 64),
    (28, 4, 128, 32896, 60, 64), (14, 2, 64, 50000, 33, 17), (40, 8, 128, 65536, 5, 128), (16, 1, 128, 65537, 34, 100),
    (4, 2, 64, 131072, 17, 700), (4, 2, 64, 131073, 17, 64), (4, 4, 64, 524288, 9, 128), (7, 1, 128, 40000, 64, 1024),
    (12, 1, 64, 30000, 50, 2)])
def test_selection_of_many_rows(Hq, H, D, n, m, top):
    assert _lib.load().ckv_block_select_workspace_size(m, Hq, H, D, n) > 0
    k, _ = context(H, n, D, seed=m)
    d = digest_of(k)
    q = queries(m, Hq, D, 3)
    p = spread_rows(n, m, 4)
    got = ops.block_select(q, d, p, top)
    assert torch.equal(got.cpu().long(), ref.select(q, d.codes, d.scale, p, top))


@pytest.mark.parametrize("n", [16400, 40000, 140000])
def test_ties_of_many_rows_go_to_the_lower_block(n):
    H, Hq, D, m = 2, 8, 64, 40
    k, _ = context(H, 64, D)
    k = k.repeat(1, n // 64 + 1, 1)[:, :n].contiguous()  # every score four blocks apart again
    d = digest_of(k)
    q = queries(m, Hq, D, 1)
    q[3] = 0  # every score equal
    p = spread_rows(n, m, 2)
    for top in (2, 3, 61, 250, 257):
        assert torch.equal(ops.block_select(q, d, p, top).cpu().long(), ref.select(q, d.codes, d.scale, p, top))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,H,D,n,m,top", [(28, 4, 128, 9000, 1, 64), (28, 4, 128, 33000, 30, 32), (14, 2, 64, 2000, 400, 9)])
def test_two_sparse_graphs_at_once_and_another_stream(Hq, H, D, n, m, top, kind):
    """Two captured calls replayed at the same time on two streams share nothing but the cache."""
    _, _, _, sparse, _ = caches(kind, H, n, D, seed=1)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    qs = [queries(m, Hq, D, s) for s in (1, 2)]
    want = [sparse(q, p, top) for q in qs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        out, lists = torch.zeros_like(q), torch.zeros((m, H, top), dtype=torch.int32, device=DEV)
        with torch.cuda.graph(g, stream=s):
            for _ in range(4):
                sparse(q, p, top, out=out, blocks=lists)
        graphs.append(g)
        outs.append((out, lists))
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, w in zip(outs, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.default_stream())
        eager = [sparse(q, p, top) for q in qs]
    streams[0].synchronize()
    for got, w in zip(eager, want):
        assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_a_digest_built_in_two_calls_at_once():
    """Each call's digest lies in its own scratch."""
    Hq, H, D, n, m, top = 14, 2, 64, 5000, 12, 20
    data = [(*context(H, n, D, seed=s), queries(m, Hq, D, s)) for s in (1, 2)]
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    want = [ops.attention_sparse(q, k, v, p, top) for k, v, q in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                k, v, q = data[i]
                got[i].append(ops.attention_sparse(q, k, v, p, top))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g[0], want[i][0]) and torch.equal(g[1], want[i][1]) for g in got[i])
