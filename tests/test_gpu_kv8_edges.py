"""Edges of the 8-bit cache, its attention and the attention over selected blocks: non-finite
rows, writes that go back, calls at the limits.  Tolerances as in tests/test_gpu_kv8.py."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402
from test_gpu_kv8 import BF, DEV, TYPES, check_attention, filled, queries  # noqa: E402
from test_gpu_sparse import caches  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


def check_nan_rows(run, q, kd, vd, p, at, blocks=None):
    """NaN in one channel of the query rows `at` (token, head): they alone come out as NaN."""
    bad = q.clone()
    for t, h in at:
        bad[t, h, 3] = float("nan")
    out = run(bad)
    nan = torch.zeros(q.shape[:2], dtype=torch.bool, device=DEV)
    for t, h in at:
        nan[t, h] = True
    assert bool(out[nan].isnan().all()) and bool(out[~nan].isfinite().all())
    # the other rows are what they are without it
    check_attention(torch.where(nan[..., None], run(q), out), q, kd, vd, p, blocks)


# a cluster; a cluster of two heads' tiles; splits and a join; row tiles over splits; the tcgen05 tiles
@pytest.mark.parametrize("Hq,H,D,n,m", [(28, 4, 128, 1500, 1), (14, 2, 64, 300, 5), (28, 4, 128, 9000, 1), (28, 4, 128, 3000, 8),
                                        (28, 4, 128, 5000, 40), (4, 2, 64, 40, 1)])
@pytest.mark.parametrize("dtype", TYPES)
def test_a_nan_query_row_gives_nan(Hq, H, D, n, m, dtype):
    c, _, _ = filled(H, n, D, dtype, seed=n)
    kd, vd = ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale)
    q = queries(m, Hq, D, 1)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    check_nan_rows(lambda x: ops.attention_kv8(x, c, p), q, kd, vd, p, [(m - 1, 1), (0, Hq - 1)])


@pytest.mark.parametrize("Hq,H,D,n,m,top", [(28, 4, 128, 2000, 1, 40), (14, 2, 64, 900, 30, 9), (4, 2, 64, 300, 3, 2)])
@pytest.mark.parametrize("kind", [BF, *TYPES])
def test_a_nan_query_row_gives_nan_over_blocks(Hq, H, D, n, m, top, kind):
    attend, kd, vd, _, _ = caches(kind, H, n, D, seed=2)
    q = queries(m, Hq, D, 1)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    blocks = torch.arange(top, dtype=torch.int32, device=DEV).expand(m, H, top).contiguous()
    check_nan_rows(lambda x: attend(x, p, blocks), q, kd, vd, p, [(m - 1, 1), (0, Hq - 1)], blocks)
