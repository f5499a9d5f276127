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


# ------------------------------------------------------------------- non-finite rows
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cuts", [(4, 5, 9), (1, 2, 3, 4, 5, 6, 7, 8), (16, 20, 24), (17, 18)])
def test_non_finite_rows_do_not_depend_on_the_pieces(cuts, dtype):
    """An infinity is the block's largest value, also of rows that come after it; it is reported once."""
    H, D, n = 2, 64, 26
    k, v = (torch.randn((H, n, D), generator=torch.Generator(device=DEV).manual_seed(s), device=DEV) for s in (1, 2))
    size = torch.arange(1, n + 1, device=DEV)[None, :, None].float()  # later rows are larger
    k, v = (k * size).to(BF), (v * size).to(BF)
    for t in (3, 18):
        k[0, t, 5], k[1, t, 6], v[0, t, 7], v[1, t, 8] = float("inf"), float("nan"), float("-inf"), float("inf")
    once = ops.KV8Cache(H, n, D, dtype, DEV, digest=True)
    ops.kv8_write(once, k, v, 0)
    assert _lib.device_error() & 0x10
    for side, x in ((once.k, k), (once.v, v)):  # the largest code of its sign
        want = torch.where(x.isposinf(), ref.QMAX[dtype], torch.where(x.isneginf(), -ref.QMAX[dtype], 0.0))
        assert torch.equal(side.float()[:, :n][~x.isfinite()], want[~x.isfinite()])
    c = ops.KV8Cache(H, n, D, dtype, DEV, digest=True)
    at = 0
    for end in (*cuts, n):
        ops.kv8_write(c, k[:, at:end], v[:, at:end], at)
        brought = not (k[:, at:end].isfinite().all() and v[:, at:end].isfinite().all())
        assert bool(_lib.device_error() & 0x10) == brought
        at = end
    for a, b in ((c.k, once.k), (c.v, once.v)):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(c.k_scale, once.k_scale) and torch.equal(c.v_scale, once.v_scale)
    assert torch.equal(c.digest.codes, once.digest.codes) and torch.equal(c.digest.scale, once.digest.scale)


# -------------------------------------------------------------------- writes that go back
def equal_caches(a, b, n):
    """Codes, scales and digests of the blocks that hold the first n tokens."""
    nb = -(-n // 16)
    for x, y in ((a.k, b.k), (a.v, b.v)):
        assert torch.equal(x.view(torch.uint8)[:, :nb * 16], y.view(torch.uint8)[:, :nb * 16])
    for x, y in ((a.k_scale, b.k_scale), (a.v_scale, b.v_scale), (a.digest.scale, b.digest.scale),
                 (a.digest.codes, b.digest.codes)):
        assert torch.equal(x[:, :nb], y[:, :nb])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,D,base,drafts,keep", [(4, 128, 28, 8, 2), (2, 64, 30, 3, 0), (2, 64, 31, 1, 0), (2, 64, 27, 5, 3), (2, 128, 20, 12, 1),
                                                  (1, 64, 40, 24, 9), (3, 64, 33, 30, 1), (2, 64, 40, 8, 0), (2, 64, 47, 16, 0)])
@pytest.mark.parametrize("device_start", [False, True])
def test_rejected_drafts_leave_nothing_behind(H, D, base, drafts, keep, dtype, device_start):
    """Drafts are appended, all but `keep` of them are rejected and others take their place: the cache
    is that of one write of the rows that stay, though a rejected row had set its block's scale."""
    n = base + drafts + 40
    k, v = (torch.randn((H, n, D), generator=torch.Generator(device=DEV).manual_seed(s), device=DEV).to(BF) for s in (3, 4))
    bad_k, bad_v = k.clone(), v.clone()
    bad_k[:, base + keep:], bad_v[:, base + keep:] = 1000 * k[:, base + keep:], 1000 * v[:, base + keep:]

    def write(c, kk, vv, a, b):
        start = torch.tensor([a], dtype=torch.int32, device=DEV) if device_start else a
        ops.kv8_write(c, kk[:, a:b], vv[:, a:b], start, b - a)

    c = ops.KV8Cache(H, n, D, dtype, DEV, digest=True)
    write(c, k, v, 0, 19)
    write(c, k, v, 19, base)
    write(c, bad_k, bad_v, base, base + drafts)
    at = base + keep
    # as many rounds of drafts as fit, every one rejected but for one row
    for _ in range(3):
        write(c, k, v, at, at + 1)
        at += 1
        write(c, bad_k, bad_v, at, at + 5)
    write(c, k, v, at, n)
    once = ops.KV8Cache(H, n, D, dtype, DEV, digest=True)
    ops.kv8_write(once, k, v, 0)
    equal_caches(c, once, n)


def test_a_second_step_back_takes_the_codes():
    """Back into the block before, then into one before that: its rows are known as codes alone."""
    H, D, n = 2, 64, 70
    k, v = (torch.randn((H, n, D), generator=torch.Generator(device=DEV).manual_seed(s), device=DEV).to(BF) for s in (5, 6))
    c = ops.KV8Cache(H, n, D, torch.int8, DEV, digest=True)
    ops.kv8_write(c, k, v, 0, 66)
    ops.kv8_write(c, k[:, 50:], v[:, 50:], 50, 3)
    rk, rv = ops.kv8_read(c, 32, 8)
    ops.kv8_write(c, k[:, 40:], v[:, 40:], 40, 4)
    for codes, scale, old, new in ((c.k, c.k_scale, rk, k), (c.v, c.v_scale, rv, v)):
        rc, rs = ref.quantize(torch.cat([old, new[:, 40:44]], 1), torch.int8)
        assert torch.equal(codes[:, 32:48].double(), rc) and torch.equal(scale[:, 2:3].double(), rs)


def test_a_cache_without_the_block_before():
    """The entry point takes null for it: appending writes are as ever."""
    H, D, n = 2, 64, 50
    k, v = (torch.randn((H, n, D), generator=torch.Generator(device=DEV).manual_seed(s), device=DEV).to(BF) for s in (7, 8))
    c, once = (ops.KV8Cache(H, n, D, torch.int8, DEV, digest=True) for _ in range(2))
    ops.kv8_write(once, k, v, 0)
    stream = torch.cuda.current_stream().cuda_stream
    for a, b in ((0, 5), (5, 40), (40, n)):
        _lib.call("ckv_kv8_write", k.data_ptr(), v.data_ptr(), n * D, D, n * D, D, n, 1, b - a, a, None, c.k.data_ptr(),
                  c.v.data_ptr(), c.k_scale.data_ptr(), c.v_scale.data_ptr(), c.tail.data_ptr(), c.tail_end.data_ptr(), None, None,
                  c.digest.codes.data_ptr(), c.digest.scale.data_ptr(), H, D, n, 0, stream)
    equal_caches(c, once, n)


# ------------------------------------------------------------- calls behind other kernels
@pytest.mark.parametrize("Hq,H,D,n,top", [(28, 4, 128, 3000, 20), (14, 2, 64, 70000, 40)])
def test_sparse_call_takes_what_the_kernels_before_it_wrote(Hq, H, D, n, top):
    """q by this library's RMSNorm (a dependent launch) and the position by a copy, directly before
    the call, both in the same buffers at every step of one graph."""
    c, _, _ = filled(H, n, D, torch.int8, seed=2, digest=True)
    steps = 24
    x = queries(steps, Hq, D, 3).view(steps, Hq * D)
    w = torch.ones(Hq * D, dtype=BF, device=DEV)
    at = torch.randint(200, n, (steps, 1), generator=torch.Generator().manual_seed(1), dtype=torch.int32).to(DEV)
    q, p = torch.zeros((1, Hq * D), dtype=BF, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    outs = torch.zeros((steps, Hq, D), dtype=BF, device=DEV)
    lists = torch.zeros((steps, 1, H, top), dtype=torch.int32, device=DEV)

    def step(i):
        p.copy_(at[i])
        ops.rmsnorm(x[i:i + 1], w, 1e-6, out=q)
        ops.attention_sparse_kv8(q.view(1, Hq, D), c, p, top, out=outs[i:i + 1], blocks=lists[i])

    step(0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i in range(steps):
            step(i)
    for _ in range(5):
        outs.zero_()
        lists.zero_()
        g.replay()
        torch.cuda.synchronize()
        for i in range(steps):
            qi = ops.rmsnorm(x[i:i + 1], w, 1e-6).view(1, Hq, D)
            torch.cuda.synchronize()
            want = ops.block_select(qi, c.digest, at[i], top)
            torch.cuda.synchronize()
            assert torch.equal(lists[i], want)
            assert torch.equal(outs[i:i + 1], ops.attention_blocks_kv8(qi, c, at[i], want))
            torch.cuda.synchronize()


# ------------------------------------------------------------------------------ lists
@pytest.mark.parametrize("kind", [BF, *TYPES])
@pytest.mark.parametrize("bad", [[5, -1, 5, -1], [-1, 3, -1, -1], [2, 4, -1, 6], [-1, -1, -1, 0]])
def test_entries_behind_the_end_of_a_list_are_reported(bad, kind):
    Hq, H, D, n = 4, 2, 64, 400
    attend, kd, vd, _, _ = caches(kind, H, n, D)
    q = queries(1, Hq, D, 1)
    p = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    lists = torch.tensor([[[1, 2, 3, -1], bad]], dtype=torch.int32, device=DEV)
    out = attend(q, p, lists)
    assert _lib.device_error() & 0x8
    kept = [b if i == 0 or bad[i - 1] != -1 else -1 for i, b in enumerate(bad)]
    check = torch.tensor([[[1, 2, 3, -1], kept]], dtype=torch.int32, device=DEV)
    want, mass = ref.attend(q, kd, vd, p, check)
    assert float(((out.double() - want).abs() - want.abs() * 2.0 ** -8 - mass * 2.0 ** -9).max()) <= 0


@pytest.mark.parametrize("kind", [BF, *TYPES])
@pytest.mark.parametrize("Hq,H,D,n,m,top", [(32, 8, 128, 4096, 1, 4096), (28, 4, 128, 300, 1, 128), (14, 2, 64, 700, 30, 300),
                                            (4, 2, 64, 9, 3, 4096)])
def test_lists_longer_than_the_context(Hq, H, D, n, m, top, kind):
    attend, kd, vd, sparse, _ = caches(kind, H, n, D, seed=1)
    q = queries(m, Hq, D, 4)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    out, blocks = sparse(q, p, top)
    nb = (p // 16 + 1).tolist()
    assert all(row[h].tolist() == [*range(b), *[-1] * (top - b)] for row, b in zip(blocks, nb) for h in range(H))
    check_attention(out, q, kd, vd, p)
    assert torch.equal(attend(q, p, blocks), out)
    # an entry behind as many as the context has blocks cannot be right
    blocks[m - 1, 0, top - 1] = 0
    assert torch.equal(attend(q, p, blocks), out) and _lib.device_error() & 0x8


@pytest.mark.parametrize("Hq,H,D,n,m,top", [(8, 2, 64, 131072, 2, 4096), (28, 4, 128, 20000, 1, 1000), (7, 1, 128, 100000, 40, 2049)])
def test_long_lists(Hq, H, D, n, m, top):
    _, kd, vd, sparse, d = caches(torch.int8, H, n, D, seed=3)
    q = queries(m, Hq, D, 5)
    p = torch.linspace(n - 1, n // 2, m, device=DEV).to(torch.int32)
    out, blocks = sparse(q, p, top)
    assert torch.equal(blocks.cpu().long(), ref.select(q, d.codes, d.scale, p, top))
    check_attention(out[:4], q[:4], kd, vd, p[:4], blocks[:4])


# --------------------------------------------------------------------- very large and small
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,H,D,n,m", [(28, 4, 128, 1500, 1), (28, 4, 128, 9000, 1), (28, 4, 128, 700, 4), (28, 4, 128, 640, 200),
                                        (14, 2, 64, 2500, 100)])
@pytest.mark.parametrize("size", [-95, 96])
def test_very_large_and_small_values(Hq, H, D, n, m, size, dtype):
    """V near the ends of what a call takes (the largest value times the keys below 2^113), and keys and
    queries whose products are ordinary though neither is."""
    k, v, q = filled(H, n, D, dtype, seed=3)[1:] + (queries(m, Hq, D, 1),)
    c = ops.KV8Cache(H, n, D, dtype, DEV, digest=True)
    ops.kv8_write(c, (k.float() * 2.0 ** -size).to(BF), (v.float() * 2.0 ** size).to(BF), 0)
    assert float(ref.values(c.v.float(), c.v_scale).abs().max()) * n < 2.0 ** 113
    q = (q.float() * 2.0 ** size).to(BF)
    p = torch.linspace(n - 1, n // 2, m, device=DEV).to(torch.int32)
    kd, vd = ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale)
    check_attention(ops.attention_kv8(q, c, p), q, kd, vd, p)
    out, blocks = ops.attention_sparse_kv8(q, c, p, 12)
    assert torch.equal(blocks.cpu().long(), ref.select(q, c.digest.codes, c.digest.scale, p, 12))
    check_attention(out, q, kd, vd, p, blocks)
