"""Block selection and attention over selected blocks against their definitions in 64 bits.

A selection is defined by whole numbers and single fp32 roundings: the lists must be equal.
Attention outputs: as tests/test_gpu_kv8.py for the 8-bit cache; over a bf16 cache P keeps 16
bits (two bf16 parts), so the same bar covers it.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402
from test_gpu_kv8 import BF, DEV, check_attention, queries, rows  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


def context(H, n, D, seed=0):
    """Keys that drift from block to block, so that blocks differ."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    nb = -(-n // 16)
    k = (torch.randn((H, nb, 1, D), generator=g, device=DEV) + 0.5 * torch.randn((H, nb, 16, D), generator=g, device=DEV))
    return k.view(H, -1, D)[:, :n].to(BF).contiguous(), rows(H, n, D, seed + 1, 0.3)


def spread_rows(n, m, seed=0):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(-1, n, (m,), generator=g, dtype=torch.int32)
    p[0] = n - 1
    if m > 2:
        p[1], p[2] = -1, 0
    return p.to(DEV)


def digest_of(k):
    d = ops.BlockDigest(k.shape[0], k.shape[1], k.shape[2], DEV)
    return ops.block_digest(k, d)


@pytest.mark.parametrize("H,n,D", [(4, 1000, 128), (2, 1, 64), (3, 17, 64), (1, 64, 128)])
def test_digest_is_its_definition_and_grows(H, n, D):
    k, _ = context(H, n, D)
    d = digest_of(k)
    dc, ds = ref.digest(k)
    assert torch.equal(d.scale.double(), ds) and torch.equal(d.codes.double(), dc)
    e = ops.BlockDigest(H, n, D, DEV)
    at = torch.zeros(1, dtype=torch.int32, device=DEV)
    for cut in range(0, n, 7):  # blocks in progress are redone from the cache
        m = min(7, n - cut)
        at.fill_(cut)
        ops.block_digest(k, e, at, m) if cut % 2 else ops.block_digest(k, e, cut, m)
    assert torch.equal(d.scale, e.scale) and torch.equal(d.codes, e.codes)


@pytest.mark.parametrize("Hq,H,D,n,m,top,sink,recent", [
    (28, 4, 128, 5000, 3, 64, 1, 1), (28, 4, 128, 600, 40, 8, 1, 1), (14, 2, 64, 9000, 20, 33, 0, 2),
    (40, 8, 128, 333, 17, 5, 2, 3), (16, 1, 128, 2000, 9, 16, 1, 1), (4, 2, 64, 40000, 5, 100, 1, 1),
    (7, 1, 128, 140000, 3, 128, 3, 1), (4, 2, 64, 100, 33, 2, 1, 1), (4, 2, 64, 100, 8, 1, 0, 1),
    (12, 1, 64, 3000, 70, 64, 0, 1), (4, 2, 64, 1, 1, 4, 1, 1)])
def test_selection_is_its_definition(Hq, H, D, n, m, top, sink, recent):
    k, _ = context(H, n, D, seed=n)
    d = digest_of(k)
    q = queries(m, Hq, D, 3)
    p = spread_rows(n, m)
    got = ops.block_select(q, d, p, top, sink, recent)
    want = ref.select(q, d.codes, d.scale, p, top, sink, recent)
    assert torch.equal(got.cpu().long(), want)


def test_selection_ties_go_to_the_lower_block():
    H, Hq, D, n = 2, 8, 64, 3000
    k, _ = context(H, 64, D)
    k = k.repeat(1, n // 64 + 1, 1)[:, :n].contiguous()  # every score four blocks apart again
    d = digest_of(k)
    q = queries(6, Hq, D, 1)
    q[3] = 0  # every score equal
    p = torch.tensor([n - 1, 1000, 500, n - 1, 15, 16], dtype=torch.int32, device=DEV)
    for top in (2, 3, 20, 61, 186, 187, 188, 200):
        assert torch.equal(ops.block_select(q, d, p, top).cpu().long(), ref.select(q, d.codes, d.scale, p, top))
    assert ops.block_select(q[3:4], d, p[3:4], 5)[0, 0].tolist() == [0, 1, 2, 3, (n - 1) // 16]


def test_selection_in_runs_of_rows(monkeypatch):
    """So many rows that the workspace holds them in several runs."""
    H, Hq, D, n, m = 8, 8, 64, 131072, 1300  # 8 * 8192 * 4 bytes a row: 1024 rows at a time
    k, _ = context(H, n, D)
    d = digest_of(k)
    q = queries(m, Hq, D, 1)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    got = ops.block_select(q, d, p, 16)
    for a, b in ((0, 20), (1010, 1040), (1290, 1300)):
        assert torch.equal(got[a:b], ops.block_select(q[a:b].contiguous(), d, p[a:b].contiguous(), 16))
    assert torch.equal(got[-2:].cpu().long(), ref.select(q[-2:], d.codes, d.scale, p[-2:], 16))


def caches(kind, H, n, D, seed=0):
    """(callable q, positions, blocks -> out, exact K, exact V, callable q, positions, top -> (out, blocks), digest)"""
    k, v = context(H, n, D, seed)
    if kind is BF:
        d = digest_of(k)
        return (lambda q, p, b, **kw: ops.attention_blocks(q, k, v, p, b, **kw), k, v,
                lambda q, p, top, **kw: ops.attention_sparse(q, k, v, p, top, digest=d, **kw), d)
    c = ops.KV8Cache(H, n, D, kind, DEV, digest=True)
    ops.kv8_write(c, k, v, 0)
    return (lambda q, p, b, **kw: ops.attention_blocks_kv8(q, c, p, b, **kw), ref.values(c.k.float(), c.k_scale)[:, :n],
            ref.values(c.v.float(), c.v_scale)[:, :n],
            lambda q, p, top, **kw: ops.attention_sparse_kv8(q, c, p, top, **kw), c.digest)


KINDS = [BF, torch.int8, torch.float8_e4m3fn]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,H,D,n,m,top", [(28, 4, 128, 3001, 1, 16), (14, 2, 64, 1203, 50, 9), (40, 8, 128, 700, 300, 20),
                                            (16, 1, 128, 500, 7, 12), (24, 1, 64, 400, 3, 10), (4, 2, 64, 33, 5, 2),
                                            (7, 1, 128, 9, 3, 4)])
def test_listed_blocks(Hq, H, D, n, m, top, kind):
    run, kd, vd, _, _ = caches(kind, H, n, D, seed=n)
    q = queries(m, Hq, D, 2)
    p = spread_rows(n, m)
    nb = -(-n // 16)
    g = torch.Generator().manual_seed(1)
    blocks = torch.full((m, H, top), -1, dtype=torch.int32)
    for i in range(m):
        for h in range(H):
            cnt = int(torch.randint(0, min(top, nb) + 1, (1,), generator=g))
            blocks[i, h, :cnt] = torch.randperm(nb, generator=g)[:cnt].sort().values.int()
    blocks = blocks.to(DEV)
    out = run(q, p, blocks)
    # a row may be listed blocks that all lie past its position: it sees nothing
    want, mass = ref.attend(q, kd, vd, p, blocks)
    assert float(((out.double() - want).abs() - want.abs() * 2.0 ** -8 - mass * 2.0 ** -9).max()) <= 0
    assert not out[mass == 0].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,H,D,n,m,top", [(28, 4, 128, 9001, 1, 64), (14, 2, 64, 5203, 30, 17), (40, 8, 128, 2100, 64, 32),
                                            (7, 1, 128, 4000, 200, 8)])
def test_selected_then_attended(Hq, H, D, n, m, top, kind):
    """The run of both, as a decode step or a blend uses them."""
    _, kd, vd, sparse, d = caches(kind, H, n, D, seed=m)
    q = queries(m, Hq, D, 5)
    p = spread_rows(n, m, 3)
    out, blocks = sparse(q, p, top)
    assert torch.equal(blocks.cpu().long(), ref.select(q, d.codes, d.scale, p, top))
    check_attention(out, q, kd, vd, p, blocks)


@pytest.mark.parametrize("kind", KINDS)
def test_all_blocks_is_dense_attention(kind):
    Hq, H, D, n, m = 28, 4, 128, 500, 20
    _, kd, vd, sparse, _ = caches(kind, H, n, D)
    q, p = queries(m, Hq, D, 1), spread_rows(n, m)
    out, blocks = sparse(q, p, 40)
    check_attention(out, q, kd, vd, p)


def test_digest_built_in_the_call():
    Hq, H, D, n, m = 14, 2, 64, 1999, 9
    k, v = context(H, n, D)
    q, p = queries(m, Hq, D, 1), spread_rows(n, m)
    a, b = ops.attention_sparse(q, k, v, p, 12), ops.attention_sparse(q, k, v, p, 12, digest=digest_of(k))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("kind", KINDS)
def test_garbage_past_the_positions(kind):
    """NaN keys and values past every row's position, and past the context's last token."""
    Hq, H, D, n, m = 14, 2, 64, 300, 4
    k, v = context(H, n, D)
    p = torch.tensor([199, 198, 190, 16], dtype=torch.int32, device=DEV)
    q = queries(m, Hq, D, 1)
    blocks = torch.arange(19, dtype=torch.int32, device=DEV).expand(m, H, 19).contiguous()
    if kind is BF:
        k2, v2 = k.clone(), v.clone()
        k2[:, 200:], v2[:, 200:] = float("nan"), float("inf")
        got, want = ops.attention_blocks(q, k2, v2, p, blocks), ops.attention_blocks(q, k, v, p, blocks)
    else:
        c = ops.KV8Cache(H, n, D, kind, DEV)
        ops.kv8_write(c, k, v, 0)
        want = ops.attention_blocks_kv8(q, c, p, blocks)
        c.k.view(torch.uint8)[:, 208:] = 0x7f
        c.v.view(torch.uint8)[:, 208:] = 0x7f
        c.k_scale[:, 13:], c.v_scale[:, 13:] = float("nan"), float("inf")
        got = ops.attention_blocks_kv8(q, c, p, blocks)
    assert torch.equal(got, want) and bool(got.isfinite().all())


@pytest.mark.parametrize("bad", [[0, 7, 7, 9], [0, 9, 7, -1], [0, 3, 1 << 20, -1], [-5, 1, 2, 3]])
def test_bad_lists_are_reported(bad):
    Hq, H, D, n = 4, 2, 64, 400
    k, v = context(H, n, D)
    q = queries(1, Hq, D, 1)
    p = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    good = torch.tensor([[[1, 2, 3, -1], [0, 5, 9, 20]]], dtype=torch.int32, device=DEV)
    lists = good.clone()
    lists[0, 1] = torch.tensor(bad)
    out = ops.attention_blocks(q, k, v, p, lists)
    assert _lib.device_error() & 0x8
    assert torch.equal(out[:, :2], ops.attention_blocks(q, k, v, p, good)[:, :2]) and bool(out.isfinite().all())


def test_sparse_decode_step_replayed_in_a_graph():
    """Write, digest, selection and attention of one token at a device position, captured once
    and replayed over the following positions."""
    Hq, H, D, n = 28, 4, 128, 700
    k, v = context(H, n, D)
    q = queries(1, Hq, D, 1)
    p = torch.tensor([600], dtype=torch.int32, device=DEV)
    c = ops.KV8Cache(H, n, D, torch.int8, DEV, digest=True)
    ops.kv8_write(c, k[:, :600], v[:, :600], 0)
    out, blocks = torch.zeros_like(q), torch.zeros((1, H, 16), dtype=torch.int32, device=DEV)

    def step():
        ops.kv8_write(c, k, v, p, by_position=True)
        ops.block_select(q, c.digest, p, 16, out=blocks)
        ops.attention_blocks_kv8(q, c, p, blocks, out=out)

    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for pos in range(600, 640):
        p.fill_(pos)
        g.replay()
        if pos % 13 == 0:
            d = ref.digest(k[:, :pos + 1])
            assert torch.equal(blocks.cpu().long(), ref.select(q, d[0], d[1], p, 16))
            kq, vq = (ref.quantize(t[:, :pos + 1], torch.int8) for t in (k, v))
            check_attention(out, q, ref.values(*kq)[:, :pos + 1], ref.values(*vq)[:, :pos + 1], p, blocks)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("Hq,H,m", [(2, 2, 40_000), (20, 1, 17_000)])
def test_more_rows_than_one_grid_holds(Hq, H, m, kind):
    """Past 32,768 row tiles (20 heads of one KV head make two) the call goes in several runs."""
    D, n, top = 64, 200, 3
    attend, kd, vd, _, _ = caches(kind, H, n, D, seed=5)
    q = queries(m, Hq, D, 6)
    g = torch.Generator().manual_seed(7)
    p = torch.randint(-1, n, (m,), generator=g, dtype=torch.int32).to(DEV)
    b0 = torch.randint(0, 4, (m, H, 1), generator=g)
    blocks = torch.cat([b0, b0 + 3, b0 + 8], -1).to(torch.int32).to(DEV)
    out = attend(q, p, blocks)
    for rows in (slice(0, 64), slice(16_300, 16_450), slice(32_700, 32_830), slice(m - 40, m)):
        if rows.start < m:
            check_attention(out[rows], q[rows], kd, vd, p[rows], blocks[rows])
