"""The 8-bit K/V cache (write, read, attention) against its definition in 64 bits.

Tolerances.  Codes and scales are defined by single fp32 roundings: they must be equal.  An
attention output is off by its own rounding to bf16 (2^-8 of the value), and by what P and
the scores lose before: P is rounded to fp16 (2^-11 of each weight), and a score is an fp32
sum of up to 128 products whose magnitudes stay below about 2^6 here (128 * 2^-24 * 2^6 =
2^-11 absolute, so 2^-11 of each weight); both act on sum_j p_j |v_j| ("mass"), together at
most 2^-10 of it, in numerator and denominator 2^-9.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402

DEV = "cuda"
BF = torch.bfloat16
TYPES = [torch.int8, torch.float8_e4m3fn]


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


def rows(H, n, D, seed, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    chan = (spread * torch.randn((H, 1, D), generator=g, device=DEV)).exp()
    return (torch.randn((H, n, D), generator=g, device=DEV) * chan).to(BF)


def queries(m, Hq, D, seed, size=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn((m, Hq, D), generator=g, device=DEV) * size).to(BF)


def filled(H, n, D, dtype, seed=0, n_ctx=None, digest=False):
    k, v = rows(H, n, D, seed, 0.5), rows(H, n, D, seed + 1, 0.3)
    c = ops.KV8Cache(H, n_ctx or n, D, dtype, DEV, digest=digest)
    ops.kv8_write(c, k, v, 0)
    return c, k, v


def check_cache(c, k, v, n):
    """Codes, scales and digest of a cache that holds rows k, v [H, n, D]."""
    for codes, scale, x in ((c.k, c.k_scale, k), (c.v, c.v_scale, v)):
        rc, rs = ref.quantize(x[:, :n], c.dtype)
        nb = rs.shape[1]
        assert torch.equal(scale[:, :nb].double(), rs)
        assert torch.equal(codes[:, :nb * 16].float().double(), rc)
        assert not codes[:, nb * 16:].float().any() and not scale[:, nb:].any()
    if c.digest is not None:
        dc, ds = ref.digest(k[:, :n])
        assert torch.equal(c.digest.scale[:, :ds.shape[1]].double(), ds)
        assert torch.equal(c.digest.codes[:, :ds.shape[1]].double(), dc)


def check_attention(out, q, k, v, positions, blocks=None, scale=None):
    want, mass = ref.attend(q, k, v, positions, blocks, scale)
    err = (out.double().view_as(want) - want).abs()
    bar = want.abs() * 2.0 ** -8 + mass * 2.0 ** -9
    worst = float((err - bar).max())
    assert worst <= 0, f"off by {float((err / (bar + 1e-30)).max()):.2f} of the bar"
    empty = positions < 0
    assert not out.view_as(want)[empty].any()


# ---------------------------------------------------------------------- write, read
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("H,n,D", [(4, 1120, 128), (2, 77, 64), (1, 1, 128), (3, 16, 64), (8, 2049, 128)])
def test_write_is_its_definition(H, n, D, dtype):
    c, k, v = filled(H, n, D, dtype, seed=n, n_ctx=n + 40, digest=True)
    check_cache(c, k, v, n)
    rk, rv = ops.kv8_read(c, 0, n)
    for got, codes, scale in ((rk, c.k, c.k_scale), (rv, c.v, c.v_scale)):
        assert torch.equal(got, ref.values(codes.float(), scale)[:, :n].float().to(BF))
    a, b = n // 3, n - n // 3
    pk, pv = ops.kv8_read(c, a, b - a)
    assert torch.equal(pk, rk[:, a:b]) and torch.equal(pv, rv[:, a:b])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("cuts", [(1, 2, 3), (15, 16, 17, 33), (7, 40, 41, 90), (64,), (5, 5, 6)])
def test_writes_in_pieces_equal_one_write(cuts, dtype):
    H, n, D = 3, 100, 128
    k, v = rows(H, n, D, 5), rows(H, n, D, 6)
    c = ops.KV8Cache(H, n + 3, D, dtype, DEV, digest=True)
    at = 0
    for end in (*cuts, n):
        ops.kv8_write(c, k[:, at:end], v[:, at:end], at)
        check_cache(c, k, v, end) if end else None
        at = end


@pytest.mark.parametrize("D", [64, 128])
def test_strided_and_by_position_sources(D):
    H, n = 4, 61
    k, v = rows(H, n, D, 1), rows(H, n, D, 2)
    # token-major rows [n, H * D] seen head-major, and a slice of a longer cache
    kt, vt = k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(0, 1).contiguous().transpose(0, 1)
    c = ops.KV8Cache(H, n, D, torch.int8, DEV)
    ops.kv8_write(c, kt, vt, 0)
    check_cache(c, k, v, n)
    big_k, big_v = torch.zeros((H, n + 9, D), dtype=BF, device=DEV), torch.zeros((H, n + 9, D), dtype=BF, device=DEV)
    big_k[:, :n], big_v[:, :n] = k, v
    c = ops.KV8Cache(H, n, D, torch.int8, DEV)
    ops.kv8_write(c, big_k, big_v, 0, 30, by_position=True)
    ops.kv8_write(c, big_k, big_v, 30, n - 30, by_position=True)
    check_cache(c, k, v, n)


def test_writing_back_into_an_earlier_block():
    """A shorter history is taken up again (a rejected draft): the tail's rows where it holds
    the block, the values of the codes where it does not."""
    H, n, D = 2, 60, 128
    c, k, v = filled(H, n, D, torch.int8, seed=3)
    new_k, new_v = rows(H, 3, D, 8), rows(H, 3, D, 9)
    ops.kv8_write(c, new_k, new_v, 52)  # block 3 (tokens 48..) is the one in the tail
    k[:, 52:55], v[:, 52:55] = new_k, new_v
    check_cache(ops.KV8Cache.wrap(c.k[:, :64], c.v, c.k_scale, c.v_scale, n), k, v, 55)
    rk, rv = ops.kv8_read(c, 0, n)
    ops.kv8_write(c, new_k, new_v, 20)  # block 1: rows 16..19 from their codes
    for codes, scale, old, new in ((c.k, c.k_scale, rk, new_k), (c.v, c.v_scale, rv, new_v)):
        rc, rs = ref.quantize(torch.cat([old[:, 16:20], new], 1), torch.int8)
        assert torch.equal(codes[:, 16:32].double(), rc) and torch.equal(scale[:, 1:2].double(), rs)


def test_device_start_replayed_in_a_graph():
    H, n, D = 2, 50, 64
    k, v = rows(H, n, D, 1), rows(H, n, D, 2)
    c = ops.KV8Cache(H, n, D, torch.float8_e4m3fn, DEV, digest=True)
    start = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.kv8_write(c, k, v, start, by_position=True)  # warm up outside the capture
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.kv8_write(c, k, v, start, by_position=True)
        start += 1
    start.zero_()
    for i in range(n):
        g.replay()
        if i in (0, 14, 15, 16, 31, n - 1):
            check_cache(c, k, v, i + 1)
    before = [t.clone() for t in (c.k.view(torch.uint8), c.k_scale)]
    g.replay()  # one past the context: recorded, nothing written
    assert _lib.device_error() & 0x8
    assert torch.equal(before[0], c.k.view(torch.uint8)) and torch.equal(before[1], c.k_scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_tiny_and_non_finite_blocks(dtype):
    H, D = 1, 64
    k = torch.zeros((H, 96, D), dtype=BF, device=DEV)
    k[:, 16:32] = 2.0 ** -101               # below the smallest block kept
    k[:, 32:48] = 2.0 ** -100               # the smallest one
    k[:, 48:64] = rows(H, 16, D, 3, 0.2) * 1e37  # large
    k[:, 64:80] = rows(H, 16, D, 4)
    k[0, 70, 5], k[0, 71, 6], k[0, 72, 7] = float("nan"), float("inf"), float("-inf")
    k[:, 80:] = float("nan")
    c = ops.KV8Cache(H, 96, D, dtype, DEV, digest=True)
    ops.kv8_write(c, k, k, 0)
    assert _lib.device_error() & 0x10
    fixed = k.clone()
    top = fixed[0, 64:80].nan_to_num(0, 0, 0).abs().amax()
    fixed[0, 70, 5], fixed[0, 71, 6], fixed[0, 72, 7] = 0, top, -top
    fixed[:, 80:] = 0
    check_cache(c, fixed, fixed, 96)
    assert c.k_scale[0, 1] == 0 and c.k_scale[0, 2] > 0 and c.k_scale[0, 5] == 0


# ------------------------------------------------------------------------ attention
SHAPES = [(28, 4, 128), (14, 2, 64), (40, 8, 128), (4, 2, 64), (7, 1, 128), (5, 5, 64), (16, 1, 128), (24, 1, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,H,D", SHAPES)
def test_one_row(Hq, H, D, dtype):
    n = 1500
    c, k, v = filled(H, n, D, dtype, seed=Hq)
    kd, vd = ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale)
    q = queries(1, Hq, D, 4)
    for pos in (0, 1, 15, 16, 700, n - 1):
        p = torch.tensor([pos], dtype=torch.int32, device=DEV)
        check_attention(ops.attention_kv8(q, c, p), q, kd, vd, p)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,H,D,n,m", [(28, 4, 128, 1200, 2), (28, 4, 128, 333, 8), (14, 2, 64, 700, 37), (40, 8, 128, 257, 130),
                                        (28, 4, 128, 1300, 300), (4, 2, 64, 5, 5), (7, 1, 128, 1, 1), (16, 1, 128, 400, 20),
                                        (24, 1, 64, 300, 11), (5, 5, 64, 513, 290), (128, 1, 64, 200, 3)])
def test_many_rows(Hq, H, D, n, m, dtype):
    c, k, v = filled(H, n, D, dtype, seed=n)
    kd, vd = ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale)
    q = queries(m, Hq, D, m)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    check_attention(ops.attention_kv8(q, c, p), q, kd, vd, p)
    g = torch.Generator().manual_seed(m)
    p = torch.randint(-1, n, (m,), generator=g, dtype=torch.int32).to(DEV)  # any order, rows that see nothing
    p[0] = -1
    check_attention(ops.attention_kv8(q, c, p), q, kd, vd, p)
    check_attention(ops.attention_kv8(q, c, torch.full_like(p, -1)), q, kd, vd, torch.full_like(p, -1))
    check_attention(ops.attention_kv8(q, c, p, scale=0.03), q, kd, vd, p, scale=0.03)


@pytest.mark.parametrize("m", [1, 3, 40, 200])
def test_what_lies_past_the_last_position_does_not_matter(m):
    """Codes of NaN and scales of NaN or infinity past every row's position."""
    Hq, H, D, n = 28, 4, 128, 900
    c, k, v = filled(H, n, D, torch.float8_e4m3fn, seed=2)
    q = queries(m, Hq, D, 3)
    p = torch.arange(500 - m, 500, dtype=torch.int32, device=DEV)
    want = ops.attention_kv8(q, c, p)
    for x, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x.view(torch.uint8)[:, 500:] = 0x7f
        s[:, 32:] = float("nan")
        s[:, 40:] = float("inf")
    assert torch.equal(ops.attention_kv8(q, c, p), want)


@pytest.mark.parametrize("m", [1, 64])
def test_scales_that_vary_widely(m):
    Hq, H, D, n = 14, 2, 64, 640
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.randn((H, n, D), generator=g, device=DEV).to(BF)
    v = torch.randn((H, n, D), generator=g, device=DEV)
    v = (v * torch.exp2(torch.randint(-8, 8, (1, n // 16, 1), generator=g, device=DEV).float()).repeat_interleave(16, 1)).to(BF)
    q = queries(m, Hq, D, 2)
    q[:, 0] *= 2.0 ** -40
    q[:, 1] = 0
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    for dtype in TYPES:
        c = ops.KV8Cache(H, n, D, dtype, DEV)
        ops.kv8_write(c, k, v, 0)
        check_attention(ops.attention_kv8(q, c, p), q, ref.values(c.k.float(), c.k_scale),
                        ref.values(c.v.float(), c.v_scale), p)


def test_sharp_rows_and_late_maxima():
    """The largest score comes last, by far more than the lazy rescale allows, or first."""
    Hq, H, D, n, m = 7, 1, 128, 800, 60
    k = torch.zeros((H, n, D), dtype=BF, device=DEV)
    k[0, :, 0] = torch.linspace(-30, 30, n, device=DEV).to(BF)
    k[0, :, 1] = torch.linspace(30, -30, n, device=DEV).to(BF)
    v = rows(H, n, D, 1, 0.2)
    q = torch.zeros((m, Hq, D), dtype=BF, device=DEV)
    q[:, ::2, 0], q[:, 1::2, 1] = 8.0, 8.0
    c = ops.KV8Cache(H, n, D, torch.int8, DEV)
    ops.kv8_write(c, k, v, 0)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    for rows_ in (1, m):
        check_attention(ops.attention_kv8(q[:rows_], c, p[:rows_]), q[:rows_], ref.values(c.k.float(), c.k_scale),
                        ref.values(c.v.float(), c.v_scale), p[:rows_], scale=None)


def test_position_past_the_context_is_reported():
    c, k, v = filled(2, 100, 64, torch.int8)
    q = queries(3, 4, 64, 1)
    p = torch.tensor([99, 100, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    out = ops.attention_kv8(q, c, p)
    assert _lib.device_error() & 0x8
    check_attention(out, q, ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale),
                    torch.full((3,), 99, dtype=torch.int32, device=DEV))


def test_no_rows_and_rows_left_alone():
    c, k, v = filled(2, 100, 64, torch.int8)
    q = queries(6, 4, 64, 1)
    p = torch.arange(94, 100, dtype=torch.int32, device=DEV)
    assert ops.attention_kv8(q, c, p, m=0).shape[0] == 0
    out = torch.full((6, 4, 64), 7.0, dtype=BF, device=DEV)
    ops.attention_kv8(q, c, p, out=out, m=4)
    assert torch.equal(out[:4], ops.attention_kv8(q, c, p)[:4]) and bool((out[4:] == 7).all())
    ops.kv8_write(c, k[:, :0], v[:, :0], 100)
    assert ops.kv8_read(c, 50, 0)[0].shape == (2, 0, 64)


def test_other_streams_and_two_graphs_at_once():
    """Two captured calls replayed at the same time on two streams share nothing."""
    Hq, H, D, n = 28, 4, 128, 4000
    c, k, v = filled(H, n, D, torch.int8, seed=1)
    p = torch.tensor([n - 1], dtype=torch.int32, device=DEV)
    qs = [queries(1, Hq, D, s) for s in (1, 2)]
    want = [ops.attention_kv8(q, c, p) for q in qs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        out = torch.zeros_like(q)
        with torch.cuda.graph(g, stream=s):
            for _ in range(8):
                ops.attention_kv8(q, c, p, out=out)
        graphs.append(g)
        outs.append(out)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.current_stream())
        got = ops.attention_kv8(qs[0], c, p)
    streams[0].synchronize()
    assert torch.equal(got, want[0])


def test_caches_past_two_gigabytes():
    """The last head's rows lie past 2^31 bytes."""
    H, D, n = 20, 128, 1 << 20
    c = ops.KV8Cache(H, n, D, torch.int8, DEV)
    x = rows(1, 300, D, 1)
    at = n - 300
    k = torch.zeros((H, 300, D), dtype=BF, device=DEV)
    k[H - 1] = x[0]
    ops.kv8_write(c, k, k, at)
    rk, _ = ops.kv8_read(c, at, 300)
    small = ops.KV8Cache(1, 300 + 4, D, torch.int8, DEV)  # the same offset in its block: n - 300 = 4 mod 16
    ops.kv8_write(small, x, x, 4)
    assert torch.equal(rk[H - 1:], ops.kv8_read(small, 4, 300)[0]) and not rk[:H - 1].any()
    q = queries(2, H, D, 1)
    p = torch.tensor([n - 1, n - 2], dtype=torch.int32, device=DEV)
    out = ops.attention_kv8(q, c, p)
    kd, vd = torch.zeros((2, 1, n, D), dtype=torch.float32, device=DEV)  # the values held, before the read's rounding
    kd[:, at:], vd[:, at:] = (ref.values(t, s)[:, 4:304].float() for t, s in ((small.k, small.k_scale), (small.v, small.v_scale)))
    check_attention(out[:, H - 1:].contiguous(), q[:, H - 1:].contiguous(), kd, vd, p)
    blocks = torch.arange(n // 16 - 20, n // 16, dtype=torch.int32, device=DEV).expand(2, H, 20).contiguous()
    out = ops.attention_blocks_kv8(q, c, p, blocks)
    check_attention(out[:, H - 1:].contiguous(), q[:, H - 1:].contiguous(), kd, vd, p, blocks[:, H - 1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 9, 70])
def test_value_scales_more_than_32_bits_of_exponent_apart(m, dtype):
    """Every third block of V lies 2^-130 below the others (their scales' ratio leaves fp32): its
    values vanish beside theirs, its weights still count in the softmax's sum."""
    H, D, n = 2, 128, 400
    k, v = rows(H, n, D, 71, 0.2), rows(H, n, D, 72, 0.2).float()
    tiny = (torch.arange(n, device=DEV) // 16 % 3 == 1)[None, :, None]
    v = torch.where(tiny, v * 2.0 ** -90, v * 2.0 ** 40).to(BF)
    c = ops.KV8Cache(H, n, D, dtype, DEV)
    ops.kv8_write(c, k, v, 0)
    q = queries(m, 4, D, 73, 0.5)
    pos = torch.linspace(n - 1, 20, m, device=DEV).to(torch.int32)
    out = ops.attention_kv8(q, c, pos)
    check_attention(out, q, ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale), pos)


@pytest.mark.parametrize("m,n", [(150, 6000), (700, 900)])
def test_tiles_in_two_graphs_at_once(m, n):
    """The same for many rows: key splits (150 rows) and a counter of work items (both)."""
    Hq, H, D = 28, 4, 128
    c, k, v = filled(H, n, D, torch.float8_e4m3fn, seed=2)
    p = torch.arange(n - m, n, dtype=torch.int32, device=DEV)
    qs = [queries(m, Hq, D, s) for s in (1, 2)]
    want = [ops.attention_kv8(q, c, p) for q in qs]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for q, s in zip(qs, streams):
        g = torch.cuda.CUDAGraph()
        out = torch.zeros_like(q)
        with torch.cuda.graph(g, stream=s):
            for _ in range(4):
                ops.attention_kv8(q, c, p, out=out)
        graphs.append(g)
        outs.append(out)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Hq,H,D,n,m", [(28, 4, 128, 900, 700), (14, 2, 64, 130, 3001), (40, 8, 128, 1300, 401), (4, 4, 128, 17, 9000),
                                        (16, 1, 64, 5000, 37), (7, 1, 128, 2500, 63), (128, 1, 64, 700, 90)])
def test_many_rows_in_tiles(Hq, H, D, n, m, dtype):
    """Shapes that the tile kernel takes: long or short contexts, half-filled tiles, odd ends."""
    c, k, v = filled(H, n, D, dtype, seed=n)
    kd, vd = ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale)
    q = queries(m, Hq, D, m)
    g = torch.Generator().manual_seed(m)
    p = torch.randint(-1, n, (m,), generator=g, dtype=torch.int32).to(DEV)
    p[0], p[m - 1] = n - 1, -1
    check_attention(ops.attention_kv8(q, c, p), q, kd, vd, p)
    check_attention(ops.attention_kv8(q, c, p.sort().values), q, kd, vd, p.sort().values)
