"""The tcgen05 tiles of the 8-bit attention, unsplit and with key splits and their join, at both head
sizes: every test asserts that its shape reaches them.  Tolerances as in tests/test_gpu_kv8.py."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

from chunkkv_b200 import _lib, ops  # noqa: E402
from oracle import kv8_oracle as ref  # noqa: E402
from test_gpu_kv8 import BF, DEV, TYPES, check_attention, filled, queries, rows  # noqa: E402


@pytest.fixture(autouse=True)
def _device_error_free():
    yield
    _lib.check_device()


# (query heads, KV heads, head dim, tokens, rows, keys in one piece)
TILES = [(28, 4, 128, 640, 200, True), (28, 4, 128, 2500, 70, False), (28, 4, 128, 4000, 40, False), (7, 1, 128, 2500, 200, False),
         (14, 2, 64, 640, 500, True), (14, 2, 64, 2500, 100, False), (16, 1, 64, 4000, 70, False), (128, 1, 64, 1300, 20, False),
         (5, 5, 64, 500, 1500, True)]
tiles = pytest.mark.parametrize("Hq,H,D,n,m,whole", TILES)
types = pytest.mark.parametrize("dtype", TYPES)


def in_tiles(Hq, H, D, n, m, whole):
    splits = _lib.load().ckv_attention_kv8_splits(m, Hq, H, D, n)
    assert splits >= 1 and (splits == 1) == whole, f"{splits} splits: the shape no longer reaches this path"


def check(c, q, p, scale=None):
    out = ops.attention_kv8(q, c, p, scale=scale)
    check_attention(out, q, ref.values(c.k.float(), c.k_scale), ref.values(c.v.float(), c.v_scale), p, scale=scale)
    return out


@types
@tiles
def test_any_positions(Hq, H, D, n, m, whole, dtype):
    in_tiles(Hq, H, D, n, m, whole)
    c, _, _ = filled(H, n, D, dtype, seed=n)
    q = queries(m, Hq, D, m)
    p = torch.randint(-1, n, (m,), generator=torch.Generator().manual_seed(m), dtype=torch.int32).to(DEV)
    p[0], p[m - 1] = n - 1, -1
    check(c, q, p)
    check(c, q, torch.arange(n - m, n, dtype=torch.int32, device=DEV).clamp_min(-1), scale=0.05)
    check(c, q, torch.full_like(p, -1))


@types
@tiles
def test_maxima_that_grow_from_tile_to_tile(Hq, H, D, n, m, whole, dtype):
    """Scores rise by some 15 powers of two a key tile (O is rescaled at each), or fall (never)."""
    in_tiles(Hq, H, D, n, m, whole)
    k = torch.zeros((H, n, D), dtype=BF, device=DEV)
    top = 5.0 * n / 128 * D ** 0.5 / 40  # 10 nats a tile of 128 keys at |q| = 40
    k[:, :, 0] = torch.linspace(-top, top, n, device=DEV).to(BF)
    k[:, :, 1] = torch.linspace(top, -top, n, device=DEV).to(BF)
    v = rows(H, n, D, 1, 0.2)
    q = torch.zeros((m, Hq, D), dtype=BF, device=DEV)
    q[:, ::2, 0], q[:, 1::2, 1] = 40.0, 40.0
    c = ops.KV8Cache(H, n, D, dtype, DEV)
    ops.kv8_write(c, k, v, 0)
    check(c, q, torch.linspace(n - 1, 0, m, device=DEV).to(torch.int32))
    check(c, q, torch.arange(n - 1, n - 1 - m, -1, dtype=torch.int32, device=DEV).clamp_min(-1))


@types
@tiles
def test_value_scales_more_than_32_bits_of_exponent_apart(Hq, H, D, n, m, whole, dtype):
    """As the test of that name for few rows: every third block of V lies 2^-130 below the others."""
    in_tiles(Hq, H, D, n, m, whole)
    k, v = rows(H, n, D, 71, 0.2), rows(H, n, D, 72, 0.2).float()
    tiny = (torch.arange(n, device=DEV) // 16 % 3 == 1)[None, :, None]
    v = torch.where(tiny, v * 2.0 ** -90, v * 2.0 ** 40).to(BF)
    c = ops.KV8Cache(H, n, D, dtype, DEV)
    ops.kv8_write(c, k, v, 0)
    check(c, queries(m, Hq, D, 73, 0.5), torch.linspace(n - 1, 20, m, device=DEV).to(torch.int32))


@types
@tiles
def test_scales_that_vary_widely(Hq, H, D, n, m, whole, dtype):
    """V's blocks over 16 powers of two; query rows of 2^-40 and of zeros among the others."""
    in_tiles(Hq, H, D, n, m, whole)
    g = torch.Generator(device=DEV).manual_seed(1)
    size = torch.exp2(torch.randint(-8, 8, (1, -(-n // 16), 1), generator=g, device=DEV).float()).repeat_interleave(16, 1)[:, :n]
    k = torch.randn((H, n, D), generator=g, device=DEV).to(BF)
    v = (torch.randn((H, n, D), generator=g, device=DEV) * size).to(BF)
    q = queries(m, Hq, D, 2)
    q[:, 0] *= 2.0 ** -40
    q[:, Hq - 1] = 0
    c = ops.KV8Cache(H, n, D, dtype, DEV)
    ops.kv8_write(c, k, v, 0)
    check(c, q, torch.arange(n - m, n, dtype=torch.int32, device=DEV).clamp_min(0))


@tiles
def test_the_same_call_gives_the_same_bits(Hq, H, D, n, m, whole):
    """Items go to the SMs as they come; their sums do not depend on it."""
    in_tiles(Hq, H, D, n, m, whole)
    c, _, _ = filled(H, n, D, torch.int8, seed=1)
    q = queries(m, Hq, D, 1)
    p = torch.linspace(n - 1, 0, m, device=DEV).to(torch.int32)
    want = ops.attention_kv8(q, c, p)
    for _ in range(20):
        assert torch.equal(ops.attention_kv8(q, c, p), want)
