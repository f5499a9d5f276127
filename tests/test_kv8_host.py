"""What the 8-bit cache and the block-sparse attention refuse, checked on the host before
anything launches, and the oracle's own arithmetic.  No GPU needed."""

from __future__ import annotations

import pytest
import torch

from chunkkv_b200 import _lib, ops
from oracle import kv8_oracle as ref

BF = torch.bfloat16


def cache(H=2, n=40, D=64, dtype=torch.int8, digest=False):
    return ops.KV8Cache(H, n, D, dtype, "cpu", digest=digest)


def test_cache_layout():
    c = cache(n=40, digest=True)
    assert c.k.shape == c.v.shape == (2, 48, 64) and c.k_scale.shape == (2, 3)
    assert c.digest.codes.shape == (2, 3, 2, 64) and c.tail.shape == (2, 2, 16, 64)
    assert c.nbytes == 2 * 2 * 48 * 64 + 2 * 2 * 3 * 4
    assert cache(dtype=torch.float8_e4m3fn).k.dtype == torch.float8_e4m3fn


def test_cache_refuses_wrong_buffers():
    with pytest.raises(NotImplementedError, match="dtype"):
        cache(dtype=torch.float16)
    with pytest.raises(ValueError):
        cache(n=0)
    c = cache()
    ok = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale, n_ctx=40)
    ops.KV8Cache.wrap(**ok)
    for bad, msg in [(dict(n_ctx=33 + 16), "shape"), (dict(v=c.v[:1]), "shape"), (dict(k_scale=c.k_scale.double()), "float32"),
                     (dict(k_scale=c.k_scale[:, :2]), "shape"), (dict(tail=torch.zeros((2, 2, 8, 64), dtype=BF)), "tail"),
                     (dict(v=c.v.view(torch.uint8).view(torch.float8_e4m3fn)), "int8"),
                     (dict(k=c.k.transpose(0, 1).contiguous().transpose(0, 1)), "contiguous"),
                     (dict(digest=ops.BlockDigest(2, 60, 64, "cpu")), "digest")]:
        with pytest.raises(ValueError, match=msg):
            ops.KV8Cache.wrap(**{**ok, **bad})
    with pytest.raises(ValueError, match="codes"):
        ops.BlockDigest.wrap(torch.zeros((2, 3, 64), dtype=torch.int8), torch.zeros((2, 3)), 40)
    with pytest.raises(ValueError, match="scale"):
        ops.BlockDigest.wrap(torch.zeros((2, 3, 2, 64), dtype=torch.int8), torch.zeros((2, 4)), 40)


def test_ops_check_arguments_before_the_device():
    c, x = cache(digest=True), torch.zeros((2, 8, 64), dtype=BF)
    pos = torch.zeros(3, dtype=torch.int32)
    q = torch.zeros((3, 4, 64), dtype=BF)
    d = c.digest
    kb = torch.zeros((2, 40, 64), dtype=BF)
    lists = torch.zeros((3, 2, 4), dtype=torch.int32)
    bad = [
        (lambda: ops.kv8_write(c, x.float(), x, 0), "bfloat16"),
        (lambda: ops.kv8_write(c, x[:1], x, 0), "shape"),
        (lambda: ops.kv8_write(c, x, x, 33), "outside"),
        (lambda: ops.kv8_write(c, x, x, -1), "outside"),
        (lambda: ops.kv8_write(c, x, x, 0, 9), "rows asked for"),
        (lambda: ops.kv8_write(c, x, x, 6, 3, by_position=True), "position 8"),
        (lambda: ops.kv8_write(c, x.transpose(1, 2).contiguous().transpose(1, 2), x, 0), "strides"),
        (lambda: ops.kv8_write(c, x, x, torch.zeros(1)), "int32"),
        (lambda: ops.kv8_read(c, 30, 11), "outside"),
        (lambda: ops.block_digest(kb, d, 39, 2), "outside"),
        (lambda: ops.block_digest(kb[:1], d), "shape"),
        (lambda: ops.attention_kv8(q[:, :3], c, pos), "multiple of 2"),
        (lambda: ops.attention_kv8(q, c, pos.long()), "int32"),
        (lambda: ops.attention_kv8(q, c, pos[:2]), "at least 3"),
        (lambda: ops.attention_kv8(q, c, pos, out=q.float()), "bfloat16"),
        (lambda: ops.attention_kv8(q, c, pos, m=4), "at least"),
        (lambda: ops.block_select(q, d, pos, 4, out=lists[:2]), "at least"),
        (lambda: ops.attention_blocks(q, kb, kb[:, :30], pos, lists), "length|shape|contiguous"),
        (lambda: ops.attention_blocks(q, kb, kb, pos, lists[:2]), "blocks"),
        (lambda: ops.attention_blocks_kv8(q, c, pos, lists.long()), "int32"),
        (lambda: ops.attention_sparse(q, kb, kb, pos, 0), "top"),
        (lambda: ops.attention_sparse(q, kb, kb, pos, 4, digest=ops.BlockDigest(2, 41, 64, "cpu")), "digest"),
        (lambda: ops.attention_sparse_kv8(q, cache(), pos, 4), "digest"),
        (lambda: ops.attention_kv8(q, c, pos), "CUDA"),
        (lambda: ops.kv8_write(c, x, x, 0), "CUDA"),
        (lambda: ops.kv8_read(c), "CUDA"),
        (lambda: ops.block_select(q, d, pos, 4), "CUDA"),
        (lambda: ops.attention_sparse(q, kb, kb, pos, 4), "CUDA"),
    ]
    for i, (call, msg) in enumerate(bad):
        with pytest.raises(ValueError, match=msg):
            call()
            pytest.fail(f"call {i} was not refused")


def test_entry_points_refuse_bad_sizes():
    """The C ABI itself: nothing is launched for any of these."""
    att = "ckv_attention_kv8"  # q, k8, v8, ks, vs, positions, out, m, Hq, H, D, n_ctx, scale, type, ws, bytes, stream
    sel = "ckv_block_select"   # q, codes, scale, positions, blocks, m, Hq, H, D, n_ctx, top, sink, recent, ws, bytes, stream
    blk = "ckv_attention_blocks"  # q, k, v, positions, blocks, out, m, Hq, H, D, n_ctx, top, scale, ws, bytes, stream
    rd = "ckv_kv8_read"  # k8, v8, ks, vs, ko, vo, H, D, n_ctx, start, m, type, stream
    P = 16
    cases = [
        (att, (P,) * 7 + (1, 5, 2, 64, 8, 1.0, 0, P, 0, None), ValueError, "bad sizes"),
        (att, (P,) * 7 + (1, 4, 2, 64, 8, 1.0, 7, P, 0, None), ValueError, "type 7"),
        (att, (P,) * 7 + (1, 4, 2, 96, 8, 1.0, 0, P, 0, None), NotImplementedError, "head_dim 96"),
        (att, (P,) * 7 + (1, 258, 2, 64, 8, 1.0, 0, P, 0, None), NotImplementedError, "129 query heads"),
        (att, (8,) + (P,) * 6 + (1, 4, 2, 64, 8, 1.0, 0, P, 0, None), ValueError, "aligned"),
        (att, (P, None) + (P,) * 5 + (1, 4, 2, 64, 8, 1.0, 0, P, 0, None), ValueError, "null"),
        (att, (P,) * 7 + (100, 4, 2, 64, 100000, 1.0, 0, P, 16, None), ValueError, "workspace of 16"),
        (sel, (P,) * 5 + (1, 4, 2, 64, 800, 2, 2, 1, P, 1 << 20, None), ValueError, "top 2"),
        (sel, (P,) * 5 + (1, 4, 2, 64, 800, 5000, 1, 1, P, 1 << 20, None), ValueError, "top 5000"),
        (sel, (P,) * 5 + (1, 4, 2, 64, 800, 4, 1, 0, P, 1 << 20, None), ValueError, "at least one last"),
        (sel, (P,) * 5 + (1, 34, 2, 64, 800, 4, 1, 1, P, 1 << 20, None), NotImplementedError, "17 query heads"),
        (sel, (P,) * 5 + (1, 4, 2, 64, 600000, 4, 1, 1, P, 1 << 30, None), NotImplementedError, "at most 524288"),
        (sel, (P,) * 5 + (100, 4, 2, 64, 800, 4, 1, 1, P, 8, None), ValueError, "workspace of 8"),
        (blk, (P,) * 6 + (1, 4, 2, 64, 800, 0, 1.0, P, 0, None), ValueError, "lists of 0"),
        (blk, (P,) * 4 + (None, P) + (1, 4, 2, 64, 800, 4, 1.0, P, 1 << 20, None), ValueError, "block list"),
        (blk, (P,) * 6 + (1, 4, 2, 256, 800, 4, 1.0, P, 1 << 20, None), NotImplementedError, "head_dim 256"),
        (rd, (P,) * 6 + (2, 64, 40, 30, 11, 0, None), ValueError, "outside"),
        (rd, (P,) * 6 + (2, 80, 40, 0, 4, 0, None), NotImplementedError, "head_dim 80"),
    ]
    for name, args, exc, msg in cases:
        with pytest.raises(exc, match=msg):
            _lib.call(name, *args)
    # nothing to do is fine, whatever the pointers
    _lib.call(att, *(None,) * 7, 0, 4, 2, 64, 8, 1.0, 0, None, 0, None)
    _lib.call(sel, *(None,) * 5, 0, 4, 2, 64, 800, 4, 1, 1, None, 0, None)
    _lib.call(blk, *(None,) * 6, 0, 4, 2, 64, 800, 4, 1.0, None, 0, None)


def test_workspace_sizes_cover_every_row_count():
    lib = _lib.load()
    for m in (1, 2, 17, 300, 5000):
        for n in (1, 16, 5248, 131072):
            assert lib.ckv_attention_kv8_workspace_size(m, 28, 4, 128, n) >= 0
            assert lib.ckv_attention_kv8_launches(m, 28, 4, 128, n) in (1, 2)
            nb = -(-n // 16)
            sel = lib.ckv_block_select_workspace_size(m, 28, 4, 128, n)
            few = m * 4 <= 32 and nb <= 4096  # one launch that keeps its scores on the SMs
            assert (sel == 0) == few and sel <= max(256 << 20, 16 * 4 * (nb + 3) * 4)
            assert lib.ckv_block_select_launches(m, 28, 4, 128, n) == 1 if few else 2
            both = lib.ckv_attention_sparse_workspace_size(m, 28, 4, 128, n, 8, 16, 1)
            assert both >= sel + 4 * nb * (2 * 128 + 4)
            assert lib.ckv_attention_sparse_workspace_size(m, 28, 4, 128, n, 8, 16, 0) >= sel
    assert lib.ckv_attention_kv8_workspace_size(1, 28, 4, 96, 100) == 0
    assert lib.ckv_block_select_workspace_size(1, 68, 4, 128, 100) == 0


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_oracle_codes_are_torch_roundings(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn((2, 37, 64), generator=g) * torch.randn((2, 37, 1), generator=g).exp()).to(BF)
    codes, scale = ref.quantize(x, dtype)
    f = torch.nn.functional.pad(x.float(), (0, 0, 0, 11)).view(2, 3, -1)
    a = f.abs().amax(-1)
    y = f * (torch.full_like(a, ref.QMAX[dtype]) / a)[..., None]
    want = y.round() if dtype is torch.int8 else y.to(dtype).float()
    assert torch.equal(want.view(2, 48, 64).double(), codes)
    assert torch.equal((a / torch.full_like(a, ref.QMAX[dtype])).double(), scale)


def test_oracle_bound_holds_every_key():
    """The digest's score bounds q . k from above, up to the rounding of both sides to 8 bits."""
    g = torch.Generator().manual_seed(2)
    k = torch.randn((1, 160, 64), generator=g).to(BF)
    q = torch.randn((1, 1, 64), generator=g).to(BF)
    dc, ds = ref.digest(k)
    a = q.double().abs().amax()
    c, _ = ref.codes_of(q.double().view(1, 64), 127.0, torch.int8)
    bound = torch.maximum(c * dc[0, :, 0], c * dc[0, :, 1]).sum(-1) * a / 127 * ds[0]
    true = (k[0].double() @ q[0, 0].double()).view(10, 16).amax(-1)
    # each of 64 products is off by half a step of either side: |q| s/2 + |k| a/254 <= a s (127/2 + 127/2 + 1/4) / 127
    assert bool((true <= bound + 64 * a * ds[0] * (127.25 / 127)).all())


def test_buffers_of_one_cache_lie_on_one_device():
    c = cache(digest=True)
    ok = dict(k=c.k, v=c.v, k_scale=c.k_scale, v_scale=c.v_scale, n_ctx=40, tail=c.tail, digest=c.digest)
    ops.KV8Cache.wrap(**ok)
    for name in ("v", "k_scale", "v_scale", "tail"):
        with pytest.raises(ValueError, match=f"{name} lies on meta"):
            ops.KV8Cache.wrap(**{**ok, name: ok[name].to("meta")})
    with pytest.raises(ValueError, match="digest lies on meta"):
        ops.KV8Cache.wrap(**{**ok, "digest": ops.BlockDigest(2, 40, 64, "meta")})
    with pytest.raises(ValueError, match="scale lies on meta"):
        ops.BlockDigest.wrap(c.digest.codes, c.digest.scale.to("meta"), 40)


def test_entry_points_refuse_scales_and_row_counts():
    """Nothing is launched for any of these."""
    P = 16
    for scale in (-1.0, float("inf"), float("nan")):
        for m in (1, 100):
            with pytest.raises(ValueError, match="scale"):
                _lib.call("ckv_attention_kv8", *(P,) * 7, m, 4, 2, 64, 100, scale, 0, P, 1 << 40, None)
        with pytest.raises(ValueError, match="scale"):
            _lib.call("ckv_attention_blocks", *(P,) * 6, 1, 4, 2, 64, 800, 4, scale, P, 1 << 40, None)
        with pytest.raises(ValueError, match="scale"):
            _lib.call("ckv_attention_blocks_kv8", *(P,) * 8, 1, 4, 2, 64, 800, 4, scale, 0, P, 1 << 40, None)
    many = (1 << 31) - 1
    with pytest.raises(ValueError, match="rows of 4 heads"):
        _lib.call("ckv_attention_blocks", *(P,) * 6, many, 4, 2, 64, 800, 4, 1.0, P, 1 << 40, None)
    with pytest.raises(ValueError, match="bad sizes"):
        _lib.call("ckv_attention_sparse", *(P,) * 8, many, 4, 2, 64, 800, 4, 1, 1, 1.0, P, 1 << 40, None)
    assert _lib.load().ckv_attention_blocks_workspace_size(many, 4, 2, 64, 4, 16) == 0
    with pytest.raises(NotImplementedError, match=f"{many} rows"):
        _lib.call("ckv_attention_kv8", *(P,) * 7, many, 4, 2, 64, 100, 1.0, 0, P, 1 << 40, None)
    assert _lib.load().ckv_attention_kv8_workspace_size(many, 4, 2, 64, 100) == 0


def test_direct_calls_convert_like_ctypes():
    """The entry points that go past ctypes (where the module is built): argument counts, ranges
    and types are checked, None is a null pointer."""
    lib = _lib.load()
    read = lib.ckv_kv8_read  # k8, v8, ks, vs, ko, vo, H, D, n_ctx, start, m, type, stream
    ok = (None,) * 6 + (4, 128, 64, 0, 0, 0, None)
    assert read(*ok) == _lib.CKV_OK
    assert read(*(None,) * 6, 4, 128, 64, 0, 1, 0, None) == _lib.CKV_ERR_ARG and "null pointer" in _lib.last_error()
    if _lib._call is None:
        pytest.skip("built without Python's headers")
    assert set(_lib._call.names) <= set(_lib.SIGNATURES)
    for bad in (ok[:-1], ok + (0,), ()):
        with pytest.raises(TypeError, match="13 expected"):
            read(*bad)
    with pytest.raises(OverflowError):
        read(*(None,) * 6, 4, 128, 1 << 31, 0, 0, 0, None)
    with pytest.raises(OverflowError):
        read(-1, *(None,) * 5, 4, 128, 64, 0, 0, 0, None)
    with pytest.raises(TypeError):
        read(*(None,) * 6, 4, 128, 64.0, 0, 0, 0, None)
    with pytest.raises(TypeError):
        lib.ckv_attention_kv8(*(None,) * 7, 0, 4, 2, 64, 8, "1.0", 0, None, 0, None)
    with pytest.raises(KeyError):
        _lib._call.bind("ckv_no_such_call", 0)
