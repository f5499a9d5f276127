"""Plans and refusals of the 8-bit cache's attention and of the attention over selected blocks, on the
host: nothing here launches.  No GPU needed."""

from __future__ import annotations

import pytest

from chunkkv_b200 import _lib

P = 16  # a pointer that is never followed
BIG = 1 << 40


def sparse(m=1, Hq=4, H=2, D=64, n=800, top=4, sink=1, recent=1, scale=1.0, ws=P, nbytes=BIG, build=False, **ptr):
    p = {k: ptr.get(k, P) for k in ("q", "k", "v", "codes", "dscale", "positions", "blocks", "out")}
    if build:
        p["codes"] = p["dscale"] = None
    return ("ckv_attention_sparse", *p.values(), m, Hq, H, D, n, top, sink, recent, scale, ws, nbytes, None)


def sparse8(m=1, Hq=4, H=2, D=64, n=800, top=4, sink=1, recent=1, scale=1.0, kind=0, ws=P, nbytes=BIG, **ptr):
    names = ("q", "k", "v", "ks", "vs", "codes", "dscale", "positions", "blocks", "out")
    return ("ckv_attention_sparse_kv8", *(ptr.get(k, P) for k in names), m, Hq, H, D, n, top, sink, recent, scale, kind, ws,
            nbytes, None)


BAD = [(dict(scale=float("nan")), ValueError, "scale"), (dict(scale=-1.0), ValueError, "scale"),
       (dict(scale=float("inf")), ValueError, "scale"), (dict(out=None), ValueError, "null"), (dict(v=8), ValueError, "aligned"),
       (dict(out=24), ValueError, "aligned"), (dict(q=8), ValueError, "aligned"), (dict(blocks=None), ValueError, "null"),
       (dict(positions=None), ValueError, "null"), (dict(Hq=34), NotImplementedError, "17 query heads"),
       (dict(n=600000), NotImplementedError, "at most 524288"), (dict(top=5000), ValueError, "top 5000"),
       (dict(top=2, sink=2), ValueError, "top 2"), (dict(recent=0), ValueError, "at least one last"),
       (dict(D=96), NotImplementedError, "head_dim 96"), (dict(m=100, nbytes=8), ValueError, "workspace of 8"),
       (dict(m=100, ws=None), ValueError, "null|workspace")]


@pytest.mark.parametrize("bad,exc,msg", BAD)
def test_sparse_calls_check_every_step_before_the_first(bad, exc, msg):
    """A call that is refused has neither built the digest nor rewritten the lists: on this host the
    first launch would fail as a CUDA error instead."""
    calls = [sparse(**bad), sparse8(**bad)]
    calls.append(sparse(**bad, build=True))
    for name, *args in calls:
        with pytest.raises(exc, match=msg):
            _lib.call(name, *args)


@pytest.mark.parametrize("bad,msg", [(dict(kind=7), "type 7"), (dict(ks=None), "null scales"), (dict(vs=None), "null scales"),
                                     (dict(codes=None), "null"), (dict(dscale=None), "null"), (dict(codes=8), "aligned")])
def test_sparse_calls_over_8_bits_check_their_own(bad, msg):
    name, *args = sparse8(**bad)
    with pytest.raises(ValueError, match=msg):
        _lib.call(name, *args)


def test_sparse_call_refuses_half_a_digest():
    name, *args = sparse(codes=None)
    with pytest.raises(ValueError, match="digest pointers"):
        _lib.call(name, *args)
    name, *args = sparse(build=True, k=8)
    with pytest.raises(ValueError, match="aligned"):
        _lib.call(name, *args)


def test_lists_longer_than_the_context_are_planned_by_its_blocks():
    """`top` may exceed the blocks that exist; no list can, so work and partials go by the latter."""
    lib = _lib.load()
    # 4096 entries over 4096 tokens: 256 blocks, which eight CTAs of a cluster share without partials
    for top in (256, 257, 1000, 4096):
        assert lib.ckv_attention_sparse_workspace_size(1, 32, 8, 128, 4096, top, 8, 0) == \
            lib.ckv_attention_sparse_workspace_size(1, 32, 8, 128, 4096, 256, 8, 0)
    for m, Hq, H, D, n in ((1, 28, 4, 128, 300), (9, 14, 2, 64, 40000), (3, 40, 8, 128, 700), (2, 7, 1, 128, 100000)):
        nb = -(-n // 16)
        for top in (1, 4, 5, 64, nb, 4096):
            for bits in (8, 16):
                size = lib.ckv_attention_blocks_workspace_size
                # what the call asks for is never more than the size for the whole list
                assert size(m, Hq, H, D, min(top, nb), bits) <= size(m, Hq, H, D, top, bits)


def test_launches_count_every_run():
    """Calls of more rows than one grid or one workspace holds go in several runs."""
    lib = _lib.load()
    blocks = lib.ckv_attention_blocks_launches
    for bits in (8, 16):
        assert blocks(32768, 2, 2, 64, 3, bits) == 1 and blocks(32769, 2, 2, 64, 3, bits) == 2
        assert blocks(100_000, 2, 2, 64, 3, bits) == 4
        assert blocks(16_384, 20, 1, 64, 3, bits) == 1 and blocks(17_000, 20, 1, 64, 3, bits) == 2  # two tiles a token
    for m, Hq, H, D, n in ((1, 28, 4, 128, 5248), (17, 28, 4, 128, 5248), (300, 28, 4, 128, 131072), (5000, 28, 4, 128, 131072),
                           (1300, 8, 8, 64, 131072)):
        nb = -(-n // 16)
        size = lib.ckv_block_select_workspace_size(m, Hq, H, D, n)
        few = m * H <= 32 and nb <= 4096
        per_token = H * ((nb + 3) // 4 * 4) * 4  # 4-byte keys, rows padded to 16 bytes
        runs = 1 if few else -(-m // (size // per_token))
        assert lib.ckv_block_select_launches(m, Hq, H, D, n) == (1 if few else 2 * runs)
    assert lib.ckv_block_select_launches(5000, 28, 4, 128, 131072) == 6


@pytest.mark.parametrize("scale", [2.5e38, 3.4e38, float("inf"), -1e-30, float("nan")])
@pytest.mark.parametrize("m,n", [(1, 100), (100, 6000)])  # streamed, in tiles
def test_softmax_scales_out_of_range(scale, m, n):
    """Past 2e38 the scale leaves fp32 in the log2 domain: refused by every form."""
    lib = _lib.load()
    assert (lib.ckv_attention_kv8_splits(m, 28, 4, 128, n) > 0) == (m > 1)
    with pytest.raises(ValueError, match="scale"):
        _lib.call("ckv_attention_kv8", *(P,) * 7, m, 28, 4, 128, n, scale, 0, P, BIG, None)
    with pytest.raises(ValueError, match="scale"):
        _lib.call("ckv_attention_blocks_kv8", *(P,) * 8, m, 28, 4, 128, n, 4, scale, 0, P, BIG, None)
    with pytest.raises(ValueError, match="scale"):
        _lib.call("ckv_attention_blocks", *(P,) * 6, m, 28, 4, 128, n, 4, scale, P, BIG, None)
