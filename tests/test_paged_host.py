"""Refusals of the paged 8-bit cache's operators (no GPU): the C ABI's checks and the Python operators'."""

from __future__ import annotations

import ctypes

import pytest
import torch

from torque_hip import _lib, ops

FAKE = 4096  # an aligned address that no refused call reads


def append_args(**changes):
    names = ("key kts khs value vts vhs kv_dtype query qts qhs q_dtype q_heads query_out tokens kv_heads dim key_pages value_pages "
             "key_scales value_scales num_pages page_size table table_stride max_pages lens starts batch cos cos_stride sin sin_stride "
             "table_dtype table_rows rotary positions wide pos_stride axes pair_axes left right flags stream").split()
    a = dict.fromkeys(names, 0)
    a.update(key=FAKE, value=FAKE, query=FAKE, query_out=FAKE, key_pages=FAKE, value_pages=FAKE, key_scales=FAKE, value_scales=FAKE,
             table=FAKE, lens=FAKE, tokens=2, batch=2, kv_heads=2, q_heads=4, dim=64, num_pages=8, page_size=16, table_stride=4,
             max_pages=4, axes=1, cos=FAKE, sin=FAKE, table_rows=10, rotary=32, starts=None, positions=None, pair_axes=None, left=None,
             right=None, stream=None)
    a.update(changes)
    return list(a.values())


@pytest.mark.parametrize("changes,message", [
    (dict(dim=96), "head dimension"),
    (dict(page_size=48), "page size"),
    (dict(num_pages=0), "num_pages"),
    (dict(kv_heads=70000, q_heads=70000), "65535"),
    (dict(tokens=3), "one token per sequence"),
    (dict(tokens=-1), "non-negative"),
    (dict(tokens=2**31, starts=FAKE), "2\\^31"),
    (dict(table_stride=3), "overlap"),
    (dict(kv_dtype=7), "dtypes"),
    (dict(q_dtype=9), "dtypes"),
    (dict(table_dtype=5), "dtypes"),
    (dict(q_heads=3), "divisible"),
    (dict(rotary=33), "rotary_dim"),
    (dict(rotary=66), "rotary_dim"),
    (dict(axes=5), "axes"),
    (dict(axes=0), "axes"),
    (dict(axes=2), "several axes"),
    (dict(axes=2, positions=FAKE, pair_axes=bytes([0, 2] * 8)), "axis"),
    (dict(positions=FAKE, flags=32), "exclude"),
    (dict(flags=32, table_rows=1), "row for each token"),
    (dict(flags=1), "unknown flags"),
    (dict(left=FAKE), "pairs"),
    (dict(flags=2), "needs signs"),
    (dict(key=None), "null"),
    (dict(query_out=None), "null"),
    (dict(cos=None), "null"),
    (dict(lens=None), "null"),
    (dict(key_pages=FAKE + 8), "aligned"),
])
def test_append_refusals(changes, message):
    with pytest.raises(ValueError, match=message):
        _lib.call("tq_paged_append", *append_args(**changes))


def test_calls_without_tokens_do_nothing():
    assert _lib.call("tq_paged_append", *append_args(tokens=0, starts=FAKE, batch=0)) == 0
    assert _lib.call("tq_paged_attention", *attention_args(tokens=0, starts=FAKE)) == 0
    assert _lib.call("tq_paged_dequantize", None, 0, None, None, None, None, 4, 16, 2, 64, None, None, 0, None) == 0


def attention_args(**changes):
    names = ("query qts qhs q_dtype tokens q_heads kv_heads dim key_pages value_pages key_scales value_scales num_pages page_size table "
             "table_stride max_pages lens starts batch max_tokens scale ws ws_bytes out ots ohs stream").split()
    a = dict.fromkeys(names, 0)
    a.update(query=FAKE, key_pages=FAKE, value_pages=FAKE, key_scales=FAKE, value_scales=FAKE, table=FAKE, lens=FAKE, out=FAKE, tokens=2,
             batch=2, kv_heads=2, q_heads=4, dim=64, num_pages=8, page_size=16, table_stride=4000, max_pages=4000, scale=0.125,
             starts=None, ws=FAKE, ws_bytes=1 << 40, stream=None)
    a.update(changes)
    return list(a.values())


@pytest.mark.parametrize("changes,message", [
    (dict(dim=80), "head dimension"),
    (dict(page_size=128), "page size"),
    (dict(tokens=5), "one token per sequence"),
    (dict(q_heads=5), "divisible"),
    (dict(q_heads=0), "divisible"),
    (dict(q_dtype=3), "dtypes"),
    (dict(scale=float("nan")), "finite"),
    (dict(scale=float("inf")), "finite"),
    (dict(out=None), "null"),
    (dict(table=None), "null"),
    (dict(value_pages=FAKE + 1), "aligned"),
    (dict(ws_bytes=64), "workspace too small"),
    (dict(ws=None), "workspace too small"),
    (dict(ws=FAKE + 4), "aligned"),
    (dict(tokens=2**30, starts=FAKE), "2\\^31"),
    (dict(tokens=2**22, batch=2**22, table_stride=8, max_pages=8), "exceed one launch"),
])
def test_attention_refusals(changes, message):
    with pytest.raises(ValueError, match=message):
        _lib.call("tq_paged_attention", *attention_args(**changes))


def test_dequantize_refusals():
    call = lambda *a: _lib.call("tq_paged_dequantize", *a, None)  # noqa: E731
    good = [FAKE, 3, FAKE, FAKE, FAKE, FAKE, 4, 16, 2, 64, FAKE, FAKE, 0]
    for at, bad, message in ((1, -1, "count"), (7, 8, "page size"), (9, 32, "head dimension"), (12, 4, "dtypes"), (0, None, "null"),
                             (10, FAKE + 2, "aligned")):
        with pytest.raises(ValueError, match=message):
            call(*good[:at], bad, *good[at + 1:])


def test_workspace_bytes():
    ws = lambda *a: int(_lib.call("tq_paged_attention_workspace_bytes", *a, 256))  # noqa: E731
    for dim, few, many in ((64, 48, 64), (128, 24, 32), (256, 12, 16)):  # as many tiles of 64 keys, and nothing to join
        assert ws(1, 1, 0, 8, 8, dim, few, 64, 1) == 0 and ws(1, 1, 0, 8, 8, dim, few + 1, 64, 1) > 0
        assert ws(32, 32, 0, 8, 8, dim, many, 64, 1) == 0 and ws(32, 32, 0, 8, 8, dim, many + 1, 64, 1) > 0
    assert ws(1, 1, 0, 32, 8, 128, 512, 64, 1) > 0
    assert ws(1, 1, 0, 30, 8, 128, 512, 64, 1) == 0 and ws(1, 1, 0, 8, 8, 100, 512, 64, 1) == 0  # refused shapes


def test_kernel_choice():
    name = lambda *a: _lib.call("tq_paged_attention_kernel", *a, 256)  # noqa: E731
    assert name(1, 1, 0, 32, 8, 128, 2000, 64, 1) == b"paged_split_kernel<128>"
    assert name(16, 1, 1, 32, 8, 128, 512, 64, 16) == b"paged_chunk_kernel<128>"  # half a unit of rows over 32768 keys
    assert name(15, 1, 1, 32, 8, 128, 9999, 64, 15) == b"paged_split_kernel<128>"
    assert name(128, 1, 1, 32, 8, 128, 32, 64, 128) == b"paged_split_kernel<128>"  # 512 rows over 2000 keys
    assert name(512, 1, 1, 32, 8, 128, 8, 64, 512) == b"paged_chunk_kernel<128>"  # enough units of rows
    assert name(64, 64, 1, 32, 8, 128, 500, 64, 0) == b"paged_split_kernel<128>"  # the most rows unknown: as if even
    assert name(1, 1, 0, 30, 8, 128, 10, 64, 1) is None and name(0, 1, 0, 8, 8, 128, 10, 64, 1) is None


def pool(count=4, kv=2, size=16, dim=64):
    return dict(key_pages=torch.zeros(count, kv, size, dim, dtype=torch.int8), value_pages=torch.zeros(count, kv, dim, size, dtype=torch.int8),
                key_scales=torch.ones(count, kv), value_scales=torch.ones(count, kv))


def test_operators_refuse_host_tensors_and_bad_pools():
    x = torch.zeros(1, 2, 64)
    batch = dict(page_table=torch.zeros(1, 2, dtype=torch.int32), context_lens=torch.ones(1, dtype=torch.int32))
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_append(x, x, **batch, **pool())
    with pytest.raises(ValueError, match="HIP device"):
        ops.paged_attention(x, **batch, **pool())
    for name, bad, message in (("key_pages", torch.zeros(4, 2, 16, 64), "int8"), ("value_pages", torch.zeros(4, 2, 16, 64, dtype=torch.int8), "transposed"),
                               ("key_scales", torch.ones(4, 3), "key_scales"), ("value_scales", torch.ones(4, 2).double(), "value_scales")):
        with pytest.raises(ValueError, match=message):
            ops.paged_dequantize(torch.zeros(1, dtype=torch.int32), **{**pool(), name: bad})


def test_header_constant_matches():
    assert _lib.TQ_TABLES_BY_TOKEN == 32
    assert ctypes.sizeof(ctypes.c_size_t) == 8
