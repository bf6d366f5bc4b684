"""The paged 8-bit cache on the GPU: appends, attention and read-back against 64 bits."""

from __future__ import annotations

import math

import paged_model as model
import pytest
import torch

from torque_hip import _lib, ops

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def starts_of(news, device="cuda"):
    return torch.tensor([sum(news[:b]) for b in range(len(news) + 1)], dtype=torch.int32, device=device)


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).cuda()


def check_attention(pool, query, news, lens, out, scale=None):
    want, off = model.attend(pool, query[: sum(news)], news, lens, scale)
    got = out[: sum(news)].double().cpu()
    assert bool(torch.isfinite(got).all())
    err = (got - want).abs().amax(-1)
    worst = float((err / off.clamp_min(1e-30)).max())
    assert bool((err <= off).all()), f"error {worst:.2f} times the bound"


ATTENTION = [
    # dim, page, dtype, kv, group, tokens each sequence adds, lengths with them
    (128, 64, "f16", 2, 4, [1], [1]),
    (128, 64, "f16", 2, 4, [1], [513]),
    (64, 16, "bf16", 1, 1, [1, 1, 1], [15, 16, 17]),
    (64, 32, "f32", 3, 5, [1, 1], [31, 700]),
    (128, 16, "bf16", 2, 8, [1] * 6, [0, 1, 63, 64, 65, 1500]),
    (256, 64, "f32", 1, 4, [1], [2100]),
    (256, 16, "f16", 2, 3, [1, 1], [129, 640]),
    (128, 32, "f16", 1, 17, [1, 1], [100, 40]),  # more query heads than a product has columns
    (64, 64, "f16", 2, 2, [5, 3, 1], [5, 200, 70]),  # drafts
    (128, 16, "f32", 1, 3, [7, 16], [900, 16]),
    (128, 64, "bf16", 1, 4, [70, 0, 33], [70, 10, 300]),  # chunks; a sequence that adds nothing
    (256, 32, "bf16", 1, 2, [130], [400]),
    (64, 16, "f32", 2, 1, [200], [777]),
    (128, 32, "f16", 2, 4, [257, 64], [257, 1000]),
]


@pytest.mark.parametrize("dim,size,dtype,kv,group,news,lens", ATTENTION)
def test_attention_against_64_bits(hip_device, dim, size, dtype, kv, group, news, lens):
    pool = model.Pool(lens, kv=kv, dim=dim, size=size, seed=3).fill()
    query = randn(5, sum(news), kv * group, dim, dtype=TYPES[dtype])
    starts = None if news == [1] * len(lens) else starts_of(news)
    out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, token_starts=starts, max_tokens=max(news), **pool.t)
    check_attention(pool, query, news, lens, out)
    again = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, token_starts=starts, max_tokens=max(news), **pool.t)
    assert torch.equal(out, again)
    if starts is None:  # the same rows, named by their offsets
        same = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
        check_attention(pool, query, news, lens, same)


@pytest.mark.parametrize("dim,size,dtype,kv,group,news,lens", [c for c in ATTENTION if max(c[5]) * c[4] < 64])
def test_cut_keys_against_64_bits(hip_device, dim, size, dtype, kv, group, news, lens):
    """A table wide enough for long sequences has the keys cut over workgroups, whatever the lengths are."""
    pool = model.Pool(lens, kv=kv, dim=dim, size=size, seed=3, width=20_000 // size).fill()
    query = randn(5, sum(news), kv * group, dim, dtype=TYPES[dtype])
    ragged = news != [1] * len(lens)
    shape = (sum(news), len(lens), int(ragged), kv * group, kv, dim, pool.table.shape[1], size, max(news), 0)
    assert _lib.call("tq_paged_attention_workspace_bytes", *shape) > 0
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news) if ragged else None, max_tokens=max(news))
    out = ops.paged_attention(query, **kw, **pool.t)
    check_attention(pool, query, news, lens, out)
    assert torch.equal(out, ops.paged_attention(query, **kw, **pool.t))


CHUNKS = [
    # dim, page, dtype, kv, group, tokens each sequence adds, lengths with them
    (128, 64, "bf16", 1, 4, [70, 0, 33], [70, 10, 300]),
    (256, 32, "bf16", 1, 2, [130], [400]),
    (256, 16, "f32", 2, 3, [45, 22], [45, 500]),
    (64, 16, "f32", 2, 1, [200], [777]),
    (128, 32, "f16", 2, 4, [257, 64], [257, 1000]),
    (128, 16, "f32", 1, 5, [31, 2, 100], [200, 2, 163]),
    (64, 64, "f16", 3, 7, [64], [65]),
    (256, 64, "f16", 1, 17, [9, 40], [9, 700]),
]


@pytest.mark.parametrize("dim,size,dtype,kv,group,news,lens", CHUNKS)
def test_chunks_against_64_bits(hip_device, dim, size, dtype, kv, group, news, lens):
    """The kernel for many rows, which a table wide enough for long sequences chooses: other pages behind the end, a page
    that is none, rows of no sequence and an output with strides."""
    pool = model.Pool(lens, kv=kv, dim=dim, size=size, seed=3, width=400_000 // size).fill()
    n = sum(news)
    shape = (n + 3, len(news), 1, kv * group, kv, dim, pool.table.shape[1], size, max(news), 0)
    assert _lib.call("tq_paged_attention_kernel", *shape) == b"paged_chunk_kernel<%d>" % dim
    query = randn(5, n + 3, kv * group, dim, dtype=TYPES[dtype])
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), max_tokens=max(news), **pool.t)
    large = torch.full((kv * group, n + 3, dim + 8), 5.0, dtype=TYPES[dtype], device="cuda")
    out = ops.paged_attention(query, out=large.transpose(0, 1)[..., 4 : dim + 4], **kw)
    check_attention(pool, query, news, lens, out)
    assert bool((large[:, n:] == 5).all()) and bool((large[..., :4] == 5).all()) and bool((large[..., dim + 4 :] == 5).all())
    again = ops.paged_attention(query, **kw)
    assert torch.equal(again[:n], out[:n]) and bool((again[n:] == 0).all())
    few = ops.paged_attention(query, **{**kw, "max_tokens": 1})  # a hint that is wrong chooses the other kernel, no more
    check_attention(pool, query, news, lens, few)
    b = len(news) - 1
    pool.table[b, (lens[b] - 1) // size // 2] = -1
    check_attention(pool, query, news, lens, ops.paged_attention(query, **kw))


def test_chunks_of_many_sequences(hip_device):
    """So many units of rows that each has a workgroup of its own, and bad queries among them."""
    g = torch.Generator().manual_seed(1)
    news = torch.randint(0, 40, (40,), generator=g).tolist()
    news[3], news[7] = 70, 0
    lens = [n + int(x) for n, x in zip(news, torch.randint(0, 90, (40,), generator=g))]
    pool = model.Pool(lens, kv=8, dim=64, size=16, seed=3, width=8192).fill()
    assert _lib.call("tq_paged_attention_kernel", sum(news), 40, 1, 8, 8, 64, 8192, 16, 70, 0) == b"paged_chunk_kernel<64>"
    assert _lib.call("tq_paged_attention_workspace_bytes", sum(news), 40, 1, 8, 8, 64, 8192, 16, 70, 0) == 0  # nothing is cut
    query = randn(5, sum(news), 8, 64, dtype=torch.bfloat16)
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), max_tokens=max(news), **pool.t)
    out = ops.paged_attention(query, **kw)
    check_attention(pool, query, news, lens, out)
    query[5, 2, 7], query[100, 0, 0] = math.inf, math.nan
    bad = ops.paged_attention(query, **kw)
    assert bool(bad[5, 2].isnan().all()) and bool(bad[100, 0].isnan().all())
    bad[5, 2], bad[100, 0] = out[5, 2], out[100, 0]
    assert torch.equal(bad, out)


def test_rows_that_see_nothing_are_zero(hip_device):
    """No tokens, more rows than tokens, a negative length, a table without pages."""
    news, lens = [1, 4, 2, 1], [0, 2, -5, 40]
    pool = model.Pool([0, 2, 0, 40], seed=1).fill()
    pool.table[3, :] = torch.tensor([-1, 10**6, -(2**31)], dtype=torch.int32)
    pool.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    query = randn(2, sum(news), 4, 64, dtype=torch.float16)
    out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
    check_attention(pool, query, news, lens, out)
    zero = out.abs().amax((1, 2)) == 0
    assert zero.tolist() == [True, True, True, False, False, True, True, True]


def test_pages_outside_the_pool_are_passed_over(hip_device):
    lens = [200, 90]
    pool = model.Pool(lens, kv=2, dim=128, size=16, seed=4).fill()
    pool.table[0, 3], pool.table[0, 12], pool.table[1, 0] = -1, pool.count, 2**31 - 1
    query = randn(6, 2, 4, 128)
    out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, **pool.t)
    check_attention(pool, query, [1, 1], lens, out)


def test_lengths_beyond_the_table_are_cut(hip_device):
    pool = model.Pool([64, 64], kv=1, dim=64, size=16, seed=4).fill()
    pool.lens = torch.tensor([2**31 - 1, 70], dtype=torch.int32, device="cuda")
    query = randn(6, 2, 2, 64)
    out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, **pool.t)
    check_attention(pool, query, [1, 1], [2**31 - 1, 70], out)


def test_nothing_behind_the_end_is_seen(hip_device):
    """NaN scales of pages not listed, and codes behind a sequence's end, change no bit."""
    lens = [37, 90]
    pool = model.Pool(lens, kv=2, dim=64, size=32, seed=8, spare=3).fill()
    query = randn(6, 2, 4, 64, dtype=torch.bfloat16)
    call = lambda: ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, **pool.t)  # noqa: E731
    want = call()
    used = set(pool.table.flatten().tolist())
    for p in range(pool.count):
        if p not in used:
            pool.t["key_scales"][p] = pool.t["value_scales"][p] = math.nan
    p = int(pool.table[0, 1])
    pool.t["key_pages"][p, :, 5:] = 127
    pool.t["value_pages"][p, :, :, 5:] = -128
    wide = torch.full((2, 9), 10**9, dtype=torch.int32, device="cuda")
    wide[:, :3] = pool.table
    pool.table = wide[:, :3]  # a table inside a wider one
    assert torch.equal(call(), want)


def test_rows_of_no_sequence(hip_device):
    """A padded call: rows behind the last sequence stay as they were in ``out``, and are zero in a new tensor."""
    news, lens = [2, 1], [50, 20]
    pool = model.Pool(lens, seed=8).fill()
    query = randn(6, 7, 4, 64)
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
    out = torch.full((7, 4, 64), 5.0, device="cuda")
    assert ops.paged_attention(query, out=out, **kw) is out
    check_attention(pool, query, news, lens, out)
    assert bool((out[3:] == 5).all())
    fresh = ops.paged_attention(query, **kw)
    assert torch.equal(fresh[:3], out[:3]) and bool((fresh[3:] == 0).all())


@pytest.mark.parametrize("news", [[1, 1], [9, 40]])
def test_strided_rows(hip_device, news):
    """Queries inside a projection's output and an output inside a larger tensor."""
    lens = [300, 45]
    pool = model.Pool(lens, kv=2, dim=128, size=16, seed=8).fill()
    both = randn(6, sum(news), 4, 256, dtype=torch.float16)
    query = both[..., 3:131]  # neither aligned nor contiguous
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
    large = torch.zeros(4, sum(news), 130, dtype=torch.float16, device="cuda")
    out = ops.paged_attention(query, out=large.transpose(0, 1)[..., 1:129], **kw)
    assert torch.equal(out, ops.paged_attention(query.contiguous(), **kw))
    check_attention(pool, query, news, lens, out)
    assert bool((large[..., 0] == 0).all()) and bool((large[..., 129] == 0).all())


def test_scale_and_bad_queries(hip_device):
    lens = [100, 64, 30]
    pool = model.Pool(lens, kv=1, dim=64, size=64, seed=2).fill()
    query = randn(6, 3, 2, 64)
    for scale in (0.0, -0.5, 0.7):
        out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, scale=scale, **pool.t)
        check_attention(pool, query, [1] * 3, lens, out, scale)
    want = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, **pool.t)
    bad = query.clone()
    bad[0, 0, 3], bad[2, 1, 0] = math.nan, math.inf
    out = ops.paged_attention(bad, page_table=pool.table, context_lens=pool.lens, **pool.t)
    assert bool(out[0, 0].isnan().all()) and bool(out[2, 1].isnan().all())
    keep = torch.ones(3, 2, dtype=torch.bool)
    keep[0, 0] = keep[2, 1] = False
    assert torch.equal(out[keep], want[keep])
    zero = torch.zeros_like(query)
    check_attention(pool, zero, [1] * 3, lens, ops.paged_attention(zero, page_table=pool.table, context_lens=pool.lens, **pool.t))


@pytest.mark.parametrize("spread", [0, 30])
@pytest.mark.parametrize("new,width", [(1, 32), (1, 4096), (100, 32), (100, 4096)])
def test_scales_far_apart(hip_device, spread, new, width):
    """Pages whose scales differ by up to 2^30, one sharp row among them."""
    lens = [500]
    pool = model.Pool(lens, kv=1, dim=64, size=16, seed=2, width=width).fill(spread=6)
    pool.t["value_scales"].mul_(torch.exp2(torch.randint(-spread, 1, pool.t["value_scales"].shape).float()).cuda())
    query = randn(6, new, 3, 64) * torch.tensor([0.01, 1.0, 8.0], device="cuda")[None, :, None]
    out = ops.paged_attention(query, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([new]), **pool.t)
    check_attention(pool, query, [new], lens, out)


def test_pool_beyond_32_bits(hip_device):
    """Pages whose byte offsets pass 2^31."""
    lens, dim, size, kv = [130], 256, 64, 8
    count = 2**31 // (dim * size * kv) + 8
    pool = model.Pool(lens, kv=kv, dim=dim, size=size, total=count)
    pool.table[0] = torch.tensor([count - 1, count - 3, 1], dtype=torch.int32)
    key, value = randn(3, 130, kv, dim, dtype=torch.float16), randn(4, 130, kv, dim, dtype=torch.float16)
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([130]), **pool.t)
    ops.paged_append(key, value, **kw)
    k, v = ops.paged_dequantize(pool.table[0].contiguous(), **pool.t)
    for x, rows in ((k, key), (v, value)):
        x = x.transpose(1, 2).reshape(-1, kv, dim)[:130]
        top = float(rows.abs().max())
        assert 127 / 32 < top <= 127 / 16  # so the largest scale is 2^-4: 127 x 2^-5 < top <= 127 x 2^-4
        worst = float((x - rows.float()).abs().max())
        assert worst <= 0.5 * 2.0**-4
    query = randn(6, 130, kv, dim, dtype=torch.float16)
    out = ops.paged_attention(query, **kw)
    check_attention(pool, query, [130], lens, out)
    one = ops.paged_attention(query[129:].contiguous(), page_table=pool.table, context_lens=pool.lens, **pool.t)
    check_attention(pool, query[129:], [1], lens, one)


# ------------------------------------------------------------------ appending


def tables(rows, rotary, dtype=torch.float32):
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv[None]
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(dtype).cuda(), angle.sin().to(dtype).cuda()


def held_rows(pool, b, lo, hi):
    """Tokens lo..hi of a sequence as the pool holds them, and their scales: [tokens, kv, dim] and [tokens, kv] each."""
    at = [(int(pool.table[b, t // pool.size]), t % pool.size) for t in range(lo, hi)]
    k = torch.stack([pool.t["key_pages"][p, :, s].double().cpu() for p, s in at])
    v = torch.stack([pool.t["value_pages"][p, :, :, s].double().cpu() for p, s in at])
    ks, vs = (torch.stack([pool.t[n][p].double().cpu() for p, _ in at]) for n in ("key_scales", "value_scales"))
    return k * ks[..., None], v * vs[..., None], ks, vs


APPEND = [
    # dim, page, dtype, kv, rotary, basis, rotated values, tokens added, lengths with them
    (128, 64, "f16", 2, 128, True, False, [1], [33]),
    (64, 16, "f32", 3, 32, False, False, [1, 1, 1], [1, 16, 17]),
    (256, 32, "bf16", 1, 64, True, True, [40, 0, 3], [40, 7, 66]),
    (128, 16, "f32", 2, 0, True, True, [100], [109]),
    (64, 64, "bf16", 2, 64, True, False, [2, 64, 65, 63], [130, 64, 66, 191]),
    (256, 64, "f32", 1, 256, False, False, [129], [140]),
    (128, 32, "f16", 1, 2, True, False, [1, 31, 32, 33], [32, 32, 32, 33]),
]


@pytest.mark.parametrize("dim,size,dtype,kv,rotary,basis,both,news,lens", APPEND)
def test_append_against_64_bits(hip_device, dim, size, dtype, kv, rotary, basis, both, news, lens):
    pool = model.Pool(lens, kv=kv, dim=dim, size=size, seed=3).fill(spread=3)
    for n in ("key_scales", "value_scales"):
        pool.t[n].mul_(0.25)  # older tokens a little smaller: some scales grow
    before = {n: t.clone() for n, t in pool.t.items()}
    olds = [held_rows(pool, b, 0, t - n) if t > n else None for b, (n, t) in enumerate(zip(news, lens))]
    tokens = sum(news)
    key, value = randn(5, tokens, kv, dim, dtype=TYPES[dtype]), randn(6, tokens, kv, dim, dtype=TYPES[dtype])
    query = randn(7, tokens, 2 * kv, dim, dtype=TYPES[dtype])
    kw = {}
    if rotary:
        kw["cos"], kw["sin"] = tables(max(lens), rotary)
    if basis:
        left, right = torch.sign(randn(8, dim)), torch.sign(randn(9, dim))
        kw.update(signs_left=left, signs_right=right, rotate_values=both)
    starts = None if news == [1] * len(lens) else starts_of(news)
    turned = ops.paged_append(key, value, query=query, page_table=pool.table, context_lens=pool.lens, token_starts=starts, **kw, **pool.t)

    had = model.hadamard(dim)
    tol = dim * 2.0**-24 * 4  # float32 sums of dim terms, relative to the largest element

    def into(x, pos, rotated):
        x = x.double().cpu()
        if pos is not None and rotary:
            x = model.turn(x, kw["cos"].double().cpu(), kw["sin"].double().cpu(), [pos] * rotary)
        if rotated:
            x = (x * right.double().cpu()) @ had * left.double().cpu()
        return x

    start, touched = 0, set()
    for b, (n, t) in enumerate(zip(news, lens)):
        if n:
            touched |= {int(pool.table[b, j]) for j in range((t - n) // size, (t - 1) // size + 1)}
            k, v, ks, vs = held_rows(pool, b, t - n, t)
            wants = []
            for i in range(n):
                wants.append((into(key[start + i], t - n + i, basis), into(value[start + i], None, both)))
                q = into(query[start + i], t - n + i, basis)
                err = (turned[start + i].double().cpu() - q).abs().max()
                assert float(err) <= float(q.abs().max()) * (tol * math.sqrt(dim) + torch.finfo(TYPES[dtype]).eps / 2)
            for got, scales, at in ((k, ks, 0), (v, vs, 1)):
                want = torch.stack([w[at] for w in wants])
                largest = want.abs().amax(-1).max(0).values
                assert bool(((got - want).abs() <= 0.5 * scales[..., None] + tol * math.sqrt(dim) * largest[None, :, None]).all())
                for h in range(kv):  # the scale: the least power of two for its tokens, or what older tokens had
                    for j in range((t - n) // size, (t - 1) // size + 1):
                        at0, at1 = max(j * size, t - n) - (t - n), min((j + 1) * size, t) - (t - n)
                        top = float(want[at0:at1, h].abs().max())
                        fresh = {model.least_scale(top * (1 - tol * 16)), model.least_scale(top * (1 + tol * 16))}
                        p, name = int(pool.table[b, j]), ("key_scales", "value_scales")[at]
                        if j * size < t - n:
                            fresh = {max(f, float(before[name][p, h])) for f in fresh}
                        assert float(pool.t[name][p, h]) in fresh
            if olds[b] is not None:  # older tokens: as they were, or half a step of a grown scale off
                k2, v2, ks2, vs2 = held_rows(pool, b, 0, t - n)
                for new, old, s_new, s_old in ((k2, olds[b][0], ks2, olds[b][2]), (v2, olds[b][1], vs2, olds[b][3])):
                    grew = (s_new > s_old)[..., None]
                    assert bool(((new - old).abs() <= torch.where(grew, 0.5 * s_new[..., None], 0.0)).all())
        start += n
    for name, t in pool.t.items():  # pages that were not written
        rest = [p for p in range(pool.count) if p not in touched]
        assert torch.equal(t[rest], before[name][rest])


def test_append_leaves_slots_behind_the_end(hip_device):
    pool = model.Pool([20], kv=1, dim=64, size=32, seed=3).fill()
    before = {n: t.clone() for n, t in pool.t.items()}
    p = int(pool.table[0, 0])
    key = randn(1, 3, 1, 64) * 1000
    ops.paged_append(key, key, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([3]), **pool.t)
    assert torch.equal(pool.t["key_pages"][p, :, 20:], before["key_pages"][p, :, 20:])
    assert torch.equal(pool.t["value_pages"][p, :, :, 20:], before["value_pages"][p, :, :, 20:])
    assert float(pool.t["key_scales"][p, 0]) == model.least_scale(float(key.abs().max()))


def test_append_special_values(hip_device):
    """Infinities, NaN, zeros, tiny and huge rows; a page filled from its first slot again forgets its scale."""
    pool = model.Pool([16] * 6, kv=1, dim=64, size=16, seed=3).fill()
    pool.t["key_scales"].fill_(math.nan)
    pool.t["value_scales"].fill_(math.inf)
    x = randn(1, 96, 1, 64).reshape(6, 16, 1, 64)
    x[0, 3, 0, 5], x[0, 4, 0, 6], x[0, 5, 0, 7] = math.inf, -math.inf, math.nan
    x[1] = 0.0
    x[2] *= 1e-20
    x[3] *= 1e30
    x[4] = math.nan
    x[5] = 127.0
    x = x.reshape(96, 1, 64)
    ops.paged_append(x, x, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([16] * 6), **pool.t)
    k, v = ops.paged_dequantize(pool.table[:, 0].contiguous(), **pool.t)
    assert torch.equal(k, v)
    k = k[:, 0]
    s = [float(pool.t["key_scales"][int(pool.table[b, 0]), 0]) for b in range(6)]
    y = x.reshape(6, 16, 64).double()
    top = [float(torch.where(y[b].isfinite(), y[b].abs(), 0.0).max()) for b in range(6)]
    assert s == [model.least_scale(t) for t in top]
    assert float(k[0, 3, 5]) == 127 * s[0] and float(k[0, 4, 6]) == -127 * s[0] and float(k[0, 5, 7]) == 0.0
    for b in (0, 1, 2, 3, 5):
        fine = y[b].isfinite()
        assert bool(((k[b].double() - y[b]).abs()[fine] <= 0.5 * s[b]).all())
    assert bool((k[4] == 0).all()) and s[1] == s[4] == model.LEAST and s[5] == 1.0 and bool((k[5] == 127).all())


@pytest.mark.parametrize("wide", [False, True])
def test_append_positions_of_several_axes(hip_device, wide):
    """Each pair is turned by its own axis's position, sections or interleaved; by token rows; by cache positions."""
    dim, kv, n, rotary = 128, 2, 21, 64
    cos, sin = tables(500, rotary, torch.bfloat16)
    key, query = randn(1, n, kv, dim, dtype=torch.bfloat16), randn(2, n, 4, dim, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(3)
    pos = torch.randint(0, 500, (3, n), generator=g).to(torch.int64 if wide else torch.int32).cuda()
    for axes in ([0] * 10 + [1] * 12 + [2] * 10, [i % 3 for i in range(32)], [2] * 32):
        pool = model.Pool([n], kv=kv, dim=dim, size=32)
        out = ops.paged_append(key, key, query=query, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([n]),
                               cos=cos, sin=sin, positions=pos, pair_axes=axes, **pool.t)
        k, _, ks, _ = held_rows(pool, 0, 0, n)
        for i in range(n):
            rows = [int(pos[a, i]) for a in axes] * 2
            c, s = cos.double().cpu(), sin.double().cpu()
            want = model.turn(query[i].double().cpu(), c, s, rows)
            assert float((out[i].double().cpu() - want).abs().max()) <= float(want.abs().max()) * (2.0**-8 + 2.0**-22)
            assert bool(((k[i] - model.turn(key[i].double().cpu(), c, s, rows)).abs() <= 0.5 * ks[i][:, None] * (1 + 1e-4)).all())
    # one axis as [tokens] and as [1, tokens], and the same rows picked beforehand
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([n]), query=query, **pool.t)
    one = ops.paged_append(key, key, cos=cos, sin=sin, positions=pos[2], **kw)
    assert torch.equal(one, out)
    assert torch.equal(one, ops.paged_append(key, key, cos=cos, sin=sin, positions=pos[2:], pair_axes=[0] * 32, **kw))
    picked = dict(cos=cos[pos[2].long()], sin=sin[pos[2].long()])
    assert torch.equal(one, ops.paged_append(key, key, tables_by_token=True, **picked, **kw))


def test_append_positions_outside_the_tables(hip_device):
    pool = model.Pool([40, 9], kv=1, dim=64, size=16, seed=3).fill()
    before = {n: t.clone() for n, t in pool.t.items()}
    cos, sin = tables(39, 64)
    key, query = randn(1, 3, 1, 64), randn(2, 3, 2, 64)
    out = ops.paged_append(key, key, query=query, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of([2, 1]),
                           cos=cos, sin=sin, **pool.t)
    p = int(pool.table[0, 2])
    assert not bool(out[0].isnan().any()) and bool(out[1].isnan().all()) and not bool(out[2].isnan().any())
    assert torch.equal(pool.t["key_pages"][p, :, 7], before["key_pages"][p, :, 7])  # position 39: no row
    assert not torch.equal(pool.t["key_pages"][p, :, 6], before["key_pages"][p, :, 6])


def test_append_bad_pages_and_lengths(hip_device):
    """Places without a page, lengths beyond the table, more rows than tokens: what has no slot is not written."""
    pool = model.Pool([48, 48, 48], kv=1, dim=64, size=16, seed=3).fill()
    pool.table[0, 1], pool.table[1, 2] = -1, pool.count + 5
    pool.lens = torch.tensor([40, 60, 2], dtype=torch.int32, device="cuda")
    news = [30, 30, 5]
    key = randn(1, sum(news), 1, 64)
    before = {n: t.clone() for n, t in pool.t.items()}
    ops.paged_append(key, key, page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
    written = {int(pool.table[0, 0]), int(pool.table[0, 2]), int(pool.table[1, 1]), int(pool.table[2, 0])}
    for p in range(pool.count):
        same = all(torch.equal(pool.t[n][p], before[n][p]) for n in pool.t)
        assert same == (p not in written)
    k, v, ks, _ = held_rows(pool, 2, 0, 2)
    assert bool(((k - key[-2:].double().cpu()).abs() <= 0.5 * ks[..., None]).all())


@pytest.mark.parametrize("dim,rotary", [(64, 64), (128, 40), (256, 128)])
def test_append_types_and_strides_of_each_operand(hip_device, dim, rotary):
    """float32 queries beside bfloat16 keys that lie unaligned in a larger tensor, expanded values, strided tables: as the
    same rows laid out plainly."""
    news, lens, kv = [37, 1, 20], [40, 1, 84], 2
    n = sum(news)
    wide = randn(1, n, 3, dim + 6, dtype=torch.bfloat16)
    key = wide[:, :2, 3 : dim + 3]
    value = randn(2, n, 1, dim, dtype=torch.bfloat16).expand(n, kv, dim)
    query = randn(3, n, 4, 2 * dim)[..., 1::2]
    cos, sin = (t[::2] for t in tables(200, rotary))
    left, right = torch.sign(randn(8, dim)), torch.sign(randn(9, dim))
    results = []
    for k, v, q, c, s in ((key, value, query, cos, sin), tuple(t.contiguous() for t in (key, value, query, cos, sin))):
        pool = model.Pool(lens, kv=kv, dim=dim, size=32, seed=3).fill()
        out = ops.paged_append(k, v, query=q, cos=c, sin=s, signs_left=left, signs_right=right, rotate_values=True, page_table=pool.table,
                               context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
        same = ops.paged_append(k, v, query=q.to(k.dtype), cos=c, sin=s, signs_left=left, signs_right=right, rotate_values=True,
                                page_table=pool.table, context_lens=pool.lens, token_starts=starts_of(news), **pool.t)
        results.append((out, same, *pool.t.values()))
    assert results[0][0].dtype is torch.float32 and results[0][1].dtype is torch.bfloat16
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_attention_refuses_outputs_that_overlap(hip_device):
    pool = model.Pool([30, 30], seed=1).fill()
    query = randn(1, 2, 4, 64)
    kw = dict(page_table=pool.table, context_lens=pool.lens, **pool.t)
    for out, message in ((query, "share memory"), (torch.zeros(1, 4, 64, device="cuda").expand(2, 4, 64), "overlap itself"),
                         (torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda"), "out must be"),
                         (torch.zeros(2, 4, 128, device="cuda")[..., ::2], "unit stride")):
        with pytest.raises(ValueError, match=message):
            ops.paged_attention(query, out=out, **kw)
    with pytest.raises(ValueError, match="no backward"):
        ops.paged_attention(query.clone().requires_grad_(), **kw)
    with pytest.raises(ValueError, match="max_tokens"):
        ops.paged_attention(query, max_tokens=0, **kw)


def test_empty_calls(hip_device):
    """No tokens, no sequences, a table without places."""
    pool = model.Pool([5, 0], seed=1).fill()
    none = torch.zeros(3, dtype=torch.int32, device="cuda")
    x = torch.zeros(0, 2, 64, device="cuda")
    before = {n: t.clone() for n, t in pool.t.items()}
    kw = dict(page_table=pool.table, context_lens=pool.lens, token_starts=none, **pool.t)
    assert ops.paged_append(x, x, query=x, **kw).shape == (0, 2, 64) and ops.paged_attention(x, **kw).shape == (0, 2, 64)
    empty = dict(page_table=pool.table[:0], context_lens=pool.lens[:0], **pool.t)
    assert ops.paged_append(x, x, **empty) is None and ops.paged_attention(x, **empty).shape == (0, 2, 64)
    assert all(torch.equal(before[n], t) for n, t in pool.t.items())
    bare = dict(page_table=pool.table[:, :0], context_lens=pool.lens, **pool.t)
    assert bool((ops.paged_attention(randn(1, 2, 4, 64), **bare) == 0).all())
    ops.paged_append(randn(1, 2, 2, 64), randn(2, 2, 2, 64), **bare)
    assert all(torch.equal(before[n], t) for n, t in pool.t.items())


def test_dequantize(hip_device):
    pool = model.Pool([200], kv=3, dim=128, size=32, seed=3).fill()
    ids = torch.tensor([3, 0, -1, pool.count, 3], dtype=torch.int32, device="cuda")
    for dtype in TYPES.values():
        k, v = ops.paged_dequantize(ids, dtype=dtype, **pool.t)
        at = ids.long().clamp(0, pool.count - 1)
        there = ((ids >= 0) & (ids < pool.count))[:, None, None, None]
        want_k = (pool.t["key_pages"][at].float() * pool.t["key_scales"][at][..., None, None] * there).to(dtype)
        want_v = (pool.t["value_pages"][at].float() * pool.t["value_scales"][at][..., None, None] * there).to(dtype)
        assert torch.equal(k, want_k) and torch.equal(v, want_v.transpose(2, 3))
    k, v = ops.paged_dequantize(ids[:0], **pool.t)
    assert k.shape == (0, 3, 32, 128) and v.shape == k.shape


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_a_run_of_steps(hip_device, dtype):
    """Prompts, drafted tokens and single tokens of a batch, one after another: every output against the pool's rows."""
    kv, group, dim, size = 2, 3, 64, 16
    final = [150, 61, 97]
    pool = model.Pool(final, kv=kv, dim=dim, size=size, seed=5)
    cos, sin = tables(200, dim)
    left, right = torch.sign(randn(8, dim)), torch.sign(randn(9, dim))
    lens = [0, 0, 0]
    for step, news in enumerate([[100, 30, 70], [3, 1, 4], [1, 1, 1], [1, 1, 1], [17, 2, 0], [1, 0, 1]]):
        lens = [a + b for a, b in zip(lens, news)]
        pool.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        n = sum(news)
        q, k, v = (randn(100 * step + i, n, h, dim, dtype=TYPES[dtype]) for i, h in enumerate((kv * group, kv, kv)))
        batch = dict(page_table=pool.table, context_lens=pool.lens, token_starts=None if news == [1] * 3 else starts_of(news))
        q = ops.paged_append(k, v, query=q, cos=cos, sin=sin, signs_left=left, signs_right=right, **batch, **pool.t)
        out = ops.paged_attention(q, max_tokens=max(news), **batch, **pool.t)
        check_attention(pool, q, news, lens, out)


def graph_step(pool, dtype, kv, group, dim, tokens, starts):
    cos, sin = tables(2000, dim)
    bufs = [torch.zeros(tokens, h, dim, dtype=dtype, device="cuda") for h in (kv * group, kv, kv)]
    batch = dict(page_table=pool.table, context_lens=pool.lens, token_starts=starts)

    def step():
        q = ops.paged_append(bufs[1], bufs[2], query=bufs[0], cos=cos, sin=sin, **batch, **pool.t)
        return ops.paged_attention(q, **batch, **pool.t)

    return bufs, step


@pytest.mark.parametrize("width", [None, 100])  # of the table: keys read by one workgroup, and cut with a workspace
@pytest.mark.parametrize("news", [[1, 1], [40, 7]])
def test_graphs_follow_the_lengths(hip_device, news, width):
    """Two captured steps replayed in turn, other lengths and rows each time, eager work between: each as the eager step."""
    kv, group, dim = 2, 2, 128
    most = 700
    pools, graphs = [], []
    for i in range(2):
        pool = model.Pool([most, most], kv=kv, dim=dim, size=32, seed=i, width=width)
        bufs, step = graph_step(pool, torch.float16, kv, group, dim, sum(news), None if news == [1, 1] else starts_of(news))
        pool.lens.copy_(torch.tensor(news, dtype=torch.int32))
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        pools.append((pool, bufs, step))
        graphs.append((graph, out))
    for turn in range(4):
        lens = [n + 150 * turn + 13 for n in news]
        for i, ((pool, bufs, step), (graph, out)) in enumerate(zip(pools, graphs)):
            pool.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            for j, b in enumerate(bufs):
                b.copy_(randn(1000 * turn + 10 * i + j, *b.shape, dtype=b.dtype))
            saved = {n: t.clone() for n, t in pool.t.items()}
            graph.replay()
            got = out.clone()
            after = {n: t.clone() for n, t in pool.t.items()}
            for n, t in pool.t.items():
                t.copy_(saved[n])
            torch.cuda.synchronize()
            want = step()
            assert torch.equal(got, want)
            assert all(torch.equal(after[n], pool.t[n]) for n in after)
            check_attention(pool, ops.paged_append(bufs[1], bufs[2], query=bufs[0], cos=tables(2000, dim)[0], sin=tables(2000, dim)[1],
                                                   page_table=pool.table, context_lens=pool.lens,
                                                   token_starts=None if news == [1, 1] else starts_of(news), **pool.t),
                            news, lens, got)


def test_streams_do_not_share(hip_device):
    """The same calls on two streams at once as one after another."""
    lens = [5000, 3000, 40]
    pool = model.Pool(lens, kv=2, dim=128, size=64, seed=3).fill()
    queries = [randn(i, 3, 8, 128, dtype=torch.float16) for i in range(12)]
    call = lambda q: ops.paged_attention(q, page_table=pool.table, context_lens=pool.lens, **pool.t)  # noqa: E731
    want = [call(q) for q in queries]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for i, q in enumerate(queries):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call(q))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
