"""The paged 8-bit cache in 64 bits, plainly: one token, one page, one head at a time (the tests' oracle)."""

from __future__ import annotations

import math

import torch

LEAST = 2.0**-40


class Pool:
    """The four tensors of a pool and a page table of pages in a random order."""

    def __init__(self, lens, *, kv=2, dim=64, size=16, seed=0, device="cuda", spare=2, width=None, total=None):
        g = torch.Generator().manual_seed(seed)
        need = [max(0, -(-n // size)) for n in lens]
        width = max([1, *need]) if width is None else width
        count = sum(need) + spare if total is None else total
        order = torch.randperm(count, generator=g)[: sum(need)].tolist()
        table = torch.full((len(lens), width), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for j in range(n):
                table[b, j] = order.pop()
        self.kv, self.dim, self.size, self.count = kv, dim, size, count
        self.t = {
            "key_pages": torch.zeros((count, kv, size, dim), dtype=torch.int8, device=device),
            "value_pages": torch.zeros((count, kv, dim, size), dtype=torch.int8, device=device),
            "key_scales": torch.full((count, kv), LEAST, device=device),
            "value_scales": torch.full((count, kv), LEAST, device=device),
        }
        self.table = table.to(device)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=device)

    def fill(self, seed=1, spread=6):
        """Random codes in every slot, scales of several powers of two."""
        g = torch.Generator(device=self.table.device).manual_seed(seed)
        for n in ("key", "value"):
            p = self.t[n + "_pages"]
            p.copy_(torch.randint(-127, 128, p.shape, generator=g, device=p.device, dtype=torch.int8))
            e = torch.randint(-spread, 1, self.t[n + "_scales"].shape, generator=g, device=p.device)
            self.t[n + "_scales"].copy_(torch.ldexp(torch.ones_like(e, dtype=torch.float32), e) / 64.0)
        return self

    def rows(self, b, n, head):
        """Keys and values of the first n tokens of sequence b in 64 bits; and which of them have a page."""
        k = torch.zeros(n, self.dim, dtype=torch.float64)
        v, there = torch.zeros_like(k), torch.zeros(n, dtype=torch.bool)
        table = self.table[b].tolist()
        for j in range(-(-n // self.size)):
            at = slice(j * self.size, min(n, (j + 1) * self.size))
            p = table[j] if j < len(table) else -1
            if not 0 <= p < self.count:
                continue
            m = at.stop - at.start
            k[at] = self.t["key_pages"][p, head, :m].double().cpu() * float(self.t["key_scales"][p, head])
            v[at] = self.t["value_pages"][p, head, :, :m].double().cpu().t() * float(self.t["value_scales"][p, head])
            there[at] = True
        return k, v, there


def attend(pool, query, news, lens, scale=None):
    """[tokens, heads, dim] outputs in 64 bits, and a bound of each row's error by its dtype (see ``bound``)."""
    heads, dim = query.shape[1], query.shape[2]
    group = heads // pool.kv
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(query.shape, dtype=torch.float64)
    off = torch.zeros(query.shape[:2], dtype=torch.float64)
    capacity = pool.table.shape[1] * pool.size
    q64 = query.detach().double().cpu()
    start = 0
    for b, (n, length) in enumerate(zip(news, lens)):
        seen_most = max(0, min(length, capacity))
        for h in range(pool.kv if seen_most else 0):
            k, v, there = pool.rows(b, seen_most, h)
            for i in range(n):
                upto = max(0, min(length - n + i + 1, seen_most))
                keep = there[:upto]
                if not bool(keep.any()):
                    continue
                kk, vv = k[:upto][keep], v[:upto][keep]
                for j in range(h * group, (h + 1) * group):
                    q = q64[start + i, j]
                    s = kk @ q * scale
                    out[start + i, j] = torch.softmax(s, 0) @ vv
                    off[start + i, j] = bound(q, kk, vv, s, scale, query.dtype)
        start += n
    return out, off


def bound(q, k, v, s, scale, dtype):
    """How far a kernel may be from 64 bits, for one row.

    The query is rounded to 127 x 256^(digits - 1) steps of its largest element (two digits for 16-bit queries, three
    for float32), so a score is off by at most half a step times sum |k|, and by a few roundings of 2^-24 relative to
    the score and to log2 of the value scale; the weights follow by exp (twice, numerator and denominator).  The weights
    of a tile of 64 are rounded to the same steps of the tile's largest: at most 64 half steps of a sum that holds that
    largest one.  float16 products (long chunks) instead round each weight by 2^-11 and each element of a float32
    query's two halves by 2^-22.  The result is rounded once, by half a step of its type.
    """
    steps = 127.0 * 256.0 ** (2 if dtype is torch.float32 else 1)
    reach = float(k.abs().sum(1).max()) * abs(scale)
    top = float(q.abs().max())
    score = reach * top * (0.5 / steps + 2.0**-22) + float(s.abs().max() + 64) * 2.0**-21
    weight = 64 * 0.5 / steps if dtype is torch.float32 else max(64 * 0.5 / steps, 2.0**-10)
    sums = 2.0**-20
    largest = float(v.abs().max())
    return (math.expm1(2 * score) + weight + sums) * largest + torch.finfo(dtype).eps / 2 * largest


def turn(x, cos, sin, rows):
    """Rotary positions in 64 bits: x [heads, dim], rows [rotary_dim] (a table row for each dimension)."""
    r = cos.shape[1]
    y = x.clone()
    for d in range(r):
        w = -x[:, d + r // 2] if d < r // 2 else x[:, d - r // 2]
        y[:, d] = x[:, d] * cos[rows[d], d] + w * sin[rows[d], d]
    return y


def hadamard(dim):
    h = torch.ones(1, 1, dtype=torch.float64)
    while h.shape[0] < dim:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h / math.sqrt(dim)


def least_scale(largest):
    """The least power of two, 2^-40 or more, of which ``largest`` is at most 127."""
    s = LEAST
    while largest > 127 * s:
        s *= 2
    return s
