"""Pages, sequences and lengths of TorquePagedKVCache, on the CPU: no call here reaches a kernel."""

from __future__ import annotations

import pytest
import torch

import torque_hip as th


def cache(**changes):
    kw = dict(kv_heads=2, head_dim=64, num_pages=6, max_sequences=3, max_tokens=100, page_size=16, device="cpu")
    return th.TorquePagedKVCache(**{**kw, **changes})


@pytest.mark.parametrize("changes,message", [
    (dict(head_dim=96), "head dimension"), (dict(page_size=128), "page_size"), (dict(kv_heads=0), "kv_heads"), (dict(num_pages=0), "num_pages"),
    (dict(max_sequences=0), "max_sequences"), (dict(max_tokens=0), "max_tokens"), (dict(rotate_values=True), "needs a rotation"),
    (dict(rotation=th.RotationSpec.from_seed(128, 1)), "does not match"),
])
def test_constructor_refusals(changes, message):
    with pytest.raises(ValueError, match=message):
        cache(**changes)


def test_pages_follow_the_sequences():
    c = cache()
    a, b = c.add_sequence(), c.add_sequence()
    assert (a, b) == (0, 1) and c.sequences == (0, 1) and c.free_pages == 6
    c.reserve([a, b], [17, 16])
    c._lengths.update({a: 17, b: 16})
    assert c.free_pages == 3 and len(set(c._pages[a] + c._pages[b])) == 3
    assert c._table[a, :2].tolist() == c._pages[a] and c._table[b, 0] == c._pages[b][0] and int(c._table[a, 2]) == -1
    c.reserve([a], [15])  # the second page has room
    assert c.free_pages == 3
    with pytest.raises(RuntimeError, match="out of pages"):
        c.reserve([a, b], [32, 33])
    assert c.free_pages == 3 and len(c._pages[a]) == 2  # nothing changed
    with pytest.raises(ValueError, match="holds 100 of each"):
        c.reserve([a], [84])
    c.truncate(a, 16)
    assert c.length(a) == 16 and c.free_pages == 4
    with pytest.raises(ValueError, match="cannot keep"):
        c.truncate(a, 17)
    c.free_sequence(a)
    assert c.free_pages == 5 and c.sequences == (1,)
    assert c.add_sequence() == 0 and c.length(0) == 0  # the slot serves again
    c.add_sequence()
    with pytest.raises(ValueError, match="3 sequences already"):
        c.add_sequence()
    with pytest.raises(ValueError, match="no sequence 7"):
        c.length(7)


def test_rows_are_dealt_to_sequences():
    c = cache()
    for _ in range(3):
        c.add_sequence()
    assert c._plan(6, None, None) == ([0, 1, 2], [2, 2, 2])
    assert c._plan(3, [2, 0], [0, 3]) == ([2, 0], [0, 3])
    for args, message in (((4, None, None), "evenly"), ((3, [0, 0], [1, 2]), "twice"), ((3, [0, 1], [1, 1]), "counts"),
                          ((3, [0, 1], [4, -1]), "counts"), ((1, [5], [1]), "no sequence 5")):
        with pytest.raises(ValueError, match=message):
            c._plan(*args)
    c._lengths.update({0: 5, 1: 6, 2: 7})
    one = c._batch([0, 1, 2], [1, 1, 1])
    assert one["token_starts"] is None and one["context_lens"].tolist() == [5, 6, 7] and one["page_table"].data_ptr() == c._table.data_ptr()
    some = c._batch([2, 0], [3, 1])
    assert some["token_starts"].tolist() == [0, 3, 4] and some["context_lens"].tolist() == [7, 5]
    assert torch.equal(some["page_table"], c._table[[2, 0], :1])  # as wide as the longest sequence


def test_refused_calls_change_no_length():
    c = cache()
    c.add_sequence()
    x = torch.zeros(2, 2, 64)
    with pytest.raises(ValueError, match="HIP device"):
        c.append(x, x)
    assert c.length(0) == 0
    with pytest.raises(ValueError, match="tables have 1 rows"):
        c.append(x, x, cos=torch.ones(1, 64), sin=torch.zeros(1, 64))
    with pytest.raises(ValueError, match="key must have shape"):
        c.append(x[0], x[0])
    with pytest.raises(ValueError, match="query must have shape"):
        c.attend(x[0])
    assert c.length(0) == 0
