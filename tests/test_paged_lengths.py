"""Slot maps of lengths at the ends of their range."""
import pytest

import modelc_b200 as mb

gpu = pytest.mark.gpu
TOP = 2 ** 31 - 1


def _t(*x):
    import torch
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@gpu
def test_positions_past_31_bits_have_no_page():
    """Such a token has no page, reads none, and takes none; the others keep theirs."""
    kv, q = _t(3, TOP - 10, TOP, 60), _t(2, 20, 5, 10)
    table = _t(7, -1, -1, -1, -1, -1, 9, -1).view(4, 2)
    step = mb.paged_slots(kv, q, table, _t(1, 2, 3, 4), _t(4), 40, 64)
    assert step.cu_q.tolist() == [0, 2, 22, 27, 37]
    assert step.new_len.tolist() == [5, TOP, TOP, 70]
    past = [min(TOP - 10 + i, TOP) for i in range(20)] + [TOP] * 5
    assert step.positions.tolist() == [3, 4] + past + list(range(60, 70)) + [0] * 3
    assert step.slots.tolist() == [7 * 64 + 3, 7 * 64 + 4] + [-1] * 25 + \
        [9 * 64 + i for i in range(60, 64)] + [4 * 64 + i for i in range(6)] + [-1] * 3
    assert step.n_free.tolist() == [3] and table[3].tolist() == [9, 4]


@gpu
def test_sums_of_new_tokens_past_31_bits():
    n = 1500  # more requests than one chunk of the scan
    kv, q = _t(*[0] * n), _t(*[1] + [TOP] * (n - 1))
    table = _t(*[-1] * (2 * n)).view(n, 2)
    step = mb.paged_slots(kv, q, table, _t(*range(2 * n)), _t(2 * n), 100, 64)
    assert step.cu_q.tolist() == [0, 1] + [TOP] * (n - 1) and step.new_len.tolist() == [1] + [TOP] * (n - 1)
    assert step.positions.tolist() == [0] + list(range(99))
    top = 2 * n - 1
    assert step.slots.tolist() == [top * 64] + [(top - 1) * 64 + i for i in range(64)] + \
        [(top - 2) * 64 + i for i in range(35)]
    assert step.n_free.tolist() == [2 * n - 1 - 2 * (n - 1)]


@gpu
def test_many_more_pages_wanted_than_there_are():
    """One-token pages: every request wants 2^20 of them, and there are three."""
    n, wide = 5, 2 ** 20
    table = _t(-1).repeat(n, wide)
    step = mb.paged_slots(_t(*[0] * n), _t(*[TOP] * n), table, _t(5, 6, 7), _t(3), 4, 1)
    assert step.slots.tolist() == [7, 6, 5, -1] and step.n_free.tolist() == [3 - n * wide]
