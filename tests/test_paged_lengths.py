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


@gpu
@pytest.mark.parametrize("tokens", [0, 1, 63, 64, 65, 200, 333, 900])
@pytest.mark.parametrize("spare", [0, 30])
def test_an_output_too_short_for_its_tokens(tokens, spare):
    """The pages taken are the ones in the table, whatever the output's length."""
    kv, q = _t(0, 30, 64, 100, 5), _t(130, 40, 300, 0, 200)
    need, have = [3, 2, 6, 2, 4], [0, 1, 1, 2, 1]
    import torch
    width, pages = 7, 12 + spare
    before = torch.full((5, width), -9, dtype=torch.int32, device="cuda")
    for z in range(5):
        before[z, :have[z]] = 100 + z
    free = torch.arange(pages, dtype=torch.int32, device="cuda")
    full, cut = before.clone(), before.clone()
    whole = mb.paged_slots(kv, q, full, free, _t(pages), 670, 64)
    short = mb.paged_slots(kv, q, cut, free, _t(pages), tokens, 64)
    assert torch.equal(cut, full) and (full >= -1).sum() == sum(need)
    for name in ("cu_q", "new_len", "n_free"):
        assert torch.equal(getattr(short, name), getattr(whole, name))
    m = min(tokens, 670)
    assert torch.equal(short.slots[:m], whole.slots[:m]) and (short.slots[m:] == -1).all()
    assert torch.equal(short.positions[:m], whole.positions[:m])


@gpu
def test_a_short_output_with_many_requests():
    """Requests of several chunks of the scan, all behind the output's end."""
    import torch
    n = 2100
    kv, q = _t(*[10] * n), _t(*[100] * n)
    table = torch.full((n, 3), -9, dtype=torch.int32, device="cuda")
    table[:, 0] = 5
    step = mb.paged_slots(kv, q, table, torch.arange(n, dtype=torch.int32, device="cuda"), _t(n), 7, 64)
    assert table[:, 1].tolist() == list(range(n - 1, -1, -1)) and (table[:, 2] == -9).all()
    assert step.n_free.tolist() == [0] and step.slots.tolist() == [5 * 64 + 10 + i for i in range(7)]
