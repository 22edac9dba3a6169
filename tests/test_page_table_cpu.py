"""The host's table of pages: what sequences hold, what is free."""
import pytest
import torch


@pytest.fixture
def table(pkg):
    from cherryq_b200.pages import PageTable
    return PageTable(3, 100, 9, 16)


def check(t):
    held = [p for s in range(t.host.shape[0]) for p in t.host[s].tolist() if p >= 0]
    assert sorted(held + t.free) == list(range(t.pages))
    for s, n in enumerate(t.held):
        row = t.host[s].tolist()
        assert all(p >= 0 for p in row[:n]) and all(p == -1 for p in row[n:])


def test_pages_come_and_go(table):
    assert table.host.shape == (3, 7) and table.host.dtype == torch.int32 and (table.host == -1).all()
    assert table.reserve({0: 1, 2: 33})
    assert table.held == [1, 0, 3] and len(table.free) == 5
    check(table)
    before = table.host.clone()
    assert not table.reserve({0: 16, 2: 48}) and torch.equal(table.host, before)      # room already
    assert not table.reserve({0: 0}) and table.held[0] == 1                           # nothing is taken away
    assert table.reserve({0: 17, 1: 64})
    check(table)
    assert table.held == [2, 4, 3] and not table.free
    table.release(1)
    check(table)
    assert table.held == [2, 0, 3] and len(table.free) == 4
    table.release(1)
    check(table)


def test_all_or_nothing(table):
    table.reserve({0: 100})
    before = table.host.clone()
    with pytest.raises(ValueError, match="3 more pages are needed, 2 of 9"):
        table.reserve({1: 16, 2: 32})
    assert torch.equal(table.host, before)
    check(table)
    with pytest.raises(ValueError, match="113 slots"):
        table.reserve({1: 113})
    assert torch.equal(table.host, before)
    assert table.reserve({1: 16, 2: 16})
    check(table)


def test_sizes(pkg):
    from cherryq_b200.pages import PageTable
    for bad in ((0, 1, 1, 16), (1, 0, 1, 16), (1, 1, 0, 16), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            PageTable(*bad)
