"""The paged cache where numbers of rows and heads are at the ends of 32 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def test_as_many_rows_as_are_taken(qc):
    """2^31 - 1 rows, one row of memory for all: the last two belong to a sequence"""
    cache = qc.KVPages.empty(2, 1, 16, 64)
    table = torch.tensor([[1]], dtype=torch.int32, device="cuda")
    n = 2 ** 31 - 1
    row = torch.arange(64, dtype=torch.half, device="cuda").view(1, 1, 64)
    cache.write(None, row.expand(n, -1, -1), (-row).expand(n, -1, -1), table, torch.tensor([3], device="cuda"), starts=torch.tensor([n - 2, n], device="cuda"))
    want = torch.zeros_like(cache.k)
    want[1, 0, 3:5] = row
    assert torch.equal(cache.k, want) and torch.equal(cache.v, -want)


def test_more_heads_than_a_number_holds(qc):
    cache = qc.KVPages.empty(2, 2, 16, 64)
    table, one = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
    row = torch.zeros(1, 1, 64, dtype=torch.half, device="cuda")
    for heads in (2 ** 31, 2 ** 32 + 2, 2 ** 17):
        q = row.expand(1, heads, 64)
        with pytest.raises(RuntimeError):
            cache.write(q, row.expand(1, 2, 64), row.expand(1, 2, 64), table, one)
