"""The paged cache where scores and values are at the ends of their types or infinite, through a cluster of CTAs and through equal ranges
whose parts a second kernel joins."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
FP16, BF16 = torch.float16, torch.bfloat16
LONG = torch.long
PAGE, SLOTS = 16, 300
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def cache_of(qc, g, KV, D, dtype):
    """SLOTS slots of one sequence: a cache, and the tables and lengths with which it is read: in a table of their own length, and with their
    pages far apart in a long one"""
    n = -(-SLOTS // PAGE)
    cache = qc.KVPages(randn(g, n, KV, PAGE, D).to(dtype), randn(g, n, KV, PAGE, D).to(dtype))
    short = torch.arange(n, device="cuda", dtype=torch.int32)[None]
    wide = torch.full((1, 40000 // PAGE), -1, dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda") * (wide.shape[1] // n)
    wide[0, at] = short[0]
    length = lambda slots: torch.tensor([slots], dtype=LONG, device="cuda")
    return cache, ((short, length(SLOTS)), (wide, length(int(at[-1]) * PAGE + SLOTS - (n - 1) * PAGE)))


def slot(x, j):
    """Slot j of all KV heads of a pool's keys or values"""
    return x[j // PAGE, :, j % PAGE]


def lost(dtype):
    """A weight in its two halves, and the few sums of these tests in 32 bits"""
    return (2.0 ** -21 if dtype == FP16 else 2.0 ** -17) + 8 * 2.0 ** -24


@pytest.mark.parametrize("dtype,big", [(FP16, 30000.0), (FP16, 3000.0), (BF16, 30000.0), (BF16, 1e17)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
def test_large_scores(qc, dtype, big, D, sign):
    """Scores of 2^24 and more, whose products are rounded to whole powers of two and coarser: one key far above the others gives its value, two
    equal ones their mean.  (The other scores are 0, or twice as far below: their weights vanish, however scores are rounded.)"""
    g, KV, G = torch.Generator(device="cuda").manual_seed(D), 2, 6
    cache, ways = cache_of(qc, g, KV, D, dtype)
    most = cache.v.abs().max().double()
    for first, second in ((0, 0), (7, 7), (299, 299), (150, 150), (3, 298), (17, 33), (64, 65)):
        q = (big * (1 + 0.3 * torch.rand(1, KV * G, D, device="cuda", generator=g))).to(dtype)
        row = (sign * big * (0.5 + 0.3 * torch.rand(KV, D, device="cuda", generator=g))).to(dtype)
        cache.k.fill_(0.0 if sign > 0 else -2 * big)
        slot(cache.k, first).copy_(row)
        slot(cache.k, second).copy_(row)
        want = (slot(cache.v, first).double() + slot(cache.v, second).double()) / 2
        want = want[:, None].expand(KV, G, D).reshape(KV * G, D)
        for table, length in ways:
            out = cache.attend(q, table, length)[0].double()
            assert bool(((out - want).abs() <= torch.finfo(dtype).eps / 2 * want.abs() + lost(dtype) * most).all()), (first, second, int(length))


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_infinite_scores(qc, dtype, D):
    """-infinity beside finite scores is a weight of 0; scores that are all -infinity have no softmax: NaN, as infinity; no slot at all gives zeros"""
    g, KV, G = torch.Generator(device="cuda").manual_seed(D + 1), 2, 4
    cache, ways = cache_of(qc, g, KV, D, dtype)
    q = randn(g, 1, KV * G, D).to(dtype)
    q[..., 0] = q[..., 0].abs() + 0.5
    q[:, 1::2, 0] *= -1                                  # every second head sees -infinity where the others see infinity
    finite = cache.k.clone()
    cache.k[..., 0] = -INF
    for table, length in ways:
        assert cache.attend(q, table, length).isnan().all()
        one = table.clone()
        one[0, 1:] = -1
        for n in (1, 5, 16, int(length)):                # a single slot, or a page's, and absent pages
            assert cache.attend(q, one, torch.tensor([n], device="cuda")).isnan().all()
        assert not cache.attend(q, torch.full_like(table, -1), length).any() and not cache.attend(q, table, length * 0).any()
    # a finite score in one place alone: of the heads that see -infinity elsewhere it has all of the weight
    for j in (0, 50, 299):
        cache.k.copy_(finite)
        cache.k[..., 0] = -INF
        slot(cache.k, j).copy_(slot(finite, j))
        for table, length in ways:
            out = cache.attend(q, table, length).view(KV, G, D)
            assert bool(((out[:, ::2].double() - slot(cache.v, j)[:, None].double()).abs() <= lost(dtype) * cache.v.abs().max().double()).all())
            assert out[:, 1::2].isnan().all()
    # a step whose own row is all that there is
    k, v = slot(cache.k, 7)[None].clone(), randn(g, 1, KV, D).to(dtype)
    for table, _ in ways:
        out = cache.step(q, k, v, None, None, None, table, torch.zeros(1, dtype=LONG, device="cuda"))
        assert out.isnan().all()


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("below", [1, 30, 100, 120, 130, 140, 148, 200, 3000])
def test_infinite_values_of_small_weights(qc, dtype, D, below):
    """A weight is not 0 however far its score, here 2^-below of the largest, lies below the others: an infinite value is infinite in its
    column, NaN where it meets the other infinity or a NaN, or where its score is -infinity; the other columns are what they are without it"""
    g, KV, G = torch.Generator(device="cuda").manual_seed(below), 2, 4
    cache, ways = cache_of(qc, g, KV, D, dtype)
    q = torch.zeros(1, KV * G, D, device="cuda", dtype=dtype)
    q[..., 0] = 8.0
    scale = math.log(2.0) / 8.0                          # the key's first column is its score in powers of two
    cache.k.zero_()
    for j in range(SLOTS):
        slot(cache.k, j)[:, 0] = -float(below)
    for top in (0, 123, 299):
        slot(cache.k, top)[:, 0] = 0.0
        clean = [cache.attend(q, table, length, scale=scale)[0] for table, length in ways]
        v = cache.v.clone()
        for low in (1, 20, 63, 64, 150, 200, 298):
            slot(cache.v, low)[:, 5] = INF
            slot(cache.v, low)[:, D - 1] = -INF
            slot(cache.v, low)[:, 9] = NAN
            slot(cache.v, low)[:, 10] = INF
            slot(cache.v, (low + 7) % 299 + (top == (low + 7) % 299))[:, 10] = -INF
            slot(cache.k, low)[:, 1] = 0.0
            for (table, length), whole in zip(ways, clean):
                out = cache.attend(q, table, length, scale=scale)[0]
                assert (out[:, 5] == INF).all() and (out[:, D - 1] == -INF).all() and out[:, 9].isnan().all() and out[:, 10].isnan().all(), (top, low)
                rest = [c for c in range(D) if c not in (5, 9, 10, D - 1)]
                assert torch.equal(out[:, rest], whole[:, rest]), (top, low)
            # a score of -infinity: 0 times infinity
            held = slot(cache.k, low).clone()
            slot(cache.k, low)[:, 0] = -INF
            for table, length in ways:
                out = cache.attend(q, table, length, scale=scale)[0]
                assert out[:, [5, 9, 10, D - 1]].isnan().all() and torch.isfinite(out[:, rest]).all()
            slot(cache.k, low).copy_(held)
            cache.v.copy_(v)
        slot(cache.k, top)[:, 0] = -float(below)


def test_infinite_values_of_long_sequences(qc):
    """One in each of two long sequences, of many tiles a CTA"""
    g, KV, H, D = torch.Generator(device="cuda").manual_seed(5), 1, 8, 128
    n = 20000
    cache = qc.KVPages(randn(g, 2 * n // 64 + 2, KV, 64, D).half(), randn(g, 2 * n // 64 + 2, KV, 64, D).half())
    table = torch.randperm(cache.pages, device="cuda", generator=g)[:2 * (n // 64 + 1)].view(2, -1).to(torch.int32)
    q, length = randn(g, 2, H, D).half(), torch.tensor([n, n - 7000], device="cuda")
    clean = cache.attend(q, table, length)
    cache.v[table[0, 100].long(), 0, 3, 17] = INF
    cache.v[table[1, 200].long(), 0, 63, 100] = -INF
    out = cache.attend(q, table, length)
    assert (out[0, :, 17] == INF).all() and (out[1, :, 100] == -INF).all()
    out[0, :, 17], out[1, :, 100] = clean[0, :, 17], clean[1, :, 100]
    assert torch.equal(out, clean)
