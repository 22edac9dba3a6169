"""The paged KV cache against plain 64-bit forms: writing, reading, attention of single tokens, steps.

Tolerance of attention, relative to the largest visible value of a sequence: the result is rounded to its type (eps / 2); a weight is kept
in two numbers of the type, 2^-21 of it lost in fp16 and 2^-17 in bf16; a score is a sum of D products in 32 bits, cut off at most
(D + 8) * 2^-23 of the products' magnitudes, which moves weights by twice that; sums over n slots take n / 16 + 32 additions in 32 bits, of
2^-24 each, of weights and of weighted values."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

FP16, BF16 = torch.float16, torch.bfloat16
LONG = torch.long


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def longs(*n):
    return torch.tensor(n, dtype=LONG, device="cuda")


def pool(qc, g, n, KV, page, D, dtype, scale=1.0):
    return qc.KVPages((randn(g, n, KV, page, D) * scale).to(dtype), (randn(g, n, KV, page, D) * scale).to(dtype))


def tables(g, B, width, n, spare=0):
    """Pages in any order, each once; the last `spare` columns of other sequences than the first have none"""
    t = torch.randperm(n, device="cuda", generator=g)[:B * width].view(B, width).to(torch.int32)
    if spare:
        t[1:, width - spare:] = -1
    return t


def seen_slots(table, page, pages, n, window, sinks):
    """Visible slots of one sequence, as (page, slot of the page)"""
    n = min(max(n, 0), len(table) * page)
    at = [j for j in range(n) if not window or j < sinks or j >= n - window]
    entries = table.tolist()
    at = [(entries[j // page], j % page) for j in at]
    return [(p, j) for p, j in at if 0 <= p < pages]


def attend_ref(cache, q, table, lengths, window=0, sinks=0, scale=None):
    """(out in 64 bits, tolerance per sequence)"""
    B, H, D = q.shape
    KV, scale = cache.n_kv_heads, scale or 1.0 / math.sqrt(D)
    out, tol = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.zeros(B, 1, 1, dtype=torch.float64, device="cuda")
    eps = torch.finfo(q.dtype).eps
    for b, n in enumerate(lengths):
        at = seen_slots(table[b], cache.page_size, cache.pages, n, window, sinks)
        if not at:
            continue
        pg, j = torch.tensor(at, device="cuda").T
        k, v = cache.k[pg, :, j].double(), cache.v[pg, :, j].double()
        qb = q[b].double().view(KV, H // KV, D)
        s = torch.einsum("kgd,skd->kgs", qb, k) * scale
        big = float(torch.einsum("kgd,skd->kgs", qb.abs(), k.abs()).max()) * scale
        out[b] = torch.einsum("kgs,skd->kgd", torch.softmax(s, -1), v).reshape(H, D)
        lost = (2.0 ** -21 if q.dtype == FP16 else 2.0 ** -17) + 2 * (D + 8) * 2.0 ** -23 * big + 2 * (len(at) / 16 + 32) * 2.0 ** -24
        tol[b] = float(v.abs().max()) * (eps / 2 + lost)
    return out, tol


def close(got, want, tol):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), (float((err - tol).max()), float(err.max()))


def rotated(x, cos, sin, pos):
    """Rows rotated at their positions, in 32 bits, each operation rounded; rows without one as they are"""
    there = (pos >= 0) & (pos < len(cos))
    p = torch.where(there, pos, 0)
    c, s = cos[p][:, None], sin[p][:, None]
    a, b = x.float().chunk(2, -1)
    return torch.where(there[:, None, None], torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype), x)


def rope(n, D):
    ang = torch.outer(torch.arange(n, device="cuda", dtype=torch.float32), 1.0 / 10000 ** (torch.arange(0, D, 2, device="cuda") / D))
    return ang.cos(), ang.sin()


# ---------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("H,KV,D,page,lengths,window,sinks", [
    (4, 4, 128, 16, (1,), 0, 0),
    (4, 4, 64, 16, (15, 16, 17), 0, 0),
    (8, 1, 128, 16, (0, 1, 63, 64, 65), 0, 0),
    (16, 2, 64, 32, (200, 0, 77, 333), 0, 0),
    (5, 1, 128, 64, (129, 511), 0, 0),
    (12, 1, 128, 32, (100, 1000), 0, 0),                  # more heads than a tile of queries holds
    (34, 2, 64, 128, (257, 31), 0, 0),
    (6, 2, 128, 256, (1500, 256, 255), 0, 0),
    (32, 32, 128, 16, (257,), 0, 0),
    (8, 8, 128, 64, (4001, 2000, 5), 0, 0),
    (64, 8, 128, 64, (3000, 17), 0, 0),
    (4, 2, 128, 16, (500, 100, 3), 37, 0),
    (4, 2, 64, 16, (500, 100, 3), 37, 5),
    (8, 2, 128, 64, (1000, 90, 70), 64, 64),
    (8, 2, 128, 64, (1000, 90, 70), 1, 1),
    (8, 2, 64, 256, (3000, 600), 1021, 4),
    (4, 1, 128, 16, (700, 20), 30, 700),                   # more sinks than slots
    (4, 1, 128, 32, (100, 33), 2 ** 31 - 1, 2 ** 31 - 1),
    (4, 2, 128, 16, (90000,), 0, 0),
    (3, 3, 64, 16, (30000, 29), 25000, 100),
])
def test_attend(qc, dtype, H, KV, D, page, lengths, window, sinks):
    g, B = gen(H * D + page), len(lengths)
    width = max(1, -(-max(lengths) // page)) + 1
    cache = pool(qc, g, B * width + 2, KV, page, D, dtype)
    table = tables(g, B, width, B * width + 2)
    q = randn(g, B, H, D).to(dtype)
    out = cache.attend(q, table, longs(*lengths), window=window, sinks=sinks)
    assert out.dtype == dtype and out.shape == q.shape
    want, tol = attend_ref(cache, q, table, lengths, window, sinks)
    close(out, want, tol)
    for b, n in enumerate(lengths):
        if n == 0:
            assert not out[b].any()
    # the same bits again
    assert torch.equal(out, cache.attend(q, table, longs(*lengths), window=window, sinks=sinks))


@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_what_a_mask_hides_may_be_anything(qc, dtype, page):
    """NaN and infinite rows behind a length, outside a window, in pages that no table names; absent pages"""
    g, D, KV, H, n = gen(3), 128, 2, 8, 6 * page + page // 2 + 3
    width = 10
    cache = pool(qc, g, 2 * width + 4, KV, page, D, dtype)
    table = tables(g, 2, width, 2 * width)
    clean = qc.KVPages(cache.k.clone(), cache.v.clone())
    window, sinks = 2 * page + 5, 3
    bad = (float("nan"), float("inf"), -float("inf"))
    for b in range(2):
        for j in list(range(sinks, n - window)) + list(range(n, width * page)):
            pg = int(table[b, j // page])
            cache.k[pg, :, j % page] = bad[j % 3]
            cache.v[pg, :, j % page] = bad[(j + 1) % 3]
    cache.k[2 * width:] = float("nan")
    q = randn(g, 2, H, D).to(dtype)
    out = cache.attend(q, table, longs(n, n), window=window, sinks=sinks)
    assert torch.equal(out, clean.attend(q, table, longs(n, n), window=window, sinks=sinks))
    close(out, *attend_ref(clean, q, table, (n, n), window, sinks))


@pytest.mark.parametrize("page", [16, 32, 128])
def test_entries_outside_the_pool(qc, page):
    """Slots of absent pages are not seen, wherever they stand; a sequence of none gets zeros"""
    g, D, KV, H = gen(4), 64, 2, 6
    cache = pool(qc, g, 40, KV, page, D, FP16)
    table = tables(g, 4, 8, 40)
    table[0, 1], table[0, 4], table[0, 7] = -1, 40, 2 ** 31 - 1
    table[1] = -5
    table[2, 0] = -2 ** 31
    table[3, 5:] = 10 ** 6
    lengths = (7 * page + 3, 8 * page, page + 1, 8 * page)
    q = randn(g, 4, H, D).half()
    for window, sinks in ((0, 0), (page + 3, 2)):
        out = cache.attend(q, table, longs(*lengths), window=window, sinks=sinks)
        close(out, *attend_ref(cache, q, table, lengths, window, sinks))
        assert not out[1].any()


def test_lengths_beyond_the_table(qc):
    g = gen(5)
    cache = pool(qc, g, 9, 1, 16, 64, BF16)
    table = tables(g, 4, 2, 9)
    q = randn(g, 4, 2, 64).bfloat16()
    lengths = (33, 2 ** 62, -1, -2 ** 63)
    close(cache.attend(q, table, longs(*lengths)), *attend_ref(cache, q, table, lengths))


def test_shared_pages(qc):
    """A prefix that all sequences share, and a page twice in a table"""
    g = gen(6)
    cache = pool(qc, g, 30, 2, 32, 128, FP16)
    table = tables(g, 3, 6, 30)
    table[:, :3] = table[0, :3]
    table[2, 4] = table[2, 3]
    q = randn(g, 3, 8, 128).half()
    close(cache.attend(q, table, longs(192, 150, 170)), *attend_ref(cache, q, table, (192, 150, 170)))


def test_strides(qc):
    """Queries with heads in front of tokens, from a wider projection, one for all sequences; a table inside a wider one"""
    g = gen(7)
    cache = pool(qc, g, 40, 2, 16, 64, FP16)
    wide = tables(g, 4, 10, 40)
    table, n = wide[:, 2:9], longs(100, 3, 112, 50)
    lengths = n.tolist()
    by_head = randn(g, 8, 4, 64).half().transpose(0, 1)
    fused = randn(g, 4, 12, 72).half()[:, 4:, 8:]
    one = randn(g, 1, 8, 64).half().expand(4, -1, -1)
    for q in (by_head, fused, one):
        out = cache.attend(q, table, n)
        assert out.is_contiguous()
        close(out, *attend_ref(cache, q, table, lengths))


def test_scores_far_apart(qc):
    """Large scores: no overflow on the way, and the weights of what is far below the largest vanish"""
    g = gen(8)
    for dtype, scale in ((FP16, 60.0), (BF16, 1e4)):
        cache = pool(qc, g, 12, 2, 64, 128, dtype, scale)
        table = tables(g, 1, 12, 12)
        q = (randn(g, 1, 4, 128) * scale).to(dtype)
        out = cache.attend(q, table, longs(700))
        assert torch.isfinite(out).all()
        top = cache.v[table[0].long()].abs().max()
        assert out.abs().max() <= top
    # values at the type's end stay finite
    cache = qc.KVPages(torch.zeros(4, 1, 16, 64, device="cuda", dtype=FP16), torch.full((4, 1, 16, 64), 65504.0, device="cuda", dtype=FP16))
    out = cache.attend(randn(g, 1, 4, 64).half(), tables(g, 1, 4, 4), longs(64))
    assert (out == 65504).all()


def test_visible_infinities(qc):
    """A visible infinite value makes its column infinite, NaN only that column; a NaN key its head's outputs"""
    g = gen(9)
    cache = pool(qc, g, 40, 2, 16, 64, FP16, 0.5)
    table = tables(g, 1, 40, 40)
    at = table[0].long()
    cache.v[at[2], 0, 3, 5] = float("inf")
    cache.v[at[30], 0, 1, 7] = -float("inf")
    cache.v[at[35], 1, 1, 9] = float("nan")
    q = randn(g, 1, 8, 64).half()
    out = cache.attend(q, table, longs(635))[0]
    assert (out[:4, 5] == float("inf")).all() and (out[:4, 7] == -float("inf")).all() and out[4:, 9].isnan().all()
    rest = torch.ones_like(out, dtype=torch.bool)
    rest[:4, 5] = rest[:4, 7] = rest[4:, 9] = False
    assert torch.isfinite(out[rest]).all()
    cache.k[at[20], 1, 0, 3] = float("nan")
    out = cache.attend(q, table, longs(635))[0]
    assert out[4:].isnan().all() and torch.isfinite(out[:4][rest[:4]]).all()


def test_offsets_beyond_32_bits(qc):
    """A pool of more than 2^32 bytes and 2^31 values"""
    pages, KV, page, D = 2 ** 31 // (8 * 256 * 128) + 40, 8, 256, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    k = torch.zeros(pages, KV, page, D, dtype=FP16, device="cuda")
    v = torch.zeros_like(k)
    cache, g = qc.KVPages(k, v), gen(10)
    table = torch.tensor([[pages - 1, 0, pages - 2], [5, pages - 3, 1]], dtype=torch.int32, device="cuda")
    T = 600
    rows = lambda: randn(g, 2 * T, KV, D).half()
    kn, vn = rows(), rows()
    cache.write(None, kn, vn, table, longs(0, 0))
    q = randn(g, 2, 16, D).half()
    close(cache.attend(q, table, longs(T, T - 1)), *attend_ref(cache, q, table, (T, T - 1)))
    got = cache.read(table, longs(0, 0), T)
    assert torch.equal(got[0].flatten(0, 1), kn) and torch.equal(got[1].flatten(0, 1), vn)
    assert int((k != 0).any(-1).any(-1).any(-1).sum()) == 6


# ---------------------------------------------------------------------------------- writing and reading
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("page,counts,firsts", [
    (16, (1,), (0,)), (16, (5, 0, 17, 40), (3, 9, 15, 0)), (64, (100, 1, 64), (60, 0, 64)), (256, (0, 300, 0, 0, 7), (1, 250, 2, 3, 255)),
    (32, (0, 0), (0, 5)),
])
def test_write_packed(qc, dtype, D, turn, page, counts, firsts):
    g, B, KV, H = gen(page + D), len(counts), 3, 6
    width = max(f + n for f, n in zip(firsts, counts)) // page + 2
    cache = pool(qc, g, B * width + 3, KV, page, D, dtype)
    table = tables(g, B, width, B * width + 3)
    before, behind = 2, 5                                    # rows of no sequence
    rows = before + sum(counts) + behind
    q, k, v = (randn(g, rows, n, D).to(dtype) for n in (H, KV, KV))
    starts = longs(before, *(before + sum(counts[:i + 1]) for i in range(B)))
    cos, sin = rope(width * page, D)
    pos = torch.randint(0, width * page, (rows,), device="cuda", generator=g)
    if sum(counts) > 3:
        pos[before + 1], pos[before + 2] = -1, width * page                    # no position: not written
    want_k, want_v = cache.k.clone(), cache.v.clone()
    kr = rotated(k, cos, sin, pos) if turn else k
    for b in range(B):
        for i in range(counts[b]):
            t, slot = before + sum(counts[:b]) + i, firsts[b] + i
            if turn and not 0 <= int(pos[t]) < len(cos):
                continue
            want_k[int(table[b, slot // page]), :, slot % page] = kr[t]
            want_v[int(table[b, slot // page]), :, slot % page] = v[t]
    args = (cos, sin, pos) if turn else (None, None, None)
    out = cache.write(q, k, v, table, longs(*firsts), *args, starts=starts)
    assert torch.equal(out, rotated(q, cos, sin, pos) if turn else q)
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)
    assert cache.write(None, k, v, table, longs(*firsts), *args, starts=starts) is None
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


def test_write_many_sequences(qc):
    """More sequences than rows of a block, one to three rows each, as single tokens and as packed ones"""
    g, B, KV, D, page = gen(20), 700, 2, 64, 16
    cache = pool(qc, g, B + 1, KV, page, D, BF16)
    table = tables(g, B, 1, B + 1)
    counts = torch.randint(0, 4, (B,), device="cuda", generator=g)
    starts = torch.cat([longs(0), counts.cumsum(0)])
    rows = int(starts[-1])
    k, v = randn(g, rows, KV, D).bfloat16(), randn(g, rows, KV, D).bfloat16()
    first = torch.randint(0, page + 1, (B,), device="cuda", generator=g)       # some rows beyond the table's end
    owner = torch.repeat_interleave(torch.arange(B, device="cuda"), counts)
    slot = first[owner] + torch.arange(rows, device="cuda") - starts[owner]
    fits = slot < page
    want_k, want_v = cache.k.clone(), cache.v.clone()
    at = (table[owner[fits], 0].long(), slice(None), slot[fits])
    want_k[at], want_v[at] = k[fits], v[fits]
    cache.write(None, k, v, table, first, starts=starts)
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v)


def test_write_outside(qc):
    """Rows without a slot or a page go nowhere: negative and huge first slots, absent pages, starts out of any order"""
    g, KV, D, page = gen(21), 2, 128, 16
    cache = pool(qc, g, 8, KV, page, D, FP16)
    table = torch.tensor([[0, -1, 1], [7, 8, 2 ** 31 - 1], [-2 ** 31, 3, 4], [5, 5, 6]], dtype=torch.int32, device="cuda")
    k, v = randn(g, 200, KV, D).half(), randn(g, 200, KV, D).half()
    before = cache.k.clone(), cache.v.clone()
    for first in ((-100, 2 ** 62, -2 ** 63, 48), (16, 16, 0, 2 ** 31), (17, 20, -17, 10 ** 12)):
        cache.write(None, k[:4], v[:4], table, longs(*first))
        assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1]), first
    cache.write(None, k[:48], v[:48], table, longs(10, 2 ** 63 - 1, -5, -2 ** 63))     # 12 rows each: some inside
    want = before[0].clone()
    want[0, :, 10:] = k[:6].transpose(0, 1)
    assert torch.equal(cache.k, want)
    for starts in ((200, 100, 50, 20, 0), (-5, -4, 300, 2, 400), (2 ** 62, 0, 0, 0, 1), (0, 0, 0, 0, 0)):
        cache.write(None, k, v, table, longs(0, 0, 0, 0), starts=longs(*starts))       # whatever is written, it is in the pool
    torch.cuda.synchronize()


def test_write_equal_shares_and_strides(qc):
    g, B, T, KV, H, D, page = gen(22), 3, 9, 2, 4, 64, 16
    cache = pool(qc, g, 10, KV, page, D, FP16)
    table = tables(g, B, 2, 10)
    fused = randn(g, B * T, H + 2 * KV, D).half()
    q, k, v = fused.split((H, KV, KV), 1)
    cos, sin = rope(40, D)
    pos = torch.arange(5, 5 + T, device="cuda").repeat(B)
    out = cache.write(q, k, v, table, longs(5, 0, 23), cos, sin, pos)
    assert torch.equal(out, rotated(q, cos, sin, pos))
    got_k, got_v = cache.read(table, longs(5, 0, 23), T)
    assert torch.equal(got_k, rotated(k, cos, sin, pos).view(B, T, KV, D)) and torch.equal(got_v, v.reshape(B, T, KV, D))
    # one value row for all tokens; tables that start on any 4 bytes
    one = randn(g, 1, KV, D).half().expand(B * T, -1, -1)
    odd = torch.empty(40 * D // 2 + 1, device="cuda")[1:].view(40, D // 2).copy_(cos)
    cache.write(None, k, one, table, longs(5, 0, 23), odd, sin, pos)
    got = cache.read(table, longs(5, 0, 23), T)
    assert torch.equal(got[0], got_k) and torch.equal(got[1], one.reshape(B, T, KV, D))


@pytest.mark.parametrize("dtype,D", [(FP16, 128), (BF16, 64)])
def test_read(qc, dtype, D):
    g, KV, page = gen(23), 5, 32
    cache = pool(qc, g, 12, KV, page, D, dtype)
    table = tables(g, 3, 4, 12)
    table[1, 1], table[2, 0] = -1, 12
    for first, count in (((0, 0, 0), 128), ((-5, 100, 31), 77), ((2 ** 62, -2 ** 63, 127), 1), ((3, 64, 1), 33)):
        k, v = cache.read(table, longs(*first), count)
        assert k.shape == v.shape == (3, count, KV, D)
        for b in range(3):
            for i in range(count):
                slot = first[b] + i
                p = int(table[b, slot // page]) if 0 <= slot < 128 else -1
                want = (cache.k[p, :, slot % page], cache.v[p, :, slot % page]) if 0 <= p < 12 else (torch.zeros(KV, D, device="cuda", dtype=dtype),) * 2
                assert torch.equal(k[b, i], want[0]) and torch.equal(v[b, i], want[1]), (b, i)


# ---------------------------------------------------------------------------------- long tables: equal ranges of all tiles, joined
def long_table(qc, D, H, KV, B, page, width, dtype, seed):
    """A small pool for a long table (pages in several places), a page of its own where each sequence's next row goes"""
    g = gen(seed)
    lengths = (torch.rand(B, device="cuda", generator=g) ** 6 * (width * page - 1)).long()
    lengths[0] = width * page - 10
    if B > 2:
        lengths[B // 2], lengths[B - 1] = 0, -3
    n = 3 * width // 4
    cache = pool(qc, g, n + B, KV, page, D, dtype)
    table = torch.randint(0, n, (B, width), device="cuda", generator=g).to(torch.int32)
    at = torch.arange(B, device="cuda")
    table[at, (lengths.clamp(min=0) // page)] = (n + at).to(torch.int32)
    return g, cache, table, lengths, randn(g, B, H, D).to(dtype)


LONG_TABLES = [
    (128, 10, 2, 1, 64, 500, FP16),            # few heads, many parts of each
    (128, 8, 8, 2, 16, 1200, BF16),
    (64, 3, 1, 40, 64, 300, FP16),
    (128, 24, 2, 33, 32, 300, BF16),           # two tiles of queries a head
    (64, 2, 1, 600, 16, 400, FP16),            # more heads than ranges
    (64, 4, 4, 260, 16, 400, BF16),
]


@pytest.mark.parametrize("D,H,KV,B,page,width,dtype", LONG_TABLES)
def test_long_tables(qc, D, H, KV, B, page, width, dtype):
    g, cache, table, lengths, q = long_table(qc, D, H, KV, B, page, width, dtype, D + B)
    out = cache.attend(q, table, lengths)
    close(out, *attend_ref(cache, q, table, lengths.tolist()))
    assert not out[lengths <= 0].any()
    k, v = (randn(g, B, KV, D).to(dtype) for _ in range(2))
    before = cache.k.clone()
    out = cache.step(q, k, v, None, None, None, table, lengths)
    close(out, *attend_ref(cache, q, table, [n + 1 if n >= 0 else 0 for n in lengths.tolist()]))
    there = lengths >= 0
    before[table[torch.arange(B, device="cuda"), lengths.clamp(min=0) // page][there].long(), :, (lengths % page)[there]] = k[there]
    assert torch.equal(cache.k, before)


@pytest.mark.parametrize("case", LONG_TABLES[::2])
def test_long_tables_whose_lengths_change(qc, case):
    """The second kernel looks at lengths while the first one runs, not while what wrote them does"""
    g, cache, table, lengths, q = long_table(qc, *case, 7)
    far = torch.full((1 << 22,), 1.0, device="cuda")
    ends = [lengths, lengths.flip(0), lengths // 3, torch.zeros_like(lengths), lengths]
    want = [cache.attend(q, table, n) for n in ends]
    torch.cuda.synchronize()
    now, outs = lengths.clone(), []

    def run():
        outs.clear()
        for n in ends:
            far.mul_(1.0)
            now.copy_(n)
            outs.append(cache.attend(q, table, now))
    run()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        run()
    for _ in range(10):
        for x in outs:
            x.fill_(float("nan"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


# ---------------------------------------------------------------------------------- steps
@pytest.mark.parametrize("dtype", [FP16, BF16])
@pytest.mark.parametrize("turn", [False, True])
@pytest.mark.parametrize("H,KV,D,page,lengths,window,sinks", [
    (4, 4, 128, 16, (0,), 0, 0),
    (8, 2, 64, 16, (0, 15, 16, 31, 200), 0, 0),
    (8, 1, 128, 64, (63, 64, 65, 500), 0, 0),
    (18, 1, 128, 32, (70, 1000), 0, 0),
    (8, 8, 128, 256, (3000, 255, 256), 0, 0),
    (4, 2, 64, 16, (300, 20), 33, 3),
    (4, 2, 128, 128, (1000, 20, 127), 1, 0),
    (32, 32, 128, 16, (256,), 0, 0),
    (64, 8, 128, 64, (2500,), 700, 4),
])
def test_step(qc, dtype, turn, H, KV, D, page, lengths, window, sinks):
    g, B = gen(H + D + page), len(lengths)
    width = max(lengths) // page + 1
    cache = pool(qc, g, B * width + 2, KV, page, D, dtype)
    table = tables(g, B, width, B * width + 2)
    q, k, v = (randn(g, B, n, D).to(dtype) for n in (H, KV, KV))
    cos, sin = rope(max(lengths) + 10, D)
    pos = longs(*lengths) + 3
    args = (cos, sin, pos) if turn else (None, None, None)
    want_k, want_v, q_before = cache.k.clone(), cache.v.clone(), q.clone()
    kr = rotated(k, cos, sin, pos) if turn else k
    for b, n in enumerate(lengths):
        want_k[int(table[b, n // page]), :, n % page] = kr[b]
        want_v[int(table[b, n // page]), :, n % page] = v[b]
    out = cache.step(q, k, v, *args, table, longs(*lengths), window=window, sinks=sinks)
    assert torch.equal(cache.k, want_k) and torch.equal(cache.v, want_v) and torch.equal(q, q_before)
    qr = rotated(q, cos, sin, pos) if turn else q
    close(out, *attend_ref(cache, qr, table, [n + 1 for n in lengths], window, sinks))
    # what write and attend give
    assert torch.equal(out, cache.attend(qr, table, longs(*lengths) + 1, window=window, sinks=sinks))


def test_step_outside(qc):
    """Rows that cannot be written: no position, no page, a full table, a negative length"""
    g, KV, H, D, page = gen(31), 2, 4, 64, 16
    cache = pool(qc, g, 20, KV, page, D, FP16)
    table = tables(g, 6, 3, 20)
    table[1, 1:] = -1
    table[2, 1] = 20
    lengths = (20, 16, 20, 48, -1, 2 ** 62)
    q, k, v = (randn(g, 6, n, D).half() for n in (H, KV, KV))
    cos, sin = rope(30, D)
    pos = longs(30, 16, 20, 7, 3, 9)                              # the first has no position
    before = cache.k.clone(), cache.v.clone()
    out = cache.step(q, k, v, cos, sin, pos, table, longs(*lengths))
    assert torch.equal(cache.k, before[0]) and torch.equal(cache.v, before[1])
    seen = [min(n + 1, 48) if n >= 0 else 0 for n in lengths]
    close(out, *attend_ref(cache, rotated(q, cos, sin, pos), table, seen))
    assert not out[4].any()
    # a NaN that the slot held is not seen once the step has written it
    cache.k[table[0, 1].long(), :, 4] = float("nan")
    cache.v[table[0, 1].long(), :, 4] = float("nan")
    pos[0] = 20
    out = cache.step(q, k, v, cos, sin, pos, table, longs(*lengths))
    close(out[:1], *attend_ref(cache, rotated(q, cos, sin, pos)[:1], table[:1], (21,)))


def test_step_infinite_row(qc):
    """The step's own value is infinite: seen as any other"""
    g = gen(32)
    cache = pool(qc, g, 4, 1, 16, 64, FP16)
    table = tables(g, 1, 4, 4)
    q, k, v = (randn(g, 1, n, 64).half() for n in (12, 1, 1))
    v[0, 0, 3] = float("inf")
    out = cache.step(q, k, v, None, None, None, table, longs(40))
    assert (out[0, :, 3] == float("inf")).all() and torch.isfinite(out[0, :, 4:]).all()


def test_sequence_grows(qc):
    """Prompts of different lengths, then steps through page after page, against the same tokens at once"""
    g, B, KV, H, D, page = gen(33), 3, 2, 8, 64, 16
    counts, more = (30, 1, 47), 40
    width = 6
    cache = qc.KVPages.empty(B * width, KV, page, D)
    assert cache.k.dtype == FP16 and cache.page_size == page and cache.pages == B * width and cache.n_kv_heads == KV and cache.head_dim == D
    table = tables(g, B, width, B * width)
    cos, sin = rope(200, D)
    new = lambda rows: [randn(g, rows, n, D).half() for n in (H, KV, KV)]
    _, k0, v0 = new(sum(counts))
    starts = longs(0, 30, 31, 78)
    pos = torch.cat([torch.arange(n, device="cuda") for n in counts])
    cache.write(None, k0, v0, table, longs(0, 0, 0), cos, sin, pos, starts)
    kept = [[rotated(k0[a:b], cos, sin, pos[a:b])] for a, b in ((0, 30), (30, 31), (31, 78))]
    length = longs(*counts)
    for _ in range(more):
        q, k, v = new(B)
        out = cache.step(q, k, v, cos, sin, length, table, length)
        kr = rotated(k, cos, sin, length)
        for b in range(B):
            kept[b].append(kr[b:b + 1])
        length += 1
    close(out, *attend_ref(cache, rotated(q, cos, sin, length - 1), table, length.tolist()))
    k, _ = cache.read(table, longs(0, 0, 0), 87)
    for b, n in enumerate(length.tolist()):
        assert torch.equal(k[b, :n], torch.cat(kept[b]))


# ---------------------------------------------------------------------------------- streams, graphs, refusals
def test_graphs_and_streams(qc):
    """A captured step follows lengths and tables; two graphs and eager calls in between keep apart"""
    g, B, KV, H, D, page = gen(34), 2, 2, 16, 128, 16
    cache = pool(qc, g, 300, KV, page, D, BF16)
    twin = qc.KVPages(cache.k.clone(), cache.v.clone())
    table = tables(g, B, 128, 300)
    cos, sin = rope(2048, D)
    q, k, v = (randn(g, B, n, D).bfloat16() for n in (H, KV, KV))
    length = longs(3, 1000)
    stream, graphs = torch.cuda.Stream(), []
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for window in (0, 100):
            cache.step(q, k, v, cos, sin, length, table, length, window=window)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                out = cache.step(q, k, v, cos, sin, length, table, length, window=window)
            graphs.append((graph, out, window))
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    cache.k.copy_(twin.k), cache.v.copy_(twin.v)
    for i in range(6):
        length.copy_(longs(i * 7, 2040 + i - 5))
        q.copy_(randn(g, B, H, D))
        table[0, 0] = 250 + i
        graph, out, window = graphs[i % 2]
        want = twin.step(q, k, v, cos, sin, length, table, length, window=window)
        graph.replay()
        assert torch.equal(out, want)
    assert torch.equal(cache.k, twin.k) and torch.equal(cache.v, twin.v)


def test_grad_inputs_are_taken(qc):
    g = gen(35)
    cache = pool(qc, g, 4, 1, 16, 64, FP16)
    q = randn(g, 1, 2, 64).half().requires_grad_()
    assert not cache.attend(q, tables(g, 1, 4, 4), longs(20)).requires_grad


def test_refusals(qc):
    z = lambda *s, dtype=FP16: torch.zeros(*s, dtype=dtype, device="cuda")
    for k, v in ((z(4, 2, 16, 64), z(4, 2, 16, 128)), (z(4, 2, 16, 64), z(4, 2, 16, 64, dtype=BF16)), (z(4, 2, 16, 96), z(4, 2, 16, 96)),
                 (z(4, 2, 24, 64), z(4, 2, 24, 64)), (z(4, 2, 8, 64), z(4, 2, 8, 64)), (z(4, 2, 512, 64), z(4, 2, 512, 64)),
                 (z(4, 2, 16, 64, dtype=torch.float32),) * 2, (z(0, 2, 16, 64), z(0, 2, 16, 64)), (z(4, 16, 2, 64).transpose(1, 2),) * 2,
                 (z(4, 2, 16, 64).cpu(), z(4, 2, 16, 64).cpu()), (z(2, 16, 64), z(2, 16, 64)), (z(1 + 4 * 2048)[1:].view(4, 2, 16, 64), z(4, 2, 16, 64))):
        with pytest.raises(RuntimeError):
            qc.KVPages(k, v)
    both = z(8, 2, 16, 64)
    with pytest.raises(RuntimeError):
        qc.KVPages(both, both)
    with pytest.raises(RuntimeError):
        qc.KVPages.empty(4, 2, 16, 64, torch.float32)
    with pytest.raises(RuntimeError):
        qc.KVPages.empty(0, 2, 16, 64)
    c = qc.KVPages.empty(8, 2, 16, 64)
    t, n, q, k = z(3, 4, dtype=torch.int32), z(3, dtype=LONG), z(3, 4, 64), z(3, 2, 64)
    tab = z(50, 32, dtype=torch.float32)
    c.attend(q, t, n)
    for bad in (dict(q=z(2, 4, 64)), dict(q=z(3, 3, 64)), dict(q=z(3, 4, 128)), dict(q=z(3, 4, 64, dtype=BF16)), dict(q=z(3, 4, 66)[:, :, 2:]),
                dict(q=z(3, 0, 64)), dict(q=z(3, 4, 128)[:, :, ::2]), dict(table=z(3, 4, dtype=LONG)), dict(table=z(2, 4, dtype=torch.int32)),
                dict(table=z(4, 3, dtype=torch.int32).T), dict(table=z(3, 0, dtype=torch.int32)), dict(table=t[0]), dict(table=t.cpu()),
                dict(length=z(3, dtype=torch.int32)), dict(length=z(2, dtype=LONG)), dict(length=n.cpu()), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
                dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(RuntimeError):
            c.attend(**{**dict(q=q, table=t, length=n), **bad})
    step = dict(q=q, k=k, v=k, cos=tab, sin=tab, positions=n, table=t, length=n)
    c.step(**step)
    for bad in (dict(k=z(3, 4, 64)), dict(v=z(2, 2, 64)), dict(cos=None), dict(positions=None), dict(sin=z(49, 32, dtype=torch.float32)),
                dict(cos=z(50, 64, dtype=torch.float32), sin=z(50, 64, dtype=torch.float32)), dict(positions=z(2, dtype=LONG)), dict(cos=tab.half(), sin=tab.half())):
        with pytest.raises(RuntimeError):
            c.step(**{**step, **bad})
    write = dict(q=q, k=k, v=k, table=t, first=n)
    c.write(**write)
    for bad in (dict(k=z(4, 2, 64)), dict(k=z(4, 2, 64), v=z(4, 2, 64), q=None), dict(starts=z(3, dtype=LONG)), dict(starts=z(4, dtype=torch.int32)),
                dict(first=z(4, dtype=LONG)), dict(cos=tab, sin=tab)):
        with pytest.raises(RuntimeError):
            c.write(**{**write, **bad})
    for count in (0, -1):
        with pytest.raises(RuntimeError):
            c.read(t, n, count)
    # nothing to write
    assert c.write(z(0, 4, 64), z(0, 2, 64), z(0, 2, 64), t, n).shape == (0, 4, 64)
