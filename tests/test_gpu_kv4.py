"""The 4-bit KV cache against plain 64-bit forms: writing, reading, attention of single tokens, accumulated weights, eviction.

Tolerances.  Attention: the result is rounded to fp16 (2^-11 of it), values and weights may be rounded to 11 bits on their way
(2^-11 of the largest value each), scores are sums of D products in 32 bits whose error stays below 2^-11 for the inputs here:
4 * 2^-11 of the largest visible value.  Accumulated weights are fp32: the relative error of one is that of its exponent, at
most (D + 8) * 2^-23 of the sum of the products' magnitudes, twice (score and maximum's sum), and 2^-20 for the exponentials
and sums."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def values(codes, scales):
    """Rows in 64 bits."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    per = u.shape[-1] // scales.shape[-2]
    s = scales.double().repeat_interleave(per, -2)
    return u * s[..., 0] + s[..., 1]


def filled(qc, g, B, KV, S, D, group, scale=1.0):
    """A cache of quantised random rows, written through the kernel."""
    cache = qc.KVCache4.empty(B, KV, S, D, group)
    S = cache.slots
    k, v = (randn(g, B * S, KV, D) * scale).half(), (randn(g, B * S, KV, D) * scale).half()
    cache.write(None, k, v, torch.zeros(B, dtype=torch.long, device="cuda"))
    return cache


def visible(S, n, window, sinks):
    j = torch.arange(S, device="cuda")
    return (j < n) & ((j < sinks) | (j >= n - window)) if window else j < n


def attend_ref(cache, q, lengths, window, sinks):
    """(out, weights (B, KV, S), magnitude of the scores' sums) in 64 bits; lengths on the host"""
    B, H, D = q.shape
    KV, S = cache.n_kv_heads, cache.slots
    out = torch.zeros(B, H, D, dtype=torch.float64, device="cuda")
    weights = torch.zeros(B, KV, S, dtype=torch.float64, device="cuda")
    big = 0.0
    for b, n in enumerate(lengths):
        at = visible(S, min(max(n, 0), S), window, sinks).nonzero().flatten()
        if not len(at):
            continue
        k, v = values(cache.k_codes[b][:, at], cache.k_scales[b][:, at]), values(cache.v_codes[b][:, at], cache.v_scales[b][:, at])
        qb = q[b].double().view(KV, H // KV, D)
        s = torch.einsum("kgd,ksd->kgs", qb, k) / math.sqrt(D)
        big = max(big, float((torch.einsum("kgd,ksd->kgs", qb.abs(), k.abs()) / math.sqrt(D)).max()))
        p = torch.softmax(s, -1)
        out[b] = torch.einsum("kgs,ksd->kgd", p, v).reshape(H, D)
        weights[b][:, at] = p.sum(1)
    return out, weights, big


def value_bound(cache, lengths, window, sinks):
    top = 0.0
    for b, n in enumerate(lengths):
        at = visible(cache.slots, min(max(n, 0), cache.slots), window, sinks).nonzero().flatten()
        if len(at):
            top = max(top, float(values(cache.v_codes[b][:, at], cache.v_scales[b][:, at]).abs().max()))
    return 4 * 2.0 ** -11 * top


def long(x):
    return torch.tensor(x, dtype=torch.long, device="cuda")


# ---------------------------------------------------------------------------------- rows
def coded(x, group):
    """(codes, scale, minimum, how near each code's quotient is to a tie) of fp16 rows in 64 bits, numpy."""
    x = x.astype(np.float64).reshape(*x.shape[:-1], -1, group)
    low = x.min(-1, keepdims=True)
    s = ((x.max(-1, keepdims=True) - low) / 15).astype(np.float16).astype(np.float64)
    r = np.divide(x - low, s, out=np.zeros_like(x), where=s > 0)
    return np.clip(np.rint(r), 0, 15), s[..., 0], low[..., 0], np.abs(np.abs(r - np.floor(r)) - 0.5)


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("B,T,H,KV,rotate", [(1, 1, 1, 1, True), (3, 5, 8, 2, True), (2, 77, 5, 5, True), (1, 33, 4, 1, False)])
def test_write_and_read(qc, D, group, B, T, H, KV, rotate):
    g = gen(D + group + T)
    S, start = 128, [7, 0, 40][:B]
    cache = qc.KVCache4.empty(B, KV, S, D, group)
    k, v = randn(g, B * T, KV, D).half(), (randn(g, B * T, KV, D) * 3).half()
    k[..., 5] *= 20
    k[0, 0, :group] = 0.25                                # a group of equal columns: scale 0
    v[-1, -1, -group:] = torch.linspace(-6e-8, 6e-8, group, device="cuda").half()     # a scale that rounds to 0
    q = torch.cat([k, k, randn(g, B * T, H, D).half()], 1)[:, :max(H, 2 * KV) // KV * KV].contiguous() if rotate else randn(g, B * T, H, D).half()
    cos, sin = torch.rand(200, D // 2, device="cuda", generator=g), randn(g, 200, D // 2)
    pos = torch.randint(0, 200, (B * T,), device="cuda", generator=g)
    out = cache.write(q, k, v, long(start), *((cos, sin, pos) if rotate else ()))
    if rotate:
        a, b = q.double().chunk(2, -1)
        c, s = cos.double()[pos][:, None], sin.double()[pos][:, None]
        want = torch.cat([a * c - b * s, b * c + a * s], -1)
        # three roundings in 32 bits of sums that may cancel, then one to fp16
        assert ((out.double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -22 * (a.abs() + b.abs()).repeat(1, 1, 2) * 3 + 2.0 ** -25).all()
        rows_k = out[:, :KV]                              # the same columns at the same positions as k
    else:
        assert torch.equal(out, q)
        rows_k = k
    rk, rv = cache.read(long(start), T)
    for rows, codes, scales, read in ((rows_k, cache.k_codes, cache.k_scales, rk), (v, cache.v_codes, cache.v_scales, rv)):
        u, s, low, tie = coded(rows.cpu().numpy(), group)
        for b in range(B):
            at = slice(start[b], start[b] + T)
            mine = codes[b][:, at].permute(1, 0, 2).cpu().numpy()
            got = np.stack([mine & 15, mine >> 4], -1).reshape(T, KV, -1, group)
            rr = slice(b * T, (b + 1) * T)
            sc = scales[b][:, at].permute(1, 0, 2, 3).double().cpu().numpy()
            assert np.array_equal(sc[..., 0], s[rr]) and np.array_equal(sc[..., 1], low[rr])
            off = np.abs(got - u[rr])
            assert off.max() <= 1 and not (off[tie[rr] > 1e-5] > 0).any()
            want = got * sc[..., :1] + sc[..., 1:]
            have = read[b].double().cpu().numpy().reshape(want.shape)
            assert (np.abs(have - want) <= 2.0 ** -11 * np.abs(want) * (1 + 2.0 ** -10) + 2.0 ** -25).all()


def test_write_takes_only_what_fits(qc):
    g = gen(1)
    cache = qc.KVCache4.empty(2, 2, 32, 64)
    k, v = randn(g, 2 * 8, 2, 64).half(), randn(g, 2 * 8, 2, 64).half()
    guard = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    cache.write(None, k, v, long([28, -5]))               # four rows fit behind 28, three behind -5
    rk, _ = cache.read(long([28, -5]), 8)
    assert (rk[0, 4:] == 0).all() and (rk[1, :5] == 0).all() and (rk[0, :4] != 0).any(-1).all() and (rk[1, 5:] != 0).any(-1).all()
    assert torch.equal(cache.k_codes[0, :, :28], guard[0][0, :, :28]) and torch.equal(cache.v_codes[1, :, 3:], guard[2][1, :, 3:])
    # positions outside the tables: queries as they are, rows not written
    cos, sin = torch.rand(4, 32, device="cuda"), torch.rand(4, 32, device="cuda")
    q = randn(g, 16, 4, 64).half()
    before = cache.k_codes.clone()
    out = cache.write(q, k, v, long([0, 0]), cos, sin, torch.full((16,), 4, device="cuda"))
    assert torch.equal(out, q) and torch.equal(cache.k_codes, before)
    out = cache.write(q, k, v, long([0, 0]), cos, sin, torch.full((16,), -1, device="cuda"))
    assert torch.equal(out, q) and torch.equal(cache.k_codes, before)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_groups_that_are_not_finite(qc, bad):
    g = gen(2)
    cache = qc.KVCache4.empty(1, 1, 32, 128, 32)
    k = randn(g, 1, 1, 128).half()
    k[0, 0, 40] = bad
    cache.write(None, k, k, long([0]))
    rk, rv = cache.read(long([0]), 1)
    for r in (rk, rv):
        assert r[0, 0, 0, 32:64].isnan().all() and r[0, 0, 0, :32].isfinite().all() and r[0, 0, 0, 64:].isfinite().all()


# ---------------------------------------------------------------------------------- attention
@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64)])
@pytest.mark.parametrize("H,KV", [(1, 1), (4, 4), (8, 1), (10, 2), (12, 1), (6, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (9, 0), (33, 4), (1, 1), (40, 70)])
def test_attend(qc, D, group, H, KV, window, sinks):
    g = gen(H * 100 + D + window)
    B, S = 4, 320
    cache = filled(qc, g, B, KV, S, D, group)
    lengths = [S, 1, 0, 131]
    q = (randn(g, B, H, D) * 2).half()
    w0 = torch.rand(B, KV, S, device="cuda", generator=g)
    w1 = torch.full_like(w0, -7.0)
    out = cache.attend(q, long(lengths), window=window, sinks=sinks, weights=w0, weights_out=w1)
    want, weights, big = attend_ref(cache, q, lengths, window, sinks)
    assert ((out.double() - want).abs() <= value_bound(cache, lengths, window, sinks) + 2.0 ** -24).all()
    assert (out[2] == 0).all()
    live = torch.arange(S, device="cuda") < long(lengths)[:, None, None]
    full = (w0.double() + weights) * live
    rel = 2 * (D + 8) * 2.0 ** -23 * big + 2.0 ** -20
    assert ((w1.double() - full).abs() <= rel * weights + 2.0 ** -23 * full).all()
    assert torch.equal(out, cache.attend(q, long(lengths), window=window, sinks=sinks))          # with and without weights
    again = w0.clone()
    cache.attend(q, long(lengths), window=window, sinks=sinks, weights=again)                      # in place
    assert torch.equal(again, w1)


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 511, 513, 1000, 2047, 4093])
@pytest.mark.parametrize("H,KV,D,B", [(8, 8, 128, 1), (16, 2, 128, 2), (7, 1, 64, 3)])
def test_attend_lengths(qc, n, H, KV, D, B):
    g = gen(n)
    cache = filled(qc, g, B, KV, 4096, D, 32)
    q = randn(g, B, H, D).half()
    for window, sinks in ((0, 0), (max(1, n // 3), 5)):
        out = cache.attend(q, long([n] * B), window=window, sinks=sinks)
        want, _, _ = attend_ref(cache, q, [n] * B, window, sinks)
        assert ((out.double() - want).abs() <= value_bound(cache, [n] * B, window, sinks)).all()


def test_lengths_outside_the_cache(qc):
    g = gen(3)
    cache = filled(qc, g, 3, 2, 64, 128, 32)
    q = randn(g, 3, 4, 128).half()
    w = torch.ones(3, 2, 64, device="cuda")
    out = cache.attend(q, long([-3, 1 << 40, 65]), weights=w)
    same = cache.attend(q, long([0, 64, 64]))
    assert torch.equal(out, same) and (out[0] == 0).all() and (w[0] == 0).all()


def test_what_is_not_visible_does_not_count(qc):
    """NaN and infinite rows behind the end and outside the window; NaN in one visible row reaches the heads that see it."""
    g = gen(4)
    n, window, sinks = 150, 60, 3
    cache = filled(qc, g, 1, 2, 256, 128, 32)
    q = randn(g, 1, 4, 128).half()
    w = torch.zeros(1, 2, 256, device="cuda")
    want = cache.attend(q, long([n]), window=window, sinks=sinks)
    hidden = ~visible(256, n, window, sinks)
    for bad in (math.nan, math.inf):
        cache.k_scales[:, :, hidden] = bad
        cache.v_scales[:, :, hidden] = bad
        w.zero_()
        assert torch.equal(cache.attend(q, long([n]), window=window, sinks=sinks, weights=w), want)
        assert w.isfinite().all()
    cache.k_scales[0, 0, 100] = math.nan
    out = cache.attend(q, long([n]), window=window, sinks=sinks)
    assert out[0, :2].isnan().all() and torch.equal(out[0, 2:], want[0, 2:])


def test_large_and_small_values(qc):
    """Values near the ends of fp16, one huge key that takes all the weight."""
    for scale in (6e-5, 1e-3, 3e4):
        g = gen(5)
        cache = qc.KVCache4.empty(1, 2, 128, 64, 32)
        k, v = randn(g, 128, 2, 64).half(), (torch.rand(128, 2, 64, device="cuda", generator=g) * 2 - 1).mul(scale).half()
        k[77] *= 50
        cache.write(None, k, v, long([0]))
        q = randn(g, 1, 8, 64).half()
        out = cache.attend(q, long([100]))
        want, _, _ = attend_ref(cache, q, [100], 0, 0)
        assert ((out.double() - want).abs() <= value_bound(cache, [100], 0, 0) + 2.0 ** -24).all()


def test_scale(qc):
    g = gen(6)
    cache = filled(qc, g, 1, 1, 64, 64, 32)
    q = randn(g, 1, 2, 64).half()
    # twice the scale on half the query: the same numbers
    assert torch.equal(cache.attend(q, long([50]), scale=0.25), cache.attend(q * 2, long([50]), scale=0.125))


@pytest.mark.parametrize("D,group,H,KV,B", [(128, 32, 8, 8, 1), (128, 64, 16, 2, 3), (64, 32, 9, 3, 2), (64, 64, 12, 1, 2)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (20, 2)])
def test_step(qc, D, group, H, KV, B, window, sinks):
    """A step is write at the slot behind the last one, then attend over one slot more, whatever was in that slot."""
    g = gen(D + B)
    S = 96
    a = filled(qc, g, B, KV, S, D, group)
    a.k_scales[:, :, 60:] = math.nan
    b = qc.KVCache4(a.k_codes.clone(), a.k_scales.clone(), a.v_codes.clone(), a.v_scales.clone())
    cos, sin = torch.rand(200, D // 2, device="cuda", generator=g), randn(g, 200, D // 2)
    for n in ([60] * B, [0] * B, [31] * B, [32] * B, [13 + 7 * i for i in range(B)]):
        q, k, v = randn(g, B, H, D).half(), randn(g, B, KV, D).half(), randn(g, B, KV, D).half()
        pos = long([100 + i for i in range(B)])
        w0 = torch.rand(B, KV, S, device="cuda", generator=g)
        w1, w2 = torch.empty_like(w0), w0.clone()
        out = a.step(q, k, v, cos, sin, pos, long(n), window=window, sinks=sinks, weights=w0, weights_out=w1)
        qr = b.write(q, k, v, long(n), cos, sin, pos)
        for i, at in enumerate(n):
            w2[i, :, at] = 0
        want = b.attend(qr, long(n) + 1, window=window, sinks=sinks, weights=w2)
        for x, y in ((a.k_codes, b.k_codes), (a.k_scales, b.k_scales), (a.v_codes, b.v_codes), (a.v_scales, b.v_scales)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
        lengths = [x + 1 for x in n]
        bound = value_bound(b, lengths, window, sinks)
        assert ((out.double() - want.double()).abs() <= 2 * bound).all()
        _, weights, big = attend_ref(b, qr, lengths, window, sinks)
        assert ((w1.double() - w2.double()).abs() <= 2 * (2 * (D + 8) * 2.0 ** -23 * big + 2.0 ** -20) * weights + 2.0 ** -22 * w2).all()
        no_turn = a.step(qr, a.read(long(n), 1)[0][:, 0], v, None, None, None, long(n), window=window, sinks=sinks)
        assert no_turn.shape == out.shape and no_turn.isfinite().all()


def test_step_into_a_full_cache(qc):
    g = gen(8)
    cache = filled(qc, g, 1, 2, 64, 128, 32)
    before = cache.k_codes.clone()
    q, k = randn(g, 1, 2, 128).half(), randn(g, 1, 2, 128).half()
    out = cache.step(q, k, k, None, None, None, long([64]))
    assert torch.equal(cache.k_codes, before) and torch.equal(out, cache.attend(q, long([64])))
    cos = torch.ones(8, 64, device="cuda")
    out = cache.step(q, k, k, cos, cos, long([8]), long([10]))          # no such position: nothing turned, nothing written
    assert torch.equal(cache.k_codes, before) and torch.equal(out, cache.attend(q, long([11])))


def test_repeats_itself_and_runs_in_a_graph(qc):
    g = gen(9)
    cache = filled(qc, g, 4, 8, 1024, 128, 32)
    q, w = randn(g, 4, 64, 128).half(), torch.zeros(4, 8, 1024, device="cuda")
    n = long([1024, 1000, 3, 700])
    first, w1 = cache.attend(q, n, weights=w, weights_out=torch.empty_like(w)), torch.empty_like(w)
    for _ in range(10):
        assert torch.equal(cache.attend(q, n, weights=w, weights_out=w1), first)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):                            # on another stream than the cache's own
        side = cache.attend(q, n)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(side, first)
    graph, w2 = torch.cuda.CUDAGraph(), torch.zeros_like(w)
    with torch.cuda.graph(graph):
        out = cache.attend(q, n, weights=w2)
    for turn in range(1, 4):
        graph.replay()
        assert torch.equal(out, first)
        assert ((w2.double() - turn * w1.double()).abs() <= 2.0 ** -22 * turn * w1).all()
    n.fill_(17)                                           # the lengths are read when the graph runs
    graph.replay()
    assert torch.equal(out, cache.attend(q, n))


def test_offsets_beyond_32_bits(qc):
    """65 heads of a million slots: codes of more than 4 GB, the last head's rows beyond them."""
    g = gen(10)
    KV, S = 65, 1 << 20
    cache = qc.KVCache4.empty(1, KV, S, 128, 64)
    n = S - 5
    k, v = randn(g, 512, KV, 128).half(), randn(g, 512, KV, 128).half()
    cache.write(None, k, v, long([n - 512]))
    q = randn(g, 1, KV, 128).half()
    out = cache.attend(q, long([n]), window=500, sinks=0)
    want, _, _ = attend_ref(cache, q, [n], 500, 0)
    assert ((out.double() - want).abs() <= value_bound(cache, [n], 500, 0)).all()
    rk, _ = cache.read(long([n - 512]), 512)
    exact = values(cache.k_codes[0, -1, n - 512:n], cache.k_scales[0, -1, n - 512:n])
    assert ((rk[0, :, -1].double() - exact).abs() <= 2.0 ** -11 * exact.abs() * (1 + 2.0 ** -10) + 2.0 ** -25).all()


# ---------------------------------------------------------------------------------- eviction
def evict_ref(w, n, keep, sinks, recent):
    """Slots that stay, by the definition; w on the host."""
    if n <= keep:
        return list(range(n))
    rank = lambda j: (0 if math.isnan(w[j]) else 1, -w[j] if not math.isnan(w[j]) else 0, j)
    middle = sorted(range(sinks, n - recent), key=rank)[:keep - sinks - recent]
    return sorted([*range(sinks), *middle, *range(n - recent, n)])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n,keep,sinks,recent", [(320, 100, 4, 30), (320, 1, 0, 0), (320, 319, 0, 0), (311, 40, 4, 36), (33, 32, 1, 2),
                                                 (5, 64, 4, 32), (0, 8, 0, 0), (320, 320, 0, 0), (320, 300, 299, 1), (257, 128, 0, 128)])
@pytest.mark.parametrize("D,group", [(64, 64), (128, 32)])
def test_evict(qc, n, keep, sinks, recent, D, group, in_place):
    g = gen(n + keep)
    B, KV, S = 2, 3, 320
    cache = filled(qc, g, B, KV, S, D, group)
    lengths = [n, min(n, max(0, n - 37))]
    w = randn(g, B, KV, S).exp()
    w[:, 0] = torch.randint(0, 3, (B, S), device="cuda", generator=g).float()       # many equal weights
    w[0, 1, 20:40] = math.nan
    w[1, 1, 10:30] = -0.0
    w[1, 1, 30:50] = 0.0
    w[1, 2] = -w[1, 2]
    old = [t.clone() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    out = cache if in_place else qc.KVCache4.empty(B, KV, (keep + 31) // 32 * 32, D, group)
    kept, left, now = cache.evict(w, long(lengths), keep, sinks=sinks, recent=recent, out=None if in_place else out)
    assert now.tolist() == [min(x, keep) for x in lengths]
    host = w.cpu()
    for b in range(B):
        for h in range(KV):
            want = evict_ref(host[b, h].tolist(), lengths[b], keep, sinks, recent)
            assert kept[b, h].tolist() == want + [-1] * (keep - len(want))
            at = torch.tensor(want, dtype=torch.long, device="cuda")
            assert torch.equal(left[b, h, :len(want)].nan_to_num(9.0), w[b, h, at].nan_to_num(9.0)) and (left[b, h, len(want):] == 0).all()
            for mine, was in zip((out.k_codes, out.k_scales, out.v_codes, out.v_scales), old):
                assert torch.equal(mine[b, h, :len(want)], was[b, h, at]) and (mine[b, h, len(want):keep] == 0).all()
                if in_place:
                    assert torch.equal(mine[b, h, keep:], was[b, h, keep:])
    if not in_place:
        for mine, was in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), old):
            assert torch.equal(mine, was)


@pytest.mark.parametrize("n,keep,sinks,recent,want", [(8, 8, 8, 2, range(8)), (5, 9, 16, 2, range(5)), (40, 10, 6, 20, [*range(6), *range(36, 40)]),
                                                      (40, 10, 16, 4, range(10)), (40, 10, 0, 2 ** 31 - 1, range(30, 40))])
def test_evict_more_than_keep_to_stay(qc, n, keep, sinks, recent, want):
    cache = filled(qc, gen(n), 1, 2, 64, 64, 32)
    w = randn(gen(1), 1, 2, 64).exp()
    kept, left, now = cache.evict(w, long([n]), keep, sinks=sinks, recent=recent, out=qc.KVCache4.empty(1, 2, 32, 64, 32))
    want = list(want)
    assert now.tolist() == [len(want)]
    for h in range(2):
        assert kept[0, h].tolist() == want + [-1] * (keep - len(want)) and torch.equal(left[0, h, :len(want)], w[0, h, want])


@pytest.mark.parametrize("n,keep", [(70000, 1000), (70001, 69990), (131072, 65536), (512, 200), (513, 200), (4000, 1000)])
def test_evict_long(qc, n, keep):
    g = gen(n)
    S = (n + 31) // 32 * 32
    cache = filled(qc, g, 1, 2, S, 64, 64)
    w = randn(g, 1, 2, S).exp()
    w[0, 1] = torch.randint(0, 1000, (S,), device="cuda", generator=g).float()
    out = qc.KVCache4.empty(1, 2, keep, 64, 64)
    kept, left, now = cache.evict(w, long([n]), keep, sinks=5, recent=100, out=out)
    for h in range(2):
        x = w[0, h, :n].cpu().numpy().copy()
        x[:5] = x[n - 100:] = np.inf
        want = np.sort(np.argsort(-x, kind="stable")[:keep])
        assert np.array_equal(kept[0, h].cpu().numpy(), want)
        at = torch.from_numpy(want).cuda()
        assert torch.equal(out.v_codes[0, h, :keep], cache.v_codes[0, h, at]) and torch.equal(out.k_scales[0, h, :keep], cache.k_scales[0, h, at])


def test_evicted_cache_goes_on(qc):
    """Prompt, attention with weights, eviction in place, steps: the same as attention over the rows that stayed."""
    g = gen(12)
    B, H, KV, D, S, n, keep = 2, 8, 2, 128, 256, 200, 64
    cache = filled(qc, g, B, KV, S, D, 32)
    w = torch.zeros(B, KV, S, device="cuda")
    for _ in range(3):
        cache.attend(randn(g, B, H, D).half(), long([n] * B), weights=w)
    assert torch.allclose(w.sum(-1), torch.full((B, KV), 3.0 * H / KV, device="cuda"), rtol=1e-4)
    kept, left, now = cache.evict(w, long([n] * B), keep, sinks=4, recent=16)
    w.zero_()
    w[:, :, :keep] = left
    for i in range(5):
        q, k = randn(g, B, H, D).half(), randn(g, B, KV, D).half()
        out = cache.step(q, k, k, None, None, None, now, weights=w)
        now += 1
        lengths = now.tolist()
        want, _, _ = attend_ref(cache, q, lengths, 0, 0)
        assert ((out.double() - want).abs() <= value_bound(cache, lengths, 0, 0)).all()
    assert torch.allclose(w.sum(-1), left.sum(-1) + 5.0 * H / KV, rtol=1e-4)


# ---------------------------------------------------------------------------------- refusals
def test_refusals(qc):
    mk = lambda *s, **o: torch.zeros(*s, device="cuda", **o)
    u8, f16 = dict(dtype=torch.uint8), dict(dtype=torch.float16)

    def cache_of(codes, scales, v_codes=None, v_scales=None):
        return qc.KVCache4(codes, scales, codes.clone() if v_codes is None else v_codes, scales.clone() if v_scales is None else v_scales)
    for codes, scales in [((1, 2, 33, 32), (1, 2, 33, 2, 2)), ((1, 2, 32, 48), (1, 2, 32, 3, 2)), ((1, 2, 32, 64), (1, 2, 32, 1, 2)),
                          ((1, 2, 32, 64), (1, 2, 64, 4, 2)), ((1, 2, 32, 64), (1, 2, 32, 8, 2)), ((2, 32, 64), (2, 32, 4, 2)), ((1, 2, 0, 64), (1, 2, 0, 4, 2))]:
        with pytest.raises(RuntimeError):
            cache_of(mk(*codes, **u8), mk(*scales, **f16))
    with pytest.raises(RuntimeError, match="dtype"):
        cache_of(mk(1, 2, 32, 64, **u8), mk(1, 2, 32, 4, 2))
    with pytest.raises(RuntimeError, match="CUDA"):
        qc.KVCache4(*[torch.zeros(1, 2, 32, 64, dtype=torch.uint8), torch.zeros(1, 2, 32, 4, 2, dtype=torch.float16)] * 2)
    with pytest.raises(RuntimeError, match="contiguous"):
        cache_of(mk(1, 32, 2, 64, **u8).transpose(1, 2), mk(1, 2, 32, 4, 2, **f16))
    c = qc.KVCache4.empty(2, 2, 40, 128)
    assert (c.sequences, c.n_kv_heads, c.slots, c.head_dim, c.group) == (2, 2, 64, 128, 32)
    q, k, n = mk(2, 4, 128, **f16), mk(2, 2, 128, **f16), mk(2, dtype=torch.long)
    w = mk(2, 2, 64)
    bad = [
        lambda: c.attend(q.float(), n), lambda: c.attend(q[:1], n), lambda: c.attend(mk(2, 3, 128, **f16), n), lambda: c.attend(mk(2, 4, 64, **f16), n),
        lambda: c.attend(q, n.int()), lambda: c.attend(q, n[:1]), lambda: c.attend(q, n.cpu()), lambda: c.attend(q.cpu(), n),
        lambda: c.attend(q, n, window=-1), lambda: c.attend(q, n, sinks=-1), lambda: c.attend(q, n, weights=w[:, :, :32].contiguous()),
        lambda: c.attend(q, n, weights=w.double()), lambda: c.attend(q, n, weights_out=w), lambda: c.attend(q.transpose(0, 1), n),
        lambda: c.attend(mk(2 * 4 * 128 + 1, **f16)[1:].view(2, 4, 128), n),
        lambda: c.step(q, k[:1], k, None, None, None, n), lambda: c.step(q, k, k, mk(8, 64), mk(8, 64), None, n),
        lambda: c.step(q, k, k, mk(8, 32), mk(8, 32), n, n), lambda: c.step(q, k, k, mk(8, 64, **f16), mk(8, 64, **f16), n, n),
        lambda: c.write(None, mk(3, 2, 128, **f16), mk(3, 2, 128, **f16), n), lambda: c.write(None, k, mk(2, 1, 128, **f16), n),
        lambda: c.write(q[:1], k, k, n), lambda: c.write(None, k, k, n[:1]), lambda: c.read(n, 0), lambda: c.read(n.float(), 1),
        lambda: c.evict(w, n, 0), lambda: c.evict(w, n, 65), lambda: c.evict(w, n, 8, sinks=-1),
        lambda: c.evict(w[:1], n, 8), lambda: c.evict(w, n, 8, out=qc.KVCache4.empty(2, 2, 64, 128, 64)),
        lambda: c.evict(w, n, 33, out=qc.KVCache4.empty(2, 2, 32, 128)), lambda: c.evict(w, n, 8, out=qc.KVCache4.empty(1, 2, 64, 128)),
        lambda: qc.KVCache4.empty(1, 1, 0, 128), lambda: qc.KVCache4.empty(1, 1, 32, 96), lambda: qc.KVCache4.empty(1, 1, 32, 128, 128),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cos_off,sin_off", [(1, 1), (3, 2), (2, 2), (0, 1), (4, 0)])
def test_tables_that_start_anywhere(qc, D, cos_off, sin_off):
    """Views whose first number lies on any 4 bytes: the same rows, queries and outputs as with tables of their own."""
    g = gen(20)
    B, T, H, KV, S, P = 2, 19, 4, 2, 64, 50
    cos, sin = randn(g, P, D // 2), randn(g, P, D // 2)

    def view(x, off):
        y = torch.empty(P * (D // 2) + off, device="cuda")[off:].view(P, D // 2)
        return y.copy_(x)
    a, b = qc.KVCache4.empty(B, KV, S, D), qc.KVCache4.empty(B, KV, S, D)
    q, k, v = randn(g, B * T, H, D).half(), randn(g, B * T, KV, D).half(), randn(g, B * T, KV, D).half()
    pos = torch.randint(0, P, (B * T,), device="cuda", generator=g)
    qa = a.write(q, k, v, long([0, 3]), cos, sin, pos)
    qb = b.write(q, k, v, long([0, 3]), view(cos, cos_off), view(sin, sin_off), pos)
    assert torch.equal(qa, qb)
    q, k, pos = randn(g, B, H, D).half(), randn(g, B, KV, D).half(), long([11, P - 1])
    oa = a.step(q, k, k, cos, sin, pos, long([T, T + 3]))
    ob = b.step(q, k, k, view(cos, cos_off), view(sin, sin_off), pos, long([T, T + 3]))
    assert torch.equal(oa, ob)
    for x, y in ((a.k_codes, b.k_codes), (a.k_scales, b.k_scales), (a.v_codes, b.v_codes), (a.v_scales, b.v_scales)):
        assert torch.equal(x, y)


def test_evict_into_a_cache_that_overlaps(qc):
    """A handle over the same storage, one sequence on: refused, where the rows would be moved over rows still to be read."""
    make = lambda *s, **o: torch.zeros(*s, device="cuda", **o)
    codes, scales = dict(dtype=torch.uint8), dict(dtype=torch.float16)
    t = make(3, 2, 64, 64, **codes), make(3, 2, 64, 4, 2, **scales), make(3, 2, 64, 64, **codes), make(3, 2, 64, 4, 2, **scales)
    a, b, c = qc.KVCache4(*(x[:2] for x in t)), qc.KVCache4(*(x[1:] for x in t)), qc.KVCache4(*(x[:2] for x in t))
    w, n = torch.ones(2, 2, 64, device="cuda"), long([64, 64])
    with pytest.raises(RuntimeError):
        a.evict(w, n, 16, out=b)
    with pytest.raises(RuntimeError):
        a.evict(w, n, 16, out=qc.KVCache4(t[0][:2], *(x.clone() for x in (t[1][:2], t[2][:2], t[3][:2]))))
    assert a.evict(w, n, 16, out=c)[2].tolist() == [16, 16]            # the same cache by another handle: in place


def test_weights_over_themselves_or_apart(qc):
    g = gen(21)
    cache = filled(qc, g, 1, 2, 64, 64, 32)
    q, n, w = randn(g, 1, 4, 64).half(), long([50]), torch.zeros(3, 2, 64, device="cuda")
    with pytest.raises(RuntimeError):
        cache.attend(q, n, weights=w.flatten()[:128].view(1, 2, 64), weights_out=w.flatten()[64:192].view(1, 2, 64))
    out = cache.attend(q, n, weights=w[:1], weights_out=w[1:2])
    assert torch.equal(out, cache.attend(q, n, weights=w[:1])) and torch.equal(w[0], w[1]) and (w[2] == 0).all()


@pytest.mark.parametrize("low", [-65504.0, -8000.0, 0.0, 4000.0])
@pytest.mark.parametrize("D,group", [(128, 32), (64, 64)])
def test_the_largest_values_stay_finite(qc, low, D, group):
    """Groups that reach to fp16's end: code 15 stands for no infinity, a column is at most half a step off, and attention over such
    values is what it is over the values that were kept."""
    g = gen(22)
    KV, n = 2, 40
    cache = qc.KVCache4.empty(1, KV, 64, D, group)
    v = (low + (65504.0 - low) * torch.rand(n, KV, D, device="cuda", generator=g)).half()
    v[..., ::group], v[..., 1::group] = 65504.0, low
    k = randn(g, n, KV, D).half()
    cache.write(None, k, v, long([0]))
    _, rv = cache.read(long([0]), n)
    assert rv.isfinite().all()
    step = (65504.0 - low) / 15
    # the scale may be 2^-11 of itself off, upwards or downwards, fifteen times, or one step of fp16 where it was lowered; then one rounding
    assert ((rv[0].double() - v.double()).abs() <= 0.5 * step * (1 + 2.0 ** -10) + 15 * step * 2.0 ** -10 + 16).all()
    q = randn(g, 1, 4, D).half()
    out = cache.attend(q, long([n]))
    want, _, _ = attend_ref(cache, q, [n], 0, 0)
    assert out.isfinite().all() and ((out.double() - want).abs() <= value_bound(cache, [n], 0, 0)).all()
    other = qc.KVCache4.empty(1, KV, 64, D, group)
    other.step(q, k[:1], v[:1], None, None, None, long([0]))
    assert torch.equal(other.v_codes[:, :, 0], cache.v_codes[:, :, 0]) and torch.equal(other.v_scales[:, :, 0], cache.v_scales[:, :, 0])
