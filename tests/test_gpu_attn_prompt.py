"""Attention of prompts and the weights of their keys against plain 64-bit forms.

Tolerances.  Outputs are rounded to fp16 (2^-11 of them), the weights to 11 bits in front of the second product (2^-11 of the
largest value), scores are sums of D products in 32 bits whose error stays below 2^-11 for the inputs here: 3 * 2^-11 of the
largest visible value.  lse and key weights are fp32: the error of a score is at most (D + 8) * 2^-23 of the sum of its
products' magnitudes, and 2^-20 for exponentials, logarithm and sums."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def seen(Tq, Tk, n, window, sinks):
    j, p = torch.arange(Tk, device="cuda"), (torch.arange(Tq, device="cuda") + Tk - Tq)[:, None]
    m = (j <= p) & (j < n) & (p < n)
    return m & ((j < sinks) | (j > p - window)) if window else m


def reference(q, k, v, lengths, window, sinks, observe=None):
    """(out, lse, key weights, magnitude of the scores' sums) in 64 bits"""
    B, Tq, H, D = q.shape
    Tk, KV = k.shape[1], k.shape[2]
    out = torch.zeros(B, Tq, H, D, dtype=torch.float64, device="cuda")
    lse = torch.full((B, H, Tq), -math.inf, dtype=torch.float64, device="cuda")
    mass = torch.zeros(B, KV, Tk, dtype=torch.float64, device="cuda")
    big = 0.0
    for b in range(B):
        n = Tk if lengths is None else min(max(lengths[b], 0), Tk)
        m = seen(Tq, Tk, n, window, sinks)
        pos = torch.arange(Tq, device="cuda") + Tk - Tq
        rows = m.any(-1)
        for h in range(H):
            kb, qb = k[b, :, h // (H // KV)].double().masked_fill((torch.arange(Tk, device="cuda") >= n)[:, None], 0), q[b, :, h].double()
            s = (qb @ kb.T / math.sqrt(D)).masked_fill(~m, -math.inf)
            big = max(big, float((qb[rows].abs() @ kb.abs().T).max() / math.sqrt(D)) if rows.any() else 0.0)
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.masked_fill(~rows, 0)[:, None])
            lse[b, h] = l
            if v is not None:
                out[b, :, h] = p @ v[b, :, h // (H // KV)].double().masked_fill((torch.arange(Tk, device="cuda") >= n)[:, None], 0)
            last = (pos >= n - (observe or Tk)) & (pos < n)
            mass[b, h // (H // KV)] += p[last].sum(0)
    return out, lse, mass, big


def make(B, Tq, Tk, H, KV, D, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)
    k = r(B, Tk, KV, D)
    k[..., 3::37] *= 3
    return (r(B, Tq, H, D) * scale).half(), k.half(), r(B, Tk, KV, D).half()


def long(x):
    return None if x is None else torch.tensor(x, dtype=torch.long, device="cuda")


def check(qc, q, k, v, lengths, window, sinks, observe=None):
    D = q.shape[-1]
    out, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks, lengths=long(lengths))
    want, l, _, big = reference(q, k, v, lengths, window, sinks)
    top = float(v.nan_to_num(0, 0, 0).abs().max())
    assert out.isfinite().all()
    assert ((out.double() - want).abs() <= 3 * 2.0 ** -11 * top).all(), float((out.double() - want).abs().max())
    empty = l == -math.inf
    assert torch.equal(lse == -math.inf, empty) and (out.transpose(1, 2)[empty] == 0).all()
    e = (D + 8) * 2.0 ** -23 * big + 2.0 ** -20
    assert ((lse.double() - l)[~empty].abs() <= e + 2.0 ** -21 * l[~empty].abs()).all()
    for last in (observe,) if observe else (None, 7):
        w = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks, lengths=long(lengths), observe=last)
        mass = reference(q, k, None, lengths, window, sinks, last)[2]
        assert ((w.double() - mass).abs() <= 3 * e * mass + 2.0 ** -30).all()
    return out


@pytest.mark.parametrize("T", [1, 2, 31, 63, 64, 65, 127, 128, 129, 191, 255, 256, 257, 300, 513])
@pytest.mark.parametrize("D,H,KV", [(128, 2, 2), (64, 6, 2)])
def test_lengths(qc, T, D, H, KV):
    check(qc, *make(2, T, T, H, KV, D, T), None, 0, 0)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (5, 3), (64, 0), (100, 4), (128, 130), (129, 64), (500, 1), (399, 0), (400, 0), (0, 9)])
@pytest.mark.parametrize("D,H,KV", [(128, 4, 1), (64, 3, 3)])
def test_windows(qc, window, sinks, D, H, KV):
    check(qc, *make(1, 400, 400, H, KV, D, window), None, window, sinks)


@pytest.mark.parametrize("Tq,Tk", [(1, 300), (5, 64), (64, 65), (100, 356), (128, 256), (129, 640), (300, 301)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (70, 2)])
def test_queries_behind_their_keys(qc, Tq, Tk, window, sinks):
    check(qc, *make(2, Tq, Tk, 4, 2, 128, Tq), None, window, sinks)


@pytest.mark.parametrize("lengths", [[300, 0, 1, 129], [64, 128, 127, 300], [-5, 400, 299, 2]])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 2)])
@pytest.mark.parametrize("Tq", [300, 77])
def test_ragged(qc, lengths, window, sinks, Tq):
    """What lies behind a prompt's end does not count, NaN and infinities included."""
    q, k, v = make(4, Tq, 300, 4, 2, 128, 5)
    want = check(qc, q, k, v, lengths, window, sinks)
    for b, n in enumerate(lengths):
        n = min(max(n, 0), 300)
        k[b, n:], v[b, n:] = math.nan, math.inf
        q[b, max(0, n - 300 + Tq):] = math.nan
    out, _ = qc.attn_prefill(q, k, v, window=window, sinks=sinks, lengths=long(lengths))
    assert torch.equal(out, want)


@pytest.mark.parametrize("H,KV", [(5, 1), (8, 1), (12, 3), (64, 8), (16, 1)])
def test_grouped_heads(qc, H, KV):
    check(qc, *make(1, 140, 140, H, KV, 64, H), None, 50, 1)


def test_strides(qc):
    """Slices of one projection's output, heads before tokens, a cache's first positions, a broadcast sequence."""
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, 200, (4 + 2 + 2) * 128 + 8, device="cuda", generator=g).half()
    q, k, v = (t.unflatten(-1, (-1, 128)) for t in (x[..., :512], x[..., 512:768], x[..., 768:1024]))
    check(qc, q, k, v, None, 0, 0)
    ht = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    check(qc, *ht, None, 60, 3)
    assert torch.equal(qc.attn_prefill(q, k, v)[0], qc.attn_prefill(*ht)[0])
    cache = torch.full((2, 512, 2, 128), math.nan, device="cuda", dtype=torch.float16)
    cache[:, :200] = k
    assert torch.equal(qc.attn_prefill(q, cache[:, :200], v)[0], qc.attn_prefill(q, k, v)[0])
    shared = k[:1].expand(2, -1, -1, -1)
    assert torch.equal(qc.attn_prefill(q, shared, v)[0], qc.attn_prefill(q, shared.contiguous(), v)[0])


def test_large_scores(qc):
    """Scores of several hundred, one key far above the rest, and equal ones."""
    q, k, v = make(1, 300, 300, 2, 2, 128, 1, scale=6.0)
    k[:, 100] *= 6
    check(qc, q, k, v, None, 0, 0)
    out, lse = qc.attn_prefill(torch.zeros_like(q), k, v)
    mean = v.double().cumsum(1) / torch.arange(1, 301, device="cuda")[:, None, None]
    assert ((out.double() - mean).abs() <= 3 * 2.0 ** -11 * float(v.abs().max())).all()
    assert ((lse.double() - torch.arange(1, 301, device="cuda").double().log()).abs() <= 2.0 ** -19).all()


@pytest.mark.parametrize("shape", [(1, 2048, 2048, 8, 8, 128, 0, 0), (1, 4096, 4096, 4, 1, 128, 1024, 4), (2, 1999, 3001, 4, 2, 64, 0, 0)])
def test_long(qc, shape):
    B, Tq, Tk, H, KV, D, window, sinks = shape
    check(qc, *make(B, Tq, Tk, H, KV, D, 3), None, window, sinks, observe=64)


def test_nan_stays_with_its_rows(qc):
    """A NaN query row is NaN, and no other; a NaN key reaches the rows that see it."""
    q, k, v = make(1, 200, 200, 2, 2, 128, 4)
    want, _ = qc.attn_prefill(q, k, v, window=50)
    q2, k2 = q.clone(), k.clone()
    q2[0, 70, 1] = math.nan
    out, _ = qc.attn_prefill(q2, k, v, window=50)
    assert out[0, 70, 1].isnan().all()
    out[0, 70, 1] = want[0, 70, 1]
    assert torch.equal(out, want)
    k2[0, 100, 0] = math.nan
    out, _ = qc.attn_prefill(q, k2, v, window=50)
    assert out[0, 100:150, 0].isnan().all() and torch.equal(out[0, :100], want[0, :100]) and torch.equal(out[0, 150:], want[0, 150:])
    assert torch.equal(out[:, :, 1], want[:, :, 1])


def test_repeats_itself_on_any_stream_and_in_a_graph(qc):
    q, k, v = make(1, 700, 700, 8, 2, 128, 6)
    first, lse = qc.attn_prefill(q, k, v, window=300, sinks=2)
    w = qc.attn_prefill_weights(q, k, lse, window=300, sinks=2)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(5):
            out, l = qc.attn_prefill(q, k, v, window=300, sinks=2)
            assert torch.equal(out, first) and torch.equal(l, lse)
            assert torch.equal(qc.attn_prefill_weights(q, k, l, window=300, sinks=2), w)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, l = qc.attn_prefill(q, k, v, window=300, sinks=2)
        gw = qc.attn_prefill_weights(q, k, l, window=300, sinks=2)
    graph.replay()
    assert torch.equal(out, first) and torch.equal(gw, w)


def test_refusals(qc):
    mk = lambda *s, dtype=torch.float16: torch.zeros(*s, device="cuda", dtype=dtype)
    q, k = mk(2, 10, 4, 128), mk(2, 10, 2, 128)
    n = mk(2, dtype=torch.long)
    bad = [
        lambda: qc.attn_prefill(q.float(), k, k), lambda: qc.attn_prefill(q, k.bfloat16(), k), lambda: qc.attn_prefill(q, k, k[:, :9]),
        lambda: qc.attn_prefill(q, k[:1], k[:1]), lambda: qc.attn_prefill(q, k[:, :9], k[:, :9]), lambda: qc.attn_prefill(mk(2, 10, 3, 128), k, k),
        lambda: qc.attn_prefill(mk(2, 10, 4, 96), mk(2, 10, 2, 96), mk(2, 10, 2, 96)), lambda: qc.attn_prefill(q, k, k, window=-1),
        lambda: qc.attn_prefill(q, k, k, sinks=-2), lambda: qc.attn_prefill(q, k, k, lengths=n[:1]), lambda: qc.attn_prefill(q, k, k, lengths=n.int()),
        lambda: qc.attn_prefill(q.transpose(1, 3), k, k), lambda: qc.attn_prefill(mk(2, 10, 4, 129)[..., 1:], k, k),
        lambda: qc.attn_prefill(mk(2, 10, 4, 132)[..., :128], k, k), lambda: qc.attn_prefill(q[0], k[0], k[0]), lambda: qc.attn_prefill(q.cpu(), k, k),
        lambda: qc.attn_prefill(mk(2, 0, 4, 128), k, k),
        lambda: qc.attn_prefill_weights(q, k, mk(2, 4, 10)), lambda: qc.attn_prefill_weights(q, k, mk(2, 4, 9, dtype=torch.float32)),
        lambda: qc.attn_prefill_weights(q, k, mk(2, 4, 10, dtype=torch.float32), observe=0),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("D,window,sinks", [(128, 0, 0), (64, 0, 0), (128, 70, 3), (64, 70, 0)])
def test_masked_values_may_be_anything(qc, bad, D, window, sinks):
    """A value that is no number, or infinite, reaches the rows that see it, in its columns, and no other."""
    q, k, v = make(2, 300, 340, 4, 2, D, 9)
    want, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
    v2 = v.clone()
    v2[0, 200, 1, 5] = v2[1, 250, 0] = v2[1, 339, 1, D - 1] = bad
    out, l = qc.attn_prefill(q, k, v2, window=window, sinks=sinks)
    assert torch.equal(l, lse)
    m = seen(300, 340, 340, window, sinks)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, :, 2:, 5] |= m[:, 200, None]
    hit[1, :, :2] |= m[:, 250, None, None]
    hit[1, :, 2:, D - 1] |= m[:, 339, None]
    assert not out[hit].isfinite().any() and out[~hit].isfinite().all()
    if not math.isnan(bad):
        assert (out[hit] == bad).all()
    top = float(v.abs().max())
    ref = reference(q, k, v, None, window, sinks)[0]
    assert ((out.double() - ref).abs()[~hit] <= 3 * 2.0 ** -11 * top).all()
    assert torch.equal(out[0, :, :2], want[0, :, :2])


def test_rows_shared_by_all_tokens(qc):
    """An expanded token: every position has the same key and value, or the same query."""
    q, k, v = make(2, 90, 150, 4, 2, 128, 10)
    for x, y, z in ((q, k[:, :1].expand(-1, 150, -1, -1), v), (q, k, v[:, 3:4].expand(-1, 150, -1, -1)), (q[:, 2:3].expand(-1, 90, -1, -1), k, v)):
        assert torch.equal(check(qc, x, y, z, None, 40, 2), qc.attn_prefill(x.contiguous(), y.contiguous(), z.contiguous(), window=40, sinks=2)[0])


def test_windows_of_any_size(qc):
    """A window or sinks up to 2^31 - 1 that leave nothing out."""
    q, k, v = make(1, 200, 260, 2, 1, 64, 11)
    want, lse = qc.attn_prefill(q, k, v)
    w = qc.attn_prefill_weights(q, k, lse)
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (5, 2 ** 31 - 1)):
        out, l = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
        assert ((out.double() - want.double()).abs() <= 2.0 ** -10 * float(v.abs().max())).all()
        assert torch.equal(qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks), w)


def test_masked_infinities_in_a_long_prompt(qc):
    """As above over several tiles and items of a CTA: the last token's values are infinite, only its own row sees them."""
    q, k, v = make(1, 1500, 1500, 40, 40, 128, 12)
    want, lse = qc.attn_prefill(q, k, v)
    v[0, 1499] = math.inf
    out, l = qc.attn_prefill(q, k, v)
    assert torch.equal(l, lse) and (out[0, 1499] == math.inf).all()
    assert ((out[0, :1499].double() - want[0, :1499].double()).abs() <= 6 * 2.0 ** -11 * float(v[0, :1499].abs().max())).all()
    assert torch.equal(out[0, :1408], want[0, :1408])


@pytest.mark.parametrize("Tq,Tk", [(1, 1), (1, 2500), (3, 1000), (8, 8), (9, 700), (33, 33), (50, 3001), (128, 1500), (129, 1500), (300, 2000)])
@pytest.mark.parametrize("H,KV,D", [(8, 1, 128), (6, 2, 64), (40, 1, 64), (4, 4, 128), (64, 8, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 70)])
def test_few_queries(qc, Tq, Tk, H, KV, D, window, sinks):
    """Heads side by side in a tile, keys in parts."""
    check(qc, *make(1, Tq, Tk, H, KV, D, Tq), None, window, sinks, observe=20)


@pytest.mark.parametrize("Tq", [5, 64, 200])
def test_few_queries_ragged(qc, Tq):
    q, k, v = make(5, Tq, 1100, 8, 2, 128, Tq)
    lengths = [1100, 0, 1100 - Tq, 1100 - Tq + 1, 1098]
    want = check(qc, q, k, v, lengths, 500, 3, observe=20)
    for b, n in enumerate(lengths):
        k[b, n:], v[b, n:] = math.nan, math.inf
        q[b, max(0, n - 1100 + Tq):] = math.nan
    out, _ = qc.attn_prefill(q, k, v, window=500, sinks=3, lengths=long(lengths))
    assert torch.equal(out, want)


@pytest.mark.parametrize("Tq,H,KV", [(20, 4, 1), (150, 2, 2)])
def test_few_queries_masked_infinities(qc, Tq, H, KV):
    q, k, v = make(1, Tq, 2000, H, KV, 128, 13)
    want, lse = qc.attn_prefill(q, k, v, window=700)
    v[0, 1999], v[0, 1100, 0, 7] = math.inf, math.nan
    out, l = qc.attn_prefill(q, k, v, window=700)
    assert torch.equal(l, lse) and (out[0, -1] == math.inf).all()
    assert ((out[0, :-1].double() - want[0, :-1].double()).abs() <= 6 * 2.0 ** -11 * float(v[0, :1100].abs().max())).all()


@pytest.mark.parametrize("Tq,Tk,H,KV,D", [(100, 1100, 8, 1, 128), (300, 2000, 4, 4, 128), (128, 1500, 8, 1, 64), (33, 700, 6, 2, 64), (200, 200, 2, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (600, 70)])
@pytest.mark.parametrize("q0,k0", [(32.0, -35.375), (64.0, -53.0)])
def test_scores_that_are_all_very_low(qc, Tq, Tk, H, KV, D, window, sinks, q0, k0):
    """Scaled scores around q0 * k0 / sqrt(D), -100 and below: a row keeps its sum also where its keys are cut into parts and it sees
    nothing of one.  The outputs' tolerance holds the scores' error too, twice that of lse, as the weights' relative error."""
    q, k, v = make(1, Tq, Tk, H, KV, D, Tq)
    q[..., 0], k[..., 0] = q0, k0
    v += 3
    out, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
    want, l, _, big = reference(q, k, v, None, window, sinks)
    e = (D + 8) * 2.0 ** -23 * big + 2.0 ** -20
    assert ((lse.double() - l).abs() <= e + 2.0 ** -21 * l.abs()).all(), float((lse.double() - l).abs().max())
    assert ((out.double() - want).abs() <= (3 * 2.0 ** -11 + 2 * e) * float(v.abs().max())).all()


@pytest.mark.parametrize("D,H,KV", [(128, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("window,sinks,observe", [(70, 0, 40), (130, 3, 9), (1, 1, 64), (0, 0, 30)])
@pytest.mark.parametrize("Tq", [400, 150])
def test_keys_that_nobody_sees_have_no_weight(qc, D, H, KV, window, sinks, observe, Tq):
    """Exactly 0, whichever tile they lie in, so that of them an eviction keeps the lowest slots."""
    lengths = [400, 300, 129]
    q, k, v = make(3, Tq, 400, H, KV, D, 14)
    out, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks, lengths=long(lengths))
    w = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks, lengths=long(lengths), observe=observe)
    cache = qc.KVCache4.empty(3, KV, 416, D)
    cache.write(None, k.reshape(-1, KV, D), v.reshape(-1, KV, D), torch.zeros(3, dtype=torch.long, device="cuda"))
    keep = 200
    kept, _, _ = cache.evict(torch.nn.functional.pad(w, (0, 16)), long(lengths), keep)
    for b, n in enumerate(lengths):
        m = seen(Tq, 400, n, window, sinks)
        pos = torch.arange(Tq, device="cuda") + 400 - Tq
        some = m[(pos >= n - observe) & (pos < n)].any(0)
        assert (w[b][:, ~some] == 0).all() and (w[b][:, some] > 0).all()
        if n > keep and int(some.sum()) <= keep:
            slots = torch.cat([some.nonzero().flatten(), (~some).nonzero().flatten()])[:keep].sort().values
            assert (kept[b].long() == slots).all()


@pytest.mark.parametrize("D,H,KV", [(128, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3), (150, 0)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_bad_lse_stays_with_the_keys_that_its_query_sees(qc, D, H, KV, window, sinks, bad):
    q, k, v = make(2, 300, 340, H, KV, D, 15)
    _, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
    want = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks)
    lse[1, H - 1, 100] = bad
    w = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks)
    m = seen(300, 340, 340, window, sinks)[100]
    hit = torch.zeros_like(w, dtype=torch.bool)
    hit[1, KV - 1] = m
    assert torch.equal(w[~hit], want[~hit])
    assert w[hit].isnan().all() if bad != bad else (w[hit] <= want[hit]).all()


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_a_query_that_is_no_number_reaches_the_weights_of_its_keys(qc, window, sinks):
    q, k, v = make(1, 300, 300, 4, 2, 128, 16)
    _, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
    want = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks)
    q[0, 130, 1] = math.nan
    _, lse = qc.attn_prefill(q, k, v, window=window, sinks=sinks)
    w = qc.attn_prefill_weights(q, k, lse, window=window, sinks=sinks)
    m = seen(300, 300, 300, window, sinks)[130]
    assert w[0, 0, m].isnan().all() and torch.equal(w[0, 0, ~m], want[0, 0, ~m]) and torch.equal(w[0, 1], want[0, 1])


@pytest.mark.parametrize("less,want", [(-math.inf, math.inf), (500.0, math.inf), (60.0, None)])
def test_weights_beyond_one(qc, less, want):
    """An lse that is not that of these scores: exp(score - lse) as it is, infinite beyond fp32."""
    q, k, v = make(1, 300, 300, 4, 2, 128, 17)
    _, lse = qc.attn_prefill(q, k, v, window=50)
    clean = qc.attn_prefill_weights(q, k, lse, window=50)
    low = lse.clone()
    low[0, 1] = low[0, 1] - less if less > 0 else less
    w = qc.attn_prefill_weights(q, k, low, window=50)
    assert torch.equal(w[0, 1], clean[0, 1])
    if want:
        assert (w[0, 0] == want).all()
        return
    _, l, mass, big = reference(q, k, None, None, 50, 0)
    other = reference(q[:, :, :1], k[:, :, :1], None, None, 50, 0)[2][0, 0]
    full = other + (mass[0, 0] - other) * math.exp(less)
    # the error of a score as in the other tests, and that of lse - 60, rounded to fp32
    e = (128 + 8) * 2.0 ** -23 * big + 2.0 ** -20 + 2.0 ** -24 * (less + float(l.abs().max()))
    assert ((w[0, 0].double() - full).abs() <= 3 * e * full).all()


def test_padding_that_is_no_number_takes_no_time(qc):
    """Rows behind a prompt's end are zeros whatever they hold; that theirs are NaN is no reason to look at rows again (twice the time)."""
    q, k, v = make(4, 1000, 1000, 64, 8, 128, 18)
    ends = [1000, 700, 300, 77]

    def median():
        for _ in range(3):
            qc.attn_prefill(q, k, v, lengths=long(ends))
        took = []
        for _ in range(15):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            n = long(ends)
            a.record()
            for _ in range(5):
                out, _ = qc.attn_prefill(q, k, v, lengths=n)
            b.record()
            torch.cuda.synchronize()
            took.append(a.elapsed_time(b))
        return sorted(took)[7], out
    finite, want = median()
    for b, n in enumerate(ends):
        q[b, n:] = k[b, n:] = v[b, n:] = math.nan
    padded, out = median()
    assert torch.equal(out, want)
    assert padded <= 1.4 * finite, (finite, padded)


@pytest.mark.parametrize("Tq,Tk,H,KV,D", [(200, 200, 8, 2, 128), (1, 1, 8, 8, 64), (60, 1500, 4, 1, 128), (300, 300, 4, 4, 64)])
@pytest.mark.parametrize("window", [0, 1, 3])
def test_the_largest_values_stay_finite(qc, Tq, Tk, H, KV, D, window):
    """An output lies between the values of its row: where all of them are fp16's largest, the weights' roundings make no infinity of it."""
    q, k, v = make(1, Tq, Tk, H, KV, D, 19, scale=2.0)
    v[:] = 65504.0
    v[..., 1::2] = -65504.0
    out, _ = qc.attn_prefill(q, k, v, window=window)
    assert out.isfinite().all()
    assert ((out.double() - v[0, 0, 0].double()).abs() <= 3 * 2.0 ** -11 * 65504).all()
    v[0, Tk - 1, :, 5] = math.inf                         # an infinite value is one
    out, _ = qc.attn_prefill(q, k, v, window=window)
    assert (out[0, -1, :, 5] == math.inf).all() and out[..., :5].isfinite().all() and out[..., 6:].isfinite().all() and out[0, :-1].isfinite().all()
