"""Adjusted logits against the same operations one by one: every operation is rounded to 32 bits, so that results are equal bit for bit,
and picked tokens with them; and against 64 bits, where each of at most five operations is off by 2^-24 of its operands, and the result by
half a step of its type."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]
LONG = torch.long


@pytest.fixture(scope="module")
def qc():
    import cherryq_b200
    return cherryq_b200.load_quant_cuda()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def reference(logits, tokens=None, length=None, prompt=None, repetition=None, presence=None, frequency=None, bias_ids=None, bias=None, mask=None,
              mask_rows=None, work=torch.float32):
    """On the host, token by token; (values before the last rounding, sum of the operands' magnitudes)"""
    x = logits.to(work, copy=True)
    big = x.abs()
    R, V = x.shape
    for r in range(R):
        if tokens is not None:
            W = tokens.shape[1]
            n = W if length is None else min(max(int(length[r]), 0), W)
            p = 0 if prompt is None else max(int(prompt[r]), 0)
            row = tokens[r].tolist()
            seen = sorted({t for t in row[:n] if 0 <= t < V})
            made = {}
            for t in row[p:n]:
                if 0 <= t < V:
                    made[t] = made.get(t, 0) + 1
            if repetition is not None and seen:
                rep, at = repetition[r].to(work), torch.tensor(seen)
                x[r, at] = torch.where(x[r, at] > 0, x[r, at] / rep, x[r, at] * rep)
                big[r, at] += x[r, at].abs()
            if made:
                at, c = torch.tensor(list(made)), torch.tensor(list(made.values())).to(work)
                if frequency is not None:
                    x[r, at] = x[r, at] - frequency[r].to(work) * c
                    big[r, at] += 2 * (frequency[r].to(work) * c).abs()
                if presence is not None:
                    x[r, at] = x[r, at] - presence[r].to(work)
                    big[r, at] += presence[r].abs().to(work)
        if bias is not None:
            for v, b in dict((int(i), float(b)) for i, b in zip(bias_ids[r], bias[r]) if 0 <= int(i) < V).items():
                x[r, v] = x[r, v] + torch.tensor(b, dtype=torch.float32).to(work)
                big[r, v] += abs(b)
        if mask is not None:
            m = r if mask_rows is None else int(mask_rows[r])
            if 0 <= m < len(mask):
                bits = ((mask[m].long()[:, None] >> torch.arange(32)) & 1).flatten()[:V]
                x[r] = torch.where(bits == 1, x[r], -float("inf"))
    return x, big


def args_of(g, R, V, W, biases=0, masks=0, strange=True):
    a = {}
    if W is not None:
        a["tokens"] = torch.randint(-3, V + 3, (R, W), generator=g) if strange else torch.randint(0, V, (R, W), generator=g)
        a["tokens"][:, ::3] = a["tokens"][:, ::3].clamp(max=max(0, min(5, V - 1)))          # some often
        if W:
            a["length"] = torch.randint(-2, W + 3, (R,), generator=g)
            a["prompt"] = torch.randint(-2, W + 3, (R,), generator=g)
        a["repetition"] = 0.5 + 1.5 * torch.rand(R, generator=g)
        a["presence"], a["frequency"] = torch.randn(R, generator=g), torch.randn(R, generator=g)
    if biases:
        a["bias_ids"] = torch.randint(-2, V + 2, (R, biases), generator=g)                  # the same twice, and outside
        a["bias"] = torch.randn(R, biases, generator=g) * 4
    if masks:
        a["mask"] = torch.randint(-2 ** 31, 2 ** 31, (masks, (V + 31) // 32), generator=g).to(torch.int32)
        a["mask_rows"] = torch.randint(-2, masks + 2, (R,), generator=g)
    return a


def on_gpu(a):
    return {k: v.cuda() for k, v in a.items()}


def check(qc, host, a, **gpu):
    """host: the logits; `gpu`: other views of the same arguments on the device"""
    out, picked = qc.adjust_logits(**{"logits": host.cuda(), **on_gpu(a), **gpu})
    want, _ = reference(host, **a)
    assert out.dtype == host.dtype and out.shape == host.shape and picked.dtype == LONG
    same = want.to(host.dtype)
    got = out.cpu()
    assert torch.equal(got.isnan(), same.isnan()) and torch.equal(got.nan_to_num(7.0, 8.0, -8.0), same.nan_to_num(7.0, 8.0, -8.0))
    assert torch.equal(picked.cpu(), want.argmax(-1))
    exact, big = reference(host.double(), work=torch.float64, **a)
    fine = exact.isfinite() & (exact.abs() < torch.finfo(host.dtype).max)
    tol = 5 * 2.0 ** -24 * big + torch.finfo(host.dtype).eps / 2 * exact.abs() + torch.finfo(host.dtype).tiny
    assert bool(((got.double() - exact).abs() <= tol)[fine].all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,W,biases,masks", [
    (1, 1, 5, 0, 0), (1, 2, 1, 1, 1), (3, 31, 40, 5, 2), (2, 33, 7, 0, 3), (5, 1000, 100, 30, 4), (1, 32000, 300, 0, 0), (2, 32000, 1, 300, 0),
    (3, 32001, 2000, 0, 1), (4, 32007, None, 7, 2), (2, 16384, 50, 3, 0), (2, 16385, 50, 3, 1), (1, 131071, 3000, 20, 1), (3, 140001, 64, 5, 2),
    (1, 300001, 500, 9, 1), (200, 1001, 20, 3, 5), (310, 5003, 9, 0, 7), (1, 8191, 0, 0, 0),
])
def test_adjust(qc, dtype, R, V, W, biases, masks):
    g = gen(R + V)
    check(qc, (torch.randn(R, V, generator=g) * 3).to(dtype), args_of(g, R, V, W, biases, masks))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,V,W,biases,masks", [
    (64, 50257, 30, 0, 0), (100, 32000, 20, 0, 0), (140, 20001, 40, 0, 2), (40, 31999, 40, 3, 1), (74, 12345, 30, 8, 3), (8, 128256, 70, 0, 2),
    (9, 100003, 50, 9, 0), (1, 200000, 3000, 0, 1), (37, 36001, 30, 0, 0), (149, 20000, 10, 0, 0),
])
def test_adjust_large_parts(qc, dtype, R, V, W, biases, masks):
    """Parts of a row with a place for every token, on more logits than are on their way at a time; in place, from odd addresses too"""
    g = gen(R + V)
    host, a = (torch.randn(R, V, generator=g) * 3).to(dtype), args_of(g, R, V, W, biases, masks)
    check(qc, host, a)
    want, picked = qc.adjust_logits(host.cuda(), **on_gpu(a))
    room = torch.full((R, V + 9), 5.0, dtype=dtype, device="cuda")
    view = room[:, 3:V + 3]
    view.copy_(host)
    got, again = qc.adjust_logits(view, **on_gpu(a), out=view)
    assert torch.equal(got, want) and torch.equal(again, picked) and bool((room[:, :3] == 5).all()) and bool((room[:, V + 3:] == 5).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_each_alone(qc, dtype):
    """Every argument without the others"""
    g, R, V, W = gen(1), 4, 3001, 60
    logits = (torch.randn(R, V, generator=g) * 3).to(dtype)
    full = args_of(g, R, V, W, 8, 3)
    check(qc, logits, {})
    for names in (["tokens"], ["tokens", "repetition"], ["tokens", "presence"], ["tokens", "frequency"], ["tokens", "length", "frequency", "presence"],
                  ["tokens", "prompt", "repetition", "presence"], ["bias_ids", "bias"], ["mask", "mask_rows"],
                  ["tokens", "length", "prompt", "repetition", "mask", "mask_rows"]):
        check(qc, logits, {n: full[n] for n in names})
    check(qc, logits, {"mask": torch.randint(-2 ** 31, 2 ** 31, (R, (V + 31) // 32), generator=g).to(torch.int32)})


@pytest.mark.parametrize("dtype", TYPES)
def test_strange_values(qc, dtype):
    """NaN and infinite logits, biases without bound, rows of which a mask leaves nothing, ties"""
    g, R, V = gen(2), 8, 4099
    nan, inf = float("nan"), float("inf")
    logits = (torch.randn(R, V, generator=g) * 3).to(dtype)
    a = args_of(g, R, V, 50, 6, 3)
    logits[0, 100], logits[0, 101] = nan, inf
    logits[1, 7] = inf
    logits[1, 4000] = inf                                      # a tie: the lower one
    logits[2, :] = -inf
    logits[3, 5:50] = torch.finfo(dtype).max
    logits[4, ::2] = -inf
    logits[5] = 2.0
    logits[6, 4098] = nan
    a["mask_rows"][:] = -1
    a["mask"][0] = 0
    a["mask"][1] = -1
    a["mask"][2] = 0
    a["mask"][2, 128] = 4                                      # token 4098 alone
    a["mask_rows"][6], a["mask_rows"][7], a["mask_rows"][0] = 0, 2, 1
    a["bias"][4, :3] = inf
    a["bias"][5, :3] = -inf
    check(qc, logits, a)
    out, picked = qc.adjust_logits(logits.cuda(), **on_gpu(a))
    assert (out[6] == -inf).all() and picked[6] == 0 and picked[7] == 4098


def test_last_bias_counts(qc):
    logits = torch.zeros(2, 100)
    ids = torch.tensor([[5, 5, 7, 5], [1, 2, 1, -1]])
    b = torch.tensor([[1.0, 2.0, 3.0, -4.0], [9.0, 1.0, 2.0, 50.0]])
    out, picked = qc.adjust_logits(logits.cuda(), bias_ids=ids.cuda(), bias=b.cuda())
    assert out[0, 5] == -4 and out[0, 7] == 3 and out[1, 1] == 2 and out[1, 2] == 1 and out.count_nonzero() == 4
    assert picked.tolist() == [7, 1]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1000, 4093])
def test_strides_and_in_place(qc, dtype, V):
    g, R = gen(3), 5
    wide = (torch.randn(R, V + 37, generator=g) * 3).to(dtype)
    a = args_of(g, R, V, 40, 4, 3)
    dev = on_gpu(a)
    for off in (0, 1, 5, 8):                                   # rows from any element on
        logits = wide[:, off:off + V]
        check(qc, logits, a, logits=wide.cuda()[:, off:off + V])
        # into a part of something wider, which keeps the rest
        to = torch.full((R, V + 20), 3.0, dtype=dtype, device="cuda")
        out, picked = qc.adjust_logits(logits.cuda(), **dev, out=to[:, 3:3 + V])
        assert out.data_ptr() == to[:, 3:].data_ptr() and (to[:, :3] == 3).all() and (to[:, 3 + V:] == 3).all()
        want, token = qc.adjust_logits(logits.cuda(), **dev)
        assert torch.equal(out, want) and torch.equal(picked, token)
        # over themselves
        mine = wide.cuda()
        out, picked = qc.adjust_logits(mine[:, off:off + V], **dev, out=mine[:, off:off + V])
        assert torch.equal(mine[:, off:off + V], want) and torch.equal(picked, token)
        assert torch.equal(mine[:, :off].cpu(), wide[:, :off]) and torch.equal(mine[:, off + V:].cpu(), wide[:, off + V:])
    # one row, one history, one list of biases for all
    logits = wide[:1, :V].expand(R, -1)
    b = {**a, "tokens": a["tokens"][:1].expand(R, -1), "bias_ids": a["bias_ids"][:1].expand(R, -1), "bias": a["bias"][:1].expand(R, -1),
         "mask": a["mask"][:1].expand(3, -1)}
    check(qc, logits, b, logits=wide.cuda()[:1, :V].expand(R, -1), tokens=dev["tokens"][:1].expand(R, -1), bias_ids=dev["bias_ids"][:1].expand(R, -1),
          bias=dev["bias"][:1].expand(R, -1), mask=dev["mask"][:1].expand(3, -1))
    # columns of something wider
    more = torch.cat([a["tokens"], a["tokens"]], 1).cuda()
    check(qc, wide[:, :V], a, logits=wide.cuda()[:, :V], tokens=more[:, :40])


def test_long_history_of_one_token(qc):
    logits = torch.zeros(2, 50, device="cuda")
    tokens = torch.full((2, 100000), 49, dtype=LONG, device="cuda")
    one = torch.ones(2, device="cuda")
    out, picked = qc.adjust_logits(logits, tokens, prompt=torch.tensor([10, 99999], device="cuda"), frequency=one)
    assert out[0, 49] == -99990 and out[1, 49] == -1 and picked.tolist() == [0, 0]


def test_repeats_itself_and_graphs(qc):
    g, R, V = gen(4), 6, 32000
    logits = (torch.randn(R, V, generator=g) * 3).half().cuda()
    a = on_gpu(args_of(g, R, V, 500, 20, 4))
    first = qc.adjust_logits(logits, **a)
    for _ in range(3):
        again = qc.adjust_logits(logits, **a)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out, picked = qc.adjust_logits(logits, **a)
    torch.cuda.current_stream().wait_stream(stream)
    for n in (0, 100, 500):
        a["length"].fill_(n)
        logits.copy_(torch.randn(R, V, generator=g) * 3)
        graph.replay()
        want = qc.adjust_logits(logits, **a)
        assert torch.equal(out, want[0]) and torch.equal(picked, want[1])


def test_refusals(qc):
    z = lambda *s, dtype=torch.float16: torch.zeros(*s, dtype=dtype, device="cuda")
    x, t, one = z(3, 100), z(3, 9, dtype=LONG), z(3, dtype=torch.float32)
    ids, b, m = z(3, 4, dtype=LONG), z(3, 4, dtype=torch.float32), z(2, 4, dtype=torch.int32)
    fine = dict(logits=x, tokens=t, length=z(3, dtype=LONG), repetition=one + 1, bias_ids=ids, bias=b, mask=m, mask_rows=z(3, dtype=LONG))
    qc.adjust_logits(**fine)
    for bad in (dict(logits=x.double()), dict(logits=x.cpu()), dict(logits=x[0]), dict(logits=z(3, 0)), dict(logits=z(100, 3).T), dict(tokens=None),
                dict(tokens=t.int()), dict(tokens=z(2, 9, dtype=LONG)), dict(tokens=z(9, 3, dtype=LONG).T), dict(length=z(3, dtype=torch.int32)), dict(length=z(2, dtype=LONG)),
                dict(repetition=z(3)), dict(repetition=z(1, dtype=torch.float32)), dict(presence=one.cpu()), dict(prompt=z(4, dtype=LONG)), dict(bias=None), dict(bias_ids=None),
                dict(bias=b.half()), dict(bias=z(3, 5, dtype=torch.float32)), dict(bias_ids=ids.int()), dict(mask=None), dict(mask=z(2, 3, dtype=torch.int32)),
                dict(mask=m.long()), dict(mask_rows=None), dict(mask_rows=z(2, dtype=LONG)), dict(out=z(3, 99)), dict(out=z(2, 100)),
                dict(out=z(3, 100, dtype=torch.float32)), dict(out=z(1, 100).expand(3, -1)), dict(out=z(100, 3).T)):
        with pytest.raises(RuntimeError):
            qc.adjust_logits(**{**fine, **bad})
    wide = z(4, 100)
    for a, o in ((wide[:3], wide[1:]), (wide.view(-1)[:300].view(3, 100), wide.view(-1)[2:302].view(3, 100))):
        with pytest.raises(RuntimeError):
            qc.adjust_logits(a, out=o)
    out, picked = qc.adjust_logits(z(0, 100))
    assert out.shape == (0, 100) and picked.shape == (0,)
