"""The decode harness on the 4-bit cache, with a sliding window, sinks and a bounded cache: against the same harness whose
cache, attention and eviction are plain torch expressions; graph replay against eager steps."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cherryq_b200 import decoder
    return decoder


def tiny(dec, kv_heads=4, head_dim=64, max_seq=256, layers=2):
    return dec.DecoderConfig(n_layers=layers, hidden=4 * head_dim, n_heads=4, n_kv_heads=kv_heads, ffn=512, vocab=1000, bits=4, group=128,
                             cherry_fraction=1 / 32, max_seq=max_seq)


def kept4(x, group):
    """The values that fp16 rows stand for in 4 bits."""
    x = x.float().unflatten(-1, (-1, group))
    low = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - low) / 15).half().float()
    return (torch.where(s > 0, ((x - low) / s).round().clamp(0, 15), 0.0) * s + low).flatten(-2)


class Plain:
    """The harness's 4-bit methods as torch expressions; every sequence's cache is a list of rows."""

    def __init__(self, d, group, other=None):
        self.d, self.group = d, group
        self.rows = {}                                  # a layer's q, k, v in the last call on the other side
        if other is not None:
            for name in ("_kv4_step", "_kv4_prompt"):
                setattr(other, name, self.noting(getattr(other, name)))
        self.k, self.v, self.w = ([None] * len(d.caches) for _ in range(3))
        for name in ("_kv4_step", "_kv4_prompt", "_kv4_evict"):
            setattr(d, name, getattr(self, name[5:]))

    def noting(self, method):
        def call(li, q, k, v, pos):
            self.rows[li] = q.clone(), k.clone(), v.clone()
            return method(li, q, k, v, pos)
        return call

    def turn(self, x, pos):
        c, s = self.d.cos[pos][:, None], self.d.sin[pos][:, None]
        a, b = x.float().chunk(2, -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1).half()

    def attend(self, q, k, v, first):
        """q (B, Tq, H, D) at slots first ..; k, v (B, KV, S, D): (out, weights per query head and query)"""
        d = self.d
        B, T, H, D = q.shape
        at, j = first + torch.arange(T, device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
        seen = j <= at
        if d.window:
            seen = seen & ((j < d.sinks) | (j > at - d.window))
        G = H // k.shape[1]
        s = torch.einsum("bthd,bhsd->bhts", q.float(), k.repeat_interleave(G, 1)) / math.sqrt(D)
        p = s.masked_fill(~seen, -math.inf).softmax(-1)
        return torch.einsum("bhts,bhsd->bthd", p, v.repeat_interleave(G, 1)).half(), p

    def per_kv(self, p, kv):
        return p.unflatten(1, (kv, -1)).sum(2)

    def prompt(self, li, q, k, v, pos):
        q, k, v = self.rows.get(li, (q, k, v))
        d, B = self.d, self.d.batch
        q, k = self.turn(q, pos), self.turn(k, pos)
        rows = lambda x: x.view(B, -1, *x.shape[1:])
        heads = lambda x: rows(x).transpose(1, 2).float()
        out, p = self.attend(rows(q), heads(k), heads(v), 0)
        self.k[li], self.v[li] = kept4(heads(k), self.group), kept4(heads(v), self.group)
        self.w[li] = self.per_kv(p, k.shape[1])[:, :, -d.kv_observe:].sum(2)
        if d.kv_budget is not None:
            self.cut(li)
            d.length.fill_(self.k[li].shape[2])
        return out.reshape(-1, *q.shape[1:]).contiguous()

    def step(self, li, q, k, v, pos):
        q, k, v = self.rows.get(li, (q, k, v))
        q, k = self.turn(q, pos), self.turn(k, pos)
        self.k[li] = torch.cat([self.k[li], kept4(k, self.group)[:, :, None]], 2)
        self.v[li] = torch.cat([self.v[li], kept4(v, self.group)[:, :, None]], 2)
        out, p = self.attend(q[:, None], self.k[li], self.v[li], self.k[li].shape[2] - 1)
        self.w[li] = torch.nn.functional.pad(self.w[li], (0, 1)) + self.per_kv(p, k.shape[1])[:, :, 0]
        return out[:, 0].contiguous()

    def cut(self, li):
        d, n, keep = self.d, self.k[li].shape[2], self.d.kv_budget
        if n <= keep:
            return
        w = self.w[li].clone()
        w[:, :, :d.sinks] = w[:, :, n - d.kv_recent:] = math.inf
        at = torch.sort(w, dim=-1, descending=True, stable=True).indices[:, :, :keep].sort(-1).values
        self.w[li] = self.w[li].gather(2, at)
        rows = at[..., None].expand(-1, -1, -1, self.k[li].shape[3])
        self.k[li], self.v[li] = self.k[li].gather(2, rows), self.v[li].gather(2, rows)

    def evict(self):
        for li in range(len(self.k)):
            self.cut(li)
        self.d.length_host = self.d.kv_budget


@pytest.mark.parametrize("batch,kv,head_dim,group", [(1, 4, 64, 32), (3, 2, 128, 64)])
@pytest.mark.parametrize("options", [dict(), dict(window=20, sinks=2), dict(kv_budget=32, kv_slack=16, sinks=2, kv_recent=8, kv_observe=16),
                                     dict(kv_budget=64, kv_slack=32)])
def test_against_torch_expressions(dec, batch, kv, head_dim, group, options):
    # With evictions one layer: its queries, keys and values follow from the tokens alone and are the same on both sides, so that
    # the weights that are ranked differ in their last bits only.  (Behind a first layer, whose outputs differ by roundings, slots
    # of nearly equal weight are ranked otherwise here and there, and other slots stay.)
    # Without evictions two layers; the torch expressions take the second layer's rows from the kernels' side, as a last bit there
    # can be another 4-bit code, which is 1/15 of the group's range.
    cfg = tiny(dec, kv, head_dim, layers=1 if "kv_budget" in options else 2)
    make = lambda: dec.CherryDecoder(cfg, seed=5, batch=batch, kv_bits=4, kv_group=group, **options)
    a, b = make(), make()
    plain = Plain(b, group, a)
    prompt = torch.randint(0, cfg.vocab, (batch, 45), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    la, lb = a.prefill(prompt), b.prefill(prompt)
    scale = float(lb.float().abs().max())
    assert float((la.float() - lb.float()).abs().max()) <= 2e-2 * scale
    for _ in range(60):
        a.tok.copy_(b.tok)
        a._kv4_room(), b._kv4_room()
        la, lb = a._step(), b._step()
        assert float((la.float() - lb.float()).abs().max()) <= 2e-2 * scale
    if a.kv_budget is not None:
        assert a.length.tolist() == [a.length_host] * batch and a.length_host == plain.k[0].shape[2] <= a.slots


@pytest.mark.parametrize("options", [dict(), dict(window=30, sinks=4), dict(kv_budget=32, kv_slack=8, sinks=4)])
def test_graph_replay_equals_eager_steps(dec, options):
    cfg = tiny(dec, 2, 128)
    prompt = torch.randint(0, cfg.vocab, (2, 50), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    a = dec.CherryDecoder(cfg, seed=7, batch=2, kv_bits=4, **options)
    a.prefill(prompt)
    eager = a.generate(60, use_graph=False)
    a.prefill(prompt)
    graphed = a.generate(60, use_graph=True)
    assert torch.equal(eager, graphed)
    a.prefill(prompt)                                     # the graph serves another prompt
    assert torch.equal(a.generate(60), eager)


def test_a_prompt_shorter_than_the_budget_loses_nothing(dec):
    cfg = tiny(dec)
    prompt = torch.randint(0, cfg.vocab, (20,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    a = dec.CherryDecoder(cfg, seed=9, kv_bits=4)
    b = dec.CherryDecoder(cfg, seed=9, kv_bits=4, kv_budget=64, kv_slack=64)
    assert torch.equal(a.prefill(prompt), b.prefill(prompt))
    assert torch.equal(a.generate(80), b.generate(80))


def test_refusals(dec):
    cfg = tiny(dec)
    for bad in (dict(kv_bits=8), dict(window=4), dict(sinks=4), dict(kv_budget=64), dict(kv_bits=4, window=-1), dict(kv_bits=4, attention="flash"),
                dict(kv_bits=4, kv_budget=0), dict(kv_bits=4, kv_budget=8, sinks=4, kv_recent=5), dict(kv_bits=4, kv_budget=8, kv_slack=0)):
        with pytest.raises(ValueError):
            dec.CherryDecoder(cfg, **bad)
    with pytest.raises(ValueError):
        dec.CherryDecoder(tiny(dec, 4, 32), kv_bits=4)
    with pytest.raises(RuntimeError):
        dec.CherryDecoder(cfg, kv_bits=4, kv_group=16)
    a = dec.CherryDecoder(cfg, kv_bits=4, kv_budget=32)
    a.prefill(torch.zeros(100, dtype=torch.long, device="cuda"))
    with pytest.raises(ValueError):
        a.generate(200)


def test_a_window_over_a_bounded_cache(dec):
    """Slots of a bounded cache are not positions once some are evicted: a window that could hide any is refused there, one that spans
    all positions changes nothing."""
    cfg = tiny(dec)
    for window in (1, 100, cfg.max_seq - 1):
        with pytest.raises(ValueError, match="window"):
            dec.CherryDecoder(cfg, kv_bits=4, kv_budget=32, kv_slack=16, window=window, sinks=2)
    prompt = torch.randint(0, cfg.vocab, (60,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    a = dec.CherryDecoder(cfg, seed=11, kv_bits=4, kv_budget=32, kv_slack=16, sinks=2)
    b = dec.CherryDecoder(cfg, seed=11, kv_bits=4, kv_budget=32, kv_slack=16, sinks=2, window=cfg.max_seq)
    assert torch.equal(a.prefill(prompt), b.prefill(prompt))
    assert torch.equal(a.generate(50), b.generate(50))


@pytest.mark.parametrize("options", [dict(), dict(window=20, sinks=2), dict(kv_budget=32, kv_slack=16, sinks=2, kv_recent=8, kv_observe=16)])
def test_two_ranks_of_a_group(dec, options, monkeypatch):
    """Each rank keeps the cache of its own heads.  Both ranks run on one device, a thread each, one behind the other on its stream; their
    slices meet on the host's side.  One layer, so that all sides quantise the same rows (see above)."""
    import threading
    cfg = tiny(dec, layers=1)
    prompt = torch.randint(0, cfg.vocab, (2, 45), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))

    def run(model, tokens):
        logits = [model.prefill(prompt).clone()]
        for i in range(40):
            if i < len(tokens):
                model.tok.copy_(tokens[i])
            else:
                tokens.append(model.tok.clone())
            model._kv4_room()
            logits.append(model._step().clone())
        return logits

    tokens = []
    want = run(dec.CherryDecoder(cfg, seed=5, batch=2, kv_bits=4, **options), tokens)
    monkeypatch.setattr("torch.distributed.get_world_size", lambda group: 2)
    monkeypatch.setattr("torch.distributed.get_rank", lambda group: group)
    ranks = [dec.CherryDecoder(cfg, seed=5, batch=2, kv_bits=4, tp_group=r, tp_gather="nccl", **options) for r in (0, 1)]
    slices, meet, got = [None, None], threading.Barrier(2, timeout=60), [None, None]

    def gather(r):
        def call(x):
            slices[r] = x
            meet.wait()
            both = torch.cat(slices, 1)
            meet.wait()
            return both
        return call

    def work(r):
        try:
            got[r] = run(ranks[r], list(tokens))
        except BaseException:
            meet.abort()
            raise
    for r in (0, 1):
        ranks[r]._gather = gather(r)
        assert ranks[r].caches[0].n_kv_heads == cfg.n_kv_heads // 2
    threads = [threading.Thread(target=work, args=(r,)) for r in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for r in (0, 1):
        assert len(got[r]) == len(want)
        for x, y in zip(got[r], want):
            assert float((x.float() - y.float()).abs().max()) <= 2e-2 * float(y.float().abs().max())
