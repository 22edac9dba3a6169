"""The decode harness on a paged cache, and with control over what is picked: against the contiguous cache, single sequences, torch
expressions on the logits; graph replay against eager steps."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cherryq_b200 import decoder
    return decoder


def tiny(dec, kv_heads=2, head_dim=64, max_seq=256, layers=2, vocab=1000):
    return dec.DecoderConfig(n_layers=layers, hidden=4 * head_dim, n_heads=4, n_kv_heads=kv_heads, ffn=512, vocab=vocab, bits=4, group=128,
                             cherry_fraction=1 / 32, max_seq=max_seq)


def tokens(cfg, *shape, seed=1):
    return torch.randint(0, cfg.vocab, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def near(x, y):
    assert float((x.float() - y.float()).abs().max()) <= 2e-2 * float(y.float().abs().max())


def step_with(model, token):
    """One eager step on the given tokens"""
    model.tok.copy_(token)
    if model.kv_page:
        model._pages_reserve({r: x + 1 for r, x in enumerate(model.held) if x})
    logits = model._step()
    model.held = [x + 1 if x else 0 for x in model.held]
    return logits


@pytest.mark.parametrize("page,kv,head_dim", [(16, 2, 64), (64, 4, 128), (256, 1, 64)])
def test_against_the_contiguous_cache(dec, page, kv, head_dim):
    cfg = tiny(dec, kv, head_dim)
    a, b = dec.CherryDecoder(cfg, seed=5, batch=3, kv_page=page), dec.CherryDecoder(cfg, seed=5, batch=3)
    prompt = tokens(cfg, 3, 45)
    near(a.prefill(prompt), b.prefill(prompt))
    for _ in range(60):
        token = b.tok.clone()
        near(step_with(a, token), step_with(b, token))


@pytest.mark.parametrize("options", [dict(), dict(window=20, sinks=2)])
def test_prompts_of_different_lengths(dec, options):
    """Each sequence of a batch gives what it gives alone"""
    cfg = tiny(dec)
    lengths = [50, 7, 33, 1]
    prompt = tokens(cfg, 4, 50)
    a = dec.CherryDecoder(cfg, seed=6, batch=4, kv_page=16, **options)
    logits = a.prefill(prompt, lengths)
    assert a.held == lengths and a.pos.tolist() == lengths and a.page_table.held == [4, 1, 3, 1]
    singles = []
    for i, n in enumerate(lengths):
        b = dec.CherryDecoder(cfg, seed=6, kv_page=32, **options)
        near(logits[i:i + 1], b.prefill(prompt[i, :n]))
        singles.append(b)
    for _ in range(40):
        token = a.tok.clone()
        logits = step_with(a, token)
        for i, b in enumerate(singles):
            near(logits[i:i + 1], step_with(b, token[i:i + 1]))


@pytest.mark.parametrize("options", [dict(), dict(window=30, sinks=4)])
def test_graph_replay_equals_eager_steps(dec, options):
    cfg = tiny(dec, 2, 128)
    prompt, lengths = tokens(cfg, 2, 50, seed=2), [50, 21]
    a = dec.CherryDecoder(cfg, seed=7, batch=2, kv_page=16, **options)
    a.prefill(prompt, lengths)
    eager = a.generate(60, use_graph=False)
    a.prefill(prompt, lengths)
    assert torch.equal(a.generate(60), eager)
    a.prefill(prompt[:, :20])                             # the graph serves other prompts, and the old ones again
    a.generate(10)
    a.prefill(prompt, lengths)
    assert torch.equal(a.generate(25), eager[:25]) and torch.equal(a.generate(35), eager[25:])


def test_sequences_come_and_go(dec):
    """A sequence gets another prompt, another one gives its pages back, while the third goes on as if alone"""
    cfg = tiny(dec)
    prompt = tokens(cfg, 3, 40, seed=3)
    alone = dec.CherryDecoder(cfg, seed=8, batch=3, kv_page=16)
    alone.prefill(prompt)
    want = torch.cat([alone.generate(10), alone.generate(10), alone.generate(10)])
    a = dec.CherryDecoder(cfg, seed=8, batch=3, kv_page=16, kv_pages=3 * 5 + 2)
    a.prefill(prompt)
    got = [a.generate(10)]
    a.prefill(tokens(cfg, 1, 25, seed=4), [20], rows=[1])
    assert a.held == [50, 20, 50] and a.pos.tolist() == [50, 20, 50]
    got.append(a.generate(10))
    a.release([2])
    assert a.page_table.held == [4, 2, 0] and a.held == [60, 30, 0]
    got.append(a.generate(10))
    got = torch.cat(got)
    assert torch.equal(got[:, 0], want[:, 0]) and torch.equal(got[:20, 2], want[:20, 2])
    # the new prompt as it is alone in a batch of the same size
    b = dec.CherryDecoder(cfg, seed=8, batch=3, kv_page=16)
    b.prefill(tokens(cfg, 1, 25, seed=4).expand(3, -1), [20] * 3)
    assert torch.equal(torch.cat([b.generate(10), b.generate(10)])[:, 1], got[10:, 1])
    # pages run out: nothing has happened
    held, table = list(a.held), a.table.clone()
    with pytest.raises(ValueError, match="pages"):
        a.generate(180)
    with pytest.raises(ValueError, match="pages"):
        a.prefill(tokens(cfg, 2, 200), rows=[1, 2])
    assert a.held == held and torch.equal(a.table, table)
    a.generate(5)


@pytest.mark.parametrize("pad", [-1, 1000, 1 << 40])
def test_what_stands_behind_a_prompt(dec, pad):
    """Any number pads a batch, on the host too"""
    cfg = tiny(dec)
    lengths = [9, 30, 1]
    prompt = tokens(cfg, 3, 30)
    a = dec.CherryDecoder(cfg, seed=6, batch=3, kv_page=16)
    a.control(repetition=1.5)
    want = a.prefill(prompt, lengths)
    told = a.generate(5)
    for r, n in enumerate(lengths):
        prompt[r, n:] = pad
    assert torch.equal(a.prefill(prompt, lengths), want) and torch.equal(a.generate(5), told)
    assert torch.equal(a.prefill(prompt.cpu(), lengths), want)


def test_released_sequences_start_anew(dec):
    """Their positions, which go on meanwhile, are none of their next prompt's"""
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=6, batch=2, kv_page=16)
    a.prefill(tokens(cfg, 2, 20))
    a.generate(100)
    a.release([0, 0])
    a.release([])
    assert a.pos.tolist() == [0, 120] and a.held == [0, 120] and a.pos_host == 120
    a.generate(100)
    assert a.held == [0, 220] and a.page_table.held == [0, 14]
    a.release([1])
    for _ in range(2):
        a.generate(200)                      # nobody is left
    assert a.held == [0, 0] and len(a.page_table.free) == a.page_table.pages
    one = a.prefill(tokens(cfg, 1, 20, seed=3), rows=[0])
    b = dec.CherryDecoder(cfg, seed=6, batch=1, kv_page=16)
    near(one, b.prefill(tokens(cfg, 1, 20, seed=3)))
    for rows in ([-1], [2], [0, 2]):
        with pytest.raises(ValueError):
            a.release(rows)
    assert a.held == [20, 0]


def test_refusals(dec):
    cfg = tiny(dec)
    for bad in (dict(kv_page=-16), dict(kv_pages=4), dict(kv_page=16, kv_pages=0), dict(kv_page=16, kv_bits=4), dict(kv_page=16, attention="flash"),
                dict(kv_page=16, kv_budget=32), dict(kv_page=16, window=-1)):
        with pytest.raises(ValueError):
            dec.CherryDecoder(cfg, **bad)
    with pytest.raises(ValueError):
        dec.CherryDecoder(tiny(dec, 4, 32), kv_page=16)
    with pytest.raises(RuntimeError):
        dec.CherryDecoder(cfg, kv_page=24)
    a, plain = dec.CherryDecoder(cfg, batch=2, kv_page=16), dec.CherryDecoder(cfg, batch=2)
    p = tokens(cfg, 2, 10)
    for lengths, rows in (([10], None), ([10, 0], None), ([11, 3], None), (None, [0]), (None, [0, 0]), (None, [1, 2]), (None, [-1, 0])):
        with pytest.raises(ValueError):
            a.prefill(p, lengths, rows)
    with pytest.raises(ValueError):
        a.prefill(tokens(cfg, 2, 256))
    for call in (lambda: plain.prefill(p, [3, 4]), lambda: plain.prefill(p, rows=[0, 1]), lambda: plain.release([0])):
        with pytest.raises(ValueError):
            call()
    a.prefill(p)
    with pytest.raises(ValueError):
        a.generate(247)


# ---------------------------------------------------------------------------------- control
def adjusted(logits, history, prompt, c):
    """What adjust_logits gives, on the host, an operation after the other in 32 bits"""
    x = logits.float().cpu()
    for r in range(len(x)):
        seen = set(history[r])
        made = {t: history[r][prompt[r]:].count(t) for t in set(history[r][prompt[r]:])}
        for t in seen:
            if "repetition" in c:
                rep = torch.tensor(c["repetition"][r], dtype=torch.float32)
                x[r, t] = x[r, t] / rep if x[r, t] > 0 else x[r, t] * rep
        for t, n in made.items():
            if "frequency" in c:
                x[r, t] = x[r, t] - torch.tensor(c["frequency"][r], dtype=torch.float32) * n
            if "presence" in c:
                x[r, t] = x[r, t] - torch.tensor(c["presence"][r], dtype=torch.float32)
        for t, b in c.get("bias", {}).items():
            x[r, t] = x[r, t] + b
    return x


@pytest.mark.parametrize("options", [dict(), dict(kv_page=16), dict(kv_bits=4)])
@pytest.mark.parametrize("control", [dict(repetition=[1.3, 2.0]), dict(presence=[0.5, 1.5], frequency=[0.2, 0.7], bias={3: 2.0, 500: -1.0}),
                                     dict(repetition=[1.1, 1.0], presence=[0.1, 0.0], frequency=[0.3, 0.1])])
def test_penalties_and_biases(dec, options, control):
    """Tokens are those that the same model's bare logits give, adjusted with the sequences' histories"""
    cfg = tiny(dec)
    a, b = (dec.CherryDecoder(cfg, seed=9, batch=2, **options) for _ in range(2))
    prompt, lengths = tokens(cfg, 2, 30, seed=5), [30, 12] if "kv_page" in options else [30, 30]
    a.control(**control)
    more = (lengths,) if "kv_page" in options else ()
    a.prefill(prompt, *more)
    bare = b.prefill(prompt, *more)
    history = [prompt[r, :n].tolist() for r, n in enumerate(lengths)]
    picked = [a.tok.clone()]
    for _ in range(30):
        want = adjusted(bare, history, lengths, control).argmax(-1).cuda()
        assert torch.equal(picked[-1], want)
        for r in range(2):
            history[r].append(int(want[r]))
        bare = step_with(b, want)
        step_with(a, picked[-1])
        picked.append(a.tok.clone())
    a.prefill(prompt, *more)
    assert torch.equal(a.generate(31), torch.stack(picked))       # and in a graph
    # without control: the bare model again
    a.control()
    b.prefill(prompt, *more), a.prefill(prompt, *more)
    assert torch.equal(a.generate(20), b.generate(20))


def test_control_in_the_middle(dec):
    """Penalties begin with a sequence's next prompt: what was not noted does not count"""
    cfg = tiny(dec)
    prompt = tokens(cfg, 2, 20, seed=8)
    a, b = (dec.CherryDecoder(cfg, seed=12, batch=2, kv_page=16) for _ in range(2))
    a.prefill(prompt), b.prefill(prompt)
    a.generate(5), b.generate(5)
    a.control(repetition=3.0, presence=2.0)
    assert torch.equal(a.generate(20), b.generate(20))
    a.prefill(prompt[:1], rows=[0]), b.prefill(prompt[:1], rows=[0])
    x, y = a.generate(20), b.generate(20)
    assert torch.equal(x[:, 1], y[:, 1]) and not torch.equal(x[:, 0], y[:, 0])
    assert len(set(x[:, 0].tolist())) > len(set(y[:, 0].tolist())) or len(set(y[:, 0].tolist())) == 20


def test_grammar(dec):
    """Sequences follow an automaton; behind a token without a next state everything is allowed; the mask of an empty state gives token 0"""
    cfg = tiny(dec, vocab=1003)
    words = (cfg.vocab + 31) // 32
    allowed = [[5, 900], [6, 1002], list(range(100, 200)), []]
    follow = torch.full((4, cfg.vocab), -1, dtype=torch.int32)
    follow[0, 5], follow[0, 900] = 1, 2
    follow[1, 6], follow[1, 1002] = 0, 0
    follow[2, 100:200] = 3
    masks = torch.zeros(4, words, dtype=torch.int64)
    for s, some in enumerate(allowed):
        for t in some:
            masks[s, t // 32] |= 1 << (t % 32)
    masks = torch.where(masks >= 1 << 31, masks - (1 << 32), masks).to(torch.int32)
    a = dec.CherryDecoder(cfg, seed=10, batch=3, kv_page=16)
    a.control(grammar=(masks, follow), frequency=0.3)
    prompt = tokens(cfg, 3, 20, seed=6)
    a.prefill(prompt, [20, 5, 11])
    eager = a.generate(40, use_graph=False)
    a.prefill(prompt, [20, 5, 11])
    out = a.generate(40)
    assert torch.equal(out, eager)
    for r in range(3):
        state = 0
        for t in out[:, r].tolist():
            if state >= 0:
                assert t in allowed[state] or (not allowed[state] and t == 0)
                state = int(follow[state, t])
    with pytest.raises(ValueError):
        a.control(grammar=(masks[:, :-1], follow))
    with pytest.raises(ValueError):
        a.control(grammar=(masks, follow + 4))
    with pytest.raises(ValueError):
        a.control(grammar=(masks, follow[:3]))


def test_everything_in_one_graph(dec):
    """A model's tokens with all of it in one graph: pages, a window, penalties"""
    cfg = tiny(dec, 4, 128, max_seq=300)
    a = dec.CherryDecoder(cfg, seed=11, batch=5, kv_page=32, kv_pages=40, window=50, sinks=4)
    a.control(repetition=1.2, frequency=[0.1, 0.2, 0.3, 0.4, 0.5])
    prompt, lengths = tokens(cfg, 5, 120, seed=7), [120, 3, 77, 64, 100]
    a.prefill(prompt, lengths)
    eager = a.generate(30, use_graph=False)
    a.prefill(prompt, lengths)
    assert torch.equal(a.generate(30), eager)
    assert eager.shape == (30, 5) and int(eager.min()) >= 0 and int(eager.max()) < cfg.vocab
