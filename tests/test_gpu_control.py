"""Control over what is picked, where calls go wrong or come in other forms: refused calls, prompts of other types and places, sequences
without a prompt."""
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
CACHES = [dict(), dict(kv_bits=4), dict(kv_page=16)]


@pytest.fixture(scope="module")
def dec():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from cherryq_b200 import decoder
    return decoder


def tiny(dec, max_seq=256, vocab=1003):
    return dec.DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, ffn=512, vocab=vocab, bits=4, group=128, cherry_fraction=1 / 32,
                             max_seq=max_seq)


def tokens(cfg, *shape, seed=1):
    return torch.randint(0, cfg.vocab, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def cycle(vocab, steps):
    """A grammar that allows tokens 10 s .. 10 s + 9 in state s, one state after the other"""
    masks, follow = torch.zeros(steps, -(-vocab // 32), dtype=torch.int64), torch.full((steps, vocab), -1, dtype=torch.int32)
    for s in range(steps):
        for t in range(10 * s, 10 * s + 10):
            masks[s, t // 32] |= 1 << (t % 32)
        follow[s, 10 * s:10 * s + 10] = (s + 1) % steps
    return torch.where(masks >= 1 << 31, masks - (1 << 32), masks).to(torch.int32), follow


@pytest.mark.parametrize("options", CACHES)
@pytest.mark.parametrize("use_graph", [False, True])
def test_refused_calls_change_nothing(dec, options, use_graph):
    """The grammar, its states and the penalties that are active stay so"""
    cfg = tiny(dec)
    a, b = (dec.CherryDecoder(cfg, seed=3, batch=2, **options) for _ in range(2))
    masks, follow = cycle(cfg.vocab, 5)
    prompt = tokens(cfg, 2, 12)
    for m in (a, b):
        m.control(grammar=(masks, follow), repetition=1.3)
        m.prefill(prompt)
        m.generate(3, use_graph)
    graph = a.graph
    for bad in (dict(grammar=(masks[:, :-1], follow)), dict(grammar=(masks, follow + 5)), dict(grammar=(masks, follow[:, :-1])),
                dict(grammar=(masks.long(), follow)), dict(repetition=[1.0, 2.0, 3.0]), dict(presence="a"), dict(bias={1: "b"}),
                dict(repetition=2.0, frequency=[0.1, 0.2, 0.3]), dict(bias={2: 1.0}, grammar=(masks[:4], follow))):
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            a.control(**bad)
    assert a.graph is graph
    x, y = a.generate(20, use_graph), b.generate(20, use_graph)
    assert torch.equal(x, y)
    for i, row in enumerate(x.tolist()):
        assert all(t // 10 == (3 + i) % 5 for t in row)
    a.prefill(prompt), b.prefill(prompt)
    assert torch.equal(a.generate(10, use_graph), b.generate(10, use_graph))
    # and a call that is not refused takes their place
    a.control(presence=0.5), b.control(presence=0.5)
    a.prefill(prompt), b.prefill(prompt)
    assert torch.equal(a.generate(10, use_graph), b.generate(10, use_graph))


@pytest.mark.parametrize("options", CACHES)
@pytest.mark.parametrize("form", ["int32", "int16", "host", "host int32"])
def test_prompts_of_other_types_and_places(dec, options, form):
    """With penalties as without them"""
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=4, batch=2, **options)
    prompt = tokens(cfg, 2, 30)
    other = prompt.to("cpu" if "host" in form else "cuda", torch.int32 if "int32" in form else torch.int16 if "int16" in form else torch.long)
    for control in (dict(), dict(repetition=1.5, presence=0.3, frequency=[0.1, 0.4])):
        a.control(**control)
        want = a.prefill(prompt), a.generate(12)
        got = a.prefill(other), a.generate(12)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    if "kv_page" in options:
        want = a.prefill(prompt[1:], [20], rows=[1]), a.generate(5)
        a.prefill(prompt), a.generate(12)
        a.prefill(prompt), a.prefill(prompt[1:], [20], rows=[1])
        want = a.generate(5)
        a.prefill(prompt), a.prefill(other[1:], [20], rows=[1])
        assert torch.equal(a.generate(5), want)


@pytest.mark.parametrize("options", CACHES)
def test_prompts_that_are_no_tokens(dec, options):
    """Refused before anything is changed"""
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=4, batch=2, **options)
    prompt = tokens(cfg, 2, 30)
    a.prefill(prompt)
    want = a.generate(10)
    a.prefill(prompt)
    for bad in (prompt.float(), prompt.half(), prompt > 5):
        with pytest.raises(ValueError, match="whole numbers"):
            a.prefill(bad)
    assert a.held == [30, 30] and a.pos.tolist() == [30, 30] and torch.equal(a.generate(10), want)


def test_repetition_is_positive(dec):
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=4, batch=2, kv_page=16)
    for bad in (0, 0.0, -1.0, [1.2, 0.0], [-0.5, 2.0], float("nan")):
        with pytest.raises(ValueError, match="repetition"):
            a.control(repetition=bad)
    assert a.controls is None
    a.control(repetition=[1e-3, 5.0], presence=-1.0, frequency=0.0)       # the others may be any number


@pytest.mark.parametrize("control", [dict(), dict(repetition=1.2, frequency=0.1)])
@pytest.mark.parametrize("use_graph", [False, True])
def test_sequences_without_a_prompt_stay_where_they_are(dec, control, use_graph):
    """Positions of released sequences, and of those that had no prompt yet, do not count up: steps look for nothing in pages that they
    do not have"""
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=5, batch=3, kv_page=16)
    if control:
        a.control(**control)
    prompt = tokens(cfg, 3, 20)
    a.prefill(prompt[:1], rows=[0])
    a.generate(10, use_graph)
    assert a.pos.tolist() == [30, 0, 0]
    a.prefill(prompt[1:], rows=[2, 1])
    a.generate(10, use_graph)
    assert a.pos.tolist() == [40, 30, 30]
    a.release([1])
    for _ in range(3):
        a.generate(20, use_graph)
    assert a.pos.tolist() == [100, 0, 90] and a.held == [100, 0, 90]
    # the next prompt counts again, as one that came first
    a.prefill(prompt[:1], rows=[1])
    got = a.generate(15, use_graph)[:, 1]
    assert a.pos.tolist() == [115, 35, 105]
    b = dec.CherryDecoder(cfg, seed=5, batch=3, kv_page=16)
    if control:
        b.control(**control)
    b.prefill(prompt[:1].expand(3, -1))
    assert torch.equal(b.generate(15, use_graph)[:, 1], got)


@pytest.mark.parametrize("options", CACHES)
def test_masks_of_any_strides(dec, options):
    """Masks whose words do not lie one behind the other"""
    cfg = tiny(dec)
    a, b = (dec.CherryDecoder(cfg, seed=6, batch=2, **options) for _ in range(2))
    masks, follow = cycle(cfg.vocab, 5)
    prompt = tokens(cfg, 2, 12)
    b.control(grammar=(masks, follow)), b.prefill(prompt)
    want = b.generate(10)
    wide = torch.zeros(5, 2 * masks.shape[1], dtype=torch.int32, device="cuda")
    wide[:, ::2] = masks.cuda()
    for form in (masks.T.contiguous().T, masks.cuda().T.contiguous().T, wide[:, ::2], masks.cuda()):
        a.control(grammar=(form, follow))
        a.prefill(prompt)
        assert torch.equal(a.generate(10), want)


def test_memory_of_a_grammar(dec):
    """4 bytes a state and token for the states that follow, a bit for the masks"""
    cfg = tiny(dec)
    a = dec.CherryDecoder(cfg, seed=6, batch=2, kv_page=16)
    masks, follow = torch.zeros(2000, 32, dtype=torch.int32), torch.full((2000, cfg.vocab), -1, dtype=torch.int64)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    a.control(grammar=(masks, follow))
    assert torch.cuda.memory_allocated() - before < 2000 * (4 * cfg.vocab + 128) + 100000


@pytest.mark.parametrize("dtype,none", [(torch.int8, -100), (torch.int32, -2 ** 31), (torch.int64, -2 ** 40), (torch.int64, -2 ** 32 + 1)])
def test_states_below_none(dec, dtype, none):
    """Any negative state is none"""
    cfg = tiny(dec)
    masks, follow = cycle(cfg.vocab, 3)
    follow[2] = -1
    got = []
    for f in (follow, torch.where(follow < 0, none, follow.long()).to(dtype)):
        a = dec.CherryDecoder(cfg, seed=6, batch=2, kv_page=16)
        a.control(grammar=(masks, f))
        a.prefill(tokens(cfg, 2, 12))
        got.append(a.generate(20))
    assert torch.equal(*got)
