"""The operators of long-context serving with a bounded 4-bit KV cache: what is timed, their plain forms and exact results.

Kinds of work and the calls that a user makes for them:
  step     `KVCache4.step`: one new token of every sequence: rotary embedding, its key and value quantised into the cache,
           attention over the cache; the written row is read back with `KVCache4.read`
  attend   `KVCache4.attend`: attention of one query per sequence over the cache, optionally with the weight that every slot
           received added to an accumulator
  write    `KVCache4.write`: a prompt's keys and values rotated and quantised into the cache, read back with `KVCache4.read`
  evict    `KVCache4.evict`: the slots with the most accumulated weight, the first and the last ones kept, in another cache;
           read back with `KVCache4.read`
  prompt   `attn_prefill`: causal attention of prompts with a sliding window and a few first tokens that stay visible
  mass     `attn_prefill_weights`: the weight that each position of a prompt received from its last queries

A cache row holds a head's D columns in 4 bits: groups of 32 or 64 columns with a scale s and a minimum m in fp16, a column's
value is s * code + m; two codes a byte, the even column in the low half.  Tensors: codes (B, KV, S, D / 2) uint8, scales
(B, KV, S, D / group, 2) fp16 = (s, m).

Head counts are those of LLaMA-2 7B / 13B / 70B (the configurations of `decoder.py`) and a small 64-wide one.
"""
import math

import torch

own = False

HEADS = {
    "7b": (32, 32, 128),
    "13b": (40, 40, 128),
    "70b": (64, 8, 128),
    "small": (16, 4, 64),
}
MAX_SCORES = 64 * 8192 * 8192          # query x key pairs of all heads that a plain form holds at once
MAX_CACHE = 1 << 29                    # columns of a cache that a plain form holds in 32 bits


def listed():
    return [
        # interactive decoding: one 7B layer, one sequence, short context: launch latency
        {"name": "step_7b_b1", "kind": "step", "heads": "7b", "group": 32, "batch": 1, "slots": 512, "held": 256, "ragged": False, "window": 0, "sinks": 0},
        # sixteen 70B sequences (grouped queries) near the end of a 4096-position cache
        {"name": "step_70b_b16", "kind": "step", "heads": "70b", "group": 32, "batch": 16, "slots": 4096, "held": 4001, "ragged": True, "window": 0, "sinks": 0},
        # a serving batch of mixed lengths whose layers look back 1021 positions and at four sinks
        {"name": "attend_13b_window", "kind": "attend", "heads": "13b", "group": 64, "batch": 8, "slots": 2304, "held": 2113, "ragged": True, "window": 1021, "sinks": 4, "weights": False},
        # long documents: four caches of 65531 positions, with the weights that an eviction goes by
        {"name": "attend_70b_long", "kind": "attend", "heads": "70b", "group": 32, "batch": 4, "slots": 65536, "held": 65531, "ragged": False, "window": 0, "sinks": 0, "weights": True},
        # a 2048-token prompt of one 13B layer into its cache
        {"name": "write_13b_2048", "kind": "write", "heads": "13b", "group": 32, "batch": 1, "slots": 4096, "tokens": 2048, "held": 0},
        # a few short follow-up prompts behind what the caches hold, 64-wide heads, an odd length
        {"name": "write_small_77", "kind": "write", "heads": "small", "group": 64, "batch": 5, "slots": 1024, "tokens": 77, "held": 333},
        # sixteen 70B caches cut from about 4000 positions to a budget of 1024
        {"name": "evict_70b_b16", "kind": "evict", "heads": "70b", "group": 32, "batch": 16, "slots": 4096, "held": 4090, "ragged": True, "keep": 1024, "sinks": 4, "recent": 256},
        # one 7B cache behind its prompt, an odd budget
        {"name": "evict_7b_b1", "kind": "evict", "heads": "7b", "group": 64, "batch": 1, "slots": 2304, "held": 2100, "ragged": False, "keep": 525, "sinks": 4, "recent": 64},
        # a 2048-token prompt of one 13B layer, full causal attention
        {"name": "prompt_13b_2048", "kind": "prompt", "heads": "13b", "batch": 1, "queries": 2048, "keys": 2048, "ragged": False, "window": 0, "sinks": 0},
        # a long 70B prompt with a sliding window and sinks
        {"name": "prompt_70b_8192_window", "kind": "prompt", "heads": "70b", "batch": 1, "queries": 8192, "keys": 8192, "ragged": False, "window": 2048, "sinks": 4},
        # the weights of a 13B prompt's positions from all of its queries
        {"name": "mass_13b_2048", "kind": "mass", "heads": "13b", "batch": 1, "queries": 2048, "keys": 2048, "ragged": False, "window": 0, "sinks": 0, "observe": 2048},
        # the same from the last 64 queries of three long 70B prompts of mixed lengths
        {"name": "mass_70b_last64", "kind": "mass", "heads": "70b", "batch": 3, "queries": 4000, "keys": 4000, "ragged": True, "window": 0, "sinks": 0, "observe": 64},
    ]


# ---------------------------------------------------------------------------------- drawn cases
def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = [work(c) for c in listed()]
    nbytes, flops = max(w["bytes"] for w in most), max(w["flops"] for w in most)
    while True:
        case = _draw(rng)
        w = work(case)
        h, kv, d = HEADS[case["heads"]]
        if w["bytes"] > nbytes or w["flops"] > flops:
            continue
        if "slots" in case and case["batch"] * kv * case["slots"] * d > MAX_CACHE:
            continue
        if "queries" in case and case["batch"] * h * case["queries"] * case["keys"] > MAX_SCORES:
            continue
        return case


def _draw(rng):
    kind = rng.choice(["step", "step", "attend", "attend", "attend", "write", "write", "evict", "evict", "prompt", "prompt", "prompt", "mass"])
    heads = rng.choice(sorted(HEADS))
    batch = _log_int(rng, 1, 32)
    if kind in ("prompt", "mass"):
        keys = _log_int(rng, 16, 8192)
        case = {"kind": kind, "heads": heads, "batch": min(batch, 4), "keys": keys,
                "queries": keys if rng.random() < 0.7 else rng.randint(1, keys), "ragged": rng.random() < 0.4}
        case.update(window=0 if rng.random() < 0.4 else _log_int(rng, 8, keys + 8), sinks=rng.choice([0, 1, 4, 64]))
        if kind == "mass":
            case["observe"] = keys if rng.random() < 0.5 else _log_int(rng, 1, 512)
        return case
    held = _log_int(rng, 1, 65536)
    case = {"kind": kind, "heads": heads, "group": rng.choice([32, 64]), "batch": batch}
    if kind == "write":
        tokens = _log_int(rng, 1, 4096)
        held = rng.randint(0, 2048)
        case.update(slots=(held + tokens + rng.randint(0, 600) + 31) // 32 * 32, tokens=tokens, held=held)
        return case
    case.update(slots=(held + 1 + rng.randint(0, 600) + 31) // 32 * 32, held=held, ragged=rng.random() < 0.5)
    if kind == "evict":
        sinks, recent = min(rng.choice([0, 4, 16]), held), rng.randint(0, held // 4)
        case.update(sinks=sinks, recent=recent, keep=min(held, sinks + recent + rng.randint(0, max(1, held // 2))))
        case["keep"] = max(1, case["keep"])
        return case
    case.update(window=0 if rng.random() < 0.5 else _log_int(rng, 8, held + 8), sinks=rng.choice([0, 1, 4, 64]))
    if kind == "attend":
        case["weights"] = rng.random() < 0.4
    return case


# ---------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _keys(g, *shape):
    """Keys as trained models have them: a few columns of a head much larger than the rest."""
    x = _normal(g, *shape)
    x[..., 3::37] *= 4.0
    return x.half()


def _lengths(case, g):
    n = case["held"] if "held" in case else case["keys"]
    length = torch.full((case["batch"],), n, device="cuda", dtype=torch.int64)
    if case.get("ragged"):
        less = torch.rand(case["batch"], device="cuda", generator=g) * (0.5 * n)
        less[0] = 0
        length -= less.long()
    return length


def _tables(positions, d):
    inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
    ang = torch.outer(torch.arange(positions, device="cuda", dtype=torch.float32), inv)
    return ang.cos(), ang.sin()


def _filled(case, g, kv, d):
    """A cache whose rows hold quantised random keys and values."""
    shape = (case["batch"], kv, case["slots"], d)
    out = []
    for make in (_keys, lambda g, *s: _normal(g, *s).half()):
        codes, scales = _quantise(make(g, *shape).float(), case["group"])
        out += [codes, scales]
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, kv, d = HEADS[case["heads"]]
    b, kind = case["batch"], case["kind"]
    st = {"case": case, "kind": kind}
    if kind in ("prompt", "mass"):
        st["q"] = _normal(g, b, case["queries"], h, d).half()
        st["k"] = _keys(g, b, case["keys"], kv, d)
        st["v"] = _normal(g, b, case["keys"], kv, d).half()
        st["lengths"] = _lengths(case, g) if case["ragged"] else None
        if kind == "mass":
            st["lse"] = _plain_prompt(st)[1]
            del st["v"]
    elif kind == "write":
        t = case["tokens"]
        st["k_codes"], st["k_scales"], st["v_codes"], st["v_scales"] = _empty_cache(b, kv, case["slots"], d, case["group"])
        st["q"] = _normal(g, b * t, h, d).half()
        st["k"] = _keys(g, b * t, kv, d)
        st["v"] = _normal(g, b * t, kv, d).half()
        st["cos"], st["sin"] = _tables(case["slots"], d)
        st["first"] = torch.full((b,), case["held"], device="cuda", dtype=torch.int64)
        st["positions"] = (case["held"] + torch.arange(t, device="cuda")).repeat(b)
    else:
        st["length"] = _lengths(case, g)
        st["k_codes"], st["k_scales"], st["v_codes"], st["v_scales"] = _filled(case, g, kv, d)
        if kind == "step":
            st["q"] = _normal(g, b, h, d).half()
            st["k"] = _keys(g, b, kv, d)
            st["v"] = _normal(g, b, kv, d).half()
            st["cos"], st["sin"] = _tables(case["slots"], d)
            st["positions"] = st["length"].clone()
        elif kind == "attend":
            st["q"] = _normal(g, b, h, d).half()
            st["weights"] = torch.rand(b, kv, case["slots"], device="cuda", generator=g) if case["weights"] else None
            st["weights_out"] = torch.zeros(b, kv, case["slots"], device="cuda") if case["weights"] else None
        else:
            # heavy-tailed, with equal weights among them (slots that no query looked at)
            w = _normal(g, b, kv, case["slots"]).mul(2).exp()
            st["weights"] = torch.where(w < 0.05, torch.zeros_like(w), w)
            st["out"] = _empty_cache(b, kv, (case["keep"] + 31) // 32 * 32, d, case["group"])
            st["zero"] = torch.zeros(b, device="cuda", dtype=torch.int64)
    if own and kind not in ("prompt", "mass"):
        import cherryq_b200
        qc = cherryq_b200.load_quant_cuda()
        st["cache"] = qc.KVCache4(st["k_codes"], st["k_scales"], st["v_codes"], st["v_scales"])
        if kind == "evict":
            st["out_cache"] = qc.KVCache4(*st["out"])
    elif own:
        import cherryq_b200
        cherryq_b200.load_quant_cuda()
    return st


def _empty_cache(b, kv, slots, d, group):
    codes = lambda: torch.zeros(b, kv, slots, d // 2, device="cuda", dtype=torch.uint8)
    scales = lambda: torch.zeros(b, kv, slots, d // group, 2, device="cuda", dtype=torch.float16)
    return codes(), scales(), codes(), scales()


# ---------------------------------------------------------------------------------- plain forms
def _quantise(x, group):
    """(codes, scales) of rows (..., D) of fp32 numbers that fit 16 bits."""
    x = x.unflatten(-1, (-1, group))
    low = x.amin(-1, keepdim=True)
    s = ((x.amax(-1, keepdim=True) - low) / 15).half()
    u = torch.where(s > 0, torch.round((x - low) / s.float()), 0.0).clamp(0, 15).to(torch.uint8).flatten(-2)
    return u[..., 0::2] | (u[..., 1::2] << 4), torch.cat([s, low.half()], -1)


def _values(codes, scales):
    """fp32 values (..., D) of codes (..., D / 2) and scales (..., D / group, 2)."""
    u = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).float().unflatten(-1, (scales.shape[-2], -1))
    return (u * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2)


def _rotate(x, cos, sin, positions):
    """Rows (T, heads, D), rotated halves, rounded to 16 bits as they are kept."""
    c, s = cos[positions][:, None], sin[positions][:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).half()


def _visible(case, length):
    j, n = torch.arange(case["slots"], device="cuda"), length[:, None]
    seen = j < n
    return seen & ((j < case["sinks"]) | (j >= n - case["window"])) if case["window"] else seen


def _plain_attend(st, q, length):
    """(output, weights per head (B, KV, G, S))"""
    case = st["case"]
    b, h, d = q.shape
    k, v = _values(st["k_codes"], st["k_scales"]), _values(st["v_codes"], st["v_scales"])
    kv = k.shape[1]
    seen = _visible(case, length)[:, None, None]         # (B, 1, 1, S)
    s = torch.matmul(q.float().view(b, kv, h // kv, d), k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, v * seen.transpose(-1, -2)).view(b, h, d).half(), p


def _prompt_scores(st, q, pos):
    """(B, KV, G, R, Tk) of the queries (B, R, H, D) at the positions (B or 1, R); -inf where a key is not seen"""
    case = st["case"]
    j, at = torch.arange(case["keys"], device="cuda"), pos[..., None]
    seen = j <= at
    if case["window"]:
        seen = seen & ((j < case["sinks"]) | (j > at - case["window"]))
    if st["lengths"] is not None:
        n = st["lengths"][:, None, None]
        seen = seen & (j < n) & (at < n)
    b, r, h, d = q.shape
    kv = st["k"].shape[2]
    q = q.float().view(b, r, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    s = torch.matmul(q, st["k"].float().permute(0, 2, 3, 1)).mul_(1.0 / math.sqrt(d))
    return s.view(b, kv, h // kv, r, -1).masked_fill_(~seen[:, None, None], -math.inf)


def _plain_prompt(st):
    b, tq, h, d = st["q"].shape
    tk = st["case"]["keys"]
    s = _prompt_scores(st, st["q"], torch.arange(tk - tq, tk, device="cuda")[None])
    top = s.amax(-1, keepdim=True)
    p = s.sub_(top.clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    kv = p.shape[1]
    o = torch.matmul(p.view(b, kv, -1, tk), st["v"].float().permute(0, 2, 1, 3)).view(b, kv, h // kv, tq, d) / total.clamp(min=1e-30)
    lse = (top + total.log()).view(b, h, tq)
    return o.permute(0, 3, 1, 2, 4).reshape(b, tq, h, d).half(), lse


def _plain_mass(st):
    """From the queries at the last positions of each prompt alone."""
    case = st["case"]
    b, tq, h, d = st["q"].shape
    first = case["keys"] - tq
    n = st["lengths"] if st["lengths"] is not None else torch.full((b,), case["keys"], device="cuda")
    pos = n[:, None] - min(case["observe"], tq) + torch.arange(min(case["observe"], tq), device="cuda")
    there = (pos >= first)[:, None, None, :, None]
    at = (pos - first).clamp(min=0)
    s = _prompt_scores(st, st["q"].gather(1, at[:, :, None, None].expand(-1, -1, h, d)), pos)
    lse = st["lse"].gather(2, at[:, None].expand(-1, h, -1)).view(*s.shape[:4], 1)
    return s.sub_(lse.clamp(min=-1e30)).exp_().masked_fill_(~there, 0.0).sum((2, 3))


def _rows(st, first, count, names=("k_codes", "k_scales", "v_codes", "v_scales")):
    """Keys and values (B, count, KV, D) of the slots first[b] .."""
    kc, ks, vc, vs = (st[n] for n in names)
    at = (torch.arange(len(first), device="cuda")[:, None], slice(None), first[:, None] + torch.arange(count, device="cuda"))
    return _values(kc[at], ks[at]).half(), _values(vc[at], vs[at]).half()


def _plain_write(st, tokens):
    """Rotated queries; the rows go into the cache."""
    case = st["case"]
    b, group = case["batch"], case["group"]
    q = _rotate(st["q"], st["cos"], st["sin"], st["positions"])
    k = _rotate(st["k"], st["cos"], st["sin"], st["positions"])
    first = st["first"] if "first" in st else st["length"]
    at = (torch.arange(b, device="cuda")[:, None], slice(None), first[:, None] + torch.arange(tokens, device="cuda"))
    st["k_codes"][at], st["k_scales"][at] = (x.unflatten(0, (b, tokens)) for x in _quantise(k.float(), group))
    st["v_codes"][at], st["v_scales"][at] = (x.unflatten(0, (b, tokens)) for x in _quantise(st["v"].float(), group))
    return q


def _plain_evict(st):
    case, w, n = st["case"], st["weights"], st["length"][:, None, None]
    j = torch.arange(case["slots"], device="cuda")
    w = torch.where((j < case["sinks"]) | (j >= n - case["recent"]), math.inf, w).masked_fill(j >= n, -math.inf)
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :case["keep"]]
    length = st["length"].clamp(max=case["keep"])
    live = torch.arange(case["keep"], device="cuda") < length[:, None, None]
    kept = torch.sort(order.masked_fill(order >= n, case["slots"]), dim=-1).values
    at = kept.clamp(max=case["slots"] - 1)
    for name, to in zip(("k_codes", "k_scales", "v_codes", "v_scales"), st["out"]):
        x = st[name]
        i = at.view(*at.shape, *[1] * (x.dim() - 3)).expand(*at.shape, *x.shape[3:])
        y = x.gather(2, i)
        to[:, :, :case["keep"]] = y.masked_fill(~live.view(*live.shape, *[1] * (x.dim() - 3)), 0)
    weights = st["weights"].gather(2, at).masked_fill(~live, 0.0)
    return kept.masked_fill(~live, -1).int(), weights, length


# ---------------------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    case, kind = st["case"], st["kind"]
    if kind == "step":
        q = _plain_write(st, 1)
        out = _plain_attend(st, q, st["length"] + 1)[0]
        return out, *_rows(st, st["length"], 1)
    if kind == "attend":
        out, p = _plain_attend(st, st["q"], st["length"])
        if st["weights"] is None:
            return out
        j = torch.arange(case["slots"], device="cuda")
        return out, torch.where(j < st["length"][:, None, None], st["weights"] + p.sum(2), 0.0)
    if kind == "write":
        q = _plain_write(st, case["tokens"])
        return q, *_rows(st, st["first"], case["tokens"])
    if kind == "evict":
        kept, weights, length = _plain_evict(st)
        names = dict(zip(("k_codes", "k_scales", "v_codes", "v_scales"), st["out"]))
        return kept, weights, length, *_rows(names, st["zero"], case["keep"])
    if kind == "prompt":
        return _plain_prompt(st)
    return _plain_mass(st)


def _run_own(st):
    from cherryq_b200 import quant_cuda as qc
    case, kind = st["case"], st["kind"]
    if kind == "step":
        out = st["cache"].step(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"], st["length"],
                               window=case["window"], sinks=case["sinks"])
        return out, *st["cache"].read(st["length"], 1)
    if kind == "attend":
        out = st["cache"].attend(st["q"], st["length"], window=case["window"], sinks=case["sinks"], weights=st["weights"],
                                 weights_out=st["weights_out"])
        return out if st["weights"] is None else (out, st["weights_out"])
    if kind == "write":
        q = st["cache"].write(st["q"], st["k"], st["v"], st["first"], st["cos"], st["sin"], st["positions"])
        return q, *st["cache"].read(st["first"], case["tokens"])
    if kind == "evict":
        kept, weights, length = st["cache"].evict(st["weights"], st["length"], case["keep"], sinks=case["sinks"],
                                                  recent=case["recent"], out=st["out_cache"])
        return kept, weights, length, *st["out_cache"].read(st["zero"], case["keep"])
    if kind == "prompt":
        return qc.attn_prefill(st["q"], st["k"], st["v"], window=case["window"], sinks=case["sinks"], lengths=st["lengths"])
    return qc.attn_prefill_weights(st["q"], st["k"], st["lse"], window=case["window"], sinks=case["sinks"],
                                   lengths=st["lengths"], observe=case["observe"])


# ---------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case, observe=None):
    """Query-key pairs that are visible in one sequence of full length, of the queries at the last `observe` positions."""
    tk, tq, w, sinks = case["keys"], case["queries"], case["window"], case["sinks"]
    first = max(tk - tq, tk - observe if observe else 0)

    def upto(n):                       # keys seen by all queries at positions 0 .. n - 1
        if not w or w >= n:
            return n * (n + 1) // 2
        total = w * (w + 1) // 2 + (n - w) * w
        out = n - w                    # queries whose window has left the first key
        return total + (min(out, sinks) * (min(out, sinks) + 1) // 2 + max(0, out - sinks) * sinks)
    return upto(tk) - upto(first)


def work(case):
    h, kv, d = HEADS[case["heads"]]
    b, kind = case["batch"], case["kind"]
    if kind in ("prompt", "mass"):
        share = 0.75 if case["ragged"] else 1.0          # mean length of mixed prompts
        tq, tk = case["queries"], case["keys"]
        if kind == "prompt":
            return {"bytes": b * share * 2 * d * (2 * tq * h + 2 * tk * kv) + b * h * tq * 4, "flops": 4.0 * d * h * b * _pairs(case) * share}
        rows = min(tq, case["observe"])
        return {"bytes": b * (rows * h * (2 * d + 4) + tk * kv * (2 * d * share + 4)), "flops": 2.0 * d * h * b * _pairs(case, case["observe"]) * share}
    row = 2 * (d // 2 + 4 * (d // case["group"]))        # a slot's key and value of one head
    if kind == "write":
        t = b * case["tokens"]
        return {"bytes": t * (2 * d * (2 * h + 4 * kv) + kv * row) + case["tokens"] * 4 * d, "flops": 6.0 * t * d * (h + 2 * kv)}
    n = case["held"] * (0.75 if case["ragged"] else 1.0)
    if kind == "evict":
        return {"bytes": b * kv * (4 * n + case["keep"] * (2 * row + 8 + 4 * d)), "flops": b * kv * (n + 4.0 * d * case["keep"])}
    seen = min(n, case["window"] + case["sinks"]) if case["window"] else n
    nbytes = b * (kv * seen * row + 4 * d * h)
    if kind == "step":
        nbytes += b * (kv * (8 * d + row) + 4 * d)
    elif case["weights"]:
        nbytes += b * kv * 8 * n
    return {"bytes": nbytes, "flops": 4.0 * d * h * b * seen}


# ---------------------------------------------------------------------------------- results in 64 bits
def _decoded(codes, scales):
    """Values of cache rows in 64 bits, column by column."""
    d = 2 * codes.shape[-1]
    col = torch.arange(d, device=codes.device)
    code = (codes[..., col // 2].int() >> (4 * (col % 2))) & 15
    pair = scales.double()[..., col // (d // scales.shape[-2]), :]
    return code * pair[..., 0] + pair[..., 1]


def _rotated64(x, st):
    half = x.shape[-1] // 2
    ang = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"]].unsqueeze(1)
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * ang
    return torch.cat([z.real, z.imag], -1).half().double()


def _coded64(x, group):
    """The values that rows stand for once they are kept in 4 bits."""
    out = torch.empty_like(x)
    for c in range(0, x.shape[-1], group):
        part = x[..., c:c + group]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        s = ((high - low) / 15).half().double()
        u = torch.where(s > 0, ((part - low) / torch.where(s > 0, s, 1.0)).round().clamp(0, 15), 0.0)
        out[..., c:c + group] = u * s + low
    return out


def _softmax64(scores):
    top = scores.max(-1, keepdim=True).values
    e = torch.exp(scores - torch.where(top > -math.inf, top, 0.0))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0), (top + total.log()).squeeze(-1)


def _attend64(st, q, k, v, length):
    """Sequence by sequence, over the visible slots alone. k, v: callables of (sequence, slots)."""
    case = st["case"]
    h, kv, d = HEADS[case["heads"]]
    out = torch.zeros(case["batch"], h, d, device="cuda", dtype=torch.float64)
    mass = torch.zeros(case["batch"], kv, case["slots"], device="cuda", dtype=torch.float64)
    for b, n in enumerate(length.tolist()):
        slots = [j for j in range(n) if not case["window"] or j < case["sinks"] or j >= n - case["window"]]
        if not slots:
            continue
        at = torch.tensor(slots, device="cuda")
        p, _ = _softmax64(torch.einsum("kgd,ksd->kgs", q[b].double().view(kv, -1, d), k(b, at)) / math.sqrt(d))
        out[b] = torch.einsum("kgs,ksd->kgd", p, v(b, at)).reshape(h, d)
        mass[b][:, at] = p.sum(1)
    return out, mass


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    h, kv, d = HEADS[case["heads"]]
    b = case["batch"]
    keys = lambda i, at: _decoded(st["k_codes"][i][:, at], st["k_scales"][i][:, at])
    vals = lambda i, at: _decoded(st["v_codes"][i][:, at], st["v_scales"][i][:, at])
    if kind in ("step", "write"):
        t = case.get("tokens", 1)
        q = _rotated64(st["q"], st)
        k, v = _coded64(_rotated64(st["k"], st), case["group"]), _coded64(st["v"].double(), case["group"])
        new = k.view(b, t, kv, d), v.view(b, t, kv, d)
        if kind == "write":
            return q, *new

        def joined(old, rows):
            def get(i, at):
                x = old(i, at.clamp(max=case["slots"] - 1))
                x[:, -1] = rows[i, 0]          # the new slot is always visible, and the last one
                return x
            return get
        out, _ = _attend64(st, q, joined(keys, new[0]), joined(vals, new[1]), st["length"] + 1)
        return out, *new
    if kind == "attend":
        out, mass = _attend64(st, st["q"], keys, vals, st["length"])
        if st["weights"] is None:
            return out
        live = torch.arange(case["slots"], device="cuda") < st["length"][:, None, None]
        return out, (st["weights"].double() + mass) * live
    if kind == "evict":
        kept = torch.full((b, kv, case["keep"]), -1, dtype=torch.int32, device="cuda")
        sums = torch.zeros(b, kv, case["keep"], dtype=torch.float64, device="cuda")
        rows = [torch.zeros(b, case["keep"], kv, d, dtype=torch.float64, device="cuda") for _ in range(2)]
        length = st["length"].clamp(max=case["keep"])
        if b * kv * case["slots"] > 1_000_000:
            return None
        for i, n in enumerate(st["length"].tolist()):
            w = st["weights"][i, :, :n].tolist()
            for g in range(kv):
                if n <= case["keep"]:
                    slots = list(range(n))
                else:
                    middle = sorted(range(case["sinks"], n - case["recent"]), key=lambda j: (-w[g][j], j))
                    more = case["keep"] - case["sinks"] - case["recent"]
                    slots = sorted([*range(case["sinks"]), *middle[:more], *range(n - case["recent"], n)])
                at = torch.tensor(slots, device="cuda")
                kept[i, g, :len(slots)] = at.int()
                sums[i, g, :len(slots)] = st["weights"][i, g, at].double()
                rows[0][i, :len(slots), g] = _decoded(st["k_codes"][i, g, at], st["k_scales"][i, g, at])
                rows[1][i, :len(slots), g] = _decoded(st["v_codes"][i, g, at], st["v_scales"][i, g, at])
        return kept, sums, length, *rows
    # prompts: head by head
    tq, tk = case["queries"], case["keys"]
    first = tk - tq
    out = torch.zeros(b, tq, h, d, dtype=torch.float64, device="cuda")
    lse = torch.full((b, h, tq), -math.inf, dtype=torch.float64, device="cuda")
    mass = torch.zeros(b, kv, tk, dtype=torch.float64, device="cuda")
    ends = st["lengths"].tolist() if st["lengths"] is not None else [tk] * b
    for i, n in enumerate(ends):
        rows = torch.arange(first, n, device="cuda") if n > first else None
        if rows is None:
            continue
        if kind == "mass":
            rows = rows[rows >= n - case["observe"]]
        cols = torch.arange(n, device="cuda")
        back = rows[:, None] - cols[None, :]
        hidden = back < 0
        if case["window"]:
            hidden |= (back >= case["window"]) & (cols >= case["sinks"])
        for g in range(h):
            kg = st["k"][i, :n, g // (h // kv)].double()
            s = (st["q"][i, rows - first, g].double() @ kg.T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            if kind == "mass":
                mass[i, g // (h // kv), :n] += torch.exp(s - st["lse"][i, g, rows - first].double()[:, None].clamp(min=-1e300)).sum(0)
                continue
            p, l = _softmax64(s)
            out[i, rows - first, g] = p @ st["v"][i, :n, g // (h // kv)].double()
            lse[i, g, rows - first] = l
    return mass if kind == "mass" else (out, lse)
