"""The operators of serving many sequences from a pool of cache pages: what is timed, their plain forms and exact results.

Kinds of work and the calls that a user makes for them:
  step     `KVPages.step`: one new token of every sequence: rotary embedding, its key and value into the sequence's last page,
           attention over the sequence's pages
  attend   `KVPages.attend`: attention of one query per sequence over its pages
  write    `KVPages.write`: packed prompts of different lengths, rotated and written into their pages
  read     `KVPages.read`: a range of slots of every sequence as one block, for a follow-up prompt
  adjust   `adjust_logits`: repetition, presence and frequency penalties, biases of single tokens, a grammar's bit mask, and the
           token with the largest logit

A page holds `page` slots of every KV head: keys and values (pages, KV, page, D) in fp16 or bf16.  A table (sequences, width) int32
names the page of every `page` slots of a sequence, -1 where there is none.

Head counts are those of LLaMA-2 7B / 13B / 70B (the configurations of `decoder.py`) and a small 64-wide one; 32000 is their vocabulary.
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
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
MAX_VALUES = 4 * 65536 * 8 * 128       # of all sequences' keys, that a plain form holds in 32 bits


def listed():
    return [
        # interactive decoding: one 7B layer, one sequence, short context: launch latency
        {"name": "step_7b_b1", "kind": "step", "heads": "7b", "type": "fp16", "page": 16, "batch": 1, "held": 256, "ragged": False, "window": 0, "sinks": 0},
        # sixteen 70B sequences (grouped queries) of mixed lengths up to about 4000 positions
        {"name": "step_70b_b16", "kind": "step", "heads": "70b", "type": "bf16", "page": 64, "batch": 16, "held": 4001, "ragged": True, "window": 0, "sinks": 0},
        # a serving batch of mixed lengths whose layers look back 1021 positions and at four sinks
        {"name": "attend_13b_window", "kind": "attend", "heads": "13b", "type": "fp16", "page": 16, "batch": 8, "held": 2113, "ragged": True, "window": 1021, "sinks": 4},
        # long documents: four sequences of 65531 positions
        {"name": "attend_70b_long", "kind": "attend", "heads": "70b", "type": "fp16", "page": 128, "batch": 4, "held": 65531, "ragged": False, "window": 0, "sinks": 0},
        # many short conversations with a small model of 64-wide heads
        {"name": "attend_small_b33", "kind": "attend", "heads": "small", "type": "bf16", "page": 32, "batch": 33, "held": 777, "ragged": True, "window": 0, "sinks": 0},
        # a 2048-token prompt of one 13B layer into its pages
        {"name": "write_13b_2048", "kind": "write", "heads": "13b", "type": "fp16", "page": 16, "batch": 1, "tokens": 2048, "held": 0, "ragged": False},
        # follow-up prompts of mixed lengths behind what the pages hold, packed
        {"name": "write_70b_packed", "kind": "write", "heads": "70b", "type": "bf16", "page": 64, "batch": 24, "tokens": 333, "held": 1001, "ragged": True},
        # what five 13B sequences hold, for the attention of their follow-up prompts
        {"name": "read_13b_2001", "kind": "read", "heads": "13b", "type": "fp16", "page": 32, "batch": 5, "held": 2001, "first": 0, "count": 2001},
        # the last 77 slots of a few short ones
        {"name": "read_small_77", "kind": "read", "heads": "small", "type": "bf16", "page": 16, "batch": 3, "held": 200, "first": 123, "count": 77},
        # one sequence's next token with penalties for what stands in front of it
        {"name": "adjust_b1", "kind": "adjust", "type": "fp16", "rows": 1, "vocab": 32000, "history": 300, "ragged": False, "penalties": True, "biases": 0, "masks": 0},
        # a serving batch with everything: penalties over long histories, biases, grammars
        {"name": "adjust_b64", "kind": "adjust", "type": "fp32", "rows": 64, "vocab": 32000, "history": 4000, "ragged": True, "penalties": True, "biases": 50, "masks": 9},
        # a large batch and a large vocabulary of odd size
        {"name": "adjust_b256", "kind": "adjust", "type": "bf16", "rows": 256, "vocab": 131071, "history": 1500, "ragged": True, "penalties": True, "biases": 0, "masks": 256},
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
        if w["bytes"] > nbytes or w["flops"] > flops:
            continue
        if case["kind"] != "adjust":
            _, kv, d = HEADS[case["heads"]]
            if case["batch"] * kv * d * _slots(case) > MAX_VALUES:
                continue
        return case


def _draw(rng):
    kind = rng.choice(["step", "step", "step", "attend", "attend", "attend", "write", "write", "read", "adjust", "adjust", "adjust"])
    if kind == "adjust":
        return {"kind": kind, "type": rng.choice(["fp16", "bf16", "fp32"]), "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 1000, 140000),
                "history": _log_int(rng, 1, 8192), "ragged": rng.random() < 0.6, "penalties": rng.random() < 0.8,
                "biases": rng.choice([0, 0, 1, 50, 300]), "masks": rng.choice([0, 1, 7, 100])}
    case = {"kind": kind, "heads": rng.choice(sorted(HEADS)), "type": rng.choice(["fp16", "bf16"]), "page": rng.choice([16, 32, 64, 128, 256]),
            "batch": _log_int(rng, 1, 64)}
    if kind == "write":
        case.update(tokens=_log_int(rng, 1, 4096), held=rng.randint(0, 2048), ragged=rng.random() < 0.6)
    elif kind == "read":
        held = _log_int(rng, 1, 16384)
        first = rng.randint(0, held - 1) if rng.random() < 0.5 else 0
        case.update(held=held, first=first, count=rng.randint(1, held - first) if rng.random() < 0.5 else held - first)
    else:
        held = _log_int(rng, 1, 65536)
        case.update(held=held, ragged=rng.random() < 0.6, window=0 if rng.random() < 0.6 else _log_int(rng, 8, held + 8), sinks=rng.choice([0, 1, 4, 64]))
    return case


def _slots(case):
    """Slots of the table's width."""
    n = case["held"] + case.get("tokens", 1)
    return -(-n // case["page"]) * case["page"]


# ---------------------------------------------------------------------------------- inputs
def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _keys(g, *shape):
    """Keys as trained models have them: a few columns of a head much larger than the rest."""
    x = _normal(g, *shape)
    x[..., 3::37] *= 4.0
    return x


def _lengths(g, batch, most, ragged):
    """`most` of each sequence, or half of it to all of it, evenly spread and in any order."""
    length = torch.full((batch,), most, device="cuda", dtype=torch.int64)
    if ragged:
        less = torch.arange(batch, device="cuda") * (most // 2) // max(1, batch - 1)
        length -= less[torch.randperm(batch, device="cuda", generator=g)]
    return length


def _prepare_adjust(case, g):
    rows, vocab, width = case["rows"], case["vocab"], case["history"]
    st = {"case": case, "kind": "adjust", "logits": (_normal(g, rows, vocab) * 2.5).to(TYPES[case["type"]])}
    args = dict.fromkeys(("tokens", "length", "prompt", "repetition", "presence", "frequency", "bias_ids", "bias", "mask", "mask_rows"))
    if case["penalties"]:
        # word frequencies of natural text: few tokens often, most of them never
        args["tokens"] = (vocab ** torch.rand(rows, width, device="cuda", generator=g)).long().clamp(max=vocab) - 1
        args["length"] = _lengths(g, rows, width, case["ragged"])
        args["prompt"] = (args["length"] * torch.rand(rows, device="cuda", generator=g)).long()
        some = lambda low, high: low + (high - low) * torch.rand(rows, device="cuda", generator=g)
        args["repetition"], args["presence"], args["frequency"] = some(1.0, 1.5), some(0.0, 1.0), some(0.0, 0.5)
    if case["biases"]:
        n = min(case["biases"], vocab)
        args["bias_ids"] = torch.rand(rows, vocab, device="cuda", generator=g).topk(n, -1).indices
        args["bias"] = _normal(g, rows, n) * 5.0
    if case["masks"]:
        # a grammar's states: some allow a few tokens, some nearly all; the last sequence has none
        share = torch.rand(case["masks"], 1, device="cuda", generator=g)
        allowed = torch.rand(case["masks"], -(-vocab // 32), 32, device="cuda", generator=g) < (share ** 4)[..., None]
        weight = torch.tensor([1 << i for i in range(32)], device="cuda", dtype=torch.int64)
        word = (allowed * weight).sum(-1)
        args["mask"] = torch.where(word >= 1 << 31, word - (1 << 32), word).to(torch.int32)
        args["mask_rows"] = torch.randint(0, case["masks"], (rows,), device="cuda", generator=g)
        args["mask_rows"][-1] = -1
    st["args"] = args
    return st


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "adjust":
        st = _prepare_adjust(case, g)
        if own:
            import cherryq_b200
            cherryq_b200.load_quant_cuda()
        return st
    h, kv, d = HEADS[case["heads"]]
    b, page, dtype = case["batch"], case["page"], TYPES[case["type"]]
    width = _slots(case) // page
    st = {"case": case, "kind": kind}
    # a pool that has served for a while: rows everywhere, pages of a sequence anywhere
    shape = (b * width + 3, kv, page, d)
    st["k_pages"], st["v_pages"] = _keys(g, *shape).to(dtype), _normal(g, *shape).to(dtype)
    if kind == "write":
        count = _lengths(g, b, case["tokens"], case["ragged"])
        st["starts"] = torch.cat([count.new_zeros(1), count.cumsum(0)])
        rows = int(st["starts"][-1])
        st["first"] = _lengths(g, b, case["held"], case["ragged"])
        need = st["first"] + count
        st["sequence"] = torch.repeat_interleave(torch.arange(b, device="cuda"), count)
        st["positions"] = st["first"][st["sequence"]] + torch.arange(rows, device="cuda") - st["starts"][st["sequence"]]
    elif kind == "read":
        rows = 0
        st["first"] = torch.full((b,), case["first"], device="cuda", dtype=torch.int64)
        need = torch.full_like(st["first"], case["held"])
    else:
        rows = b
        st["length"] = _lengths(g, b, case["held"], case["ragged"])
        need = st["length"] + 1
        st["positions"] = st["length"].clone()
    table = torch.randperm(shape[0], device="cuda", generator=g)[:b * width].view(b, width)
    st["table"] = torch.where(torch.arange(width, device="cuda") * page < need[:, None], table, -1).to(torch.int32)
    if rows:
        st["q"] = _normal(g, rows, h, d).to(dtype)
    if kind in ("write", "step"):
        st["k"], st["v"] = _keys(g, rows, kv, d).to(dtype), _normal(g, rows, kv, d).to(dtype)
        inv = 1.0 / (10000.0 ** (torch.arange(0, d, 2, device="cuda", dtype=torch.float32) / d))
        ang = torch.outer(torch.arange(_slots(case), device="cuda", dtype=torch.float32), inv)
        st["cos"], st["sin"] = ang.cos(), ang.sin()
    if own:
        import cherryq_b200
        st["pages"] = cherryq_b200.load_quant_cuda().KVPages(st["k_pages"], st["v_pages"])
    return st


# ---------------------------------------------------------------------------------- plain forms
def _rotate(x, st):
    """Rows (T, heads, D), rotated halves, rounded to 16 bits as they are kept."""
    c, s = st["cos"][st["positions"]][:, None], st["sin"][st["positions"]][:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1).to(x.dtype)


def _plain_write(st, sequence, slot):
    """The rows of k and v into the pages; rotated queries."""
    q, k = _rotate(st["q"], st), _rotate(st["k"], st)
    page = st["case"]["page"]
    at = (st["table"][sequence, slot // page].long(), slice(None), slot % page)
    st["k_pages"][at] = k
    st["v_pages"][at] = st["v"]
    return q


def _gathered(pages, table):
    """(sequences, KV, slots, D) in 32 bits; absent pages as page 0"""
    return pages[table.long().clamp(min=0)].permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _plain_attend(st, q, length):
    case = st["case"]
    b, h, d = q.shape
    k, v = _gathered(st["k_pages"], st["table"]), _gathered(st["v_pages"], st["table"])
    kv, slots = k.shape[1], k.shape[2]
    j, n = torch.arange(slots, device="cuda"), length[:, None]
    seen = j < n
    if case["window"]:
        seen = seen & ((j < case["sinks"]) | (j >= n - case["window"]))
    seen = seen[:, None, None]
    s = torch.matmul(q.float().view(b, kv, h // kv, d), k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    return torch.matmul(p, v * seen.transpose(-1, -2)).view(b, h, d).to(q.dtype)


def _plain_read(st):
    case = st["case"]
    slot = st["first"][:, None] + torch.arange(case["count"], device="cuda")
    page = st["table"].long().gather(1, slot // case["page"])
    at = (page, slice(None), slot % case["page"])
    return st["k_pages"][at], st["v_pages"][at]


def _plain_adjust(st):
    a, logits = st["args"], st["logits"]
    rows, vocab = logits.shape
    x = logits.float()
    if a["tokens"] is not None:
        i = torch.arange(a["tokens"].shape[1], device="cuda")
        there = i < a["length"][:, None]
        made = there & (i >= a["prompt"][:, None])
        count = lambda which: torch.zeros(rows, vocab, device="cuda").scatter_add_(1, a["tokens"], which.float())
        c_all, c_out = count(there), count(made)
        rep = a["repetition"][:, None]
        x = torch.where(c_all > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - a["frequency"][:, None] * c_out
        x = torch.where(c_out > 0, x - a["presence"][:, None], x)
    if a["bias_ids"] is not None:
        x = x + torch.zeros_like(x).scatter_(1, a["bias_ids"], a["bias"])
    if a["mask"] is not None:
        v = torch.arange(vocab, device="cuda")
        bits = (a["mask"][a["mask_rows"].clamp(min=0)][:, v // 32] >> (v % 32)) & 1
        x = torch.where((bits == 1) | (a["mask_rows"] < 0)[:, None], x, -math.inf)
    return x.to(logits.dtype), x.argmax(-1)


# ---------------------------------------------------------------------------------- one pass
def run(st):
    return _run_own(st) if own else _run_plain(st)


def _run_plain(st):
    kind = st["kind"]
    if kind == "adjust":
        return _plain_adjust(st)
    if kind == "read":
        return _plain_read(st)
    if kind == "write":
        return _plain_write(st, st["sequence"], st["positions"]), st["k_pages"], st["v_pages"]
    if kind == "step":
        q = _plain_write(st, torch.arange(st["case"]["batch"], device="cuda"), st["length"])
        return _plain_attend(st, q, st["length"] + 1), st["k_pages"], st["v_pages"]
    return _plain_attend(st, st["q"], st["length"])


def _run_own(st):
    from cherryq_b200 import quant_cuda as qc
    case, kind = st["case"], st["kind"]
    if kind == "adjust":
        return qc.adjust_logits(st["logits"], **st["args"])
    pages = st["pages"]
    if kind == "read":
        return pages.read(st["table"], st["first"], case["count"])
    if kind == "write":
        q = pages.write(st["q"], st["k"], st["v"], st["table"], st["first"], st["cos"], st["sin"], st["positions"], st["starts"])
        return q, st["k_pages"], st["v_pages"]
    if kind == "step":
        out = pages.step(st["q"], st["k"], st["v"], st["cos"], st["sin"], st["positions"], st["table"], st["length"],
                         window=case["window"], sinks=case["sinks"])
        return out, st["k_pages"], st["v_pages"]
    return pages.attend(st["q"], st["table"], st["length"], window=case["window"], sinks=case["sinks"])


# ---------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "adjust":
        rows, vocab = case["rows"], case["vocab"]
        share = 0.75 if case["ragged"] else 1.0          # mean length of mixed sequences
        item = 4 if case["type"] == "fp32" else 2
        nbytes = rows * (2 * vocab * item + 8)
        if case["penalties"]:
            nbytes += rows * (8 * case["history"] * share + 28)
        nbytes += rows * 12 * case["biases"]
        if case["masks"]:
            nbytes += min(rows, case["masks"]) * (vocab / 8) + 8 * rows
        return {"bytes": nbytes, "flops": 2.0 * rows * vocab}
    h, kv, d = HEADS[case["heads"]]
    b = case["batch"]
    share = 0.75 if case.get("ragged") else 1.0
    if kind == "write":
        t = b * case["tokens"] * share
        return {"bytes": t * (2 * 2 * d * (h + 2 * kv) + 8) + case["tokens"] * 4 * d, "flops": 3.0 * t * d * (h + kv)}
    if kind == "read":
        return {"bytes": b * case["count"] * 8 * d * kv, "flops": 0.0}
    n = case["held"] * share
    seen = min(n, case["window"] + case["sinks"]) if case["window"] else n
    nbytes = b * (kv * seen * 4 * d + 4 * d * h + 8 + 4 * seen / case["page"])
    if kind == "step":
        nbytes += b * (kv * 8 * d + 4 * d + 8)
    return {"bytes": nbytes, "flops": 4.0 * d * h * b * seen}


# ---------------------------------------------------------------------------------- results in 64 bits
def _rotated64(x, st):
    """What rows are kept as: the rotation in 64 bits, rounded to their type."""
    half = x.shape[-1] // 2
    ang = torch.complex(st["cos"].double(), st["sin"].double())[st["positions"]].unsqueeze(1)
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * ang
    return torch.cat([z.real, z.imag], -1)


def _attend64(st, q, length, fresh=None):
    """Sequence by sequence and page by page, over the visible slots alone. fresh: (keys, values) of the last slot."""
    case = st["case"]
    h, kv, d = HEADS[case["heads"]]
    out = torch.zeros(case["batch"], h, d, device="cuda", dtype=torch.float64)
    for b, n in enumerate(length.tolist()):
        slots = torch.arange(n, device="cuda")
        if case["window"]:
            slots = slots[(slots < case["sinks"]) | (slots >= n - case["window"])]
        if not len(slots):
            continue
        where = st["table"][b].long()[slots // case["page"]], slots % case["page"]
        k, v = (x[where[0], :, where[1]].double() for x in (st["k_pages"], st["v_pages"]))
        if fresh is not None:
            k[-1], v[-1] = fresh[0][b], fresh[1][b]
        s = torch.einsum("kgd,skd->kgs", q[b].double().view(kv, -1, d), k) / math.sqrt(d)
        out[b] = torch.einsum("kgs,skd->kgd", torch.softmax(s, -1), v).reshape(h, d)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "adjust":
        return _adjust64(st)
    if kind == "attend":
        return _attend64(st, st["q"], st["length"])
    if kind == "read":
        k, v = [], []
        for b, f in enumerate(st["first"].tolist()):
            line = torch.arange(f, f + case["count"], device="cuda")
            page = st["table"][b].long()[line.div(case["page"], rounding_mode="floor")]
            k.append(st["k_pages"][page, :, line.remainder(case["page"])].double())
            v.append(st["v_pages"][page, :, line.remainder(case["page"])].double())
        return torch.stack(k), torch.stack(v)
    q, k, v = _rotated64(st["q"], st), _rotated64(st["k"], st), st["v"].double()
    if kind == "write":
        owner, slots = st["sequence"].tolist(), st["positions"].tolist()
    else:
        owner, slots = range(case["batch"]), st["length"].tolist()
        # attention is computed on the rows as they are kept
        kept = lambda x: x.to(st["q"].dtype).double()
        q = _attend64(st, kept(q), st["length"] + 1, (kept(k), v))
    table = st["table"].tolist()
    page = torch.tensor([table[s][j // case["page"]] for s, j in zip(owner, slots)], device="cuda")
    line = torch.tensor([j % case["page"] for j in slots], device="cuda")
    pools = st["k_pages"].double(), st["v_pages"].double()
    for pool, rows in zip(pools, (k, v)):
        pool[page, :, line] = rows
    return q, *pools


def _adjust64(st):
    a = st["args"]
    x = st["logits"].double()
    rows, vocab = x.shape
    if rows * vocab > 50_000_000:
        return None
    for r in range(rows):
        if a["tokens"] is not None:
            n, p = int(a["length"][r]), int(a["prompt"][r])
            rep, pres, freq = (float(a[k][r]) for k in ("repetition", "presence", "frequency"))
            seen = torch.unique(a["tokens"][r, :n])
            x[r, seen] = torch.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
            made, times = torch.unique(a["tokens"][r, p:n], return_counts=True)
            x[r, made] -= freq * times.double() + pres
        if a["bias_ids"] is not None:
            x[r, a["bias_ids"][r]] += a["bias"][r].double()
        state = int(a["mask_rows"][r]) if a["mask"] is not None else -1
        if state >= 0:
            bits = torch.stack([(a["mask"][state].long() >> i) & 1 for i in range(32)], -1).flatten()[:vocab]
            x[r, bits == 0] = -math.inf
    return x, x.argmax(-1)
