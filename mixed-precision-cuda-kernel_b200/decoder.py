"""Minimal LLaMA-architecture decode harness around the CherryQ quantized linear.

The reference evaluates its kernels inside a vendored Hugging Face LLaMA
(llama/modeling_llama_quant.py:724-785 decoder layer, :251 MLP, :371-419 attention of the
reference project; protocol of benchmark_perplexity.py:92-113).  This module keeps only what
a decode benchmark needs: RMSNorm fused with the residual add, rotary embeddings (HF "rotate
half" convention) fused with the KV-cache write, SwiGLU (three small CUDA kernels of the
library), an fp16 KV cache, an unquantised fp16 lm_head, greedy sampling, and the seven quantized
projections per layer as `QuantLinear` modules (q, k, v, o, gate, up, down - separate, as in
the reference, each with its own cherry columns).  Weights are random (no checkpoint can be
loaded offline): dense ~ N(0, 0.02), cherry columns ~ N(0, 0.2), packed on the GPU layer by
layer so that the fp16 model never exists in memory.

One decode step (embedding lookup -> layers -> logits -> argmax -> cache / position update)
touches only device tensors, so it is captured once in a CUDA graph and replayed.
Decode attention is a single-query kernel of the library that reads the current position on the
device (so the captured graph serves every step); prefill attention is torch's
scaled_dot_product_attention.  Both are plumbing here, not the measured path.

`tp_group` shards every projection along its output rows over the ranks of a process group
(column parallel: heads for q / k / v, output features for o / gate / up / down) and gathers the
slices with an NCCL all-gather where the next op needs the whole vector (attention output, o,
SwiGLU output, down): four collectives per layer.  Every output element is still computed by
exactly the single-GPU arithmetic, so the tokens are identical for every group size (with the 4-bit
cache up to the rounding of attention's sums, whose split goes by the heads of a rank); all ranks
draw the full random weight and pack only their rows.

`kv_bits=4` keeps keys and values in 4 bits (`quant_cuda.KVCache4`): prompts go through `attn_prefill`, steps through
`KVCache4.step`, both with a sliding `window` and the first `sinks` positions visible if asked for.  `kv_budget` bounds the cache: a
prompt's positions are weighed by its last `kv_observe` queries (`attn_prefill_weights`), every step adds what each slot
received, and whenever the `kv_budget + kv_slack` slots of a layer are full the heaviest `kv_budget` stay (`KVCache4.evict`; the
first `sinks` and the last `kv_recent` always do).  Keys keep the rotation of their own positions.  Slots are not positions any more then,
so that a `window` that hides any and `kv_budget` exclude one another.

`kv_page=64` keeps the fp16 cache in pages of so many slots (`quant_cuda.KVPages`), `kv_pages` of them for all sequences of a layer:
prompts may have different lengths (`prefill(tokens, lengths)`), single sequences get a new one while the others go on
(`prefill(tokens, lengths, rows)`) or give their pages back (`release`), and a `window` with `sinks` can be asked for.

`control(...)` puts `quant_cuda.adjust_logits` behind the logits of every step: penalties for tokens that occurred in a sequence, biases
of single tokens, and a grammar as bit masks with a table of the states that follow.

`dense=True` builds the parity twin: the same packed buffers, every projection computed as
F.linear(x, unpack()) the way the reference's dense mode does (llama/qlinear.py:183-195).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from types import SimpleNamespace

import torch
import torch.nn.functional as F

from . import load_quant_cuda
from .qlinear import QuantLinear, forward_normed_input, forward_shared_input


@dataclass
class DecoderConfig:
    n_layers: int = 32
    hidden: int = 4096
    n_heads: int = 32
    n_kv_heads: int = 32
    ffn: int = 11008
    vocab: int = 32000
    bits: int = 4
    group: int = 128
    cherry_fraction: float = 1 / 256
    max_seq: int = 512
    rope_theta: float = 10000.0
    eps: float = 1e-5

    @property
    def head_dim(self) -> int:
        return self.hidden // self.n_heads


LLAMA2_7B = DecoderConfig()
LLAMA2_13B = DecoderConfig(n_layers=40, hidden=5120, n_heads=40, n_kv_heads=40, ffn=13824, bits=3)
LLAMA2_70B = DecoderConfig(n_layers=80, hidden=8192, n_heads=64, n_kv_heads=8, ffn=28672, bits=3)


def linear_algorithmic_bytes(k: int, n: int, bits: int, group: int, fraction: float, m: int = 1) -> int:
    """Bytes one call of a quantized linear has to move (reference-format sizes)."""
    c = math.ceil(k * fraction) // 8 * 8
    kc = k - c
    return kc // 8 * bits * n + math.ceil(kc / group) * n * 2 + c * n * 2 + c * 2 + m * k * 2 + m * n * 2


class CherryDecoder:
    PROJ = ("q", "k", "v", "o", "gate", "up", "down")

    def __init__(self, cfg: DecoderConfig, device="cuda", seed: int = 0, dense: bool = False,
                 release_reference_buffers: bool = False, tp_group=None, tp_gather: str = "peer", batch: int = 1,
                 attention: str = "auto", kv_bits: int = 16, kv_group: int = 32, window: int = 0, sinks: int = 0,
                 kv_budget: int = None, kv_slack: int = 256, kv_recent: int = None, kv_observe: int = 64, kv_page: int = 0,
                 kv_pages: int = None):
        if not torch.cuda.is_available():
            raise RuntimeError("CherryDecoder needs a CUDA device (there is no CPU path)")
        if batch < 1:
            raise ValueError("batch must be at least 1")
        self.cfg, self.dev, self.dense = cfg, torch.device(device), dense
        self.batch = batch          # sequences decoded in lockstep (same prompt length, one position counter)
        # decode attention over the KV cache: "own" = this library's kernels (cq_attn_decode); "flash" = the
        # flash_attn package's flash_attn_with_kvcache (a library call, like the lm_head's cuBLAS matmul);
        # "auto" = own, except for grouped-query models with caches of more than 1024 positions whose heads the tensor-core
        # kernel does not take, where that package imports.  Measured on B200 with cold caches, own against flash_attn:
        # 7B at 256 positions 4.9 us and 9.5; 13B shapes at 2100 positions, batch 8, 70 and 159; 8 query heads per KV head
        # at 4000 positions 12.5 and 20 at batch 1, 20 and 27 at 4, 50 and 64 at 16, 93 and 194 at 32.
        if attention not in ("auto", "own", "flash"):
            raise ValueError("attention is 'auto', 'own' or 'flash'")
        if kv_bits not in (4, 16):
            raise ValueError("kv_bits is 16 or 4")
        if window < 0 or sinks < 0:
            raise ValueError("window and sinks must not be negative")
        if kv_bits == 16 and (((window or sinks) and not kv_page) or kv_budget is not None):
            raise ValueError("window, sinks and kv_budget need the 4-bit cache (kv_bits=4); window and sinks a paged one (kv_page)")
        if kv_page < 0 or (kv_pages is not None and (not kv_page or kv_pages < 1)):
            raise ValueError("kv_page and kv_pages must be positive, and come together")
        if kv_page and (kv_bits != 16 or attention == "flash" or cfg.head_dim not in (64, 128)):
            raise ValueError("the paged cache is fp16 and has its own attention, for heads 64 or 128 wide")
        if kv_bits == 4 and (attention == "flash" or cfg.head_dim not in (64, 128)):
            raise ValueError("the 4-bit cache has its own attention, for heads 64 or 128 wide")
        self.kv_bits, self.window, self.sinks, self.kv_budget, self.kv_observe = kv_bits, window, sinks, kv_budget, kv_observe
        self.kv_page = kv_page
        if kv_budget is not None:
            self.kv_recent = kv_budget // 4 if kv_recent is None else kv_recent
            if not (kv_budget > 0 and kv_slack > 0 and kv_observe > 0 and self.kv_recent >= 0 and sinks + self.kv_recent <= kv_budget):
                raise ValueError("kv_budget must hold the sinks and the recent positions, and kv_slack and kv_observe be positive")
            if 0 < window < cfg.max_seq:
                # a step's window counts slots, which are positions only until the first eviction
                raise ValueError("a window cannot be kept over a bounded cache (kv_budget), whose slots are not positions")
        self._flash = None
        grouped = cfg.n_heads // cfg.n_kv_heads
        if attention == "flash" or (attention == "auto" and kv_bits == 16 and not kv_page and cfg.max_seq > 1024 and
                                    grouped > (8 if cfg.head_dim in (64, 128) else 1)):
            try:
                from flash_attn import flash_attn_with_kvcache
                self._flash = flash_attn_with_kvcache
            except Exception:
                if attention == "flash":
                    raise
        self.qc = load_quant_cuda()
        self.group = tp_group
        if tp_group is not None:
            import torch.distributed as dist
            self.tp, self.rank = dist.get_world_size(tp_group), dist.get_rank(tp_group)
        else:
            self.tp, self.rank = 1, 0
        # exchange step of the sharded projections: "peer" = this library's peer-memory kernel for
        # slices that fit its landing area (decode batches), NCCL for the rest (prefill); "nccl" = NCCL only
        self.peer = None
        if self.tp > 1 and tp_gather == "peer":
            from .parallel import PeerAllGather
            try:
                self.peer = PeerAllGather(tp_group, self.dev)
            except RuntimeError as e:       # raised on every rank together: all of them take NCCL
                import warnings
                warnings.warn(f"peer-memory exchange unavailable ({e}); the sharded projections use NCCL")
        elif tp_gather not in ("peer", "nccl"):
            raise ValueError("tp_gather is 'peer' or 'nccl'")
        g = torch.Generator(device=self.dev).manual_seed(seed)
        hd, h, kv = cfg.head_dim, cfg.n_heads, cfg.n_kv_heads
        shapes = {"q": (cfg.hidden, h * hd), "k": (cfg.hidden, kv * hd), "v": (cfg.hidden, kv * hd),
                  "o": (h * hd, cfg.hidden), "gate": (cfg.hidden, cfg.ffn), "up": (cfg.hidden, cfg.ffn),
                  "down": (cfg.ffn, cfg.hidden)}
        if h % self.tp or kv % self.tp or any(n % (8 * self.tp) for _, n in shapes.values()):
            raise ValueError(f"{self.tp} ranks do not divide the heads / output features of this configuration")
        self.full_shapes = shapes
        self.shapes = {name: (k, n // self.tp) for name, (k, n) in shapes.items()}    # this rank's shards
        self.h_local, self.kv_local = h // self.tp, kv // self.tp
        self.layers = []
        for _ in range(cfg.n_layers):
            lay = {name: self._make_linear(k, n, g) for name, (k, n) in self.full_shapes.items()}
            lay["norm1"] = torch.ones(cfg.hidden, dtype=torch.float16, device=self.dev)
            lay["norm2"] = torch.ones(cfg.hidden, dtype=torch.float16, device=self.dev)
            if release_reference_buffers and not dense:
                for name in self.PROJ:
                    lay[name].release_reference_buffers()
            self.layers.append(lay)
        self.embed = (torch.randn(cfg.vocab, cfg.hidden, device=self.dev, generator=g) * 0.02).half()
        self.lm_head = (torch.randn(cfg.vocab, cfg.hidden, device=self.dev, generator=g) * 0.02).half()
        self.final_norm = torch.ones(cfg.hidden, dtype=torch.float16, device=self.dev)
        inv = 1.0 / (cfg.rope_theta ** (torch.arange(0, hd, 2, device=self.dev, dtype=torch.float32) / hd))
        ang = torch.outer(torch.arange(cfg.max_seq, device=self.dev, dtype=torch.float32), inv)
        self.cos, self.sin = ang.cos(), ang.sin()                      # (max_seq, hd / 2)
        if kv_bits == 4:
            slots = cfg.max_seq if kv_budget is None else kv_budget + kv_slack
            make = lambda n: self.qc.KVCache4.empty(batch, self.kv_local, n, hd, kv_group, self.dev)
            self.caches = [make(slots) for _ in range(cfg.n_layers)]
            self.slots = slots
            self.zero = torch.zeros(batch, dtype=torch.long, device=self.dev)
            if kv_budget is not None:
                self.prompt_cache = make(cfg.max_seq)        # of one layer at a time
                self.kv_weights = torch.zeros(cfg.n_layers, batch, self.kv_local, self.caches[0].slots, device=self.dev)
                # slots that hold a position, on the device and on the host
                self.length, self.length_host = torch.zeros(batch, dtype=torch.long, device=self.dev), 0
        elif kv_page:
            from .pages import PageTable
            each = -(-cfg.max_seq // kv_page)
            self.page_table = PageTable(batch, cfg.max_seq, batch * each if kv_pages is None else kv_pages, kv_page)
            self.table = self.page_table.host.to(self.dev)           # the same for all layers
            self.pages = [self.qc.KVPages.empty(self.page_table.pages, self.kv_local, kv_page, hd, torch.float16, self.dev)
                          for _ in range(cfg.n_layers)]
            self.zero = torch.zeros(batch, dtype=torch.long, device=self.dev)
        else:
            self.k_cache = torch.zeros(cfg.n_layers, batch, cfg.max_seq, self.kv_local, hd, dtype=torch.float16, device=self.dev)
            self.v_cache = torch.zeros_like(self.k_cache)
        # state of the decode loop, all on the device: next token and position of every sequence
        self.tok = torch.zeros(batch, dtype=torch.long, device=self.dev)
        self.pos = torch.zeros(batch, dtype=torch.long, device=self.dev)
        self.pos_host = 0           # the host's copy of `pos` (the largest): every step is checked against max_seq before it is launched
        self.held = [0] * batch     # positions of each sequence, with pages
        # what a step adds to the positions: nothing where a sequence has no pages, which would be looked for in more and more places
        self.moves = torch.zeros(batch, dtype=torch.long, device=self.dev) if kv_page else 1
        self.graph = None
        self.controls = self.follow = None

    # ------------------------------------------------------------------ construction
    def _make_linear(self, k: int, n: int, g: torch.Generator) -> QuantLinear:
        cfg = self.cfg
        w = (torch.randn(n, k, device=self.dev, generator=g) * 0.02).half()
        c = math.ceil(k * cfg.cherry_fraction) // 8 * 8
        idx = torch.randperm(k, device=self.dev, generator=g)[:c].to(torch.int32)
        if c:
            w[:, idx.long()] = (torch.randn(n, c, device=self.dev, generator=g) * 0.2).half()
        if self.tp > 1:            # this rank's output rows of the same full matrix
            n = n // self.tp
            w = w[self.rank * n:(self.rank + 1) * n].contiguous()
        ql = QuantLinear(cfg.bits, cfg.group, None, cfg.cherry_fraction, k, n, bias=False).to(self.dev)
        ql.pack(SimpleNamespace(weight=w, bias=None, cherry_indices=idx, group_size=cfg.group))
        if self.dense:
            ql.dense_weight = ql.unpack()
        return ql

    def quantized_bytes_per_token(self) -> int:
        cfg = self.cfg
        per_layer = sum(linear_algorithmic_bytes(k, n, cfg.bits, cfg.group, cfg.cherry_fraction)
                        for k, n in self.shapes.values())
        return per_layer * cfg.n_layers

    def lm_head_bytes(self) -> int:
        return self.cfg.vocab * self.cfg.hidden * 2

    # ------------------------------------------------------------------ building blocks
    def _lin(self, ql: QuantLinear, x: torch.Tensor) -> torch.Tensor:
        if self.dense:
            return F.linear(x, ql.dense_weight)
        return ql(x)

    def _lins(self, lay, names, x: torch.Tensor):
        """The projections `names` of one layer on the same input: one launch where the kernel allows."""
        if self.dense:
            return [F.linear(x, lay[n].dense_weight) for n in names]
        return forward_shared_input([lay[n] for n in names], x)

    def _lin_gather(self, ql: QuantLinear, x: torch.Tensor) -> torch.Tensor:
        """A sharded projection followed by the exchange of its slices; for decode batches of up to four rows
        both happen in one launch of the row-tile kernel."""
        if self.tp > 1 and self.peer is not None and not self.dense and x.shape[0] <= 4 and x.dtype == torch.float16:
            row = ql.row_layer()
            if row is not None and self.peer.fits(x.shape[0], ql.out_features):
                return self.peer.matvec_gather(row, x.contiguous())
        return self._gather(self._lin(ql, x))

    def _gather(self, x: torch.Tensor) -> torch.Tensor:
        """(t, n_local) slices of all ranks -> (t, tp * n_local), in rank order."""
        if self.tp == 1:
            return x
        import torch.distributed as dist
        t, nl = x.shape
        if self.peer is not None and x.dtype == torch.float16 and self.peer.fits(t, nl):
            return self.peer(x.contiguous())
        out = torch.empty(self.tp, t, nl, dtype=x.dtype, device=x.device)
        dist.all_gather_into_tensor(out, x.contiguous(), group=self.group)
        return out.view(1, self.tp * nl) if t == 1 else out.permute(1, 0, 2).reshape(t, self.tp * nl)

    def _norm(self, h: torch.Tensor, delta, w: torch.Tensor):
        """(rmsnorm(h + delta) * w, h + delta): the residual add rides in the norm kernel."""
        if delta is None:
            return self.qc.rmsnorm(h, None, w, self.cfg.eps, False)[0], h
        y, hs = self.qc.rmsnorm(h, delta, w, self.cfg.eps, True)
        return y, hs

    def _norm_lins(self, lay, names, h: torch.Tensor, delta, w: torch.Tensor):
        """The projections `names` of rmsnorm(h + delta) * w, and h + delta: one row in one launch."""
        if self.dense:
            xn, h = self._norm(h, delta, w)
            return self._lins(lay, names, xn), h
        return forward_normed_input([lay[n] for n in names], h, delta, w, self.cfg.eps)

    def _layer(self, li: int, h: torch.Tensor, delta, pos: torch.Tensor, decode: bool):
        """One decoder layer on the residual stream h with the previous layer's MLP output `delta`
        still to be added; returns (h, delta) in the same form."""
        cfg, lay = self.cfg, self.layers[li]
        t, nh, kv, hd, nb = h.shape[0], self.h_local, self.kv_local, cfg.head_dim, self.batch
        (q, k, v), h = self._norm_lins(lay, ("q", "k", "v"), h, delta, lay["norm1"])
        q, k, v = q.view(t, nh, hd), k.view(t, kv, hd), v.view(t, kv, hd)
        if self.kv_bits == 4:
            a = (self._kv4_step if decode else self._kv4_prompt)(li, q, k, v, pos).view(t, nh * hd)
        elif self.kv_page:
            a = (self._pages_step if decode else self._pages_prompt)(li, q, k, v, pos).view(t, nh * hd)
        elif decode and self._flash is None:
            a = self.qc.attn_decode_step(q, k, v, self.cos, self.sin, pos, self.k_cache[li], self.v_cache[li]).view(t, nh * hd)
        else:
            self.qc.rope_cache(q, k, v, self.cos, self.sin, pos, self.k_cache[li], self.v_cache[li])
            if decode:
                a = self._flash(q.view(t, 1, nh, hd), self.k_cache[li], self.v_cache[li],
                                cache_seqlens=(pos + 1).to(torch.int32), causal=True).view(t, nh * hd)
            else:
                ts = t // nb              # tokens per sequence; rows are (sequence, token)
                a = F.scaled_dot_product_attention(q.view(nb, ts, nh, hd).transpose(1, 2), k.view(nb, ts, kv, hd).transpose(1, 2),
                                                   v.view(nb, ts, kv, hd).transpose(1, 2), is_causal=True, enable_gqa=(kv != nh))
                a = a.transpose(1, 2).reshape(t, nh * hd)
        (gate, up), h = self._norm_lins(lay, ("gate", "up"), h, self._lin_gather(lay["o"], self._gather(a)), lay["norm2"])
        if self.tp == 1 and not self.dense and t <= 16:
            # one GPU, decode batch: the SwiGLU rides in the down projection's input staging
            return h, lay["down"].forward_swiglu(gate, up)
        act = self.qc.silu_mul(gate, up)
        return h, self._lin_gather(lay["down"], self._gather(act))

    # ------------------------------------------------------------------ 4-bit cache
    def _kv4_step(self, li: int, q, k, v, pos):
        weights = None if self.kv_budget is None else self.kv_weights[li]
        return self.caches[li].step(q, k, v, self.cos, self.sin, pos, pos if self.kv_budget is None else self.length,
                                    window=self.window, sinks=self.sinks, weights=weights)

    def _kv4_prompt(self, li: int, q, k, v, pos):
        """Attention of the prompts on their fp16 keys and values; the cache takes them in 4 bits, all or the budget's."""
        nb, (t, nh, hd), kv = self.batch, q.shape, k.shape[1]
        cache = self.caches[li] if self.kv_budget is None else self.prompt_cache
        turned = cache.write(torch.cat([q, k], 1), k, v, self.zero, self.cos, self.sin, pos).view(nb, t // nb, nh + kv, hd)
        q, k, v = turned[:, :, :nh], turned[:, :, nh:], v.view(nb, t // nb, kv, hd)
        out, lse = self.qc.attn_prefill(q, k, v, window=self.window, sinks=self.sinks)
        if self.kv_budget is not None:
            weights = torch.zeros(nb, kv, cache.slots, device=self.dev)
            weights[:, :, :t // nb] = self.qc.attn_prefill_weights(q, k, lse, window=self.window, sinks=self.sinks, observe=self.kv_observe)
            _, left, length = cache.evict(weights, self.zero + t // nb, self.kv_budget, sinks=self.sinks, recent=self.kv_recent,
                                          out=self.caches[li])
            self.kv_weights[li, :, :, :self.kv_budget] = left
            self.length.copy_(length)
        return out

    def _kv4_evict(self):
        """Every layer's cache down to the budget; the slots that stay keep their weights."""
        for li, cache in enumerate(self.caches):
            _, left, length = cache.evict(self.kv_weights[li], self.length, self.kv_budget, sinks=self.sinks, recent=self.kv_recent)
            self.kv_weights[li, :, :, :self.kv_budget] = left
        self.length.copy_(length)
        self.length_host = self.kv_budget

    def _kv4_room(self):
        """A free slot for the next position."""
        if self.kv_budget is not None:
            if self.length_host == self.slots:
                self._kv4_evict()
            self.length_host += 1

    def _kv4_rows(self):
        """What a step at positions 0, 1 and 2 changes."""
        rows = [x[:, :, :3] for c in self.caches for x in (c.k_codes, c.k_scales, c.v_codes, c.v_scales)]
        return rows if self.kv_budget is None else rows + [self.kv_weights, self.length]

    # ------------------------------------------------------------------ paged cache
    def _pages_step(self, li: int, q, k, v, pos):
        return self.pages[li].step(q, k, v, self.cos, self.sin, pos, self.table, pos, window=self.window, sinks=self.sinks)

    def _pages_prompt(self, li: int, q, k, v, pos):
        """Attention of the prompts on their own keys and values, which go into their sequences' pages (rows behind a prompt's end
        have no position and go nowhere)."""
        table, lengths = self.prompts
        nb, (t, nh, hd), kv = len(lengths), q.shape, k.shape[1]
        turned = self.pages[li].write(torch.cat([q, k], 1), k, v, table, self.zero[:nb], self.cos, self.sin, pos).view(nb, t // nb, nh + kv, hd)
        return self.qc.attn_prefill(turned[:, :, :nh], turned[:, :, nh:], v.view(nb, t // nb, kv, hd), window=self.window, sinks=self.sinks,
                                    lengths=lengths)[0]

    def _pages_reserve(self, slots):
        """Pages for the first slots[s] positions of the sequences named."""
        if self.page_table.reserve(slots):
            self.table.copy_(self.page_table.host)

    def release(self, rows):
        """These sequences' pages are free for others; their steps are computed, on nothing, until they get a prompt."""
        if not self.kv_page:
            raise ValueError("only a paged cache (kv_page) has pages to give back")
        rows = [int(r) for r in rows]
        if any(not 0 <= r < self.batch for r in rows):
            raise ValueError(f"rows must be sequences of the {self.batch}")
        if not rows:
            return
        for r in rows:
            self.page_table.release(r)
            self.held[r] = 0
        self.table.copy_(self.page_table.host)
        at = torch.tensor(rows, device=self.dev)
        self.pos[at] = self.moves[at] = 0            # (nothing is looked for in pages that they no longer have)
        self.pos_host = max(self.held)

    # ------------------------------------------------------------------ control over what is picked
    def control(self, repetition=None, presence=None, frequency=None, bias=None, grammar=None):
        """From here on tokens are picked from adjusted logits.  repetition, presence, frequency: a number for all sequences or
        one for each (repetition positive), from a sequence's next prompt on; presence and frequency count what was generated, repetition the prompt too.  bias:
        {token: number}.  (prefill's logits are adjusted ones then.)  grammar: (masks (states, words) int32 with a bit for each token, follow (states, vocab) integers: the state
        behind a token, -1 for none; kept in 32 bits, 128 KB a state for 32000 tokens); sequences start in state 0, here and with every
        prompt.  Without arguments: the bare logits again."""
        if all(x is None for x in (repetition, presence, frequency, bias, grammar)):
            self.controls = self.follow = self.graph = None
            return
        each = lambda x: None if x is None else torch.broadcast_to(torch.as_tensor(x, dtype=torch.float32), (self.batch,)).contiguous().to(self.dev)
        c, states = {"repetition": each(repetition), "presence": each(presence), "frequency": each(frequency)}, None
        if repetition is not None and not bool((c["repetition"] > 0).all()):
            raise ValueError("repetition must be positive")
        if bias is not None:
            ids, numbers = list(bias.keys()), list(bias.values())
            c["bias_ids"] = torch.tensor(ids, dtype=torch.long, device=self.dev).expand(self.batch, -1)
            c["bias"] = torch.tensor(numbers, dtype=torch.float32, device=self.dev).expand(self.batch, -1)
        if grammar is not None:
            masks, follow = grammar
            if masks.dtype != torch.int32 or masks.dim() != 2 or masks.shape[0] < 1 or masks.shape[1] < -(-self.cfg.vocab // 32) or \
                    tuple(follow.shape) != (masks.shape[0], self.cfg.vocab) or int(follow.max()) >= masks.shape[0]:
                raise ValueError("grammar is (masks (states, words) int32, follow (states, vocab) of states or -1)")
            c["mask"], states = masks.to(self.dev).contiguous(), (follow.clamp(min=-1) if follow.dtype == torch.long else follow).to(self.dev, torch.int32)
            c["mask_rows"] = torch.zeros(self.batch, dtype=torch.long, device=self.dev)
        if any(c[n] is not None for n in ("repetition", "presence", "frequency")):
            # a sequence's tokens by position, up to the one that is read next
            c["tokens"] = torch.zeros(self.batch, self.cfg.max_seq, dtype=torch.long, device=self.dev)
            c["length"], c["prompt"] = (torch.zeros(self.batch, dtype=torch.long, device=self.dev) for _ in range(2))
        # (nothing has changed so far: a call that is refused leaves the present control, and the graph, as they are)
        self.controls, self.follow, self.graph = c, states, None

    def _pick(self, logits: torch.Tensor, rows=None) -> torch.Tensor:
        """The next token of every sequence (of `rows`); logits are adjusted in place."""
        c = self.controls
        if c is None:
            return logits.argmax(-1)
        mine = c if rows is None else {n: x if x is None or n == "mask" else x[rows] for n, x in c.items()}
        _, picked = self.qc.adjust_logits(logits, **mine, out=logits)
        if self.follow is not None:
            state = mine["mask_rows"]
            behind = torch.where(state >= 0, self.follow[state.clamp(min=0), picked], state)
            if rows is None:
                state.copy_(behind)
            else:
                c["mask_rows"][rows] = behind
        return picked

    def _remember(self):
        """The token that a step reads, in the history."""
        c = self.controls
        if c is not None and c.get("tokens") is not None:
            c["tokens"].scatter_(1, self.pos.clamp(max=self.cfg.max_seq - 1)[:, None], self.tok[:, None])
            c["length"].copy_(torch.where(c["prompt"] > 0, self.pos + 1, 0))       # (0: its prompt was not noted)

    def _logits(self, h: torch.Tensor, delta) -> torch.Tensor:
        return F.linear(self._norm(h, delta, self.final_norm)[0], self.lm_head)

    # ------------------------------------------------------------------ prefill / decode
    @torch.inference_mode()
    def prefill(self, tokens: torch.Tensor, lengths=None, rows=None) -> torch.Tensor:
        """Runs the prompts (T,) or (batch, T), integers of any type on any device, through the model, fills the caches, returns the last
        position's logits (batch, vocab).  With a paged cache: lengths[i] of the T tokens are prompt i's, and prompt i is that of
        sequence rows[i] while the others keep what they have."""
        if tokens.is_floating_point() or tokens.is_complex() or tokens.dtype == torch.bool:
            raise ValueError(f"tokens must be whole numbers, not {tokens.dtype}")
        if tokens.dim() == 1:
            tokens = tokens[None]
        if not self.kv_page and (lengths is not None or rows is not None):
            raise ValueError("prompts of different lengths, and of some sequences alone, need a paged cache (kv_page)")
        some = rows is not None
        rows = list(range(self.batch)) if rows is None else [int(r) for r in rows]
        if tokens.shape[0] != len(rows):
            raise ValueError(f"{tokens.shape[0]} prompts for a decoder of batch {self.batch}" if not some else f"{tokens.shape[0]} prompts for {len(rows)} sequences")
        if len(set(rows)) != len(rows) or any(not 0 <= r < self.batch for r in rows):
            raise ValueError(f"rows must be different sequences of the {self.batch}")
        n, t = tokens.shape
        ends = [t] * n if lengths is None else [int(x) for x in lengths]
        if len(ends) != n or t == 0 or any(not 0 < x <= t for x in ends) or max(ends) >= self.cfg.max_seq:
            if lengths is not None:
                raise ValueError(f"lengths must be 1 to {min(t, self.cfg.max_seq - 1)}, one for each prompt")
            raise ValueError(f"a prompt of {t} tokens does not fit max_seq = {self.cfg.max_seq} (one position must stay free)")
        t = min(t, max(ends))
        tokens = tokens[:, :t].to(self.dev, torch.long)
        place = torch.arange(t, device=self.dev)
        if self.kv_page:
            old = [self.page_table.held[r] for r in rows]
            need = sum(-(-x // self.kv_page) for x in ends)
            if need > len(self.page_table.free) + sum(old):
                raise ValueError(f"{need} pages are needed, {len(self.page_table.free) + sum(old)} of {self.page_table.pages} are free")
            for r in rows:
                self.page_table.release(r)
            self.page_table.reserve(dict(zip(rows, ends)))
            self.table.copy_(self.page_table.host)
            end = torch.tensor(ends, dtype=torch.long, device=self.dev)
            self.prompts = self.table[rows] if some else self.table, end
            inside = place < end[:, None]
            tokens, pos = torch.where(inside, tokens, 0), torch.where(inside, place, -1).reshape(-1)
        else:
            pos = place.repeat(n)
        h, delta = self.embed[tokens.reshape(-1)], None
        for li in range(self.cfg.n_layers):
            h, delta = self._layer(li, h, delta, pos, decode=False)
        last = torch.tensor([i * t + x - 1 for i, x in enumerate(ends)], device=self.dev)
        logits = self._logits(h[last].contiguous(), delta[last].contiguous())
        self._check_exchange()
        for r, x in zip(rows, ends):
            self.held[r] = x
        self.pos_host = max(self.held)
        if self.kv_budget is not None:
            self.length_host = min(t, self.kv_budget)
        at = torch.tensor(rows, device=self.dev)
        filled = torch.tensor(ends, dtype=torch.long, device=self.dev)
        self.pos[at] = filled
        if self.kv_page:
            self.moves[at] = 1
        c = self.controls
        if c is not None and c.get("tokens") is not None:
            c["tokens"][at, :t] = tokens
            c["length"][at], c["prompt"][at] = filled, filled
        if c is not None and c.get("mask_rows") is not None:
            c["mask_rows"][at] = 0
        self.tok[at] = self._pick(logits, at if some else None)
        return logits

    @torch.inference_mode()
    def _step(self) -> torch.Tensor:
        """One greedy decode step on the device-side state; returns the logits (1, vocab)."""
        self._remember()
        h, delta = self.embed[self.tok], None
        for li in range(self.cfg.n_layers):
            h, delta = self._layer(li, h, delta, self.pos, decode=True)
        logits = self._logits(h, delta)
        self.tok.copy_(self._pick(logits))
        self.pos.add_(self.moves)
        if self.kv_budget is not None:
            self.length.add_(1)
        return logits

    @torch.inference_mode()
    def capture(self):
        """Captures one decode step in a CUDA graph (the state tensors are saved and restored)."""
        if self.cfg.max_seq < 4:
            raise ValueError("max_seq must be at least 4")
        # the warm-up and the captured step run at positions 0, 1, 2: always inside the cache, whatever
        # the current position is (state and those cache rows are restored below)
        # (with pages no sequence has any meanwhile)
        rows = self._kv4_rows() if self.kv_bits == 4 else [self.table] if self.kv_page else [self.k_cache[:, :, :3], self.v_cache[:, :, :3]]
        if self.controls is not None:
            rows = rows + [x[:, :3] if n == "tokens" else x for n, x in self.controls.items() if n in ("tokens", "length", "mask_rows") and x is not None]
        saved = [x.clone() for x in (self.tok, self.pos, *rows)]
        self.pos.zero_()
        if self.kv_page:
            self.table.fill_(-1)
        if self.kv_budget is not None:
            self.length.zero_()
        s = torch.cuda.Stream(device=self.dev)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for _ in range(2):          # warm-up: first-use re-packs and allocations happen here
                self._step()
            s.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=s):
                self.graph_logits = self._step()
        torch.cuda.current_stream().wait_stream(s)
        torch.cuda.synchronize()
        for dst, src in zip((self.tok, self.pos, *rows), saved):
            dst.copy_(src)

    @torch.inference_mode()
    def generate(self, n_tokens: int, use_graph: bool = True) -> torch.Tensor:
        """Greedy continuation after `prefill`: returns the n_tokens generated ids, (n_tokens,) for one
        sequence and (n_tokens, batch) for more (the first one is the prefill's argmax)."""
        if n_tokens < 0 or self.pos_host + n_tokens > self.cfg.max_seq:
            raise ValueError(f"{n_tokens} more tokens after position {self.pos_host} do not fit max_seq = "
                             f"{self.cfg.max_seq}: the KV cache holds max_seq positions")
        if self.kv_page:
            self._pages_reserve({r: x + n_tokens for r, x in enumerate(self.held) if x})
        out = torch.empty(n_tokens, self.batch, dtype=torch.long, device=self.dev)
        if use_graph and self.graph is None:
            self.capture()
        for i in range(n_tokens):
            out[i:i + 1].copy_(self.tok)
            if self.kv_bits == 4:
                self._kv4_room()
            if use_graph:
                self.graph.replay()
            else:
                self._step()
        self.held = [x + n_tokens if x else 0 for x in self.held]
        self.pos_host = max(self.held) if self.kv_page else self.pos_host + n_tokens
        self._check_exchange()
        return out[:, 0] if self.batch == 1 else out

    def _check_exchange(self):
        """Raises if a peer never delivered a slice (the kernel fills that output with NaN and sets a
        status bit) or a bounded device-side wait of a projection ran out: one host read per call."""
        if self.peer is not None:
            self.peer.check()
        if self.qc.device_timed_out(self.dev.index if self.dev.index is not None else torch.cuda.current_device()):
            raise RuntimeError("a bounded device-side wait of a quantized projection ran out")
