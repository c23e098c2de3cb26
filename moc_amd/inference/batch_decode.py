"""Decode of a batch of sequences with a DecoderModel over a paged 8-bit cache:
ragged prompts in one forward, then one token a sequence and step, drawn with
temperature, top-k, top-p and min-p.  The reference decodes one sequence
greedily over a static bf16 cache (benchmark_decode.py:366-420,
moc_amd/inference/decode_model.py); layers, weights and FFN forms are those.

A step of a layer: norm, q/k/v projection, K.paged_append (RoPE, keys and values
into the pages), K.paged_attention, out_proj, residual, then the FFN half.  A
whole step, the draw included, is captured in one HIP graph: the sequences'
lengths, page tables and tokens are device buffers that it reads.
"""
from __future__ import annotations

import math
from typing import Sequence

import torch

from .. import kernels as K
from .decode_model import DecoderModel


class BatchDecoder:
    """`slots` sequences over one pool of pages for each layer.

    codes: float8_e4m3fn or int8, what keys and values are held in; page: tokens a
    page (a power of two from 16 to 256); pages: of the pool, by default enough
    for every slot at the model's max_seq."""

    def __init__(self, model: DecoderModel, slots: int, *, page: int = 64, pages: int | None = None,
                 codes: torch.dtype = torch.float8_e4m3fn):
        cfg, w = model.cfg, model.embed.weight
        if w.dtype != torch.bfloat16:
            raise ValueError(f"BatchDecoder runs bf16 models, got {w.dtype}")
        if slots < 1:
            raise ValueError("BatchDecoder: at least one slot")
        width = -(-cfg.max_seq // page)
        self.model, self.slots, self.page = model, slots, page
        self.pages = slots * width if pages is None else pages
        self.heads, self.head_dim = cfg.heads, cfg.hidden // cfg.heads
        self.kv = [K.paged_kv(self.pages, self.heads, page, self.head_dim, dtype=codes, device=w.device)
                   for _ in model.layers]
        zeros = lambda *s, dtype=torch.int32: torch.zeros(*s, dtype=dtype, device=w.device)  # noqa: E731
        self.table, self.lens = zeros(slots, width), zeros(slots)
        self.live = zeros(slots)                       # 1: the slot takes a token a step
        self.room = zeros(slots)                       # positions that it has a place and an angle for
        self.tokens = zeros(slots, dtype=torch.int64)  # the last token of each
        # what the last step drew for each: the id; -1: its logits are NaN; -2: it took none
        self.drawn = zeros(slots, dtype=torch.int64)
        self._none = torch.full_like(self.drawn, -2)
        self.release()

    def release(self) -> None:
        """Every page back to the pool, every slot out of use."""
        self._free = list(range(self.pages - 1, -1, -1))
        self._held: list[list[int]] = [[] for _ in range(self.slots)]
        self._live = [False] * self.slots
        self._upload()
        self.lens.zero_()
        self.drawn.copy_(self._none)

    def _upload(self) -> None:
        # -1: no page; a token there is not stored and its logits are NaN
        rows = [h + [-1] * (self.table.shape[1] - len(h)) for h in self._held]
        self.table.copy_(torch.tensor(rows, dtype=torch.int32))
        self.live.copy_(torch.tensor(self._live, dtype=torch.int32))
        room = [min(len(h) * self.page, self.model.cfg.max_seq) for h in self._held]
        self.room.copy_(torch.tensor(room, dtype=torch.int32))

    def _more(self, what: str, tokens: Sequence[int], held: Sequence[list[int]], free: int) -> list[int]:
        """Pages that the slots want beside the ones they hold, if there are so many."""
        if max(tokens) > self.model.cfg.max_seq:
            raise ValueError(f"{what}: {max(tokens)} tokens, the model has {self.model.cfg.max_seq} positions")
        more = [max(-(-n // self.page) - len(h), 0) for n, h in zip(tokens, held)]
        if sum(more) > free:
            raise ValueError(f"{what}: {sum(more)} pages wanted, {free} are free")
        return more

    def reserve(self, tokens: Sequence[int]) -> None:
        """Pages for tokens[slot] tokens of each slot.  0: out of use; the slot
        keeps its pages, its length and its token, and goes on when a later call
        names it again."""
        if len(tokens) != self.slots:
            raise ValueError(f"reserve: {self.slots} slots, got {len(tokens)}")
        more = self._more("reserve", tokens, self._held, len(self._free))
        for held, m in zip(self._held, more):
            held.extend(self._free.pop() for _ in range(m))
        self._live = [n > 0 for n in tokens]
        self._upload()

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, cu: torch.Tensor | None = None,
                lens: torch.Tensor | None = None) -> torch.Tensor:
        """Hidden states [tokens, hidden] of new tokens whose sequences' lengths
        (self.lens or the ones given, these tokens counted) are set; cu as in
        K.paged_append."""
        x = self.model.embed(tokens)
        lens = self.lens if lens is None else lens
        scale = 1.0 / math.sqrt(self.head_dim)
        for layer, kv in zip(self.model.layers, self.kv):
            a = layer.attn
            q, k, v = a.qkv_proj(layer.attn_norm(x)).view(-1, 3 * self.heads, self.head_dim).split(self.heads, dim=1)
            q = K.paged_append(q, k, v, a.rope_cos, a.rope_sin, kv, self.table, lens, cu)
            o = K.paged_attention(q, kv, self.table, lens, cu, scale=scale)
            x = x + a.out_proj(o.flatten(1))
            if layer.fuse:
                x = layer.ffn.fused_decode_residual(x, layer.ffn_norm.weight, layer.ffn_norm.eps)
            else:
                x = x + layer._ffn(layer.ffn_norm(x)[None])[0]
        return x

    @torch.no_grad()
    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return self.model.lm_head(self.model.final_norm(x))

    @torch.no_grad()
    def prompt(self, prompts: Sequence[torch.Tensor], room: int = 0) -> torch.Tensor:
        """Starts the first slots with these prompts (1-D token ids, at least one
        token each) and pages for `room` tokens more; logits [prompts, vocab] behind
        their last tokens, from which the caller draws self.tokens.  What ran before
        ends in every slot, unless the prompts are refused."""
        n = [int(p.numel()) for p in prompts]
        if not n or min(n) < 1 or len(n) > self.slots:
            raise ValueError(f"prompt: 1 to {self.slots} prompts of at least one token")
        if room < 0:
            raise ValueError(f"prompt: room for {room} tokens")
        empty = [0] * (self.slots - len(n))
        wanted = [t + room for t in n] + empty
        self._more("prompt", wanted, [[]] * self.slots, self.pages)
        self.release()
        self.reserve(wanted)
        self.lens.copy_(torch.tensor(n + empty, dtype=torch.int32))
        cu = torch.tensor([0, *n, *empty], dtype=torch.int32).cumsum(0, dtype=torch.int32).to(self.lens.device)
        x = self.forward(torch.cat([p.reshape(-1) for p in prompts]).to(self.tokens.device), cu)
        return self.logits(x.index_select(0, cu[1:len(n) + 1].long() - 1))

    @torch.no_grad()
    def step(self, u: torch.Tensor, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
        """One token more of each live slot: self.tokens go in, are replaced by
        the drawn ones (K.sample_tokens with the uniform numbers u [slots]) and
        returned.  Slots out of use keep theirs.  So does one whose pages are full,
        which goes on once reserve gives it room.  One whose logits are NaN gets
        token 0.  self.drawn tells these from a drawn token."""
        takes = self.lens < self.room * self.live  # it has a place for its token
        lens = self.lens + takes
        # a slot that takes none has its token still to store: of no length, it stores nothing
        logits = self.logits(self.forward(self.tokens, lens=lens * takes))
        drawn = K.sample_tokens(logits, u, temperature, top_k, top_p, min_p)
        self.lens.copy_(lens)  # only now: a step that is refused is none
        torch.where(takes, drawn, self._none, out=self.drawn)
        torch.where(takes, drawn.clamp_min(0), self.tokens, out=self.tokens)
        return self.tokens

    @torch.no_grad()
    def generate(self, prompts: Sequence[torch.Tensor], length: int, *, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0,
                 generator: torch.Generator | None = None, graph: bool = True) -> torch.Tensor:
        """`length` tokens behind each prompt, int64 [prompts, length].  Settings
        are numbers, or tensors [slots] (K.sample_tokens); temperature 0 is
        greedy.  graph: the step is captured once and replayed.  A sequence whose
        logits are NaN goes on with token 0 (self.drawn: of the last token)."""
        if length < 1:
            raise ValueError("generate: at least one token")
        n, dev = len(prompts), self.lens.device
        u = torch.rand(length, self.slots, generator=generator, device=dev)
        settings = (temperature, top_k, top_p, min_p)
        first = self.prompt(prompts, room=length - 1)
        of = [s[:n] if isinstance(s, torch.Tensor) else s for s in settings]
        self.drawn[:n] = K.sample_tokens(first, u[0, :n], *of)
        self.tokens[:n] = self.drawn[:n].clamp_min(0)
        out = torch.empty(n, length, dtype=torch.int64, device=dev)
        out[:, 0] = self.tokens[:n]
        now, step = torch.empty_like(u[0]), None
        if graph and length > 2:
            step = self._capture(now, settings)
        for i in range(1, length):
            now.copy_(u[i])
            if step is None:
                self.step(now, *settings)
            else:
                step.replay()
            out[:, i] = self.tokens[:n]
        return out

    def _capture(self, u: torch.Tensor, settings) -> torch.cuda.CUDAGraph:
        """The step as a HIP graph.  The warm-up runs change nothing: with no
        live slot and lengths of 0 no key is stored and no token replaced.  They
        bring what the FFNs derive from their weights up to date, so that the
        capture makes none of it and the model need not be frozen."""
        lens, live, drawn = self.lens.clone(), self.live.clone(), self.drawn.clone()
        self.lens.zero_()
        self.live.zero_()
        try:
            with torch.cuda.device(u.device):
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                try:
                    with torch.cuda.stream(side):
                        for _ in range(2):
                            self.step(u, *settings)
                finally:
                    torch.cuda.current_stream().wait_stream(side)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    self.step(u, *settings)
        finally:
            self.lens.copy_(lens)
            self.live.copy_(live)
            self.drawn.copy_(drawn)
        return graph
