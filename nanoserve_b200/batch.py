"""Several sequences at once on a `Qwen2Runner`'s weights: continuations of one common prefix, sampled.

The reference serves one sequence at a time, greedily (``python/nanoserve/qwen.py:12,166-178``).  Here the common prefix is run
once and its keys and values are stored once, in whole pages that every sequence's table begins with; what is left of it and the
sequences' own prompts follow as one ragged batch of rows.  A decode step takes one row per sequence through the quantized linears
(`w4_linear` at M = number of sequences), `paged_kv_append`, `shared_prefix_attention` and `sample`; one CUDA graph serves every
step, since lengths, step and random numbers are read on the device.
"""
from typing import List, Optional, Sequence

import torch
import torch.nn.functional as F

from .qwen import Qwen2Runner


class Batch:
    """`n_seqs` sequences of up to `max_own` tokens each behind a common prefix of up to `max_prefix`, on one GPU."""

    def __init__(self, runner: Qwen2Runner, n_seqs: int, max_prefix: int, max_own: int, page: int = 64):
        if runner.world != 1:
            raise ValueError("a batch runs on one GPU")
        cfg, dev = runner.cfg, runner.dev
        if n_seqs < 1 or max_own < 1 or max_prefix < 0:
            raise ValueError(f"{n_seqs} sequences of up to {max_own} tokens behind up to {max_prefix}")
        if page not in (16, 32, 64, 128, 256, 512, 1024) or cfg.head_dim not in (64, 128):
            raise ValueError(f"pages of {page} tokens, heads of {cfg.head_dim}: a power of two from 16 to 1024, and 64 or 128")
        self.r, self.k, self.B, self.page, self.max_own = runner, runner.k, n_seqs, page, max_own
        self.heads = (cfg.n_heads, cfg.n_kv_heads, cfg.head_dim)
        self.n_shared = max_prefix // page
        own = -(-(max_own + page) // page)  # (what is left of the prefix goes to every sequence's own pages)
        shape = (cfg.n_layers, self.n_shared + n_seqs * own, cfg.n_kv_heads, page, cfg.head_dim)
        self.cache_k, self.cache_v = (torch.zeros(shape, dtype=torch.bfloat16, device=dev).unbind(0) for _ in range(2))
        self.own_table = self.n_shared + torch.arange(n_seqs * own, dtype=torch.int32, device=dev).view(n_seqs, own)
        self.shared = -1  # tokens of the prefix in its pages; set by prefill, as the tables that depend on it
        self.prefix_len = torch.zeros(1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(n_seqs, dtype=torch.int32, device=dev)
        self.step_no = torch.zeros(1, dtype=torch.int64, device=dev)
        self.left = 0  # steps that there is room for
        self.tokens = torch.zeros(max_own, n_seqs, dtype=torch.int64, device=dev)
        self.last = torch.zeros(n_seqs, dtype=torch.int64, device=dev)
        self.u = torch.zeros(max_own, n_seqs, device=dev)
        self.logits = torch.zeros(n_seqs, cfg.vocab, dtype=torch.bfloat16, device=dev)
        self.sampling = dict(temperature=0.0)
        self.graph: Optional[torch.cuda.CUDAGraph] = None

    def _layers(self, x, attend):
        """The decoder layers over rows x [T, H]; attend(layer, qkv) -> [T, Hq D].  Returns the final norm of the rows."""
        r, k, cfg = self.r, self.k, self.r.cfg
        h = k.rmsnorm(x, None, r.layers[0]["ln_in"], cfg.rms_eps)
        for li, L in enumerate(r.layers):
            a = attend(li, r.linear(h, L["qkv"]))
            h = k.rmsnorm(x, r.linear(a, L["o"]), L["ln_post"], cfg.rms_eps)
            if r.gu_block == 16:
                act = k.w4_linear_swiglu(h, L["gu"][0], L["gu"][1], cfg.group)
            else:
                act = k.swiglu_blocks(r.linear(h, L["gu"]), r.gu_block)
            nxt = r.layers[li + 1]["ln_in"] if li + 1 < cfg.n_layers else r.final_norm
            h = k.rmsnorm(x, r.linear(act, L["d"]), nxt, cfg.rms_eps)
        return h

    def _append(self, li, qkv, table, lens, cu=None):
        return self.k.paged_kv_append(qkv, self.r.layers[li]["bias"], self.r.inv_freq, self.cache_k[li], self.cache_v[li], table,
                                      lens, *self.heads, cu_tokens=cu)

    def _pick(self, h):
        """One token per row of h [B, H]: logits (the vocabulary projection takes eight rows at a time), then the draw."""
        for b in range(0, self.B, 8):
            self.k.lm_head(h[b:b + 8], self.r.lm_head, logits=self.logits[b:b + 8])
        u = self.u.index_select(0, self.step_no)[0]
        self.k.sample(self.logits, u, out=self.last, **self.sampling)
        self.tokens.index_copy_(0, self.step_no, self.last[None])
        self.step_no.add_(1).clamp_(max=self.max_own - 1)  # (a captured step replayed beyond the room goes on writing the last row)

    @torch.no_grad()
    def prefill(self, prefix: torch.Tensor, prompts: Sequence[torch.Tensor]):
        """Runs the prefix [P] once and every sequence's prompt behind it, and draws the first token of each."""
        if len(prompts) != self.B:
            raise ValueError(f"{len(prompts)} prompts for {self.B} sequences")
        P, dev = prefix.numel(), self.r.dev
        shared = min(max(P - 1, 0) // self.page, self.n_shared) * self.page  # (every sequence has a row of its own to draw from)
        own = [torch.cat([prefix[shared:], p]) for p in prompts]
        n = [o.numel() for o in own]
        if min(n) < 1 or max(n) > self.own_table.shape[1] * self.page:
            raise ValueError("a sequence has no token, or more than its pages hold")
        if shared != self.shared:  # (else a captured step goes on reading the tables that are there)
            self.graph, self.shared = None, shared
            self.prefix_len.fill_(shared)
            self.prefix_table = torch.arange(shared // self.page, dtype=torch.int32, device=dev)
            self.table = torch.cat([self.prefix_table[None].expand(self.B, -1), self.own_table], 1).contiguous()
        self.lens.copy_(torch.tensor([shared + x for x in n], dtype=torch.int32))
        self.step_no.zero_()
        self.left = min(self.max_own - 1, self.own_table.shape[1] * self.page - max(n))
        ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
        if shared:
            cu, lens, table = ints(0, shared), ints(shared), self.prefix_table[None]

            def attend(li, qkv):
                q = self._append(li, qkv, table, lens, cu)
                return self.k.paged_attention(q, self.cache_k[li], self.cache_v[li], table, lens, *self.heads, cu_tokens=cu)
            self._layers(F.embedding(prefix[:shared], self.r.embed), attend)
        ends = torch.tensor(n).cumsum(0)
        cu = ints(0, *ends.tolist())

        def attend(li, qkv):
            q = self._append(li, qkv, self.table, self.lens, cu)
            return self.k.paged_attention(q, self.cache_k[li], self.cache_v[li], self.table, self.lens, *self.heads, cu_tokens=cu,
                                          max_tokens=max(n))
        h = self._layers(F.embedding(torch.cat(own), self.r.embed), attend)
        self._pick(h[(ends - 1).to(dev)].contiguous())

    @torch.no_grad()
    def step(self):
        """The next token of every sequence (nothing of it on the host: it can be captured; replays beyond the room write the last row
        of `tokens`, and keys that find no page are left out).  A row without a token (-1: its logits were not numbers) goes on from
        token 0."""
        if self.left < 1:
            raise ValueError("no prefill, or no room for another token")
        self.left -= 1
        self.lens += 1
        first = self.shared // self.page
        own_lens = self.lens - self.prefix_len

        def attend(li, qkv):
            q = self._append(li, qkv, self.table, self.lens)
            if not self.shared:
                return self.k.paged_attention(q, self.cache_k[li], self.cache_v[li], self.table, self.lens, *self.heads)
            return self.k.shared_prefix_attention(q, self.cache_k[li], self.cache_v[li], self.prefix_table, self.prefix_len,
                                                  self.table[:, first:], own_lens, *self.heads)
        self._pick(self._layers(F.embedding(self.last.clamp(min=0), self.r.embed), attend))

    def generate(self, prefix: torch.Tensor, prompts: Sequence[torch.Tensor], n_new: int, temperature: float = 1.0, top_k: int = 0,
                 top_p: float = 1.0, min_p: float = 0.0, u: Optional[torch.Tensor] = None, seed: int = 0,
                 use_graph: bool = True) -> List[List[int]]:
        """`n_new` tokens of every sequence.  u [n_new, n_seqs]: the random numbers, uniform in [0, 1); else drawn from `seed`.
        Returns a list of ids per sequence."""
        most = self.own_table.shape[1] * self.page
        longest = max(p.numel() for p in prompts) + prefix.numel() - min(max(prefix.numel() - 1, 0) // self.page,
                                                                         self.n_shared) * self.page
        if n_new < 1 or n_new > self.max_own or longest + n_new - 1 > most:
            raise ValueError(f"{n_new} tokens do not fit behind {longest} in pages for {most}")
        sampling = dict(temperature=float(temperature), top_k=int(top_k), top_p=float(top_p), min_p=float(min_p))
        if sampling != self.sampling:
            self.graph = None  # they are part of it
        self.sampling = sampling
        if u is None:
            u = torch.rand(n_new, self.B, device=self.r.dev, generator=torch.Generator(device=self.r.dev).manual_seed(seed))
        stream = self.r.stream  # split linears of one device share scratch: everything runs on the runner's own stream
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            self.u[:n_new].copy_(u)
            self.prefill(prefix, prompts)
            if use_graph and self.graph is None and n_new > 1:
                lens, step_no, last, left = self.lens.clone(), self.step_no.clone(), self.last.clone(), self.left
                self.step()  # (warms what the capture needs; its token is drawn again)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                self.left = left
                with torch.cuda.graph(graph, stream=stream):
                    self.step()
                self.graph, self.left = graph, left
                self.lens.copy_(lens)
                self.step_no.copy_(step_no)
                self.last.copy_(last)
            for _ in range(n_new - 1):
                if use_graph:
                    self.left -= 1
                    self.graph.replay()
                else:
                    self.step()
        torch.cuda.synchronize()
        self.r.check_status()
        return self.tokens[:n_new].T.tolist()
