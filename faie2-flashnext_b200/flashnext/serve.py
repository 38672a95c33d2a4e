"""Serving requests of different lengths: the batched decode step over the paged 4-bit KV cache.

BatchDecodeModel steps its sequences at one position over dense fp32 caches. Here every place of the batch holds a request at a
position of its own: its keys and values live in pages of 4-bit codes (flashnext/kv4.py), a finished request's pages go back
to the pool and its place to the next request, whose DeltaNet states start from zero. Pages, slots and lengths are planned
on the GPU, so a step is one CUDA graph whatever the lengths are.

    m = ServeModel(fn, cfg, W, batch=8, pages=512, max_ctx=4096)
    outs = m.generate(prompts, n_new=[64, 200, ...])        # any number of requests; a list of token arrays

A prompt is fed a token per step, as in the other decode models (the DeltaNet core and the MoE layer take a token per
sequence and step)."""

from __future__ import annotations

import numpy as np

from model import HD, BatchDecodeModel


class OutOfPages(RuntimeError):
    """A step found too few free pages. outs: what generate would have returned, None for requests that were not finished."""

    def __init__(self, message, outs):
        super().__init__(message)
        self.outs = outs


class ServeModel(BatchDecodeModel):
    def __init__(self, fn, cfg: dict, W: dict, batch: int, pages: int, max_ctx: int = 512, page_size: int = 64):
        """pages: of the pool, for each attention layer (one table serves them all); idle places use one each."""
        import torch

        import kv4
        self.page_size, self.n_pages = page_size, pages
        self.ws, self.planner = kv4.KV4Workspace(fn), kv4.KV4Planner(fn, page_size)
        if pages < batch:
            raise ValueError("a page per place of the batch is wanted at least")
        super().__init__(fn, cfg, W, batch, max_ctx)
        dev = self.h.device
        i32 = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=dev)  # noqa: E731
        self.inputs, self.zero, self.drop, self.ones, self.ctx = i32(batch), i32(1), i32(batch), i32(batch) + 1, i32(batch)
        self.table = i32(batch, -(-max_ctx // page_size)) - 1
        self.free_ids = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_count = i32(1) + pages
        self.K = torch.zeros(batch, cfg["nkv"], HD, device=dev)
        self.free_plan, self.plan = kv4.KV4Plan(batch, 0, dev), kv4.KV4Plan(batch, batch, dev)

    def _caches(self, dev):
        import kv4
        return dict(cache=kv4.KV4Cache(self.fn, self.cfg["nkv"], HD, self.page_size, self.n_pages, self.ws))

    def launches_per_step(self) -> int:
        """As the batched step's; two plans instead of the step counter, four attention kernels (norm + RoPE, store, attention
        and its join, which a single place of up to 128 tokens does without) instead of two."""
        attn = sum(L["kind"] != "G" for L in self.layers)
        join = self.B > 1 or self.table.shape[1] * self.page_size > 128
        return super().launches_per_step() + (1 + join) * attn + 1

    def _embed(self, s):
        """The step's plan (places that are dropped give their pages back, then every place gets a row), then its inputs."""
        f, p, d = self.planner, self.plan, self.free_plan
        f.plan(self.ctx, self.drop, self.table, self.free_ids, self.free_count, 0, out=d)
        f.plan(d.ctx, self.ones, self.table, self.free_ids, d.free_count, self.B, out=p)
        self.fn.embed_batch(self.cfg["embed"], self.E.data_ptr(), self.cfg["D"], self.inputs.data_ptr(), 1,
                            self.zero.data_ptr(), self.h.data_ptr(), self.B, s)

    def _attention(self, L, s):
        nh, nkv, B = self.cfg["nh"], self.cfg["nkv"], self.B
        qg = self.proj[:, :nh * 2 * HD].unflatten(1, (nh, 2 * HD))
        k, v = (self.proj[:, nh * 2 * HD + i * nkv * HD:nh * 2 * HD + (i + 1) * nkv * HD].unflatten(1, (nkv, HD)) for i in (0, 1))
        ps, q = self.proj.shape[1], self.Q.view(B, nh, HD)
        self.fn.qk_rope_rows(qg.data_ptr(), ps, 2 * HD, k.data_ptr(), ps, HD, L["q_norm"].data_ptr(), L["k_norm"].data_ptr(),
                             self.inv_freq.data_ptr(), self.plan.positions.data_ptr(), B, nh, nkv, q.data_ptr(),
                             self.K.data_ptr(), self.cfg["eps"], s)
        L["cache"].store(self.K, v, self.plan.slots)
        L["cache"].attn(q, self.plan.cu, self.plan.kv_len, self.table, max_new=1, gate=qg[..., HD:], out=self.att.view(B, nh, HD))

    def _advance(self, s):
        """The lengths and the pool of the next step."""
        import torch
        with torch.cuda.stream(torch.cuda.ExternalStream(s)):
            self.ctx.copy_(self.plan.ctx)
            self.free_count.copy_(self.plan.free_count)

    def launch_step(self, s: int):
        import torch
        with torch.cuda.stream(torch.cuda.ExternalStream(s)):  # the kv4 layer launches on the current stream
            super().launch_step(s)

    def start(self, prompts, stream):
        """Every place idle: no request, no pages taken."""
        import torch
        with torch.cuda.stream(stream):
            self.inputs.zero_()
            self.ctx.zero_()
            self.drop.fill_(-1)
            self.table.fill_(-1)
            self.free_ids.copy_(torch.arange(self.n_pages, dtype=torch.int32))
            self.free_count.fill_(self.n_pages)
        for g in self.gdns:
            self.fn.gdn_reset(g, stream.cuda_stream)

    def generate(self, prompts, n_new, stream, logits=None, wait=False):
        """Greedy decode of any number of requests, as many at a time as the batch has places. prompts: a list of token id
        arrays (of any lengths); n_new: tokens to generate, one number or one per request. Returns a list of arrays, prompt
        then new tokens. logits: an optional callback(request, position, row [vocab]) per step. wait: a request is admitted, in order,
        when the pages that it may come to need fit beside those of the requests before it and one for each idle place; without
        it requests take places as they come free, and a step that finds no page raises OutOfPages."""
        import torch
        if self.graph is None:
            raise RuntimeError("capture() the step first")
        prompts = [np.asarray(p, np.int32).reshape(-1) for p in prompts]
        n_new = [n_new] * len(prompts) if np.ndim(n_new) == 0 else list(n_new)
        if len(n_new) != len(prompts) or any(len(p) < 1 or n < 1 or len(p) + n > self.max_ctx for p, n in zip(prompts, n_new)):
            raise ValueError("every request wants a prompt and new tokens within the context")
        need = [-(-(len(p) + n - 1) // self.page_size) for p, n in zip(prompts, n_new)]  # the last token is not fed
        if wait and max(need, default=0) + self.B - 1 > self.n_pages:
            raise ValueError("a request wants more pages than there are beside one for each other place")
        self.start(None, stream)
        waiting, place, seq = list(range(len(prompts))), [None] * self.B, [p.tolist() for p in prompts]
        at = [0] * self.B  # tokens fed of the place's request
        inputs, drop = np.zeros(self.B, np.int32), np.full(self.B, -1, np.int32)
        while waiting or any(r is not None for r in place):
            for b in range(self.B):
                drop[b] = -1 if place[b] is None else 0
                held = [need[r] for r in place if r is not None]
                if place[b] is None and waiting and (
                        not wait or sum(held) + need[waiting[0]] + self.B - len(held) - 1 <= self.n_pages):
                    place[b], at[b] = waiting.pop(0), 0
                    for g in self.gdns:
                        self.fn.gdn_reset_seq(g, b, stream.cuda_stream)
                inputs[b] = 0 if place[b] is None else seq[place[b]][at[b]]
            with torch.cuda.stream(stream):
                self.inputs.copy_(torch.from_numpy(inputs))
                self.drop.copy_(torch.from_numpy(drop))
                self.graph.replay()
            self.fn.sync(stream.cuda_stream)
            if int(self.plan.status):
                done = [np.array(s, np.int32) if len(s) == len(p) + n else None for s, p, n in zip(seq, prompts, n_new)]
                raise OutOfPages(f"out of pages: {int(self.plan.status)} of the batch found none (of {self.n_pages})", done)
            new = self.next.cpu().numpy()
            for b, r in enumerate(place):
                if r is None:
                    continue
                if logits is not None:
                    logits(r, at[b], self.logits[b])
                at[b] += 1
                if at[b] == len(seq[r]):
                    seq[r].append(int(new[b]))
                if len(seq[r]) == len(prompts[r]) + n_new[r]:
                    place[b] = None
        return [np.array(s, np.int32) for s in seq]
