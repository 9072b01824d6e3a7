"""Several sessions decoded together under a cache budget.

A small random decoder (grouped-query attention, gated MLP)
whose sessions share one pool of pages per layer.  The prompts, each of its
own length, are appended in one call per layer; every step then appends one
row per session, attends over each session's slots while the attention weight
of every slot accumulates, and samples under per-session penalties, biases and
an allow mask.  A session that has grown `slack` slots past its budget keeps
its first tokens, its latest ones and the heaviest of the rest.

    python -m examples.paged_batch --sessions 8 --steps 200 --budget 192 --kv k8v4
"""
from __future__ import annotations

import argparse

import torch

from rec_b200 import paged, sampling

KV_FORMATS = {"bf16": (16, 16), "k8v8": (8, 8), "k8v4": (8, 4), "k4v4": (4, 4)}


class Decoder:
    """Weights and the residual stream are fp32; q, the cache and the
    attention's output are bf16, as the kernels take them."""

    def __init__(self, layers=2, hidden=256, heads=8, kv_heads=2, head_dim=64, vocab=1000, seed=0):
        self.layers, self.hidden, self.heads, self.kv_heads, self.head_dim = layers, hidden, heads, kv_heads, head_dim
        g = torch.Generator(device="cuda").manual_seed(seed)

        def matrix(n, k):
            return torch.randn(n, k, device="cuda", generator=g) * k ** -0.5

        self.embedding, self.head = matrix(vocab, hidden) * hidden ** 0.5, matrix(vocab, hidden)
        line = (heads + 2 * kv_heads) * head_dim
        self.blocks = [dict(qkv=matrix(line, hidden), o=matrix(hidden, heads * head_dim),
                            up=matrix(4 * hidden, hidden), down=matrix(hidden, 2 * hidden)) for _ in range(layers)]
        self.frequency = 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda", dtype=torch.float64) / head_dim)

    @staticmethod
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)

    def rope(self, x, positions):
        angle = positions.double()[:, None, None] * self.frequency
        cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)
        a, b = x.chunk(2, -1)
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    def qkv(self, block, x, positions):
        q, k, v = (self.norm(x) @ block["qkv"].T).unflatten(1, (-1, self.head_dim)).split(
            [self.heads, self.kv_heads, self.kv_heads], 1)
        return self.rope(q, positions), self.rope(k, positions), v

    def finish(self, block, x, attended):
        x = x + attended.flatten(1).to(x.dtype) @ block["o"].T
        gate, up = (self.norm(x) @ block["up"].T).chunk(2, -1)
        return x + (torch.nn.functional.silu(gate) * up) @ block["down"].T

    def logits(self, x):
        return 2.0 * self.norm(x) @ self.head.T


class PagedBatch:
    """The sessions' caches and one step of all of them."""

    def __init__(self, model: Decoder, sessions: int, budget: int, *, slack=32, page=16, kv="bf16", recent=32, first=4,
                 decay=0.98):
        if kv not in KV_FORMATS or not 0 < first + recent < budget or slack < 1:
            raise ValueError("kv must be one of " + ", ".join(KV_FORMATS) + "; first + recent below the budget")
        self.model, self.budget, self.slack, self.recent, self.first, self.decay = model, budget, slack, recent, first, decay
        self.page, self.sessions = page, sessions
        self.kv = kv
        self.i32 = dict(device="cuda", dtype=torch.int32)
        self.lengths = torch.zeros(sessions, **self.i32)
        self.positions = torch.zeros(sessions, **self.i32)  # of the next token
        self.longest = 0
        self.steps = torch.arange(sessions + 1, **self.i32)
        self.logits = None

    def _reserve(self, slots: int) -> None:
        width = -(-slots // self.page)
        pages = width * self.sessions
        m, (kb, vb) = self.model, KV_FORMATS[self.kv]
        # any order will do; sessions that grow by turns get theirs interleaved
        self.table = torch.arange(pages, **self.i32).reshape(width, self.sessions).T.contiguous()
        self.caches = [paged.PagedKV.allocate(pages, m.kv_heads, self.page, m.head_dim, k_bits=kb, v_bits=vb)
                       for _ in range(m.layers)]
        per_slot = (pages, m.kv_heads, self.page)
        self.weights = [torch.zeros(per_slot, device="cuda") for _ in range(m.layers)]
        self.places = [torch.zeros(per_slot, **self.i32) for _ in range(m.layers)]

    def prefill(self, prompts) -> torch.Tensor:
        """Every session's prompt (a list of ids each); logits [sessions, vocab]."""
        counts = [len(p) for p in prompts]
        if len(counts) != self.sessions or min(counts) < 1:
            raise ValueError("one prompt of at least one token per session")
        self._reserve(max(max(counts), self.budget + self.slack))
        ids = torch.tensor([t for p in prompts for t in p], device="cuda")
        n = torch.tensor(counts, **self.i32)
        cu = torch.cat([self.steps[:1], n.cumsum(0).int()])
        session = torch.repeat_interleave(torch.arange(self.sessions, device="cuda"), n.long())
        positions = torch.arange(len(ids), **self.i32) - cu[session]
        x, last = self.model.embedding[ids], (cu[1:] - 1).long()
        zeros = torch.zeros_like(n)
        for block, cache, weights, places in zip(self.model.blocks, self.caches, self.weights, self.places):
            q, k, v = self.model.qkv(block, x, positions)
            q, k, v = q.bfloat16(), k.bfloat16(), v.bfloat16()
            paged.paged_append(cache, k, v, self.table, zeros, cu, weights=weights, positions=places)
            # a prompt token attends as a session of its own length would, up to 4,096 of them a call
            attended = torch.cat([paged.paged_attn_decode(cache, q[i:i + 4096], self.table[session[i:i + 4096]],
                                                          positions[i:i + 4096] + 1) for i in range(0, len(ids), 4096)])
            # the last token's weights are what the first eviction goes by
            paged.paged_attn_decode(cache, q[last], self.table, n, weights=weights)
            x = self.model.finish(block, x, attended)
        self.lengths, self.positions, self.longest = n, n.clone(), max(counts)
        self._evict()
        self.logits = self.model.logits(x[last])
        return self.logits

    def step(self, ids: torch.Tensor) -> torch.Tensor:
        """One token per session; logits [sessions, vocab]."""
        x = self.model.embedding[ids.long()]
        lengths = self.lengths + 1
        for block, cache, weights, places in zip(self.model.blocks, self.caches, self.weights, self.places):
            q, k, v = self.model.qkv(block, x, self.positions)
            paged.paged_append(cache, k.bfloat16(), v.bfloat16(), self.table, self.lengths, self.steps, weights=weights,
                               positions=places, first_positions=self.positions)
            attended = paged.paged_attn_decode(cache, q.bfloat16(), self.table, lengths, weights=weights, decay=self.decay)
            x = self.model.finish(block, x, attended)
        self.lengths, self.positions, self.longest = lengths, self.positions + 1, self.longest + 1
        self._evict()
        self.logits = self.model.logits(x)
        return self.logits

    def _evict(self) -> None:
        if self.longest < self.budget + self.slack:
            return
        for cache, weights, places in zip(self.caches, self.weights, self.places):
            lengths = paged.paged_evict(cache, self.table, self.lengths, self.budget, weights, positions=places,
                                        keep_from=self.positions - self.recent, keep_below=self.first)
        self.lengths, self.longest = lengths, self.budget

    def generate(self, prompts, steps: int, *, temperature=0.8, top_k=50, top_p=0.95, seed=0, repetition=1.1,
                 frequency=0.1, presence=0.1, bias=None, banned=()) -> torch.Tensor:
        """ids int32 [sessions, steps].  bias: {id: value}; banned: ids that
        no session may sample."""
        logits = self.prefill(prompts)
        vocab = logits.shape[1]
        n = max(len(p) for p in prompts)
        history = torch.zeros(self.sessions, n + steps, **self.i32)
        for b, p in enumerate(prompts):
            history[b, :len(p)] = torch.tensor(p, **self.i32)
        prompt_len = self.positions.clone()
        used = prompt_len.clone()
        allowed = torch.ones(-(-vocab // 32) * 32, dtype=torch.int64)
        allowed[torch.tensor(list(banned), dtype=torch.int64)] = 0
        words = (allowed.reshape(-1, 32) << torch.arange(32)).sum(1).to(torch.uint32).view(torch.int32).cuda()
        allow = words.expand(self.sessions, -1)
        bias = bias or {-1: 0.0}
        bias_ids = torch.tensor([list(bias)], **self.i32).repeat(self.sessions, 1)
        bias_values = torch.tensor([list(bias.values())], device="cuda").float().repeat(self.sessions, 1)
        rows = torch.arange(self.sessions, device="cuda")
        plain = sampling.params(temperature, top_k, top_p)
        for i in range(steps):
            ruled = sampling.process_logits(logits.bfloat16(), history, used, prompt_len, repetition, frequency, presence,
                                            bias_ids, bias_values, allow)
            u = sampling.uniforms(self.sessions, vocab, seed + i, "cuda") if temperature > 0 else None
            ids = sampling.sample_logits(ruled, plain, u)
            history[rows, used.long()] = ids
            used = used + 1
            if i + 1 < steps:
                logits = self.step(ids)
        paged.check_status()
        return torch.stack([history[b, p:p + steps] for b, p in enumerate(prompt_len.tolist())])


def main(argv=None) -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--sessions", type=int, default=8)
    ap.add_argument("--steps", type=int, default=200)
    ap.add_argument("--budget", type=int, default=192)
    ap.add_argument("--kv", choices=KV_FORMATS, default="k8v4")
    ap.add_argument("--temperature", type=float, default=0.8)
    ap.add_argument("--seed", type=int, default=0)
    args = ap.parse_args(argv)
    model = Decoder(seed=args.seed)
    g = torch.Generator().manual_seed(args.seed)
    prompts = [torch.randint(0, 1000, (40 + 37 * b,), generator=g).tolist() for b in range(args.sessions)]
    batch = PagedBatch(model, args.sessions, args.budget, kv=args.kv)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    ids = batch.generate(prompts, args.steps, temperature=args.temperature, seed=args.seed)
    end.record()
    end.synchronize()
    for b, row in enumerate(ids.tolist()):
        print(f"session {b}: prompt {len(prompts[b])}, cache {int(batch.lengths[b])} of "
              f"{int(batch.positions[b])} tokens, ids {row[:8]} ...")
    print(f"{args.sessions * args.steps} tokens in {start.elapsed_time(end):.1f} ms")


if __name__ == "__main__":
    main()
