"""Serving ragged requests over paged 4-bit caches, with the model of harness.py.

The reference runs one batch of equally long sequences per cache
(cache.py:59-336); a server has requests of any length that come and go. A
step here is

  plan      PageTables.plan: pages, slots and positions of the step's tokens
  layers    Int4PagedKVCache.append, then .attend, for every layer
  logits    of the rows that are needed
  logprobs  token_logprobs: of given tokens, with entropy and alternatives

all on the GPU: ``forward_paged`` takes prompts, parts of prompts and single
tokens in one step, whatever ``plan`` placed. ``PagedServer`` generates and
scores: new prompts in parts, all of them together, then one token a step for
every running request;

    python -m sunshape_mlx_b200.serving

serves a few random prompts on a small random model.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

from .harness import Decoder, DecoderConfig
from .logprobs import TokenLogprobs, token_logprobs
from .paged import Int4PagedKVCache, PageTables, StepPlan

__all__ = ["make_paged_caches", "forward_paged", "PagedServer"]


def make_paged_caches(model: Decoder, tables: PageTables) -> list[Int4PagedKVCache]:
    """One 4-bit paged cache per layer, all placed by ``tables``."""
    return [Int4PagedKVCache(tables, model.cfg.n_kv_heads, model.cfg.head_dim) for _ in model.layers]


def _rope(model: Decoder, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
    """Decoder._rope for tokens x (n, heads, d) at positions of their own."""
    ang = torch.outer(positions.float(), model._inv_freq)[:, None]
    cos, sin = ang.cos(), ang.sin()
    h = x.shape[-1] // 2
    a, b = x[..., :h].float(), x[..., h:].float()
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


@torch.no_grad()
def forward_paged(model: Decoder, ids: torch.Tensor, plan: StepPlan, caches: list[Int4PagedKVCache], *,
                  max_q: int, rows: torch.Tensor | None = None) -> torch.Tensor:
    """Logits (n or rows, vocab) in the model's dtype of the step's tokens ids
    (n,), which ``plan`` placed. Every layer stores their keys and values and
    attends over all that the requests hold. ``rows`` selects the tokens whose
    logits are needed."""
    cfg = model.cfg
    n, H, Hk, d = ids.shape[0], cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    h = model.embed[ids]
    for layer, cache in zip(model.layers, caches):
        qkv = (model._rms(h, layer["n1"]) @ layer["wqkv"]).view(n, H + 2 * Hk, d)
        q = _rope(model, qkv[:, :H], plan.positions)
        k = _rope(model, qkv[:, H:H + Hk], plan.positions)
        cache.append(k, qkv[:, H + Hk:], plan)
        o = cache.attend(q, plan, 1.0 / math.sqrt(d), max_q=max_q)
        h = h + o.view(n, H * d) @ layer["wo"]
        h = h + model._mlp(h, layer)
    if rows is not None:
        h = h[rows]
    return model._rms(h, model.norm) @ model.lm_head


class PagedServer:
    """A server's loop over at most ``max_requests`` requests at a time.

    ``start`` takes prompts into free rows and runs them (in parts of at most
    ``chunk`` tokens each, together; requests that run already wait until the
    last part is in), ``step`` generates one token for every running request,
    ``stop`` frees the pages of requests. The host keeps what a scheduler knows
    anyway (lengths, free rows and pages); ``start`` waits for the GPU when it
    copies its prompts, no other call does.
    """

    def __init__(self, model: Decoder, *, n_pages: int, page_size: int = 64, max_requests: int = 16,
                 max_tokens: int = 4096, chunk: int = 512, top_k: int = 0):
        self.model, self.chunk, self.top_k = model, chunk, top_k
        self.tables = PageTables(n_pages, page_size, max_requests, -(-max_tokens // page_size), model.device)
        self.caches = make_paged_caches(model, self.tables)
        self.max_tokens = max_tokens
        self.lens: dict[int, int] = {}                      # running requests: tokens held
        self.next_ids = torch.zeros(max_requests, dtype=torch.int64, device=model.device)

    def _pages(self, tokens: int) -> int:
        return -(-tokens // self.tables.page_size)

    def _run(self, new: dict[int, int], ids: torch.Tensor, rows: torch.Tensor | None):
        """One step of `new` tokens per request, in the order of the request rows. One that
        raises leaves lengths and pages as they were."""
        for r, q in new.items():
            if self.lens[r] + q > self.max_tokens:
                raise ValueError(f"request {r} would hold more than {self.max_tokens} tokens")
        if sum(self._pages(n + new.get(r, 0)) for r, n in self.lens.items()) > self.tables.n_pages:
            raise RuntimeError("the page pool has too few free pages")
        q = torch.zeros(self.tables.block_table.shape[0], dtype=torch.int32)
        for r, c in new.items():
            q[r] = c
        t = self.tables
        before = t.seq_lens, t.n_free
        try:
            plan = t.plan(q.to(self.model.device, non_blocking=True), ids.shape[0])
            logits = forward_paged(self.model, ids, plan, self.caches, max_q=max(new.values()), rows=rows)
        except BaseException:
            t.seq_lens, t.n_free = before  # a plan changes nothing else but table entries past these lengths
            raise
        for r, c in new.items():
            self.lens[r] += c
        return logits

    def start(self, prompts: list[torch.Tensor]) -> tuple[list[int], list[TokenLogprobs]]:
        """Takes prompts (1-D tensors of at least one id of the vocabulary) in
        and runs them. Returns their request numbers and, per prompt, the log
        probabilities of its tokens after the first (entropy and alternatives
        are those of the position before each)."""
        dev = self.model.device
        free = [r for r in range(self.tables.block_table.shape[0]) if r not in self.lens]
        if len(prompts) > len(free):
            raise RuntimeError(f"{len(prompts)} prompts for {len(free)} free rows")
        if any(p.dim() != 1 or not p.numel() for p in prompts):
            raise ValueError("prompts must be 1-D and hold a token at least")
        vocab = self.model.cfg.vocab
        if any(int(p.min()) < 0 or int(p.max()) >= vocab for p in prompts):  # no kernel looks at them before the embedding
            raise ValueError(f"prompts must hold ids from 0 to {vocab - 1}")
        reqs = free[: len(prompts)]
        prompts = [p.to(dev, torch.int64) for p in prompts]
        for r in reqs:
            self.lens[r] = 0
        done, parts = [0] * len(prompts), [[] for _ in prompts]
        try:
            while any(d < p.numel() for d, p in zip(done, prompts)):
                take = [min(self.chunk, p.numel() - d) for d, p in zip(done, prompts)]
                ids = torch.cat([p[d:d + c] for p, d, c in zip(prompts, done, take)])
                # the token after each one; none (-1) after a prompt's last
                nxt = torch.cat([F.pad(p, (0, 1), value=-1)[d + 1:d + 1 + c] for p, d, c in zip(prompts, done, take)])
                logits = self._run({r: c for r, c in zip(reqs, take) if c}, ids, None)
                lp = token_logprobs(logits, nxt, top_k=self.top_k)
                at = 0
                for i, c in enumerate(take):
                    if c:
                        parts[i].append(TokenLogprobs(*(t[at:at + c] for t in lp)))
                        at += c
                        done[i] += c
                        if done[i] == prompts[i].numel():
                            self.next_ids[reqs[i]] = logits[at - 1].argmax()
        except Exception:
            self.stop(reqs)
            raise
        return reqs, [TokenLogprobs(*(torch.cat(t)[:-1] for t in zip(*p))) for p in parts]

    def step(self) -> tuple[torch.Tensor, TokenLogprobs]:
        """Feeds every running request its next token. Returns the ids that
        were fed (in the order of the request numbers) and what
        ``token_logprobs`` says of the greedy token after each. Raises, with
        nothing changed, while a request holds ``max_tokens`` or the pool has
        too few pages for all: ``stop`` one first."""
        reqs = sorted(self.lens)
        if not reqs:
            raise RuntimeError("no request is running")
        at = torch.tensor(reqs).to(self.model.device, non_blocking=True)
        ids = self.next_ids[at]
        logits = self._run({r: 1 for r in reqs}, ids, None)
        best = logits.argmax(-1)
        self.next_ids[at] = best
        return ids, token_logprobs(logits, best, top_k=self.top_k)

    def stop(self, reqs: list[int]) -> None:
        """Ends requests: their pages are free again."""
        done = torch.zeros(self.tables.block_table.shape[0], dtype=torch.bool)
        for r in reqs:
            if self.lens.pop(r, None) is not None:
                done[r] = True
        self.tables.release(done.to(self.model.device, non_blocking=True))


def main() -> None:
    g = torch.Generator().manual_seed(0)
    model = Decoder(DecoderConfig(n_layers=4, hidden=1024, n_heads=8, n_kv_heads=2, ffn=2816, vocab=32000), seed=1)
    server = PagedServer(model, n_pages=256, max_requests=8, top_k=3)
    reqs, scored = server.start([torch.randint(32000, (n,), generator=g) for n in (700, 1, 65, 1200)])
    for r, s in zip(reqs, scored):
        mean = float(s.logprobs.mean()) if s.logprobs.numel() else float("nan")
        print(f"request {r}: {server.lens[r]} tokens, mean log probability {mean:.3f}")
    for _ in range(8):
        ids, lp = server.step()
    print("last ids", ids.tolist(), "log probabilities", [round(x, 3) for x in lp.logprobs.tolist()])
    server.stop(reqs[:2])
    server.tables.check()
    print(f"{int(server.tables.n_free)} of {server.tables.n_pages} pages free, caches of "
          f"{sum(c.nbytes for c in server.caches) / 1e6:.1f} MB")


if __name__ == "__main__":
    main()
