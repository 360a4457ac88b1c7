"""Plain references of the paged 4-bit operators: Python loops for the plan,
the byte layout word by word, attention and log probabilities in 64 bits."""

import math

import numpy as np
import torch


def plan(seq_lens, q_lens, table, free, n_free, page, n_tokens):
    """(cu_q, positions, requests, slots, lens, n_free, status, table) as lists / arrays."""
    table = table.copy()
    pages = lambda x: -(-x // page)  # noqa: E731
    q_lens = [max(0, q) for q in q_lens]
    need = [pages(s + q) - pages(s) for s, q in zip(seq_lens, q_lens)]
    status = (1 if sum(need) > n_free else 0) | (2 if any(pages(s + q) > table.shape[1] for s, q in zip(seq_lens, q_lens)) else 0)
    status |= 4 if sum(q_lens) > n_tokens else 0
    pos, req, slot = [0] * n_tokens, [-1] * n_tokens, [-1] * n_tokens
    if status:
        return [0] * (len(q_lens) + 1), pos, req, slot, list(seq_lens), n_free, status, table
    cu, t = [0], 0
    for b, (s, q) in enumerate(zip(seq_lens, q_lens)):
        for i in range(need[b]):
            n_free -= 1
            table[b, pages(s) + i] = free[n_free]
        for p in range(s, s + q):
            pos[t], req[t], slot[t] = p, b, int(table[b, p // page]) * page + p % page
            t += 1
        cu.append(t)
    return cu, pos, req, slot, [s + q for s, q in zip(seq_lens, q_lens)], n_free, 0, table


def stored(x: torch.Tensor) -> torch.Tensor:
    """What the pages stand for after rows x (..., D) were written: the formula's
    fp32 differences and quotients, then code * s + z in 64 bits."""
    g = x.double().reshape(*x.shape[:-1], -1, 32)
    nan = g.isnan().any(-1, keepdim=True)
    g = g.clamp(-32768.0, 32768.0)
    z = g.amin(-1, keepdim=True)
    fifteen = torch.full_like(z, 15.0).float()  # a tensor: torch multiplies by the inverse of a number
    s = ((g.amax(-1, keepdim=True).float() - z.float()) / fifteen).half().double()
    z = z.float().half().double()
    c = torch.where(s > 0, ((g.float() - z.float()) / torch.where(s > 0, s, 1.0).float()).round().clamp(0, 15).double(), 0.0)
    return torch.where(nan, math.nan, c * s + z).flatten(-2)


def read_block(blk: np.ndarray, d: int):
    """(keys, values) (16, D) float32 of one block's 20 D bytes, by the layout's definition."""
    g_n, w_n = d // 32, d // 64
    n = min(g_n, 4)
    k, v = np.zeros((16, d), np.float32), np.zeros((16, d), np.float32)
    half = lambda at: np.float32(blk[at:at + 2].view(np.float16)[0])  # noqa: E731
    for t in range(16):
        hi, j2, lo = t // 8, t % 8 // 2, t % 2
        for dim in range(d):
            g, j, nb = dim // 32, dim % 32 // 8, dim % 8
            at = ((g // n * 16 + t) * 4 + j) * n * 4 + g % n * 4 + nb // 2
            sz = 8 * d + (t * g_n + g) * 4
            k[t, dim] = np.float32((blk[at] >> (4 * (nb % 2))) & 15) * half(sz) + half(sz + 2)
            x = dim // 8
            q = (hi * 2 + lo) * w_n + x % w_n
            at = 10 * d + (q // 4) * 512 + (x // w_n * 4 + j2) * 16 + q % 4 * 4 + nb // 2
            sz = 18 * d + (((g * 4 + j2) * 2 + hi) * 2 + lo) * 4
            v[t, dim] = np.float32((blk[at] >> (4 * (nb % 2))) & 15) * half(sz) + half(sz + 2)
    return k, v


def attention(q, k, v, len_, scale, causal=True, window=0):
    """One request: q (nq, hq, D), k and v (T, hkv, D) with T >= len_. Returns
    out and lse in 64 bits, sum p |v| and the bound sum scale |q| |k| of each row."""
    nq, hq, d = q.shape
    grp = hq // k.shape[1]
    k, v = (x[:len_].double().repeat_interleave(grp, 1) for x in (k, v))
    z = torch.einsum("qhd,thd->qht", q.double(), k) * scale
    pos = len_ - nq + torch.arange(nq, device=q.device)[:, None, None]
    t = torch.arange(len_, device=q.device)
    see = torch.ones_like(z, dtype=torch.bool)
    if causal:
        see &= t <= pos
    if window:
        see &= t > pos - window
    z = z.masked_fill(~see, -math.inf)
    some = see.any(-1, keepdim=True)
    p = torch.where(some, torch.softmax(z, -1), 0.0)
    mag = (torch.einsum("qhd,thd->qht", q.double().abs(), k.abs()) * abs(scale)).masked_fill(~see, 0).amax(-1) if len_ else z.sum(-1)
    return (torch.einsum("qht,thd->qhd", p, v), torch.logsumexp(z, -1) if len_ else z.sum(-1) - math.inf,
            torch.einsum("qht,thd->qhd", p, v.abs()), mag)


def logprobs(x, targets, top):
    """(logprobs, entropy, ids, top logprobs) in 64 bits; NaN, +inf and all -inf rows by their definition."""
    n, vocab = x.shape
    x = x.double()
    bad = ~(x < math.inf).all(-1)
    none = (x == -math.inf).all(-1)
    y = torch.log_softmax(x, -1)
    h = -torch.where(y > -math.inf, y.exp() * y, 0.0).sum(-1)
    y[none], h[none] = -math.inf, 0.0
    y[bad], h[bad] = math.nan, math.nan
    lp = y.gather(1, targets.clamp(0, vocab - 1)[:, None])[:, 0]
    lp = torch.where(targets < 0, 0.0, torch.where(targets >= vocab, math.nan, lp))
    ids = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]
    tl = y.gather(1, ids)
    ids = ids.int()
    ids[bad] = -1
    if top > vocab:
        ids = torch.nn.functional.pad(ids, (0, top - vocab), value=-1)
        tl = torch.nn.functional.pad(tl, (0, top - vocab), value=-math.inf)
        tl[bad] = math.nan
    return lp, h, ids, tl
