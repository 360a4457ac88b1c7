"""Operators of a serving step over a paged KV cache held in 4 bits, as measured cases.

plan       block tables and slot maps of ragged requests, from their lengths
write      new keys and values quantised into the pages by slot, then read back as stored
attention  attention over the pages: single tokens, several, long prompts; ragged requests
logprobs   log probabilities of given tokens, entropy and the most probable alternatives

Format of the pages: groups of 32 dims of one token and head share an fp16 scale s and an fp16
zero z, value = code * s + z with a 4-bit code. A page of one head is a sequence of blocks of 16
tokens, each 20 * head_dim bytes: key codes, key (s, z) pairs, value codes, value (s, z) pairs,
in the byte order that `_pack` writes.

Where `own` is false, `run` computes everything with elementary torch operations in 32 bits.
"""

import math
import random

import torch

own = False

GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one decode step of a small server: 64 requests, a token each
        dict(name="plan_decode", op="plan", n=64, ctx_lo=1, ctx_hi=8192, q_lo=1, q_hi=1, page=64, salt=1),
        # a large scheduler step: prompts and decodes mixed, some requests idle
        dict(name="plan_mixed", op="plan", n=1500, ctx_lo=0, ctx_hi=4096, q_lo=0, q_hi=80, page=16, salt=2),
        # the new tokens of a decode step, 32 requests
        dict(name="write_decode", op="write", n=32, hkv=8, d=128, page=64, dtype="bf16", skip=0, salt=3),
        # the tokens of many prompts at once, an odd number, some of them padding
        dict(name="write_prompt", op="write", n=49999, hkv=8, d=128, page=64, dtype="fp16", skip=7, salt=4),
        # the smallest decode: one request with a short context, where latency counts
        dict(name="decode_one", op="attention", n=1, ctx_lo=776, ctx_hi=776, q_lo=1, q_hi=1, hq=32, hkv=8, d=128,
             page=64, dtype="fp16", causal=True, window=0, salt=5),
        # an ordinary decode batch with ragged contexts
        dict(name="decode_batch", op="attention", n=32, ctx_lo=500, ctx_hi=16384, q_lo=1, q_hi=1, hq=32, hkv=8, d=128,
             page=64, dtype="bf16", causal=True, window=0, salt=6),
        # one very long context, eight query heads to a key head
        dict(name="decode_long", op="attention", n=1, ctx_lo=524287, ctx_hi=524287, q_lo=1, q_hi=1, hq=64, hkv=8, d=128,
             page=128, dtype="fp16", causal=True, window=0, salt=7),
        # prompt chunks and decoding requests in one step, smaller heads, a sliding window
        dict(name="mixed_window", op="attention", n=12, ctx_lo=0, ctx_hi=2500, q_lo=1, q_hi=900, hq=21, hkv=3, d=64,
             page=16, dtype="fp16", causal=True, window=1000, salt=8),
        # one long prompt, causal
        dict(name="prompt_long", op="attention", n=1, ctx_lo=0, ctx_hi=0, q_lo=8192, q_hi=8192, hq=32, hkv=8, d=128,
             page=64, dtype="bf16", causal=True, window=0, salt=9),
        # the logits of one token
        dict(name="logprobs_one", op="logprobs", n=1, vocab=128256, top=20, dtype="bf16"),
        # an odd vocabulary in 32 bits, as small models and reference runs have it
        dict(name="logprobs_fp32", op="logprobs", n=333, vocab=50257, top=5, dtype="fp32"),
        # scoring the tokens of a prompt
        dict(name="logprobs_prompt", op="logprobs", n=2047, vocab=128256, top=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "write", "decode", "decode", "prompt", "prompt", "logprobs", "logprobs"])
    salt = rng.randrange(1 << 20)
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        n, q = _log(rng, 1, 1500), _log(rng, 1, 400)
        q = max(1, min(q, 120000 // n))
        return dict(op="plan", n=n, ctx_lo=rng.choice([0, 1]), ctx_hi=_log(rng, 1, 8192), q_lo=rng.choice([0, 1]), q_hi=q, page=page, salt=salt)
    dtype = rng.choice(["bf16", "fp16"])
    d = rng.choice([64, 128, 128, 256])
    if op == "write":
        hkv = rng.choice([1, 2, 3, 4, 8, 16])
        n = min(_log(rng, 1, 50000), 50000 * 8 * 128 // (hkv * d))
        return dict(op="write", n=n, hkv=hkv, d=d, page=page, dtype=rng.choice(["bf16", "fp16", "fp32"]), skip=rng.choice([0, 0, 3, 50]), salt=salt)
    if op == "logprobs":
        n, vocab = _log(rng, 1, 2047), _log(rng, 1000, 131072)
        return dict(op="logprobs", n=n, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 32]), dtype=rng.choice(["bf16", "fp16", "fp32"]))
    hkv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 4, 7, 8, 16])
    if op == "decode":
        n = _log(rng, 1, 128)
        most = max(64, 4_000_000 * 128 // (n * hkv * d))
        hi = _log(rng, 16, min(131072, most))
        return dict(op="attention", n=n, ctx_lo=rng.choice([0, hi // 4]), ctx_hi=hi, q_lo=1, q_hi=rng.choice([1, 1, 1, 2, 4]), hq=hkv * group, hkv=hkv, d=d,
                    page=page, dtype=dtype, causal=True, window=rng.choice([0, 0, 0, _log(rng, 16, 4096)]), salt=salt)
    n = _log(rng, 1, 16)
    q = _log(rng, 17, 4096 // n)
    ctx = rng.choice([0, 0, _log(rng, 16, 4096)])
    hkv = min(hkv, max(1, 32 // group))
    return dict(op="attention", n=n, ctx_lo=0, ctx_hi=ctx, q_lo=rng.choice([1, q // 2]), q_hi=q, hq=hkv * group, hkv=hkv, d=d,
                page=page, dtype=dtype, causal=rng.choice([True, True, True, False]), window=0, salt=salt)


def _lens(c):
    """(tokens held before, new tokens) of each request: they belong to the case, not to the seed."""
    r = random.Random(c["salt"])
    old = [r.randint(c["ctx_lo"], c["ctx_hi"]) for _ in range(c["n"])]
    new = [r.randint(c["q_lo"], c["q_hi"]) for _ in range(c["n"])]
    if not sum(new):
        new[0] = 1
    return old, new


def _pages(tokens, page):
    return -(-tokens // page)


# ------------------------------------------------------------------ the page format, in elementary operations

def _quantise(x):
    """(codes, s, z) of x (..., D): codes as numbers (..., G, 32), s and z fp16 (..., G)."""
    x = x.float().unflatten(-1, (-1, GROUP)).clamp(-32768.0, 32768.0)
    lo, hi = x.amin(-1), x.amax(-1)
    s, z = ((hi - lo) / torch.full_like(lo, 15.0)).half(), lo.half()  # a quotient: by a number torch multiplies by its inverse
    sf, zf = s.float().unsqueeze(-1), z.float().unsqueeze(-1)
    c = torch.where(sf > 0, ((x - zf) / sf).round().clamp(0.0, 15.0), torch.zeros_like(x))
    return c, s, z


def _pack(kc, ks, kz, vc, vs, vz):
    """Pages (P, H, bytes) of codes (P, H, page, G, 32) and scales (P, H, page, G)."""
    p, h, page, g, _ = kc.shape
    d, nb = g * GROUP, page // 16
    w = d // 64
    n = min(g, 4)
    nib = lambda c: c.to(torch.uint8).unflatten(-1, (-1, 4, 2))  # noqa: E731  words, bytes, nibbles
    by = lambda c: (c[..., 0] | (c[..., 1] << 4))                # noqa: E731
    k = by(nib(kc))                                              # (P, H, page, G, 4 j, 4 B)
    k = k.reshape(p, h, nb, 16, g // n, n, 4, 4).permute(0, 1, 2, 4, 3, 6, 5, 7).reshape(p, h, nb, 8 * d)
    sz = lambda s, z: torch.stack([s, z], -1).view(torch.uint8)  # noqa: E731  (..., G, 4 B)
    ksz = sz(ks, kz).reshape(p, h, nb, 2 * d)
    v = by(nib(vc)).reshape(p, h, nb, 2, 4, 2, 8, w, 4)          # hi, j, lo, i, word, byte
    v = v.permute(0, 1, 2, 6, 4, 3, 5, 7, 8).reshape(p, h, nb, 32, w, 16).transpose(3, 4).reshape(p, h, nb, 8 * d)
    vsz = sz(vs, vz).reshape(p, h, nb, 2, 4, 2, g, 4).permute(0, 1, 2, 6, 4, 3, 5, 7).reshape(p, h, nb, 2 * d)
    return torch.cat([k, ksz, v, vsz], -1).reshape(p, h, nb * 20 * d).contiguous()


def _values(codes, sz):
    """code * s + z in 32 bits: codes (..., G, 32), sz bytes (..., G, 4)."""
    sz = sz.contiguous().view(torch.float16).float()
    return (codes.float() * sz[..., :1] + sz[..., 1:]).flatten(-2)


def _unpack(pages, d):
    """Keys and values (..., page, D) in 32 bits of pages (..., bytes)."""
    lead, g, w = pages.shape[:-1], d // GROUP, d // 64
    n = min(g, 4)
    b = pages.reshape(*lead, -1, 20 * d)
    nb = b.shape[-2]
    f = math.prod(lead) * nb
    b = b.reshape(f, 20 * d)
    nib = lambda x: torch.stack([x & 15, x >> 4], -1).flatten(-2)  # noqa: E731
    k = b[:, : 8 * d].reshape(f, g // n, 16, 4, n, 4).permute(0, 2, 1, 4, 3, 5)
    k = _values(nib(k).reshape(f, 16, g, GROUP), b[:, 8 * d: 10 * d].reshape(f, 16, g, 4))
    v = b[:, 10 * d: 18 * d].reshape(f, w, 32, 16).transpose(1, 2).reshape(f, 8, 4, 2, 2, w, 4).permute(0, 3, 2, 4, 1, 5, 6)
    vsz = b[:, 18 * d:].reshape(f, g, 4, 2, 2, 4).permute(0, 3, 2, 4, 1, 5).reshape(f, 16, g, 4)
    v = _values(nib(v).reshape(f, 16, g, GROUP), vsz)
    return k.reshape(*lead, nb * 16, d), v.reshape(*lead, nb * 16, d)


# ------------------------------------------------------------------ inputs

def _kv(gen, shape, dtype):
    """Keys with a few strong channels, as rotary keys have them, and plain values."""
    k = torch.randn(shape, generator=gen, device="cuda")
    k[..., 3::16] *= 3.0
    k[..., 5::32] += 2.0
    v = torch.randn(shape, generator=gen, device="cuda") * 0.7
    return k.to(dtype), v.to(dtype)


def _pool(gen, pages, hkv, page, d, valid):
    """A pool of pages; places that hold no token yet (from `valid` of a page on) hold stale bits: NaN scales."""
    out = torch.empty((pages, hkv, page * 20 * d // 16), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (hkv * page * d))
    for a in range(0, pages, step):
        b = min(pages, a + step)
        k, v = _kv(gen, (b - a, hkv, page, d), torch.float32)
        kq, vq = _quantise(k), _quantise(v)
        stale = torch.arange(page, device="cuda")[None, None, :, None] >= valid[a:b, None, None, None]
        for q in (kq, vq):
            q[1].masked_fill_(stale, float("nan"))
            q[2].masked_fill_(stale, float("nan"))
        out[a:b] = _pack(*kq, *vq)
    return out


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    if c["op"] == "logprobs":
        n, vocab = c["n"], c["vocab"]
        x = torch.randn((n, vocab), generator=gen, device="cuda") * 2.0
        # a few tokens stand out, and a few are banned
        x.scatter_add_(1, torch.randint(vocab, (n, 24), generator=gen, device="cuda"), torch.rand((n, 24), generator=gen, device="cuda") * 14)
        x[:, torch.randint(vocab, (5,), generator=gen, device="cuda")] = float("-inf")
        targets = torch.randint(vocab, (n,), generator=gen, device="cuda")
        targets[5::50] = -1
        return dict(c=c, logits=x.to(DTYPES[c["dtype"]]), targets=targets)
    page = c["page"]
    if c["op"] == "write":
        n, hkv, d = c["n"], c["hkv"], c["d"]
        pages = _pages(n, page) + 3
        k, v = _kv(gen, (n, hkv, d), DTYPES[c["dtype"]])
        order = torch.randperm(pages, generator=gen, device="cuda")
        t = torch.arange(n, device="cuda")
        slots = order[t // page] * page + t % page
        if c["skip"]:
            slots[c["skip"] // 2::c["skip"]] = -1
        return dict(c=c, k=k, v=v, slots=slots, pages=torch.full((pages, hkv, page * 20 * d // 16), 255, dtype=torch.uint8, device="cuda"))
    old, new = _lens(c)
    if c["op"] == "plan":
        held = [_pages(o, page) for o in old]
        need = [_pages(o + q, page) for o, q in zip(old, new)]
        width = max(need) + 1
        total = sum(need) + 11
        order = torch.randperm(total, generator=gen, device="cuda").int()
        first = torch.tensor([0] + held, device="cuda").cumsum(0)[:-1]
        j = torch.arange(width, device="cuda")
        has = _ints(held)
        table = torch.where(j[None] < has[:, None], order[(first[:, None] + j[None]).clamp(max=total - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
        free = torch.zeros(total, dtype=torch.int32, device="cuda")
        left = total - sum(held)
        free[:left] = order[sum(held):]
        return dict(c=c, seq_lens=_ints(old), q_lens=_ints(new), table=table, free=free, n_free=_ints([left]), n_tokens=sum(new) + 5)
    lens = [o + q for o, q in zip(old, new)]
    need = [_pages(x, page) for x in lens]
    total, width = sum(need) + 2, max(need) + 1
    order = torch.randperm(total, generator=gen, device="cuda").int()
    first = torch.tensor([0] + need, device="cuda").cumsum(0)[:-1]
    j = torch.arange(width, device="cuda")
    table = torch.where(j[None] < _ints(need)[:, None], order[(first[:, None] + j[None]).clamp(max=total - 1)], torch.full((), -1, dtype=torch.int32, device="cuda"))
    valid = torch.zeros(total, dtype=torch.int64, device="cuda")
    left = (_ints(lens)[:, None] - j[None] * page).clamp(0, page)
    valid[table[table >= 0].long()] = left[table >= 0].long()
    pages = _pool(gen, total, c["hkv"], page, c["d"], valid)
    q = torch.randn((sum(new), c["hq"], c["d"]), generator=gen, device="cuda").to(DTYPES[c["dtype"]])
    return dict(c=c, q=q, pages=pages, table=table, seq_lens=_ints(lens), cu_q=_ints([0] + new).cumsum(0).int(), max_q=max(new), max_len=max(lens),
                scale=1.0 / math.sqrt(c["d"]))


# ------------------------------------------------------------------ one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    import sunshape_mlx_b200 as ss

    op = s["c"]["op"]
    if op == "plan":
        p = ss.plan_step(s["seq_lens"], s["q_lens"], s["table"], s["free"], s["n_free"], page_size=s["c"]["page"], n_tokens=s["n_tokens"])
        return dict(cu_q=p.cu_q, positions=p.positions, requests=p.requests, slots=p.slots, seq_lens=p.seq_lens, n_free=p.n_free, table=s["table"])
    if op == "write":
        ss.int4_append(s["k"], s["v"], s["slots"], s["pages"])
        k, v = ss.int4_fetch(s["slots"], s["pages"], s["c"]["d"], dtype=s["k"].dtype)
        return dict(k=k, v=v)
    if op == "attention":
        c = s["c"]
        o, lse = ss.int4_attention(s["q"], s["pages"], s["table"], s["seq_lens"], s["cu_q"], s["scale"], max_q=s["max_q"], causal=c["causal"], window=c["window"], return_lse=True)
        return dict(out=o, lse=lse)
    r = ss.token_logprobs(s["logits"], s["targets"], top_k=s["c"]["top"])
    return dict(logprobs=r.logprobs, entropy=r.entropy, top_ids=r.top_ids, top_logprobs=r.top_logprobs)


def _run_plain(s):
    return {"plan": _plain_plan, "write": _plain_write, "attention": _plain_attention, "logprobs": _plain_logprobs}[s["c"]["op"]](s)


def _plain_plan(s):
    page, table, n_free = s["c"]["page"], s["table"], s["n_free"]
    new = s["q_lens"].clamp(min=0)
    lens = s["seq_lens"] + new
    held, want = (s["seq_lens"] + page - 1) // page, (lens + page - 1) // page
    need = want - held
    off = need.cumsum(0) - need
    cu = torch.cat([torch.zeros_like(n_free), new.cumsum(0)]).int()
    j = torch.arange(table.shape[1], device="cuda")[None]
    fresh = (j >= held[:, None]) & (j < want[:, None])
    at = (n_free - 1 - off)[:, None] - (j - held[:, None])
    table.copy_(torch.where(fresh, s["free"][at.clamp(0, s["free"].shape[0] - 1)], table))
    t = torch.arange(s["n_tokens"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(cu, t, right=True) - 1
    live = t < cu[-1]
    b = b.clamp(max=new.shape[0] - 1)
    pos = torch.where(live, s["seq_lens"][b] + t - cu[b], 0)
    slots = table[b, (pos // page).long()].long() * page + pos % page
    return dict(cu_q=cu, positions=pos, requests=torch.where(live, b, -1).int(), slots=torch.where(live, slots, -1), seq_lens=lens.int(), n_free=(n_free - need.sum()).int(), table=table)


def _plain_write(s):
    pages, slots, d = s["pages"], s["slots"], s["c"]["d"]
    n_pages, hkv, page = pages.shape[0], pages.shape[1], s["c"]["page"]
    live = slots >= 0
    # the tokens in the order of the pool's places, the pool's own bits where no token goes
    place = torch.full((n_pages * page + 1,), -1, dtype=torch.long, device="cuda")
    place[torch.where(live, slots, n_pages * page)] = torch.arange(slots.shape[0], device="cuda")
    place = place[:-1].reshape(n_pages, page)
    fill = lambda x: x[place.clamp(min=0)].transpose(1, 2)  # noqa: E731  (P, H, page, ...)
    kq, vq = _quantise(s["k"]), _quantise(s["v"])
    packed = _pack(*[fill(x) for x in kq], *[fill(x) for x in vq])
    one = torch.full((n_pages, 1, page, d // GROUP, GROUP), 15.0, device="cuda") * (place >= 0)[:, None, :, None, None]
    bits = one[..., 0].to(torch.int16).clamp(max=1).neg().view(torch.float16)  # all ones where a token goes
    mask = _pack(one, bits, bits, one, bits, bits)
    pages.copy_((packed & mask) | (pages & ~mask))
    k, v = _unpack(pages, d)
    at = slots.clamp(min=0)
    take = lambda x: torch.where(live[:, None, None], x.transpose(1, 2).reshape(-1, hkv, d)[at], 0.0).to(s["k"].dtype)  # noqa: E731
    return dict(k=take(k), v=take(v))


def _plain_attention(s):
    c, q, cu, lens = s["c"], s["q"], s["cu_q"], s["seq_lens"]
    page, hkv, d = c["page"], c["hkv"], c["d"]
    n, hq, grp = c["n"], c["hq"], c["hq"] // c["hkv"]
    used = _pages(s["max_len"], page)
    k, v = _unpack(s["pages"][s["table"][:, :used].clamp(min=0).long()], d)   # (B, P, H, page, D)
    k, v = (x.transpose(1, 2).reshape(n, hkv, used * page, d) for x in (k, v))
    kpos = torch.arange(used * page, device="cuda")
    there = kpos[None] < lens[:, None]
    k, v = (torch.where(there[:, None, :, None], x, 0.0) for x in (k, v))
    nq = cu[1:] - cu[:-1]
    i = torch.arange(s["max_q"], device="cuda")
    rows = (cu[:-1, None] + i[None]).clamp(max=q.shape[0] - 1).long()
    x = q[rows].float().reshape(n, s["max_q"], hkv, grp, d).permute(0, 2, 3, 1, 4).reshape(n, hkv, grp * s["max_q"], d)
    z = (x @ k.transpose(-1, -2)) * s["scale"]
    qpos = (lens - nq)[:, None] + i[None]
    see = there[:, None, :].expand(n, s["max_q"], -1)
    if c["causal"]:
        see = see & (kpos[None, None] <= qpos[:, :, None])
    if c["window"]:
        see = see & (kpos[None, None] > qpos[:, :, None] - c["window"])
    see = see[:, None, None]
    z = z.reshape(n, hkv, grp, s["max_q"], -1).masked_fill_(~see, float("-inf"))
    m = z.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = (z - m).exp_()
    del z
    tot = p.sum(-1, keepdim=True)
    o = (p.reshape(n, hkv, -1, used * page) @ v).reshape(n, hkv, grp, s["max_q"], d) / tot.clamp(min=1e-38)
    lse = torch.where(tot > 0, m + tot.log(), float("-inf"))[..., 0]
    t = torch.arange(q.shape[0], device="cuda", dtype=torch.int32)
    b = (torch.searchsorted(cu, t, right=True) - 1).long()
    r = (t - cu[b]).long()
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], hq, d)[b, r]
    return dict(out=o.to(q.dtype), lse=lse.permute(0, 3, 1, 2).reshape(n, s["max_q"], hq)[b, r])


def _plain_logprobs(s):
    x, t, k = s["logits"].float(), s["targets"], s["c"]["top"]
    m = x.amax(-1, keepdim=True)
    y = x - m
    e = y.exp()
    tot = e.sum(-1, keepdim=True)
    lse = m + tot.log()
    h = tot.log() - (e * y.clamp(min=torch.finfo(torch.float32).min)).sum(-1, keepdim=True) / tot
    lp = torch.where(t >= 0, (x.gather(1, t.clamp(min=0)[:, None]) - lse)[:, 0], 0.0)
    if not k:
        none = x.new_zeros((x.shape[0], 0))
        return dict(logprobs=lp, entropy=h[:, 0], top_ids=none.int(), top_logprobs=none)
    top, ids = x.sort(stable=True, dim=-1, descending=True)  # ties in the order of the indices
    return dict(logprobs=lp, entropy=h[:, 0], top_ids=ids[:, :k].int(), top_logprobs=top[:, :k] - lse)


# ------------------------------------------------------------------ work of a pass

def work(case):
    c = case
    if c["op"] == "logprobs":
        es = 4 if c["dtype"] == "fp32" else 2
        return dict(bytes=c["n"] * (c["vocab"] * es + 8 + 8 + 8 * c["top"]), flops=c["n"] * c["vocab"] * 6)
    if c["op"] == "write":
        es = 4 if c["dtype"] == "fp32" else 2
        live = c["n"] - (len(range(c["skip"] // 2, c["n"], c["skip"])) if c["skip"] else 0)
        e = 2 * c["hkv"] * c["d"]
        return dict(bytes=c["n"] * (8 + e * es) + live * e * (es + 2 * 0.625), flops=live * e * 8)
    old, new = _lens(c)
    if c["op"] == "plan":
        fresh = sum(_pages(o + q, c["page"]) - _pages(o, c["page"]) for o, q in zip(old, new))
        return dict(bytes=4 * 4 * c["n"] + 8 * fresh + 16 * (sum(new) + 5), flops=sum(new) * 4)
    pairs = keys = 0
    for o, q in zip(old, new):
        w = c["window"] or o + q
        keys += min(o + q, q + w - 1) if q else 0
        if not c["causal"]:
            pairs += q * (o + q)
        else:  # row i sees min(o + i + 1, w) keys
            full = max(0, min(q, w - o))
            pairs += full * o + full * (full + 1) // 2 + (q - full) * w
    es = 2
    return dict(bytes=keys * c["hkv"] * c["d"] * 1.25 + sum(new) * c["hq"] * (2 * c["d"] * es + 4), flops=4 * c["d"] * c["hq"] * pairs)


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_groups(x):
    """What a group of 32 stands for after it was stored: numpy-style, 64 bits."""
    x = x.double().reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    x = torch.minimum(torch.maximum(x, torch.full_like(x, -2.0 ** 15)), torch.full_like(x, 2.0 ** 15))
    z = x.min(-1, keepdim=True).values
    s = ((x.max(-1, keepdim=True).values - z) / 15).to(torch.float16).double()
    z = z.to(torch.float16).double()
    code = torch.round((x - z) / torch.where(s > 0, s, torch.ones_like(s)))
    code = torch.minimum(torch.maximum(code, torch.zeros_like(code)), torch.full_like(code, 15))
    return (torch.where(s > 0, code, torch.zeros_like(code)) * s + z).flatten(-2)


def _exact_block(blk, d):
    """Keys and values (16, D) of many blocks (M, 20 D bytes), a word at a time by the format's definition."""
    m, g, w, n = blk.shape[0], d // 32, d // 64, min(d // 32, 4)
    k = torch.empty((m, 16, d), dtype=torch.float64, device=blk.device)
    v = torch.empty_like(k)
    sz = blk.reshape(m, -1, 2).view(torch.float16)[..., 0].double()
    tok = torch.arange(16, device=blk.device)
    for dim in range(d):
        gr, j, nb = dim // 32, dim % 32 // 8, dim % 8
        byte = (((gr // n * 16 + tok) * 4 + j) * n + gr % n) * 4 + nb // 2
        code = (blk[:, byte].int() >> (4 * (nb % 2))) & 15
        half = 4 * d + (tok * g + gr) * 2
        k[:, :, dim] = code.double() * sz[:, half] + sz[:, half + 1]
        hi, j, lo = tok // 8, tok % 8 // 2, tok % 2
        i, wi = dim // 8 // w, dim // 8 % w
        q = (hi * 2 + lo) * w + wi
        byte = 10 * d + ((q // 4) * 32 + i * 4 + j) * 16 + (q % 4) * 4 + nb // 2
        code = (blk[:, byte].int() >> (4 * (nb % 2))) & 15
        half = 9 * d + (((gr * 4 + j) * 2 + hi) * 2 + lo) * 2
        v[:, :, dim] = code.double() * sz[:, half] + sz[:, half + 1]
    return k, v


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "plan":
        return None
    if c["op"] == "write":
        if c["n"] * c["hkv"] * c["d"] > 1 << 26:
            return None
        gone = (s["slots"] < 0)[:, None, None]
        return dict(k=_exact_groups(s["k"]).masked_fill(gone, 0), v=_exact_groups(s["v"]).masked_fill(gone, 0))
    if c["op"] == "logprobs":
        lp, ent, top = [], [], []
        for a in range(0, c["n"], 256):
            x, t = s["logits"][a:a + 256].double(), s["targets"][a:a + 256]
            y = torch.log_softmax(x, -1)
            p = y.exp()
            ent.append(-torch.where(p > 0, p * y, torch.zeros_like(y)).sum(-1))
            lp.append(torch.where(t < 0, torch.zeros_like(ent[-1]), y[torch.arange(y.shape[0], device=y.device), t.clamp(min=0)]))
            top.append(torch.topk(y, c["top"], -1).values)  # the values of a row's best are the same whichever of equals is taken
        return dict(logprobs=torch.cat(lp), entropy=torch.cat(ent), top_ids=None, top_logprobs=torch.cat(top))
    old, new = _lens(c)
    grp, d = c["hq"] // c["hkv"], c["d"]
    if work(c)["flops"] > 1.2e13 or sum(old) + sum(new) > 3_000_000:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for b, (o, nq) in enumerate(zip(old, new)):
        used = _pages(o + nq, c["page"])
        for h in range(c["hkv"]):
            raw = s["pages"][s["table"][b, :used].long(), h].reshape(-1, 20 * d)
            k, v = (x.reshape(-1, d)[: o + nq] for x in _exact_block(raw, d))
            for a in range(0, nq, 1024):
                e = min(nq, a + 1024)
                x = s["q"][row + a: row + e, h * grp: (h + 1) * grp].double()
                z = torch.einsum("qgd,td->qgt", x, k) * s["scale"]
                at = torch.arange(o + a, o + e, device="cuda")[:, None, None]
                t = torch.arange(o + nq, device="cuda")
                if c["causal"]:
                    z.masked_fill_(t > at, -math.inf)
                if c["window"]:
                    z.masked_fill_(t <= at - c["window"], -math.inf)
                lse[row + a: row + e, h * grp: (h + 1) * grp] = torch.logsumexp(z, -1)
                out[row + a: row + e, h * grp: (h + 1) * grp] = torch.einsum("qgt,td->qgd", torch.softmax(z, -1), v)
        row += nq
    return dict(out=out, lse=lse)
