"""The paged 4-bit operators on the GPU against plain references.

Tolerances, from the number formats: u = 2^-11 is the relative rounding of
fp16, u_out that of the output (2^-11 fp16, 2^-8 bf16). Keys, values and
probabilities may each be rounded to fp16 inside the kernel, so a logit is off
by at most dz = u * max_t scale sum |q_d k_td|, and an output element by
u_out |o| + (4 u + 2 dz) sum p |v|; over all elements the rounding errors are
independent and the 2-norm error stays below that of the output format, u_out.
Integers and stored codes are equal."""

import math

import numpy as np
import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ss(cuda_ok):
    import sunshape_mlx_b200 as ss

    return ss


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ plan

@pytest.mark.parametrize("n,page,qs,ctx", [(1, 16, [1], 0), (1, 16, [0], 5), (3, 16, [1, 0, 17], 40), (64, 64, [1], 3000),
                                           (513, 16, [0, 1, 5, 33], 100), (1500, 32, [0, 3, 64], 700), (5, 48, [100, 1, 0], 97),
                                           (2, 16, [5000], 31), (9000, 16, [0, 1], 40)])
def test_plan_step(ss, n, page, qs, ctx):
    rng = np.random.default_rng(n + page)
    lens = rng.integers(0, ctx + 1, n).tolist()
    new = [int(qs[i % len(qs)]) for i in range(n)]
    new[-1] = -3 if n > 2 else new[-1]  # negative: none
    held = [-(-s // page) for s in lens]
    width = max(-(-(s + max(0, q)) // page) for s, q in zip(lens, new)) + 2
    pool = sum(held) + sum(width for _ in range(1)) + sum(-(-max(0, q) // page) + 1 for q in new) + 3
    order = rng.permutation(pool).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    free = np.full(pool, -7, np.int32)
    free[:pool - at] = order[at:]
    n_tokens = sum(max(0, q) for q in new) + 4
    want = R.plan(lens, new, table, free, pool - at, page, n_tokens)
    wide = torch.full((n, width + 3), -9, dtype=torch.int32, device="cuda")  # rows of a wider table
    gt = wide[:, :width]
    gt.copy_(torch.from_numpy(table))
    args = _i32(lens), _i32(new), gt, torch.from_numpy(free).cuda(), _i32([pool - at])
    for _ in range(2):  # a repeated call repeats its result
        p = ss.plan_step(*args, page_size=page, n_tokens=n_tokens)
        for got, w in zip((p.cu_q, p.positions, p.requests, p.slots, p.seq_lens), want):
            assert got.tolist() == list(w)
        assert (p.n_free.item(), p.status.item()) == want[5:7]
        assert np.array_equal(gt.cpu().numpy(), want[7])
        assert (wide[:, width:] == -9).all()


@pytest.mark.parametrize("free,width,n_tokens,status", [(2, 9, 99, 1), (50, 3, 99, 2), (50, 9, 49, 4), (1, 2, 3, 7)])
def test_plan_that_does_not_fit_changes_nothing(ss, free, width, n_tokens, status):
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    table[0, 0] = 50
    lens = _i32([7, 0])
    p = ss.plan_step(lens, _i32([20, 60] if status != 4 else [10, 40]), table, torch.arange(51, dtype=torch.int32, device="cuda"),
                     _i32([free]), page_size=16, n_tokens=n_tokens)
    assert p.status.item() == status and p.n_free.item() == free
    assert p.seq_lens.tolist() == [7, 0] and p.cu_q.tolist() == [0, 0, 0]
    assert (p.slots == -1).all() and (p.requests == -1).all() and (p.positions == 0).all()
    assert table[0].tolist() == [50] + [-1] * (width - 1) and (table[1] == -1).all()


def test_tables_allocate_release_and_check(ss):
    t = ss.PageTables(n_pages=10, page_size=16, max_requests=3, max_pages=6, device="cuda")
    p = t.plan(_i32([33, 0, 16]), 49)
    assert t.block_table[0, :3].tolist() == [0, 1, 2] and t.block_table[2, 0].item() == 3
    assert t.n_free.item() == 6 and p.slots[48].item() == 3 * 16 + 15
    t.plan(_i32([1, 1, 1]), 3)
    assert t.seq_lens.tolist() == [34, 1, 17] and t.n_free.item() == 4
    t.check()
    t.release(torch.tensor([True, False, True], device="cuda"))
    assert t.seq_lens.tolist() == [0, 1, 0] and t.n_free.item() == 9
    assert (t.block_table[0] == -1).all() and (t.block_table[2] == -1).all()
    left = t.free_pages[:9].tolist() + t.block_table[1, :1].tolist()
    assert sorted(left) == list(range(10))
    t.plan(_i32([0, 200, 0]), 200)
    with pytest.raises(RuntimeError, match="table row"):
        t.check()
    t.check()  # reported once
    assert t.seq_lens.tolist() == [0, 1, 0]
    q = t.plan(_i32([70, 0, 3]), 73)  # and the server goes on
    assert t.status.item() == 0 and q.seq_lens.tolist() == [70, 1, 3]


# ------------------------------------------------------------------ write and read

def _slots(n, pages, page, seed, skip=()):
    s = torch.randperm(pages * page, generator=_gen(seed), device="cuda")[:n]
    for i in skip:
        s[i] = -1
    return s


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,h,d,page", [(1, 1, 64, 16), (1, 8, 128, 64), (37, 3, 64, 16), (130, 2, 128, 48), (19, 2, 256, 32)])
def test_append_then_read(ss, n, h, d, page, dtype):
    g = _gen(n + d)
    pages = -(-n // page) + 2
    pool = torch.full((pages, h, page * d * 5 // 4), 0xA5, dtype=torch.uint8, device="cuda")
    before = pool.clone()
    k = (torch.randn((n, h, d), generator=g, device="cuda") * 3 + 1).to(dtype)
    v = (torch.randn((n, h, d), generator=g, device="cuda") * 0.1).to(dtype)
    skip = (0,) if n > 2 else ()
    slots = _slots(n, pages, page, n, skip)
    ss.int4_append(k, v, slots, pool)
    kr, vr = ss.int4_fetch(slots, pool, d)
    live = slots >= 0
    assert torch.equal(kr[live], R.stored(k)[live].float()) and torch.equal(vr[live], R.stored(v)[live].float())
    assert (kr[~live] == 0).all() and (vr[~live] == 0).all()
    # the bytes are where the layout says, and nothing else was touched
    host, old = pool.cpu().numpy(), before.cpu().numpy()
    used = {int(s) for s in slots[live].tolist()}
    for s in list(used)[:3]:
        blk = host[s // page, h - 1].reshape(-1, 20 * d)[s % page // 16]
        rk, rv = R.read_block(blk, d)
        i = (slots == s).nonzero()[0, 0]
        assert np.array_equal(rk[s % 16], kr[i, h - 1].cpu().numpy()) and np.array_equal(rv[s % 16], vr[i, h - 1].cpu().numpy())
    assert (host != old).sum() <= len(used) * h * d * 5 // 4
    other = torch.tensor([s for s in range(pages * page) if s not in used], device="cuda")
    a, b = ss.int4_fetch(other, pool, d), ss.int4_fetch(other, before, d)
    for x, y in zip(a, b):
        assert torch.equal(x.nan_to_num(1e9), y.nan_to_num(1e9))
    h16 = ss.int4_fetch(slots, pool, d, dtype=torch.float16)
    assert torch.equal(h16[0], kr.half()) and torch.equal(h16[1], vr.half())


def test_append_strides_and_alignment(ss):
    g = _gen(3)
    big = torch.randn((9, 2, 5, 64 * 3 + 1), generator=g, device="cuda").half()
    k, v = big[:, 0, 1:4, 1:65], big[:, 1, :3, 67:131]  # unaligned views, strides of their own
    pool = ss.int4_pool(2, 3, 16, 64)
    slots = torch.arange(9, device="cuda") + 3
    ss.int4_append(k, v, slots, pool)
    kr, vr = ss.int4_fetch(slots, pool, 64)
    assert torch.equal(kr, R.stored(k).float()) and torch.equal(vr, R.stored(v).float())
    wide = torch.zeros((2, 5, 16 * 80 + 64), dtype=torch.uint8, device="cuda")
    view = wide[:, 1:4, : 16 * 80]  # pool strides of their own
    ss.int4_append(k, v, slots, view)
    assert torch.equal(view, torch.where(view != 0, pool, view))
    assert (wide[:, 0] == 0).all() and (wide[:, 4] == 0).all() and (wide[:, :, 16 * 80:] == 0).all()


def test_append_edge_values(ss):
    d = 64
    x = torch.zeros((8, 1, d), device="cuda")
    x[0] = 1.5                       # constant: scale 0
    x[1, 0, 3] = math.nan            # marks its group
    x[2, 0, 5] = math.inf
    x[2, 0, 6] = -math.inf
    x[3, 0, 40] = 3e38               # saturates
    x[4] = torch.linspace(-7.5, 7.5, 64, device="cuda")  # ties between codes
    x[5] = 1e-30                     # scale underflows to 0
    x[6, 0, ::2] = 65504.0
    x[7, 0, :32] = torch.arange(32, device="cuda") * 6e-8  # fp16 subnormal range
    pool = ss.int4_pool(1, 1, 16, d)
    slots = torch.arange(8, device="cuda")
    ss.int4_append(x, x, slots, pool)
    k, v = ss.int4_fetch(slots, pool, d)
    want = R.stored(x).float()
    for got in (k, v):
        assert torch.equal(got.isnan(), want.isnan()) and got[1, 0, :32].isnan().all() and not got[1, 0, 32:].isnan().any()
        assert torch.equal(got.nan_to_num(0), want.nan_to_num(0))
    assert k.nan_to_num(0).abs().max() <= 32768 * 1.001 and not k.isinf().any()


def test_append_far_into_a_large_pool(ss):
    d, page, h = 256, 128, 16  # 640 KiB a page: page 8000 lies past 4 GiB
    pool = ss.int4_pool(8200, h, page, d)
    assert pool.numel() > 1 << 32
    k = torch.randn((3, h, d), generator=_gen(1), device="cuda").bfloat16()
    slots = torch.tensor([8199 * page + 127, 5, 8000 * page], device="cuda")
    ss.int4_append(k, k, slots, pool)
    kr, vr = ss.int4_fetch(slots, pool, d)
    assert torch.equal(kr, R.stored(k).float()) and torch.equal(vr, kr)
    q = torch.randn((1, h, d), generator=_gen(2), device="cuda").half()
    table = _i32([[8000]])
    o = ss.int4_attention(q, pool, table, _i32([1]), _i32([0, 1]), 0.1, max_q=1)
    assert torch.equal(o[0], kr[2].half())  # one key: its value


def test_nothing_to_write(ss):
    pool = ss.int4_pool(1, 2, 16, 64).fill_(7)
    e = torch.empty((0, 2, 64), device="cuda")
    s = torch.empty(0, dtype=torch.int64, device="cuda")
    ss.int4_append(e, e, s, pool)
    k, v = ss.int4_fetch(s, pool, 64)
    assert k.shape == v.shape == (0, 2, 64) and (pool == 7).all()
    x = torch.ones((3, 2, 64), device="cuda")
    ss.int4_append(x, x, torch.tensor([-1, 16, 1 << 40], device="cuda"), pool)  # outside the pool
    assert (pool == 7).all()


# ------------------------------------------------------------------ attention

def _setup(ss, old, new, hkv, d, page, seed, dtype, grp, pad=0):
    """A pool with the requests' tokens written by the framework, stale NaN elsewhere."""
    g = _gen(seed)
    lens = [o + q for o, q in zip(old, new)]
    need = [-(-x // page) for x in lens]
    total, width = sum(need) + 1, max(max(need), 1)
    order = torch.randperm(total, generator=g, device="cuda").int()
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at, slots = 0, []
    for b, x in enumerate(need):
        table[b, :x] = order[at:at + x]
        at += x
        t = torch.arange(lens[b], device="cuda")
        slots.append(table[b, t // page].long() * page + t % page)
    slots = torch.cat(slots)
    pool = ss.int4_pool(total, hkv, page, d).fill_(255)  # NaN scales wherever nothing is written
    k = torch.randn((slots.shape[0], hkv, d), generator=g, device="cuda")
    k[..., ::16] *= 4
    v = torch.randn((slots.shape[0], hkv, d), generator=g, device="cuda") + 0.3
    ss.int4_append(k, v, slots, pool)
    kr, vr = ss.int4_fetch(slots, pool, d)
    first = np.concatenate([[0], np.cumsum(lens)])
    kv = [(kr[first[b]:first[b + 1]], vr[first[b]:first[b + 1]]) for b in range(len(lens))]
    q = torch.randn((sum(new) + pad, hkv * grp, d), generator=g, device="cuda").to(dtype)
    return pool, table, _i32(lens), _i32([0] + list(np.cumsum(new))), q, kv


def _check(o, lse, q, kv, old, new, scale, causal, window):
    u, u_out = 2.0 ** -11, 2.0 ** -11 if q.dtype == torch.float16 else 2.0 ** -8
    at, num, den = 0, 0.0, 0.0
    for (k, v), o0, nq in zip(kv, old, new):
        if not nq:
            continue
        want, wl, pv, mag = R.attention(q[at:at + nq], k, v, o0 + nq, scale, causal, window)
        got, gl = o[at:at + nq].double(), lse[at:at + nq].double()
        dz = u * mag
        assert torch.isfinite(got).all()
        assert ((got - want).abs() <= u_out * want.abs() + (4 * u + 2 * dz[..., None]) * pv + 1e-7).all(), (o0, nq)
        none = wl == -math.inf
        assert torch.equal(gl == -math.inf, none) and (got[none] == 0).all()
        assert ((gl - wl)[~none].abs() <= dz[~none] + 1e-5 * (1 + wl[~none].abs())).all()
        num += float((got - want).square().sum())
        den += float(want.square().sum())
        at += nq
    assert math.sqrt(num) <= u_out * math.sqrt(den), math.sqrt(num / max(den, 1e-300)) / u_out
    assert (o[at:] == 0).all() and (lse[at:] == -math.inf).all()


CASES = [
    # old, new, hkv, grp, d, page, dtype, causal, window
    ([0], [1], 1, 1, 128, 16, torch.float16, True, 0),
    ([15, 16, 17, 0, 63], [1, 1, 1, 1, 1], 2, 4, 128, 16, torch.bfloat16, True, 0),
    ([776], [1], 8, 4, 128, 64, torch.float16, True, 0),
    ([5000, 3, 1200, 129], [1, 1, 0, 1], 2, 8, 128, 128, torch.bfloat16, True, 0),
    ([100, 2000], [1, 1], 1, 16, 128, 32, torch.float16, True, 0),
    ([300, 40, 0], [1, 1, 1], 3, 7, 64, 16, torch.float16, True, 0),
    ([1111, 48], [1, 1], 2, 5, 256, 48, torch.bfloat16, True, 0),
    ([900, 30], [4, 3], 2, 4, 128, 64, torch.float16, True, 0),            # several tokens at once
    ([900, 30, 5], [1, 1, 1], 2, 4, 128, 64, torch.float16, True, 20),     # window
    ([70, 0, 1000], [33, 17, 1], 2, 4, 128, 16, torch.bfloat16, True, 0),  # prompt chunks beside a decode
    ([0], [257], 2, 4, 128, 64, torch.float16, True, 0),
    ([0, 128], [128, 129], 1, 1, 128, 128, torch.bfloat16, True, 0),
    ([0, 500], [200, 100], 2, 7, 64, 16, torch.float16, True, 50),
    ([0, 40], [100, 3], 1, 2, 256, 32, torch.float16, True, 0),
    ([0, 40], [300, 20], 2, 4, 128, 64, torch.bfloat16, False, 0),
    ([10, 40], [300, 20], 2, 4, 64, 64, torch.float16, False, 33),
    ([0, 0, 0], [600, 0, 31], 1, 16, 128, 16, torch.float16, True, 0),
]


@pytest.mark.parametrize("old,new,hkv,grp,d,page,dtype,causal,window", CASES)
def test_attention(ss, old, new, hkv, grp, d, page, dtype, causal, window):
    pool, table, lens, cu, q, kv = _setup(ss, old, new, hkv, d, page, sum(old) + d, dtype, grp, pad=3)
    scale = 1 / math.sqrt(d)
    o, lse = ss.int4_attention(q, pool, table, lens, cu, scale, max_q=max(new), causal=causal, window=window, return_lse=True)
    _check(o, lse, q, kv, old, new, scale, causal, window)
    again = ss.int4_attention(q, pool, table, lens, cu, scale, max_q=max(new), causal=causal, window=window)
    assert torch.equal(again, o)  # the same bits every time


def test_attention_max_q_is_a_hint(ss):
    old, new = [50, 0, 7], [40, 1, 20]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 2, 128, 16, 3, torch.float16, 4)
    for hint in (1, 2, 16, 40, 5000):
        o, lse = ss.int4_attention(q, pool, table, lens, cu, 0.08, max_q=hint, return_lse=True)
        _check(o, lse, q, kv, old, new, 0.08, True, 0)


def test_attention_rows_without_keys(ss):
    # lengths below the number of query rows: the first rows stand before the first key
    pool, table, _, cu, q, kv = _setup(ss, [0, 0, 0], [5, 40, 2], 2, 64, 16, 4, torch.float16, 3)
    lens = [2, 0, 1]
    o, lse = ss.int4_attention(q, pool, table, _i32(lens), cu, 0.1, max_q=40, return_lse=True)
    at = 0
    for (k, v), ln, nq in zip(kv, lens, [5, 40, 2]):
        for i in range(nq):
            seen = ln - nq + i + 1
            if seen <= 0:
                assert (o[at + i] == 0).all() and (lse[at + i] == -math.inf).all()
            else:
                want, wl, _, _ = R.attention(q[at + i:at + i + 1], k, v, seen, 0.1)
                assert (o[at + i].double() - want[0]).abs().max() < 4e-3 * (1 + want.abs().max())  # 8 u of values near 4
                assert (lse[at + i].double() - wl[0]).abs().max() < 1e-2
        at += nq


def test_attention_bad_table_entries_hide_their_keys(ss):
    old, new = [60], [1]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 1, 128, 16, 6, torch.float16, 4)
    (k, v), = kv
    for entry in (-1, pool.shape[0], 1 << 30):
        t = table.clone()
        t[0, 1] = entry
        o = ss.int4_attention(q, pool, t, lens, cu, 0.09, max_q=1)
        keep = torch.cat([torch.arange(16), torch.arange(32, 61)]).cuda()
        want, _, _, _ = R.attention(q, k[keep], v[keep], 45, 0.09)
        assert (o.double() - want).abs().max() < 4e-3 * (1 + want.abs().max())


def test_attention_large_and_special_values(ss):
    d = 128
    pool, table, lens, cu, q, kv = _setup(ss, [70, 200], [1, 1], 1, d, 16, 7, torch.bfloat16, 4)
    (k0, v0), (k1, v1) = kv
    # queries far outside fp16's range: one key takes all the weight
    big = (q.float() * 1e6).to(torch.bfloat16)
    o = ss.int4_attention(big, pool, table, lens, cu, 1.0, max_q=1)
    for b, (k, v) in enumerate(kv):
        z = torch.einsum("hd,td->ht", big[b].double(), k[:, 0].double())
        want = v[z.argmax(-1), 0].double()  # values may pass through fp16 on their way to bf16: the bound above with dz = 0
        assert ((o[b].double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -11) * want.abs()).all()
    # tiny ones: the mean of the values
    o = ss.int4_attention((q.float() * 1e-30).to(torch.bfloat16), pool, table, lens, cu, 1.0, max_q=1)
    for b, (k, v) in enumerate(kv):
        want = v[:, 0].double().mean(0)
        assert ((o[b].double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -11 * v[:, 0].double().abs().mean(0)).all()
    # NaN of one request stays there; a zero query is an ordinary one
    q2 = q.clone()
    q2[0, 1] = math.nan
    q2[1] = 0
    o = ss.int4_attention(q2, pool, table, lens, cu, 0.1, max_q=1)
    assert o[0, 1].isnan().all() and torch.isfinite(o[0, [0, 2, 3]]).all() and torch.isfinite(o[1]).all()
    # a key with NaN reaches every row that sees it, values with NaN their dims
    nan = torch.zeros((1, 1, d), device="cuda")
    nan[0, 0, 40] = math.nan
    one = torch.ones((1, 1, d), device="cuda")
    slot = (table[0, 1].long() * 16 + 3)[None]
    for kk, vv in ((nan, one), (one, nan)):
        pool2 = pool.clone()
        ss.int4_append(kk, vv, slot, pool2)
        o = ss.int4_attention(q, pool2, table, lens, cu, 0.1, max_q=1)
        assert torch.isfinite(o[1]).all()
        if kk is nan:
            assert o[0].isnan().all()
        else:
            assert o[0, :, 32:64].isnan().all() and torch.isfinite(o[0, :, :32]).all() and torch.isfinite(o[0, :, 64:]).all()


def test_attention_scales_of_tiny_and_large_values(ss):
    # values of 1e-3 and of 1e3 next to ordinary keys: the output keeps its relative precision
    for mag in (1e-3, 1e3):
        g = _gen(8)
        pool = ss.int4_pool(20, 2, 16, 128).fill_(255)
        n = 300
        slots = torch.arange(n, device="cuda")
        k = torch.randn((n, 2, 128), generator=g, device="cuda")
        v = torch.randn((n, 2, 128), generator=g, device="cuda") * mag
        ss.int4_append(k, v, slots, pool)
        kr, vr = ss.int4_fetch(slots, pool, 128)
        q = torch.randn((40, 8, 128), generator=g, device="cuda").half()
        table = torch.arange(20, dtype=torch.int32, device="cuda")[None]
        for nq in (1, 40):
            x = q[:nq].contiguous()
            o, lse = ss.int4_attention(x, pool, table, _i32([n]), _i32([0, nq]), 0.09, max_q=nq, return_lse=True)
            want, wl, pv, mag_ = R.attention(x, kr, vr, n, 0.09)
            dz = 2.0 ** -11 * mag_[..., None]
            # fp16 results below 2^-14 keep 2^-25 absolutely
            assert ((o.double() - want).abs() <= 2.0 ** -11 * want.abs() + (4 * 2.0 ** -11 + 2 * dz) * pv + 2.0 ** -24).all()


def test_attention_wide_heads_with_few_and_many_units(ss):
    # 256 dims: units of 8 rows, one or two CTAs on an SM, and in turn on one workspace
    cases = []
    for i, (old, new, hkv, grp, window) in enumerate([([2000], [5], 8, 4, 0), ([0, 30, 200], [150, 90, 1], 8, 4, 0),
                                                      ([900] * 40, [1] * 40, 8, 2, 300), ([4000], [1], 4, 8, 0)]):
        for dtype in (torch.float16, torch.bfloat16):
            cases.append((_setup(ss, old, new, hkv, 256, 32, 40 + i, dtype, grp, pad=2), old, new, window))
    for _ in range(2):
        for (pool, table, lens, cu, q, kv), old, new, window in cases:
            o, lse = ss.int4_attention(q, pool, table, lens, cu, 0.06, max_q=max(new), window=window, return_lse=True)
            _check(o, lse, q, kv, old, new, 0.06, True, window)


def test_attention_launches_of_every_shape_share_a_workspace(ss):
    """Units cut into parts, by launches with one and two CTAs on an SM and
    units of 4, 8 and 16 rows, in turn on one stream: every one finds its
    counters at zero."""
    cases = []
    for i, (old, new, grp) in enumerate([([40000], [1], 4), ([3000] * 24, [1] * 24, 4), ([20000, 9000], [2, 2], 8), ([50000], [1], 8),
                                         ([2500] * 40, [1] * 40, 8), ([30000], [4], 4)]):
        cases.append((_setup(ss, old, new, 8, 128, 64, 20 + i, torch.bfloat16, grp), old, new))
    first = None
    for _ in range(3):
        out = [ss.int4_attention(q, pool, t, ln, cu, 0.09, max_q=max(new), return_lse=True) for (pool, t, ln, cu, q, kv), old, new in cases]
        if first is None:
            first = out
            for ((pool, t, ln, cu, q, kv), old, new), (o, lse) in zip(cases, out):
                _check(o, lse, q, kv, old, new, 0.09, True, 0)
        for (o, lse), (o1, lse1) in zip(out, first):
            assert torch.equal(o, o1) and torch.equal(lse, lse1)


@pytest.mark.parametrize("old,new,hkv,grp,d,dtype,causal,window", [
    ([4000], [64], 8, 4, 128, torch.bfloat16, True, 0),        # 16 units of 32 tiles
    ([5001], [37], 8, 4, 128, torch.float16, True, 0),         # ragged rows and keys
    ([3000, 900, 0], [40, 50, 130], 4, 8, 64, torch.float16, True, 0),  # units of 1 to 24 tiles
    ([2500, 2500], [40, 1], 8, 4, 64, torch.bfloat16, True, 1300),      # a window, and a decoding request
    ([2000], [200], 2, 3, 128, torch.float16, False, 0),
    ([20000], [1200], 1, 1, 128, torch.bfloat16, True, 0),
    ([3000] * 4, [32] * 4, 8, 4, 128, torch.float16, True, 0),  # tiles for the length of their keys
    ([3000, 70, 3000], [12, 12, 11], 8, 4, 64, torch.bfloat16, True, 0),  # and just not
])
def test_attention_few_tiles_are_cut_along_the_keys(ss, old, new, hkv, grp, d, dtype, causal, window):
    pool, table, lens, cu, q, kv = _setup(ss, old, new, hkv, d, 64, sum(old) + d, dtype, grp, pad=3)
    first = None
    for _ in range(3):  # the order of arrival does not matter, and counters are left as they were found
        o, lse = ss.int4_attention(q, pool, table, lens, cu, 0.09, max_q=max(new), causal=causal, window=window, return_lse=True)
        if first is None:
            first = o, lse
            _check(o, lse, q, kv, old, new, 0.09, causal, window)
        assert torch.equal(o, first[0]) and torch.equal(lse, first[1])


def test_attention_cut_tiles_wait_that_runs_out_then_recovers(ss):
    """Parts that give up still arrive: the counters of their units end at zero."""
    import ctypes as C

    from sunshape_mlx_b200 import _lib as L
    from sunshape_mlx_b200.paged import _workspace

    L.check_device_errors()
    old, new = [4000], [64]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 8, 128, 16, 15, torch.bfloat16, 4)
    out, ws = torch.empty_like(q), _workspace(pool, 128)
    a = L.Int4AttnArgs(q.data_ptr(), L.SS_BF16, q.stride(0), q.stride(1), q.shape[0], 32, 8, 128, pool.data_ptr(), pool.shape[0],
                       pool.stride(0), pool.stride(1), 16, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(),
                       cu.data_ptr(), 1, 64, 0.09, 1, 0, out.data_ptr(), None, ws.data_ptr(), ws.numel(), 1_000_000, 2 + 1)
    L.call("ss_int4_attention", C.byref(a), L.stream_ptr(q.device))
    torch.cuda.synchronize()
    args = (q, pool, table, lens, cu, 0.09)
    with pytest.raises(L.SunShapeCudaError, match="int4_attention tile wait"):
        ss.int4_attention(*args, max_q=64)
    o, lse = ss.int4_attention(*args, max_q=64, return_lse=True)
    _check(o, lse, q, kv, old, new, 0.09, True, 0)
    L.check_device_errors()


@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_attention_any_scale(ss, scale):
    for old, new, d in (([200, 30], [1, 1], 128), ([0, 60], [400, 300], 64)):
        pool, table, lens, cu, q, kv = _setup(ss, old, new, 2, d, 16, 11, torch.bfloat16, 4)
        o, lse = ss.int4_attention(q, pool, table, lens, cu, scale, max_q=max(new), return_lse=True)
        _check(o, lse, q, kv, old, new, scale, True, 0)


def test_attention_tiles_and_units_share_a_batch(ss):
    # requests on both sides of the rule that sends rows to the tile kernel, empty ones, and wrong pages
    old, new = [0, 3000, 17, 0, 64, 500], [700, 1, 0, 300, 2, 36]
    for dtype, window in ((torch.float16, 0), (torch.bfloat16, 130)):
        pool, table, lens, cu, q, kv = _setup(ss, old, new, 8, 128, 64, 12, dtype, 4, pad=7)
        o, lse = ss.int4_attention(q, pool, table, lens, cu, 0.088, max_q=700, window=window, return_lse=True)
        _check(o, lse, q, kv, old, new, 0.088, True, window)
    t = table.clone()
    t[0, 3] = -1  # keys 192 .. 255 of the first request disappear
    o = ss.int4_attention(q, pool, t, lens, cu, 0.088, max_q=700)
    (k, v) = kv[0]
    for row in (100, 300, 699):
        keep = torch.tensor([i for i in range(row + 1) if not 192 <= i < 256], device="cuda")
        want, _, _, _ = R.attention(q[row:row + 1], k[keep], v[keep], len(keep), 0.088, causal=False)
        assert (o[row].double() - want[0]).abs().max() < 2.0 ** -7 * (1 + want.abs().max())


def test_attention_tiles_special_values(ss):
    d = 128
    pool, table, lens, cu, q, kv = _setup(ss, [0, 0], [300, 300], 2, d, 16, 13, torch.bfloat16, 4)
    q2 = q.clone()
    q2[5, 1] = math.nan
    q2[7] = 0
    q2[8] = (q2[8].float() * 1e30).to(q.dtype)   # one key takes all the weight
    q2[9] = (q2[9].float() * 1e-37).to(q.dtype)
    o, lse = ss.int4_attention(q2, pool, table, lens, cu, 1.0, max_q=300, return_lse=True)
    assert o[5, 1].isnan().all() and torch.isfinite(o[5, [0] + list(range(2, 8))]).all()
    keep = [i for i in range(600) if i != 5]
    assert torch.isfinite(o[keep]).all()
    (k, v), _ = kv
    for h in range(8):
        z = torch.einsum("d,td->t", q2[8, h].double(), k[:9, h // 4].double())
        want = v[z.argmax(), h // 4].double()
        assert ((o[8, h].double() - want).abs() <= (2.0 ** -8 + 4 * 2.0 ** -11) * want.abs()).all()
    for row in (7, 9):  # the mean of the values
        want = v[:row + 1].double().mean(0).repeat_interleave(4, 0)
        pv = v[:row + 1].double().abs().mean(0).repeat_interleave(4, 0)
        assert ((o[row].double() - want).abs() <= 2.0 ** -8 * want.abs() + 4 * 2.0 ** -11 * pv).all()
        assert (lse[row] - math.log(row + 1)).abs().max() < 1e-5
    # the widest groups that pages hold: codes times scales reach fp16's largest
    pool2 = ss.int4_pool(4, 1, 64, d).fill_(255)
    x = torch.zeros((200, 1, d), device="cuda")
    x[:, 0, ::2], x[:, 0, 1::2] = 32768.0, -32768.0
    ss.int4_append(x, x * 1e-3, torch.arange(200, device="cuda"), pool2)
    kr, vr = ss.int4_fetch(torch.arange(200, device="cuda"), pool2, d)
    qq = torch.randn((200, 16, d), generator=_gen(3), device="cuda").half()
    t = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    o, lse = ss.int4_attention(qq, pool2, t, _i32([200]), _i32([0, 200]), 1e-6, max_q=200, return_lse=True)
    _check(o, lse, qq, [(kr, vr)], [0], [200], 1e-6, True, 0)


def test_attention_strided_queries_other_stream_and_pool_view(ss):
    old, new = [200, 31], [2, 1]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 2, 128, 16, 9, torch.float16, 4)
    want = ss.int4_attention(q, pool, table, lens, cu, 0.1, max_q=2)
    qkv = torch.zeros((3, 8 + 4, 128), dtype=torch.float16, device="cuda")
    qkv[:, :8] = q
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=torch.float16, device="cuda")[1:].view(3, 8, 128)
    odd.copy_(q)  # 2-byte aligned
    swapped = q.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((table.shape[0], table.shape[1] + 5), 1 << 29, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    big = torch.full((pool.shape[0], 4, pool.shape[2] + 16), 255, dtype=torch.uint8, device="cuda")
    big[:, 1:3, :pool.shape[2]] = pool
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ss.int4_attention(x, pool, table, lens, cu, 0.1, max_q=2) for x in (qkv[:, :8], odd, swapped)]
        got.append(ss.int4_attention(q, big[:, 1:3, :pool.shape[2]], wide[:, :table.shape[1]], lens, cu, 0.1, max_q=2))
    s.synchronize()
    for x in got:
        assert torch.equal(x, want)


def test_attention_in_a_cuda_graph(ss):
    old, new = [500, 31], [1, 1]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 2, 128, 16, 10, torch.float16, 4)
    want = ss.int4_attention(q, pool, table, lens, cu, 0.1, max_q=1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ss.int4_attention(q, pool, table, lens, cu, 0.1, max_q=1)
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        out = ss.int4_attention(q, pool, table, lens, cu, 0.1, max_q=1)
    for ln in ([501, 32], [17, 1], [490, 16]):  # lengths change under the graph
        lens.copy_(_i32(ln))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ss.int4_attention(q, pool, table, lens, cu, 0.1, max_q=1))
    lens.copy_(_i32([501, 32]))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_attention_wait_that_runs_out_is_reported_then_recovers(ss):
    """The tile kernel's waits are bounded: with one tile never announced and a
    bound of 1 ms the launch gives up, the next call says so, and the one
    after is right."""
    import ctypes as C

    from sunshape_mlx_b200 import _lib as L
    from sunshape_mlx_b200.paged import _workspace

    L.check_device_errors()
    old, new = [0, 100], [900, 400]
    pool, table, lens, cu, q, kv = _setup(ss, old, new, 4, 128, 16, 14, torch.float16, 4)
    out, ws = torch.empty_like(q), _workspace(pool, 128)
    a = L.Int4AttnArgs(q.data_ptr(), L.SS_F16, q.stride(0), q.stride(1), q.shape[0], 16, 4, 128, pool.data_ptr(), pool.shape[0],
                       pool.stride(0), pool.stride(1), 16, table.data_ptr(), table.stride(0), table.shape[1], lens.data_ptr(),
                       cu.data_ptr(), 2, 900, 0.09, 1, 0, out.data_ptr(), None, ws.data_ptr(), ws.numel(), 1_000_000, 2 + 1)
    L.call("ss_int4_attention", C.byref(a), L.stream_ptr(q.device))
    torch.cuda.synchronize()
    args = (q, pool, table, lens, cu, 0.09)
    with pytest.raises(L.SunShapeCudaError, match="int4_attention tile wait") as e:
        ss.int4_attention(*args, max_q=900)
    assert e.value.code == L.SS_ERR_TIMEOUT
    o, lse = ss.int4_attention(*args, max_q=900, return_lse=True)
    _check(o, lse, q, kv, old, new, 0.09, True, 0)
    L.check_device_errors()


def test_no_queries(ss):
    pool = ss.int4_pool(1, 2, 16, 64)
    q = torch.empty((0, 4, 64), dtype=torch.float16, device="cuda")
    o, lse = ss.int4_attention(q, pool, _i32([[0]]), _i32([5]), _i32([0, 0]), 1.0, max_q=1, return_lse=True)
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals(ss):
    pool = ss.int4_pool(2, 2, 16, 64)
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device="cuda")
    t, ln, cu = _i32([[0]]), _i32([1]), _i32([0, 1])
    ok = dict(queries=q, pages=pool, block_table=t, seq_lens=ln, cu_q=cu, scale=1.0, max_q=1)
    ss.int4_attention(**ok)
    for bad, err in [(dict(queries=q.float()), TypeError), (dict(queries=q.cpu()), ValueError), (dict(queries=q[:, :3]), ValueError),
                     (dict(queries=q[..., :32]), ValueError), (dict(queries=q[0]), ValueError), (dict(pages=pool[:, :, :80]), ValueError),
                     (dict(pages=pool.view(torch.int8)), ValueError), (dict(block_table=t.long()), ValueError),
                     (dict(block_table=_i32([[0], [1]])), ValueError), (dict(seq_lens=ln.cpu()), ValueError), (dict(cu_q=_i32([0])), ValueError),
                     (dict(max_q=0), ValueError), (dict(window=-1), ValueError), (dict(queries=q.transpose(1, 2)), ValueError)]:
        with pytest.raises(err):
            ss.int4_attention(**{**ok, **bad})
    x, s = torch.zeros((3, 2, 64), device="cuda"), torch.arange(3, device="cuda")
    for bad in [(x, x[:2], s, pool), (x, x.half(), s, pool), (x[:, :1], x[:, :1], s, pool), (x, x, s.int(), pool), (x, x, s[:2], pool),
                (x[..., :60], x[..., :60], s, pool), (x.cpu(), x.cpu(), s, pool), (x, x, s, pool[:, :, 1:])]:
        with pytest.raises(ValueError):
            ss.int4_append(*bad)
    with pytest.raises(TypeError):
        ss.int4_append(x.double(), x.double(), s, pool)
    with pytest.raises(ss._lib.SunShapeCudaError, match="multiples of 16"):
        ss.int4_append(x, x, s, torch.zeros(2 * 2 * 16 * 80 + 1, dtype=torch.uint8, device="cuda")[1:].view(2, 2, -1))
    with pytest.raises(ValueError):
        ss.int4_fetch(s.int(), pool, 64)
    with pytest.raises(ValueError):
        ss.int4_fetch(s, pool, 96)
    f, nf = _i32([0, 1]), _i32([2])
    for bad in [dict(page_size=8), dict(n_tokens=-1), dict(q_lens=_i32([1, 2])), dict(free_pages=f.long()), dict(seq_lens=ln.cpu())]:
        with pytest.raises(ValueError):
            ss.plan_step(**{**dict(seq_lens=ln, q_lens=ln, block_table=t, free_pages=f, n_free=nf, page_size=16, n_tokens=4), **bad})
    with pytest.raises(ValueError):
        ss.PageTables(4, 20, 1, 1)
