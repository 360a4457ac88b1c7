"""The paged 4-bit operators where a value, a size or a launch is at the end
of its range: each against its definition in 64 bits. u = 2^-11 is the
relative rounding of fp16."""

import math

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
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def _filled(ss, k, v, page=64):
    """A pool that holds k, v (T, hkv, D) in order, and the row of its table."""
    pages = -(-k.shape[0] // page)
    pool = ss.int4_pool(pages, k.shape[1], page, k.shape[2]).fill_(255)
    ss.int4_append(k, v, torch.arange(k.shape[0], device="cuda"), pool)
    return pool, torch.arange(pages, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ one key far above all others

@pytest.mark.parametrize("nats", [16.0, 17.0, 18.0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n_req,nq,grp,d,keys", [(320, 1, 4, 128, 16384), (320, 1, 8, 128, 16384), (320, 1, 4, 64, 16384), (320, 1, 4, 256, 16384),
                                                 (1, 640, 32, 128, 65536), (1, 640, 32, 64, 65536), (1, 64, 32, 128, 65536)])
def test_attention_one_key_above_a_long_context(ss, n_req, nq, grp, d, keys, dtype, nats):
    """The first key is `nats` above all others and its value is 0: the output
    is what the others leave. Keys and queries are powers of two, so logits
    are exact. A probability keeps fp16's relative rounding down to 2^-24 of the
    largest and is off by 4 u at most down to 2^-26 (18 nats). Sums of n terms
    in fp32 are off by n 2^-24, and a row has four of them at least."""
    k = torch.zeros((keys, 1, d), device="cuda")
    k[0] = 0.5
    v = torch.randn((keys, 1, d), generator=_gen(keys + d), device="cuda") + 1.0
    v[0] = 0.0
    pool, row = _filled(ss, k, v)
    kr, vr = ss.int4_fetch(torch.arange(keys, device="cuda"), pool, d)
    assert torch.equal(kr, k) and (vr[0] == 0).all()
    q = torch.full((n_req * nq, grp, d), 2.0, dtype=dtype, device="cuda")
    cu = torch.arange(n_req + 1, dtype=torch.int32, device="cuda") * nq
    o, lse = ss.int4_attention(q, pool, row.expand(n_req, -1).contiguous(), _i32([keys] * n_req), cu, nats / d, max_q=nq, causal=False, return_lse=True)
    want, wl, pv, _ = R.attention(q[:1], kr, vr, keys, nats / d, causal=False)
    u, u_out = 2.0 ** -11, 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    sums = keys / 4 * 2.0 ** -24
    assert ((o.double() - want).abs() <= u_out * want.abs() + (4 * u + sums) * pv + keys * 2.0 ** -37 * vr.abs().max()).all()
    assert ((lse.double() - wl).abs() <= sums + 1e-5 * (1 + wl.abs())).all()


# ------------------------------------------------------------------ launches inside graphs

def _batch(ss, old, new, d, grp, seed, dtype=torch.bfloat16):
    lens = [a + b for a, b in zip(old, new)]
    need = [-(-x // 64) for x in lens]
    k = torch.randn((sum(need) * 64, 8, d), generator=_gen(seed), device="cuda")
    v = torch.randn((sum(need) * 64, 8, d), generator=_gen(seed + 1), device="cuda")
    pool, row = _filled(ss, k, v)
    table = torch.full((len(old), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, x in enumerate(need):
        table[b, :x] = row[at:at + x]
        at += x
    cu = [0]
    for x in new:
        cu.append(cu[-1] + x)
    q = torch.randn((cu[-1], 8 * grp, d), generator=_gen(seed + 2), device="cuda").to(dtype)
    return (q, pool, table, _i32(lens), _i32(cu), 0.09), max(new)


def _stale_memory(pool, stream, nbytes):
    """Leaves nbytes of ones in the free memory that a graph pool has for a stream."""
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool, stream=stream):
        x = torch.full((nbytes,), 255, dtype=torch.uint8, device="cuda")
    g.replay()
    torch.cuda.synchronize()
    del x
    return g


@pytest.mark.parametrize("d", [64, 128, 256])
def test_attention_captured_without_a_call_before(ss, d):
    """Two graphs whose first call is the captured one, replayed in the other
    order, in memory that held something else: units are cut into parts, so
    every output waits on counters that must start at zero."""
    decode, m1 = _batch(ss, [3000, 9000], [1, 1], d, 4, 1)
    mixed, m2 = _batch(ss, [3000, 20, 4000], [1, 300, 40], d, 4, 2)  # both kernels, one launch beside the other
    want = [ss.int4_attention(*decode, max_q=m1), ss.int4_attention(*mixed, max_q=m2)]
    mem = torch.cuda.graph_pool_handle()
    stream = torch.cuda.Stream()  # no call ran on it
    keep = _stale_memory(mem, stream, 128 << 20)
    first, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(first, pool=mem, stream=stream):
        a = [ss.int4_attention(*decode, max_q=m1), ss.int4_attention(*mixed, max_q=m2)]
    with torch.cuda.graph(second, pool=mem, stream=stream):
        b = [ss.int4_attention(*mixed, max_q=m2), ss.int4_attention(*decode, max_q=m1)]
    second.replay()
    torch.cuda.synchronize()
    assert torch.equal(b[0], want[1]) and torch.equal(b[1], want[0])
    for _ in range(2):
        first.replay()
        torch.cuda.synchronize()
        assert torch.equal(a[0], want[0]) and torch.equal(a[1], want[1])
    # a call on that stream, outside any graph, before and after
    with torch.cuda.stream(stream):
        c = ss.int4_attention(*decode, max_q=m1)
    stream.synchronize()
    assert torch.equal(c, want[0])
    del keep


def test_attention_graphs_of_one_stream_replayed_side_by_side(ss):
    """Graphs captured on one stream, and calls on it, may run at the same time: each has counters of its own."""
    calls = [_batch(ss, [20000, 9000], [1, 1], 128, 4, 3), _batch(ss, [3000, 20, 4000], [1, 300, 40], 128, 4, 4)]
    want = [ss.int4_attention(*x, max_q=m) for x, m in calls]
    s = torch.cuda.Stream()
    graphs, outs = [], []
    for x, m in calls:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(ss.int4_attention(*x, max_q=m))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(30):
        for o in outs:
            o.fill_(math.nan)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        with torch.cuda.stream(s):
            eager = ss.int4_attention(*calls[0][0], max_q=1)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])


# ------------------------------------------------------------------ written values

@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_groups_across_the_largest_magnitude(ss, d, dtype):
    """Codes are those of the clamped values, also where others of the group
    lie so near 2^15 that its zero is rounded up to it."""
    g = _gen(d)
    n = 500
    near = 32768.0 - torch.rand((n, 2, d), generator=g, device="cuda") * torch.rand((n, 2, 1), generator=g, device="cuda") * 300
    x = torch.where(torch.rand((n, 2, d), generator=g, device="cuda") < 0.1, 33000 + torch.rand((n, 2, d), generator=g, device="cuda") * 20000, near)
    x[0, 0] = 32760.0
    x[0, 0, 7::32] = 40000.0
    x[1, 0, 3::32] = math.inf
    x[2, 0] = 65000.0
    x[3, 0, 5::32] = -math.inf
    k, v = x.to(dtype), (-x).to(dtype)
    pool, slots = ss.int4_pool(-(-n // 16), 2, 16, d), torch.arange(n, device="cuda")
    ss.int4_append(k, v, slots, pool)
    kr, vr = ss.int4_fetch(slots, pool, d)
    assert torch.equal(kr, R.stored(k).float()) and torch.equal(vr, R.stored(v).float())


# ------------------------------------------------------------------ small keys

@pytest.mark.parametrize("nq", [1, 60])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("steps", [1, 3, 1025])
def test_attention_keys_of_the_smallest_scales(ss, steps, d, nq):
    """Scales of `steps` times fp16's smallest: units of few rows take such
    keys exactly, tiles to 2^-24 where code and scale are both odd."""
    s = steps * 2.0 ** -24
    t = 200
    codes = (torch.arange(t, device="cuda") % 8 * 2)[:, None].expand(t, 32).clone().float()
    codes[:, 0], codes[:, 1] = 0.0, 15.0
    k = (codes * s)[:, None].repeat(1, 1, d // 32).contiguous()
    pool, row = _filled(ss, k, torch.randn((t, 1, d), generator=_gen(1), device="cuda"))
    kr, vr = ss.int4_fetch(torch.arange(t, device="cuda"), pool, d)
    assert torch.equal(kr, k)
    size = 2.0 ** 17 / steps
    size = 2.0 ** math.floor(math.log2(size))
    q = torch.full((nq, 32, d), size, dtype=torch.bfloat16, device="cuda")
    o, lse = ss.int4_attention(q, pool, row[None], _i32([t]), _i32([0, nq]), 128 / d, max_q=nq, causal=False, return_lse=True)
    _, wl, _, _ = R.attention(q, kr, vr, t, 128 / d, causal=False)
    odd = d // 32 if nq > 1 and steps % 2 else 0
    assert ((lse.double() - wl).abs() <= 128 / d * odd * size * 2.0 ** -24 + 1e-5 * (1 + wl.abs())).all()


# ------------------------------------------------------------------ arguments

def test_pools_without_heads_are_refused(ss):
    pool = torch.zeros((2, 0, 1280), dtype=torch.uint8, device="cuda")
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device="cuda")
    s = torch.zeros(1, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        ss.int4_attention(q, pool, _i32([[0]]), _i32([1]), _i32([0, 1]), 1.0, max_q=1)
    with pytest.raises(ValueError):
        ss.int4_fetch(s, pool, 64)
    with pytest.raises(ValueError):
        ss.int4_append(q[:, :0].float(), q[:, :0].float(), s, pool)
    for bad in ((0, 2, 16, 64), (2, 0, 16, 64), (2, 2, 24, 64)):
        with pytest.raises(ValueError):
            ss.int4_pool(*bad)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("old,new,seen", [(100, 1, 101), (0, 300, 300), (0, 300, 40), (0, 8, 3)])
def test_attention_windows_past_every_key_hide_nothing(ss, old, new, seen, causal):
    """Also where requests have more query rows than keys, and for numbers that no 32 bits hold."""
    k = torch.randn((old + new, 2, 64), generator=_gen(1), device="cuda")
    pool, row = _filled(ss, k, torch.randn_like(k))
    q = torch.randn((new, 8, 64), generator=_gen(2), device="cuda").half()
    args = q, pool, row[None], _i32([seen]), _i32([0, new]), 0.1
    want = ss.int4_attention(*args, max_q=new, causal=causal)
    ref = R.attention(q, *ss.int4_fetch(torch.arange(old + new, device="cuda"), pool, 64), seen, 0.1, causal)[0]
    assert (want.double() - ref).abs().max() < 4e-3 * (1 + ref.abs().max())
    for window in (seen, 10 ** 6, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5):
        assert torch.equal(ss.int4_attention(*args, max_q=new, causal=causal, window=window), want)
    assert torch.equal(ss.int4_attention(*args, max_q=2 ** 32 + 1, causal=causal), ss.int4_attention(*args, max_q=2 ** 31 - 1, causal=causal))


def test_sizes_past_32_bits_are_refused(ss):
    i = _i32([1])
    with pytest.raises(ValueError, match="page_size"):
        ss.plan_step(i, i, i[None], i, i, page_size=2 ** 32 + 16, n_tokens=1)
    with pytest.raises(ValueError, match="page_size"):
        ss.release_pages(i, i.bool(), i[None], i, i, page_size=2 ** 32 + 16)
    x = torch.empty((1, 2 ** 31 + 8), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="vocab"):
        ss.token_logprobs(x, torch.zeros(1, dtype=torch.int64, device="cuda"))


def test_single_elements_of_any_stride(ss):
    """A dimension of one element is contiguous whatever its stride says."""
    wide = lambda x: torch.stack([_i32(x)] * 3, -1)[..., 0]  # noqa: E731  stride 3
    k = torch.randn((20, 2, 64), generator=_gen(1), device="cuda")
    pool, _ = _filled(ss, k, k)
    q = torch.randn((1, 4, 64), generator=_gen(2), device="cuda").half()
    want = ss.int4_attention(q, pool, _i32([[0]]), _i32([20]), _i32([0, 1]), 0.1, max_q=1)
    table = torch.zeros((1, 3), dtype=torch.int32, device="cuda")[:, ::3]
    assert torch.equal(ss.int4_attention(q, pool, table, wide([20]), _i32([0, 1]), 0.1, max_q=1), want)
    p = ss.plan_step(wide([5]), wide([2]), torch.as_strided(_i32([7]), (1, 1), (0, 9)), _i32(range(8)), wide([1]), page_size=16, n_tokens=2)
    assert p.status.item() == 0 and p.slots.tolist() == [7 * 16 + 5, 7 * 16 + 6]
    lens, left, status = ss.release_pages(wide([5]), torch.tensor([True], device="cuda"), torch.as_strided(_i32([1]), (1, 1), (0, 9)), _i32([0, 0]), wide([1]),
                                          page_size=16)
    assert (lens.item(), left.item(), status.item()) == (0, 2, 0)


def test_refused_head_dims_leave_no_memory_behind(ss):
    pool = ss.int4_pool(2, 2, 16, 64)
    q = torch.zeros((1, 4, 100_000), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError):
        ss.int4_attention(q, pool, _i32([[0]]), _i32([1]), _i32([0, 1]), 1.0, max_q=1)
    assert torch.cuda.memory_allocated() - before < 1 << 20


def test_inputs_that_want_gradients_are_refused(ss):
    k = torch.randn((20, 2, 64), generator=_gen(1), device="cuda")
    pool, row = _filled(ss, k, k)
    q = torch.randn((1, 4, 64), generator=_gen(2), device="cuda").half().requires_grad_()
    args = pool, row[None], _i32([20]), _i32([0, 1]), 0.1
    x = torch.randn((3, 50), generator=_gen(3), device="cuda").requires_grad_()
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="gradient"):
        ss.int4_attention(q, *args, max_q=1)
    with pytest.raises(ValueError, match="gradient"):
        ss.token_logprobs(x, t)
    with torch.no_grad():
        assert torch.equal(ss.int4_attention(q, *args, max_q=1), ss.int4_attention(q.detach(), *args, max_q=1))
        assert torch.equal(ss.token_logprobs(x, t).logprobs, ss.token_logprobs(x.detach(), t).logprobs)


def test_server_refuses_ids_outside_the_vocabulary(ss):
    from sunshape_mlx_b200.harness import Decoder, DecoderConfig
    from sunshape_mlx_b200.serving import PagedServer

    model = Decoder(DecoderConfig(n_layers=1, hidden=128, n_heads=2, n_kv_heads=1, ffn=128, vocab=97), seed=1)
    server = PagedServer(model, n_pages=4, page_size=16, max_requests=2, max_tokens=32)
    fine = torch.arange(5)
    for bad in (torch.tensor([3, 97]), torch.tensor([-1, 4]), torch.tensor([3, 97], device="cuda"), torch.tensor([2 ** 40])):
        with pytest.raises(ValueError, match="ids from 0 to 96"):
            server.start([fine, bad])
        assert not server.lens and server.tables.n_free.item() == 4
    reqs, _ = server.start([fine, torch.tensor([0, 96], device="cuda")])
    assert reqs == [0, 1]


def test_server_goes_on_after_a_step_that_failed(ss, monkeypatch):
    """A layer that raises leaves the requests where they were: the next step is the one that failed."""
    from sunshape_mlx_b200.harness import Decoder, DecoderConfig
    from sunshape_mlx_b200.paged import Int4PagedKVCache
    from sunshape_mlx_b200.serving import PagedServer

    model = Decoder(DecoderConfig(n_layers=2, hidden=256, n_heads=4, n_kv_heads=2, ffn=256, vocab=97), seed=1)
    prompts = [torch.arange(15), torch.arange(32) % 7]  # the next token of either one takes a page

    def serve(fail):
        server = PagedServer(model, n_pages=8, page_size=16, max_requests=2, max_tokens=64, top_k=3)
        server.start(prompts)
        got = [server.step()]
        if fail:
            real = Int4PagedKVCache.append

            def broken(self, *a):
                if self is server.caches[1]:
                    raise torch.cuda.OutOfMemoryError("no memory")
                real(self, *a)

            with monkeypatch.context() as m:
                m.setattr(Int4PagedKVCache, "append", broken)
                before = dict(server.lens), server.tables.n_free.item()
                for _ in range(2):
                    with pytest.raises(torch.cuda.OutOfMemoryError):
                        server.step()
                assert (server.lens, server.tables.n_free.item()) == before
        got += [server.step() for _ in range(3)]
        server.tables.check()
        assert server.lens == {0: 19, 1: 36} and server.tables.n_free.item() == 3
        return got

    for (a, la), (b, lb) in zip(serve(True), serve(False)):
        assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(la, lb))


def test_the_same_results_without_the_native_lane(ss, monkeypatch):
    from sunshape_mlx_b200 import _lib as L

    k = torch.randn((200, 2, 64), generator=_gen(1), device="cuda")
    q = torch.randn((200, 8, 64), generator=_gen(2), device="cuda").half()
    x = torch.randn((5, 3000), generator=_gen(3), device="cuda")

    def run():
        table, free = torch.full((2, 8), -1, dtype=torch.int32, device="cuda"), torch.arange(20, dtype=torch.int32, device="cuda")
        p = ss.plan_step(_i32([0, 0]), _i32([130, 70]), table, free, _i32([20]), page_size=32, n_tokens=200)
        pool = ss.int4_pool(20, 2, 32, 64).fill_(255)
        ss.int4_append(k, k, p.slots, pool)
        kv = ss.int4_fetch(p.slots, pool, 64)
        o = ss.int4_attention(q, pool, table, p.seq_lens, p.cu_q, 0.1, max_q=130, return_lse=True)
        return [*p, table, pool, *kv, *o, *ss.token_logprobs(x, torch.arange(5, device="cuda"), top_k=4)]

    want = run()
    monkeypatch.setattr(L, "_fast", L._NoFast())
    for a, b in zip(run(), want):
        assert torch.equal(a, b)


# ------------------------------------------------------------------ what no test reached

def test_append_into_a_view_of_a_larger_pool(ss):
    g = _gen(3)
    k, v = torch.randn((2, 9, 3, 64), generator=g, device="cuda").half()
    wide = torch.full((2, 5, 16 * 80 + 64), 0x5A, dtype=torch.uint8, device="cuda")
    view, slots = wide[:, 1:4, :16 * 80], torch.arange(9, device="cuda") + 12  # of both pages
    dense = view.clone()
    ss.int4_append(k, v, slots, view)
    kr, vr = ss.int4_fetch(slots, view, 64)
    assert torch.equal(kr, R.stored(k).float()) and torch.equal(vr, R.stored(v).float())
    ss.int4_append(k, v, slots, dense)
    assert torch.equal(view, dense)
    assert (wide[:, [0, 4]] == 0x5A).all() and (wide[:, :, 16 * 80:] == 0x5A).all()


@pytest.mark.parametrize("n,page", [(1, 16), (7, 32), (700, 16), (9000, 48)])
def test_release_pages(ss, n, page):
    """Against the definition: pages of ended requests on the stack in the order of the requests and of their tables."""
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, 5 * page, (n,), generator=g)
    done = torch.rand(n, generator=g) < 0.4
    held = (lens + page - 1) // page
    pool = int(held.sum()) + 5
    order = torch.randperm(pool, generator=g).int()
    table = torch.full((n, 6), -1, dtype=torch.int32)
    at = 0
    for b in range(n):
        table[b, :held[b]] = order[at:at + held[b]]
        at += int(held[b])
    free = torch.full((pool,), -7, dtype=torch.int32)
    free[:pool - at] = order[at:]
    gt, gf, left = table.cuda(), free.cuda(), _i32([pool - at])
    got_lens, got_left, status = ss.release_pages(lens.int().cuda(), done.cuda(), gt, gf, left, page_size=page)
    stack = free[:pool - at].tolist()
    for b in range(n):
        if done[b]:
            stack += table[b, :held[b]].tolist()
            table[b, :held[b]] = -1
    assert status.item() == 0 and got_left.item() == len(stack) and gf[:len(stack)].tolist() == stack
    assert (gf[len(stack):].cpu() == -7).all() and torch.equal(gt.cpu(), table)
    assert torch.equal(got_lens.cpu().long(), torch.where(done, 0, lens))


def test_release_of_more_pages_than_are_out_changes_nothing(ss):
    table, free = _i32([[3, 4], [5, -1]]), _i32([0, 1, 2, 9, 9, 9])
    lens, left, status = ss.release_pages(_i32([20, 9]), torch.tensor([True, True], device="cuda"), table, free, _i32([4]), page_size=16)
    assert status.item() == 8 and left.item() == 4 and lens.tolist() == [20, 9]
    assert table.tolist() == [[3, 4], [5, -1]] and free.tolist() == [0, 1, 2, 9, 9, 9]
    t = ss.PageTables(n_pages=4, page_size=16, max_requests=2, max_pages=4)
    t.seq_lens = _i32([40, 0])  # three pages that were never handed out
    t.release(torch.tensor([True, False], device="cuda"))
    with pytest.raises(RuntimeError, match="released"):
        t.check()


@pytest.mark.parametrize("d,nq", [(64, 300), (128, 300), (128, 60), (256, 700)])
def test_attention_many_rows_of_any_stride(ss, d, nq):
    k = torch.randn((1000 + nq, 2, d), generator=_gen(1), device="cuda")
    pool, row = _filled(ss, k, torch.randn_like(k))
    qkv = torch.randn((nq, 12, d), generator=_gen(2), device="cuda").half()
    q = qkv[:, :8]
    odd = torch.zeros(nq * 8 * d + 1, dtype=torch.float16, device="cuda")[1:].view(nq, 8, d)
    odd.copy_(q)  # 2-byte aligned
    args = pool, row[None], _i32([1000 + nq]), _i32([0, nq]), 0.1
    o, lse = ss.int4_attention(q.contiguous(), *args, max_q=nq, return_lse=True)
    for x in (q, odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        o2, lse2 = ss.int4_attention(x, *args, max_q=nq, return_lse=True)
        assert torch.equal(o2, o) and torch.equal(lse2, lse)
    kr, vr = ss.int4_fetch(torch.arange(1000 + nq, device="cuda"), pool, d)
    want, wl, pv, mag = R.attention(q, kr, vr, 1000 + nq, 0.1)
    u = 2.0 ** -11
    assert ((o.double() - want).abs() <= u * want.abs() + (4 * u + 2 * u * mag[..., None]) * pv + 1e-7).all()
    assert ((lse.double() - wl).abs() <= u * mag + 1e-5 * (1 + wl.abs())).all()
