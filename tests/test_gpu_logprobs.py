"""token_logprobs against 64 bits.

Tolerance: a logit's distance y to the row's largest is exact to 2^-24 |y|, an
exponential to 2^-22, and a sum of n terms kept by a thread of at most 600
terms to 600 * 2^-24 relatively: 4e-5 covers them in log units; the entropy
weights the same errors by the distances, up to the entropy itself. Ids are
equal."""

import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ss(cuda_ok):
    import sunshape_mlx_b200 as ss

    return ss


def _check(ss, x, t, top):
    r = ss.token_logprobs(x, t, top_k=top)
    lp, h, ids, tl = R.logprobs(x, t, top)
    assert torch.equal(r.top_ids, ids)
    for got, want in ((r.logprobs, lp), (r.entropy, h), (r.top_logprobs, tl)):
        got = got.double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got == -math.inf, want == -math.inf)
        fin = torch.isfinite(want)
        assert ((got - want)[fin].abs() <= 4e-5 * (1 + h.nan_to_num(0).max()) + 2.0 ** -22 * want[fin].abs()).all()
    again = ss.token_logprobs(x, t, top_k=top)
    for a, b in zip(r, again):
        assert torch.equal(a.nan_to_num(7), b.nan_to_num(7))
    return r


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,vocab,top", [(1, 1, 1), (1, 1, 0), (3, 2, 5), (5, 31, 32), (2, 1000, 20), (7, 4097, 8), (1, 50257, 20),
                                         (300, 33, 4), (1, 128256, 32), (65, 128256, 5), (40, 50257, 32), (700, 2000, 1), (3, 262144, 8)])
def test_logprobs(ss, n, vocab, top, dtype):
    g = torch.Generator(device="cuda").manual_seed(n + vocab)
    x = (torch.randn((n, vocab), generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(vocab, (n,), generator=g, device="cuda")
    _check(ss, x, t, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [97, 5000, 70001])
def test_orders_and_ties(ss, vocab, dtype):
    i = torch.arange(vocab, device="cuda")
    rows = [torch.zeros(vocab, device="cuda"), (i // 7).float() % 5, i.float() % 200, -(i.float() % 200), (i == vocab - 1).float() * 3,
            torch.where(i % 512 == 3, 9.0, 0.0), torch.where(i < 40, 5.0, -1.0), torch.where(i >= vocab - 40, 5.0, -1.0),
            torch.where(i % 512 == 5, 5.0 + (i % 4096) / 1024.0, 0.0), i.float() / vocab * 8, -i.float() / vocab * 8]
    x = torch.stack(rows).to(dtype)
    t = torch.arange(len(rows), device="cuda") * 3
    for top in (1, 20, 32):
        _check(ss, x, t, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [61, 128256])
def test_masked_rows_and_special_values(ss, vocab, dtype):
    low = torch.finfo(dtype).min
    inf = math.inf
    x = torch.randn((12, vocab), generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
    x[0] = -inf                       # nothing is possible
    x[1] = -inf
    x[1, 50] = 2.0                    # one token is
    x[2, ::2] = -inf
    x[3] = low                        # masked by the type's lowest value: uniform
    x[4, 3:] = low
    x[5, 7] = math.nan
    x[6, vocab - 1] = inf
    x[7, :40] = -inf
    x[8] = -inf
    x[8, [5, 9, 44]] = torch.tensor([1.0, 3.0, 3.0], device="cuda").to(dtype)
    x[9] = x[9] * 0 - 0.0
    x[9, ::3] = 0.0                   # +0 and -0 are equal
    x[10] = torch.finfo(dtype).max
    x[11, 0] = math.nan
    x[11, 1] = inf
    t = torch.tensor([0, 50, 1, 2, 0, 7, 3, 5, 9, -1, vocab, 3], device="cuda")
    for top in (0, 5, 32):
        r = _check(ss, x, t, top)
    assert r.logprobs[9] == 0 and r.logprobs[10].isnan() and r.entropy[0] == 0 and r.entropy[1] == 0


def test_strides_alignment_and_stream(ss):
    g = torch.Generator(device="cuda").manual_seed(2)
    big = torch.randn((6, 3, 1009), generator=g, device="cuda")
    t = torch.arange(6, device="cuda") * 100
    for dt in (torch.float32, torch.float16, torch.bfloat16):
        x = big.to(dt)[:, 1, 1:1004]  # rows start anywhere
        want = ss.token_logprobs(x.contiguous(), t, top_k=7)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = ss.token_logprobs(x, t, top_k=7)
        s.synchronize()
        assert torch.equal(got.top_ids, want.top_ids)
        _check(ss, x, t, 7)
    e = torch.empty((0, 10), device="cuda")
    r = ss.token_logprobs(e, torch.empty(0, dtype=torch.int64, device="cuda"), top_k=3)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 3)


def test_one_row_repeated(ss):
    # rows of stride 0: every row gives what one row gives
    x = torch.randn((1, 5000), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda").half()
    t = torch.full((9,), 77, device="cuda")
    r = ss.token_logprobs(x.expand(9, 5000), t, top_k=4)
    one = ss.token_logprobs(x, t[:1], top_k=4)
    for a, b in zip(r, one):
        assert torch.equal(a, b.expand_as(a))


def test_refusals(ss):
    x, t = torch.zeros((3, 8), device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in [(x.cpu(), t), (x[0], t), (x, t.int()), (x, t[:2]), (x[:, ::2], t), (x[:, :0], t), (x, t.cpu())]:
        with pytest.raises(ValueError):
            ss.token_logprobs(*bad)
    with pytest.raises(TypeError):
        ss.token_logprobs(x.double(), t)
    for k in (-1, 33):
        with pytest.raises(ValueError):
            ss.token_logprobs(x, t, top_k=k)
