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
