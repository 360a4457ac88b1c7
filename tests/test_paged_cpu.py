"""Checks of the paged 4-bit operators that need no GPU: the argument block
mirrors the C struct, bad calls are refused before a device is touched, and
the plan's reference agrees with a second statement of it."""

import ctypes as C
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

import paged_ref as R
from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "sunshape_b200.h")


@pytest.fixture(scope="module")
def lib():
    from sunshape_mlx_b200 import build, _lib as L

    build.build()
    return L.load()


def test_attention_args_layout_matches_header():
    from sunshape_mlx_b200 import _lib as L

    fields = [f for f, _ in L.Int4AttnArgs._fields_]
    prog = "#include <cstdio>\n#include <cstddef>\n#include \"%s\"\nint main(){printf(\"%%zu\", sizeof(ss_int4_attn_args));%s}\n" % (
        HEADER, "".join(f'printf(" %zu", offsetof(ss_int4_attn_args, {f}));' for f in fields))
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "l.cpp"), os.path.join(d, "l")
        open(src, "w").write(prog)
        subprocess.run(["g++", src, "-o", exe], check=True)
        got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(L.Int4AttnArgs)] + [getattr(L.Int4AttnArgs, f).offset for f in fields]


def _args(**kw):
    from sunshape_mlx_b200 import _lib as L

    p = C.c_void_p(4096)  # never read: the calls are refused
    a = L.Int4AttnArgs(p, L.SS_F16, 1024, 128, 1, 8, 2, 128, p, 4, 2 * 16 * 160, 16 * 160, 16, p, 4, 4, p, p, 1, 1, 1.0, 1, 0, p, p, p, 1 << 30)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("bad,word", [(dict(q=None), "null"), (dict(out=None), "null"), (dict(dtype=0), "fp16 or bf16"), (dict(d=96), "head_dim"),
                                      (dict(hq=7), "multiple of the kv heads"), (dict(hkv=0), "kv heads"), (dict(n_pages=0), "empty"),
                                      (dict(page_size=24), "page_size"), (dict(page_stride=8), "multiples of 16"), (dict(window=-1), "window"),
                                      (dict(n_tokens=-1), "empty"), (dict(width=0), "empty")])
def test_attention_refuses_without_a_device(lib, bad, word):
    from sunshape_mlx_b200 import _lib as L

    assert lib.ss_int4_attention(C.byref(_args(**bad)), None) == 1
    assert word in L.last_error()


def test_other_entry_points_refuse_without_a_device(lib):
    from sunshape_mlx_b200 import _lib as L

    p = C.c_void_p(4096)
    assert lib.ss_int4_attention(None, None) == 1
    plan = lambda *, n=1, page=16, width=4, q=p: lib.ss_plan_step(p, q, n, p, 4, width, p, 4, p, page, 8, p, p, p, p, p, p, p, None)  # noqa: E731
    assert plan(n=0) == 1 and "requests" in L.last_error()
    assert plan(n=16385) == 1 and plan(page=20) == 1 and plan(width=5) == 1 and plan(q=None) == 1
    assert lib.ss_release_pages(p, p, 1, p, 4, 4, p, 4, p, 8, p, p, p, None) == 1
    app = lambda *, d=64, dt=0, pool=p, page=16: lib.ss_int4_append(p, p, dt, 64, 64, 64, 64, p, 1, 1, d, pool, 1, 1280, 1280, page, None)  # noqa: E731
    assert app(d=80) == 1 and "head_dim" in L.last_error()
    assert app(dt=3) == 1 and app(pool=None) == 1 and app(page=0) == 1 and app(pool=C.c_void_p(4097)) == 1
    assert lib.ss_int4_fetch(p, -1, 1, 64, p, 1, 1280, 1280, 16, p, p, 0, None) == 1
    assert lib.ss_int4_fetch(p, 1, 1, 64, p, 1, 1280, 1280, 16, C.c_void_p(4100), p, 0, None) == 1
    lp = lambda *, x=p, dt=0, vocab=9, top=1: lib.ss_token_logprobs(x, dt, 1, 9, vocab, p, top, p, p, p, p, None)  # noqa: E731
    assert lp(x=None) == 1 and lp(dt=7) == 1 and lp(vocab=0) == 1 and lp(top=33) == 1 and lp(top=-1) == 1
    # nothing to do is not an error
    assert lib.ss_int4_append(None, None, 0, 0, 0, 0, 0, None, 0, 1, 64, None, 0, 0, 0, 16, None) == 0
    assert lib.ss_token_logprobs(None, 0, 0, 0, 0, None, 0, None, None, None, None, None) == 0


def test_python_layer_refuses_cpu_tensors():
    import sunshape_mlx_b200 as ss

    x = torch.zeros((1, 2, 64))
    pool = torch.zeros((1, 2, 1280), dtype=torch.uint8)
    i = torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ss.int4_append(x, x, i.long(), pool), lambda: ss.int4_fetch(i.long(), pool, 64),
                 lambda: ss.int4_attention(x.half(), pool, i[None], i, torch.zeros(2, dtype=torch.int32), 1.0, max_q=1),
                 lambda: ss.plan_step(i, i, i[None], i, i, page_size=16, n_tokens=1), lambda: ss.token_logprobs(x[0], i.long())):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_plan_reference_hands_out_each_page_once():
    rng = np.random.default_rng(0)
    n, page, pool = 7, 16, 60
    lens, table, free, left = [0] * n, np.full((n, 12), -1, np.int32), np.arange(pool, dtype=np.int32)[::-1].copy(), pool
    for _ in range(12):
        q = rng.integers(0, 25, n).tolist()
        cu, pos, req, slot, lens2, left2, status, table2 = R.plan(lens, q, table, free, left, page, sum(q) + 2)
        if status:
            assert (table2 == table).all() and lens2 == lens and left2 == left
            break
        used = table2[table2 >= 0].tolist()
        assert len(set(used)) == len(used) == pool - left2 and len({s for s in slot if s >= 0}) == sum(q)
        assert cu[-1] == sum(q) and slot[-2:] == [-1, -1]
        lens, table, left = lens2, table2, left2
    else:
        raise AssertionError("the pool never ran out")
