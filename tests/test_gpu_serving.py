"""The serving loop over paged 4-bit caches: every attention of every step
equals softmax attention over what the pages hold, the scored prompts equal
token_logprobs of the model's own logits, and pages come back."""

import math

import pytest
import torch

import paged_ref as R

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def model(cuda_ok):
    from sunshape_mlx_b200.harness import Decoder, DecoderConfig

    return Decoder(DecoderConfig(n_layers=2, hidden=512, n_heads=4, n_kv_heads=2, ffn=1024, vocab=1003), seed=3)


def test_serving_steps_attend_over_their_pages(model, monkeypatch):
    from sunshape_mlx_b200.paged import Int4PagedKVCache
    from sunshape_mlx_b200.serving import PagedServer

    seen = []
    real = Int4PagedKVCache.attend

    def spy(self, q, plan, scale, **kw):
        out, lse = real(self, q, plan, scale, return_lse=True, **kw)
        t = self.tables
        cu, lens = plan.cu_q.tolist(), plan.seq_lens.tolist()
        for b, n in enumerate(lens):
            x = q[cu[b]:cu[b + 1]]
            if not x.shape[0]:
                continue
            pos = torch.arange(n, device=q.device)
            slots = t.block_table[b, pos // t.page_size].long() * t.page_size + pos % t.page_size
            k, v = self.fetch(slots)
            want, wl, pv, mag = R.attention(x, k, v, n, scale)
            u = 2.0 ** -11  # fp16 steps inside, bf16 outside
            bound = 2.0 ** -8 * want.abs() + (4 * u + 2 * u * mag[..., None]) * pv + 1e-7
            assert ((out[cu[b]:cu[b + 1]].double() - want).abs() <= bound).all()
            seen.append(x.shape[0])
        return out

    monkeypatch.setattr(Int4PagedKVCache, "attend", spy)
    g = torch.Generator().manual_seed(1)
    server = PagedServer(model, n_pages=20, page_size=16, max_requests=5, max_tokens=160, chunk=48, top_k=4)
    prompts = [torch.randint(1003, (n,), generator=g) for n in (100, 1, 33, 48)]
    reqs, scored = server.start(prompts)
    server.step()
    assert reqs == [0, 1, 2, 3] and server.lens == {0: 101, 1: 2, 2: 34, 3: 49}
    assert [s.logprobs.shape[0] for s in scored] == [99, 0, 32, 47]
    server.stop([0, 2])
    more, _ = server.start([torch.randint(1003, (120,), generator=g)])
    assert more == [0]
    for _ in range(3):
        ids, lp = server.step()
        assert ids.shape == (3,) and lp.top_ids.shape == (3, 4)
        # the greedy token is the best alternative
        assert torch.equal(lp.logprobs, lp.top_logprobs[:, 0])
    server.tables.check()
    assert {1, 33, 48} <= set(seen)
    held = sum(-(-n // 16) for n in server.lens.values())
    assert server.tables.n_free.item() == 20 - held
    with pytest.raises(RuntimeError, match="free pages"):
        server.start([torch.randint(1003, (150,), generator=g), torch.randint(1003, (150,), generator=g)])
    assert sorted(server.lens) == [0, 1, 3]
    server.stop([0, 1, 3])
    assert server.tables.n_free.item() == 20
    with pytest.raises(RuntimeError, match="no request"):
        server.step()


def test_scored_prompt_is_the_models_own(model):
    """In parts or whole, beside other requests or alone, a prompt gets the same scores up to bf16 steps of the model."""
    from sunshape_mlx_b200.serving import PagedServer

    g = torch.Generator().manual_seed(2)
    p = torch.randint(1003, (70,), generator=g)
    alone = PagedServer(model, n_pages=8, page_size=16, max_requests=1, max_tokens=128, chunk=128)
    _, (a,) = alone.start([p])
    both = PagedServer(model, n_pages=40, page_size=32, max_requests=3, max_tokens=128, chunk=19)
    _, (_, b) = both.start([torch.randint(1003, (90,), generator=g), p])
    # dense attention over the uncompressed keys: what 4 bits change is small beside the entropy
    dense = torch.stack([model.forward(p[None, :i + 1].cuda(), None, 0)[0] for i in range(1, 69, 9)])
    lp, _, _, _ = R.logprobs(dense, p[2:70:9].cuda(), 0)
    assert (a.logprobs - b.logprobs).abs().max() < 0.15
    assert (a.logprobs[1:69:9].double() - lp).abs().max() < 0.5 and math.log(1003) * 0.5 < a.entropy.mean() < math.log(1003)


def test_example_runs(cuda_ok, capsys):
    from sunshape_mlx_b200 import serving

    serving.main()
    out = capsys.readouterr().out
    assert "request 3: 1200 tokens" in out and "pages free" in out


def test_refusals(model):
    from sunshape_mlx_b200.serving import PagedServer

    s = PagedServer(model, n_pages=8, page_size=16, max_requests=1, max_tokens=32)
    for bad, err in (([torch.zeros(0, dtype=torch.int64)], ValueError), ([torch.zeros((1, 3), dtype=torch.int64)], ValueError),
                     ([torch.zeros(33, dtype=torch.int64)], ValueError), ([torch.zeros(3, dtype=torch.int64)] * 2, RuntimeError)):
        with pytest.raises(err):
            s.start(bad)
        assert not s.lens and s.tables.n_free.item() == 8
