"""The serving loop of nutllm_b200.paged_demo against the same layers on a
contiguous cache in 64 bits, and its bookkeeping of pages."""
import pytest

import nutllm_b200 as nb  # noqa: F401

HEADS, KV, D, LAYERS = 8, 2, 32, 2


def plain(torch, weights, prompts, steps):
    """decode() with whole caches in 64 bits, one sequence at a time."""
    def norm(x):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)

    got = []
    for p in prompts:
        x, caches, rows = p.double().cpu(), [([], []) for _ in weights], []
        h = None
        inputs = [x[i] for i in range(len(x))]
        for t in range(len(inputs) + steps):
            y = inputs[t] if t < len(inputs) else h
            freq = 10000.0 ** (-torch.arange(0, D, 2).double() / D)
            turn = torch.polar(torch.ones(D // 2).double(), t * freq)

            def rotate(v):
                return torch.view_as_real(torch.view_as_complex(v.reshape(-1, D // 2, 2).contiguous()) * turn).reshape(-1, D)

            for (wq, wo), (ks, vs) in zip(weights, caches):
                qkv = (norm(y) @ wq.double().cpu()).reshape(-1, D)
                ks.append(rotate(qkv[HEADS:HEADS + KV]))
                vs.append(qkv[HEADS + KV:])
                k, v = torch.stack(ks, 1), torch.stack(vs, 1)  # [KV][t][D]
                q = rotate(qkv[:HEADS]).reshape(KV, HEADS // KV, D)
                w = torch.softmax(q @ k.transpose(1, 2) / D ** 0.5, -1)
                y = y + (w @ v).reshape(-1) @ wo.double().cpu()
            h = norm(y)
            if t >= len(inputs):
                rows.append(h)
        got.append(torch.stack(rows))
    return torch.stack(got, 1)


def setup(torch, lens):
    from nutllm_b200 import paged_demo as demo
    weights = demo.random_weights(LAYERS, HEADS, KV, D)
    g = torch.Generator(device="cuda").manual_seed(3)
    return demo, weights, [torch.randn(n, HEADS * D, generator=g, device="cuda") for n in lens]


@pytest.mark.gpu
@pytest.mark.parametrize("more", [{}, dict(budget=64, sinks=2, recent=8), dict(sparse_pages=8)], ids=["dense", "budget", "sparse"])
def test_decode_matches_whole_caches(gpu, more):
    """With a budget and page count that nothing outgrows, all three ways are the exact attention.  The fp32 loop differs
    from 64 bits by rounding only: 30 tokens of 2 layers stay within 1e-4 (2^-24 times some hundred operations and a
    growth of less than 10 a layer)."""
    import torch
    lens, steps = [19, 1, 33], 10
    demo, weights, prompts = setup(torch, lens)
    session = demo.PagedSession(3, LAYERS, HEADS, KV, D, pages=16, max_pages=8, dtype=torch.float32, **more)
    got = demo.decode(session, weights, prompts, steps)
    session.check()
    want = plain(torch, weights, prompts, steps)
    assert float((got.double().cpu() - want).abs().max()) < 1e-4
    assert session.length == [29, 11, 43]


@pytest.mark.gpu
def test_trimmed_sequences_give_their_pages_back(gpu):
    import torch
    lens, steps, budget = [100, 20, 70], 30, 48
    demo, weights, prompts = setup(torch, lens)
    session = demo.PagedSession(3, LAYERS, HEADS, KV, D, pages=20, max_pages=8, budget=budget, sinks=2, recent=8)
    got = demo.decode(session, weights, prompts, steps)
    session.check()
    assert bool(torch.isfinite(got).all())
    assert all(n < budget + session.page_size for n in session.length)
    held = [p for pages in session.owned for p in pages]
    assert sorted(held + session.free) == list(range(20))
    assert [len(p) for p in session.owned] == [-(-n // 16) for n in session.length]
    for t in session.layers:
        for s, n in enumerate(session.length):
            for h in range(KV):
                kept = t["positions"][s, h, :n]
                assert int(kept.unique().numel()) == n
                # the sinks and the newest tokens are still there
                assert {0, 1, *range(session.seen[s] - 8, session.seen[s])} <= set(kept.tolist())
            assert bool((t["positions"][s, :, n:] == -1).all()) and not bool(t["weights"][s, :, n:].any())
    with pytest.raises(RuntimeError, match="out of pages"):
        session.extend([1000, 0, 0])
