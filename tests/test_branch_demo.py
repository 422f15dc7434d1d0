"""The branching operators together, as a serving loop uses them: beam search
and drafted trees against the same model without a cache, and a beam step as
a captured graph."""
import pytest

pytestmark = pytest.mark.gpu


def plain_hidden(torch, model, tokens):
    """The model on whole sequences [S][n], no cache: fp64."""
    S, n = tokens.shape
    H, KV, D = model.heads, model.kv_heads, model.head_dim
    angle = torch.arange(n, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    turn = torch.polar(torch.ones_like(angle), angle).cuda()[None, :, None]
    x = model.embedding[tokens].double()
    norm = lambda y: y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-5)  # noqa: E731
    for qkv_weight, out_weight in model.layers:
        qkv = (norm(x) @ qkv_weight.double()).reshape(S, n, H + 2 * KV, D)
        qk = torch.view_as_real(torch.view_as_complex(qkv[:, :, :H + KV].reshape(S, n, H + KV, D // 2, 2).contiguous()) * turn)
        q, k = qk.reshape(S, n, H + KV, D).split([H, KV], 2)
        k, v = (y.repeat_interleave(H // KV, 2) for y in (k, qkv[:, :, H + KV:]))
        z = torch.einsum("sihd,sjhd->shij", q, k) / D ** 0.5
        z = z.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -torch.inf)
        x = x + torch.einsum("shij,sjhd->sihd", z.softmax(-1), v).reshape(S, n, H * D) @ out_weight.double()
    return norm(x) @ model.head.double()


def plain_beams(torch, model, prompt, steps, beams, eos):
    """Beam search by the definition, each step from scratch."""
    kept = [(0.0, [], False)]
    for _ in range(steps):
        found = []
        live = [i for i, k in enumerate(kept) if not k[2]]
        if live:
            logits = plain_hidden(torch, model, torch.tensor([prompt + kept[i][1] for i in live], device="cuda"))[:, -1]
            logp = dict(zip(live, torch.log_softmax(logits, -1)))
        for i, (score, path, done) in enumerate(kept):
            if done:
                found.append((-score, i, eos, path, True))
                continue
            best = torch.topk(logp[i], beams)
            found += [(-(score + v), i, t, path + [t], t == eos) for v, t in zip(best.values.tolist(), best.indices.tolist())]
        found.sort(key=lambda c: c[:3])
        kept = [(-f[0], f[3], f[4]) for f in found[:beams]]
    return [(k[0], k[1]) for k in kept]


@pytest.mark.parametrize("beams,page_size,eos", [(1, 16, 3), (4, 4, 5), (5, 16, 0)])
def test_beam_search_matches_the_model_without_a_cache(beams, page_size, eos):
    torch = pytest.importorskip("torch")
    from nutllm_b200 import branch_demo as demo
    model = demo.Model(vocab=60, layers=2, heads=4, kv_heads=2, head_dim=32, seed=3)
    prompts = [[5, 9, 31, 7, 22, 50, 1, 2, 40], [11], list(range(17))]
    got = demo.beam_search(model, prompts, 9, beams, eos, dtype=torch.float32, page_size=page_size)
    for prompt, best in zip(prompts, got):
        # Paths may tie: behind one token, any path of the same two tokens attends to the same two values.  So the
        # scores are compared, and each path is scored by the definition.
        want = plain_beams(torch, model, prompt, 9, beams, eos)
        for (score, path), (b, other) in zip(best, want):
            said = torch.log_softmax(plain_hidden(torch, model, torch.tensor([prompt + path], device="cuda"))[0], -1)
            own = sum(float(said[len(prompt) - 1 + i, t]) for i, t in enumerate(path))
            assert len(path) == 9 or path[-1] == eos
            assert abs(score - own) <= 1e-4 * (1 + abs(own)) and abs(score - b) <= 1e-4 * (1 + abs(b))
            near = [w for w, _ in want if abs(w - b) <= 1e-4 * (1 + abs(b))]
            assert path == other or len(near) > 1 or abs(want[-1][0] - b) <= 1e-4 * (1 + abs(b))
        assert len({tuple(path) for _, path in best}) == beams


@pytest.mark.parametrize("widths,page_size", [([1], 16), ([3, 2], 4), ([4, 2, 1, 1], 16), ([40], 8)])
def test_drafted_trees_give_the_greedy_tokens(widths, page_size):
    torch = pytest.importorskip("torch")
    from nutllm_b200 import branch_demo as demo
    model = demo.Model(vocab=60, layers=2, heads=4, kv_heads=2, head_dim=32, seed=4)
    prompts = [[5, 9, 31, 7, 22, 50, 1, 2, 40], [11], list(range(17))]
    tokens, passes = demo.tree_greedy(model, prompts, 12, widths, dtype=torch.float32, page_size=page_size)
    plain, most = demo.tree_greedy(model, prompts, 12, [], dtype=torch.float32, page_size=page_size)
    assert tokens == plain and passes <= most
    if widths == [40]:  # of 60 tokens: most of them are drafted
        assert passes < most
    for prompt, path in zip(prompts, plain):
        said = plain_hidden(torch, model, torch.tensor([prompt + path[:-1]], device="cuda"))[0].argmax(-1).tolist()
        assert said[len(prompt) - 1:] == path


def test_a_beam_step_as_a_graph():
    """select, update, copy, append and attention captured once and replayed: the steps of the loop without it."""
    torch = pytest.importorskip("torch")
    import nutllm_b200 as nb
    from nutllm_b200 import branch_demo as demo
    beams, requests, steps = 3, 2, 14
    S = beams * requests
    model = demo.Model(vocab=80, layers=2, heads=4, kv_heads=2, head_dim=32, seed=5)
    prompts = [[5, 9, 31], [11, 12, 13, 14, 15, 16, 17]]

    def start():
        s = demo.BranchSession(model, S, 80, 8, 8, page_size=4, dtype=torch.bfloat16, max_positions=64)
        x = s.prompts([prompts[i // beams] if i % beams == 0 else [] for i in range(S)])
        logits = torch.zeros(S, 80, device="cuda")
        logits[::beams] = model.logits(x[torch.tensor([2, 9], device="cuda")])
        scores = torch.full((requests, beams), -torch.inf, device="cuda")
        scores[:, 0] = 0.0
        state = dict(logits=logits, scores=scores, rows=torch.zeros(S, dtype=torch.int32, device="cuda"),
                     tokens=torch.zeros(S, dtype=torch.int32, device="cuda"), one=torch.ones(S, dtype=torch.int32, device="cuda"),
                     starts=torch.arange(S + 1, dtype=torch.int32, device="cuda"))
        return s, nb.BeamSearch(requests, beams, 80, beams), state

    def step(s, search, t):
        search.select(t["logits"].data_ptr(), t["scores"].data_ptr(), t["scores"].data_ptr(), t["rows"].data_ptr(),
                      t["tokens"].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        s.update(parent=t["rows"], add=t["one"])
        t["logits"].copy_(model.logits(s.forward(t["tokens"], t["starts"], 1)))

    def run(graphed):
        s, search, t = start()
        seen, graph = [], None
        for i in range(steps):
            if graphed and i == 2:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step(s, search, t)
            if graph is not None:
                graph.replay()
            else:
                step(s, search, t)
            seen.append((t["rows"].tolist(), t["tokens"].tolist(), t["scores"].clone(), s.lengths.tolist()))
        s.check()
        assert sorted(s.free[:int(s.count)].tolist()) == [p for p, n in enumerate(s.refs.tolist()) if n == 0]
        return seen

    for a, b in zip(run(False), run(True)):
        assert a[0] == b[0] and a[1] == b[1] and a[3] == b[3] and torch.equal(a[2], b[2])


def test_demo_runs():
    import subprocess
    import sys
    out = subprocess.run([sys.executable, "-m", "nutllm_b200.branch_demo", "--prompts", "40,5", "--steps", "6", "--layers", "2",
                          "--vocab", "500"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    assert "beam search" in out.stdout and "2 of 2 sequences" in out.stdout
