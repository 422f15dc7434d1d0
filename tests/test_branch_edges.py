"""Branching decode (test_branch.py) where its definitions and its kernels'
short cuts could part: logits and scores that are no numbers or tie, values
that are none and hardly weigh, logits far from zero and next to it, long sums,
books and caches of several layers, and numbers beyond their fields."""
import math
import random

import numpy as np
import pytest

import nutllm_b200 as nb
from test_branch import PAIRS, UNIT, Book, Tree, paths, plain_beams, run_beams, same_beams
from test_paged import EPS, KINDS, Pool, dtypes

gpu = pytest.mark.gpu


@pytest.fixture
def torch_cuda():
    return pytest.importorskip("torch")


# ---------------------------------------------------------------------------
# beams


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [3, 40, 1025, 5003])
@pytest.mark.parametrize("n", [3, 33])
@pytest.mark.parametrize("case", ["all", "few left", "few left beside infinity", "-infinity among them", "one beam", "the end"])
def test_beam_select_nan_are_candidates(torch_cuda, kind, V, n, case):
    """NaN counts as -infinity: its token is chosen, the lowest first, where nothing better is left."""
    torch = torch_cuda
    B = 1 if case in ("few left", "few left beside infinity") else 2
    logits = torch.full((B, V), math.nan)
    scores = torch.tensor([[-1.0, -0.5][:B]])
    if case.startswith("few left"):
        logits[0, V // 2], logits[0, V - 1] = 1.0, 2.0
        if case == "few left beside infinity":  # (whatever lane has it has NaN too)
            logits[0, V // 3] = math.inf
    elif case == "-infinity among them":
        logits[0, ::2] = -math.inf
        logits[1, 1::2] = -math.inf
    elif case == "one beam":  # an ended beam beside it: one candidate
        logits[1, :] = 0.5
    elif case == "the end":
        logits[:, :2] = 1.0
    ended = torch.tensor([[0, 1]]) if case == "one beam" else None
    logits = logits.to(dtypes(torch)[kind])
    got = run_beams(torch, logits.cuda(), scores.cuda(), n, ended.to(torch.uint8).cuda() if ended is not None else None,
                    1 if ended is not None else -1)
    same_beams(got, plain_beams(torch, logits, scores, ended, 1 if ended is not None else -1, n))


@gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("low", [-math.inf, math.nan])
@pytest.mark.parametrize("V", [5, 3000, 70000])
def test_beam_select_ties_of_beams_without_a_score(torch_cuda, kind, low, V):
    """All tokens of a beam whose score is -infinity tie, whatever their logits: the lowest ones are chosen."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(8, V, generator=g).to(dtypes(torch)[kind])
    scores = torch.tensor([[-1.0, low, -2.0, low], [low, low, low, low]])
    ended = torch.tensor([[1, 0, 1, 0], [0, 1, 0, 0]])
    got = run_beams(torch, logits.cuda(), scores.cuda(), 12, ended.to(torch.uint8).cuda(), 4)
    same_beams(got, plain_beams(torch, logits, scores, ended, 4, 12))


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [31, 1023, 5000])
@pytest.mark.parametrize("n", [1, 8, 31, 64])
def test_beam_select_equal_logits_around_zero(torch_cuda, kind, V, n):
    """+0 and -0 are equal logits, next to the least numbers of either sign and to a few levels."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(V + n)
    dt = dtypes(torch)[kind]
    least = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps  # the least subnormal
    scores = torch.tensor([[-1.0, -1.0], [-3.0, -0.25]])
    for levels in ([0.0, -0.0], [-0.0, -least], [0.0, -0.0, -least, least], [-1.0, -0.0, 0.0], [-1.0, -2.0, -0.0]):
        logits = torch.tensor(levels, dtype=dt)[torch.randint(len(levels), (4, V), generator=g)]
        got, want = run_beams(torch, logits.cuda(), scores.cuda(), n), plain_beams(torch, logits, scores, None, -1, n)
        if least not in (abs(v) for v in levels):
            same_beams(got, want)
            continue
        # What is less than 2^-100 rounds to nothing beside a score of 1/4 or more, so that all tokens of a beam tie in 64
        # bits, and the interface leaves open which go first; fp16's 2^-24 is less than what separates two beams' sums
        # (40 roundings of 2^-24).  So: different candidates, with the scores as defined
        for r, row in enumerate(want):
            chosen = [c for c in zip(got[1][r].tolist(), got[2][r].tolist()) if c[0] >= 0]
            assert len(set(chosen)) == len(chosen) and all(0 <= t < V for _, t in chosen)
            for x, c in zip(got[0][r].tolist(), row):
                assert x == c[0] or abs(x - c[0]) <= 40 * EPS + abs(c[0]) * EPS


# ---------------------------------------------------------------------------
# tree attention


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("length,low", [(70, "first"), (70, "last"), (5000, "first"), (5000, "last")])
def test_tree_values_that_are_no_numbers_and_hardly_weigh(torch_cuda, cache, rows, D, length, low):
    """An infinity or NaN among the values that a row sees shows in that dimension, also where its slot's weight, beside
    others 256 nats greater, is 0 in any format; in one block, and in a part of several blocks that weighs nothing."""
    torch = torch_cuda
    n, H, KV = 9, 4, 2
    pool = Pool(torch, [length], H, KV, D, 16, cache, seed=6)
    k = torch.zeros(KV, length, D)
    few = length // 2 if low == "first" else length - length // 2
    if low == "first":
        k[:, :few, 0] = -256.0
        odd = few // 4  # in the prefix
    else:
        k[:, few:, 0] = -256.0
        odd = length - n + 4  # a drafted token
    v = pool.v[0].float().clone()
    v[:, odd, 3], v[:, odd, 5], v[:, odd, 7] = math.nan, math.inf, -math.inf
    dt = dtypes(torch)[cache]
    pool.put(0, k.to(dt), v.to(dt), 0)
    pool.k[0], pool.v[0] = k.to(dt), v.to(dt)
    pool.cache.reserve_tree(n)
    seen = [[j for j in range(i + 1) if j != 4 or i % 2] for i in range(n)]
    tree = Tree(torch, pool, [n], rows, masks=[seen])
    tree.q_cpu.zero_()
    tree.q_cpu[:, :, 0] = 1.0
    tree.q.copy_(tree.q_cpu.reshape(n, -1))
    tree.run(scale=1.0)
    pool.cache.check()
    out = tree.out.reshape(n, H, D).float().cpu()
    rest = [d for d in range(D) if d not in (3, 5, 7)]
    for i in range(n):
        shows = low == "first" or 4 in seen[i]
        assert bool(out[i, :, 3].isnan().all()) == shows, i
        assert bool((~out[i][:, [5, 7]].isfinite()).all()) == shows, i
        assert bool(out[i][:, rest].isfinite().all()), i
        if not shows:
            assert bool(out[i].isfinite().all()), i


# ---------------------------------------------------------------------------
# the loops of branch_demo


def test_empty_prompts_are_refused(torch_cuda):
    """Their first token was taken from the row of the prompt before."""
    from nutllm_b200 import branch_demo as demo
    for prompts in ([[]], [[1, 2], []], [[], [3]]):
        with pytest.raises(ValueError, match="empty prompt"):
            demo.beam_search(None, prompts, 4, 2, 0)
        with pytest.raises(ValueError, match="empty prompt"):
            demo.tree_greedy(None, prompts, 4, [2])


# ---------------------------------------------------------------------------
# numbers beyond their fields


def test_numbers_beyond_their_fields_are_refused():
    """ctypes would keep their low 64 bits."""
    book = dict(sequences=4, max_pages=8, n_pages=30, page_size=16)
    for name in book:
        for wrap in (1 << 64, 3 << 64, -1 << 64):
            with pytest.raises(ValueError, match="field"):
                nb.PageBook(16, 16, 16, 16, 16, **(book | {name: book[name] + wrap}))
    for k in range(5):
        for at in ((1 << 64) + 16, (-1 << 64) + 16):
            with pytest.raises(ValueError, match="field"):
                nb.PageBook(*(at if i == k else 16 for i in range(5)), **book)
    cache = dict(sequences=4, max_pages=8, n_pages=30, page_size=16, heads=8, kv_heads=2, head_dim=64, max_rows=0, page_stride=0,
                 head_stride=0, slot_stride=0)
    for name in cache:
        with pytest.raises(ValueError, match="field"):
            nb.PagedCache(16, 16, 16, 16, **(cache | {name: cache[name] + (1 << 64)}))
    for more in (dict(dtype=1 << 32), dict(device=1 << 32)):
        with pytest.raises(ValueError, match="field"):
            nb.PagedCache(16, 16, 16, 16, **cache, **more)
    with pytest.raises(ValueError, match="field"):
        nb.PageBook(16, 16, 16, 16, 16, **book, device=1 << 32)
    for name in ("bounds", "bound_scales"):
        with pytest.raises(ValueError, match="field"):
            nb.PagedCache(16, 16, 16, 16, **cache, **{name: (1 << 64) + 16})
    for name in ("sequences", "beams", "vocab", "n_out"):
        with pytest.raises(ValueError, match="field"):
            nb.BeamSearch(**(dict(sequences=1, beams=1, vocab=10, n_out=1) | {name: (1 << 64) + 1}))


@gpu
def test_row_positions_beyond_an_address_are_refused(torch_cuda):
    torch = torch_cuda
    pool = Pool(torch, [30], 4, 2, 64, 16, "f16")
    x = torch.zeros(1, 256, dtype=torch.float16, device="cuda")
    starts = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    for at in ((1 << 64) + starts.data_ptr(), (-1 << 64) + starts.data_ptr()):
        with pytest.raises(ValueError, match="field"):
            pool.cache.append(0, x.data_ptr(), x.data_ptr(), starts.data_ptr(), 1, 1, dtype=nb.F16, row_position=at)
    pool.cache.check()


# ---------------------------------------------------------------------------
# caches of several layers, and their book


@gpu
def test_compact_of_every_layer_then_the_book(torch_cuda):
    """Layers share table and lengths: each is compacted from the lengths as they were, into an array that the next
    update keeps; in place for the last alone."""
    torch = torch_cuda
    S, M, P, ps, KV, D, n = 3, 8, 40, 4, 2, 64, 7
    lens = [9, 17, 12]
    book = Book(torch, S, M, P, ps)
    book.plain(None, None, [a + n for a in lens])
    book.update(None, None, [a + n for a in lens])
    g = torch.Generator().manual_seed(3)
    layers = [torch.randn(2, P, KV, ps, D, generator=g).half().cuda() for _ in range(3)]
    caches = [nb.PagedCache(x[0].data_ptr(), x[1].data_ptr(), book.dev["table"].data_ptr(), book.dev["lengths"].data_ptr(), sequences=S,
                            max_pages=M, n_pages=P, page_size=ps, heads=4, kv_heads=KV, head_dim=D, dtype=nb.F16) for x in layers]
    lists = [[0, 3, 6], [2], []]
    starts = torch.tensor([0, n, 2 * n, 3 * n], dtype=torch.int32, device="cuda")
    accepted = paths(torch, lists, 4)
    left = torch.zeros(S, dtype=torch.int32, device="cuda")

    def rows(x, s, slots):
        pages = torch.tensor([book.table[s][t // ps] for t in slots], device="cuda").long()
        return x[:, pages, :, torch.tensor([t % ps for t in slots], device="cuda")]

    want = [[rows(x, s, list(range(lens[s])) + [lens[s] + j for j in lists[s]]).clone() for s in range(S)] for x in layers]
    for cache in caches:
        cache.compact(starts.data_ptr(), accepted.data_ptr(), 4, new_lengths=left.data_ptr())
        cache.check()
        assert left.tolist() == [a + len(x) for a, x in zip(lens, lists)]
        assert book.dev["lengths"].tolist() == [a + n for a in lens]
    for x, kept in zip(layers, want):
        for s in range(S):
            assert torch.equal(rows(x, s, range(lens[s] + len(lists[s]))), kept[s])
    # the update gives back the pages behind what is kept
    keep = [a + len(x) for a, x in zip(lens, lists)]
    copies = book.plain(None, keep, [1] * S)
    book.update(None, keep, [1] * S)
    book.same(copies)
    assert book.count == P - sum(book.pages(k + 1) for k in keep)
    book.book.check()


@gpu
@pytest.mark.parametrize("seed", [0, 1, 2, 3])
def test_refused_updates_say_why(torch_cuda, seed):
    """LengthError where the free pages do not suffice, IndexError where a sequence outgrows its table (or both)."""
    torch = torch_cuda
    S, M, P, ps = 9, 6, 30, 4
    book, r, met = Book(torch, S, M, P, ps, seed), random.Random(seed), set()
    for _ in range(40):
        parent = [r.randrange(S) for _ in range(S)] if r.random() < 0.5 else list(range(S))
        keep = [r.randrange(M * ps + 1) for _ in range(S)]
        add = [r.choice([0, 1, 2, 5, 9, 20]) for _ in range(S)]
        outgrown = any(min(w, book.lengths[p]) + a > M * ps for p, w, a in zip(parent, keep, add))
        want = book.plain(parent, keep, add)
        book.update(parent, keep, add)
        book.same(want)
        if want is None:
            met.add(outgrown)
            with pytest.raises(IndexError if outgrown else nb.LengthError):
                book.book.check()
        book.book.check()
    assert met == {False, True}


@gpu
@pytest.mark.parametrize("beams,eos,seed", [(1, 3, 3), (1, 0, 8), (3, 5, 3), (4, 0, 9)])
def test_beam_search_paths(torch_cuda, beams, eos, seed):
    """Paths and not scores alone: equal to those of the search by the definition wherever every choice of it was clear,
    that is, no two neighbours among a step's beams + 1 best within 1e-3 of one another (scores are within 1e-4)."""
    torch = torch_cuda
    from nutllm_b200 import branch_demo as demo
    from test_branch_demo import plain_hidden
    model = demo.Model(vocab=60, layers=2, heads=4, kv_heads=2, head_dim=32, seed=seed)
    prompts = [[5, 9, 31, 7, 22, 50, 1, 2, 40], [11], list(range(17)), [3, 3], [59, 0, 1, 30]]
    got = demo.beam_search(model, prompts, 6, beams, eos, dtype=torch.float32, page_size=4)
    clear = 0
    for prompt, best in zip(prompts, got):
        kept, gap = [(0.0, [], False)], math.inf
        for _ in range(6):
            found = []
            for i, (score, path, done) in enumerate(kept):
                if done:
                    found.append((-score, i, eos, path, True))
                    continue
                logits = plain_hidden(torch, model, torch.tensor([prompt + path], device="cuda"))[0, -1]
                top = torch.topk(torch.log_softmax(logits, -1), beams + 1)
                found += [(-(score + v), i, t, path + [t], t == eos) for v, t in zip(top.values.tolist(), top.indices.tolist())]
            found.sort(key=lambda c: c[:3])
            gap = min([gap] + [b[0] - a[0] for a, b in zip(found[:beams], found[1:])])
            kept = [(-f[0], f[3], f[4]) for f in found[:beams]]
        for (score, _), (b, _, _) in zip(best, kept):
            assert abs(score - b) <= 1e-4 * (1 + abs(b))
        if gap > 1e-3:
            clear += 1
            assert [path for _, path in best] == [k[1] for k in kept]
    assert clear >= 1


@gpu
@pytest.mark.parametrize("cache,rows", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("D", [8, 16, 24, 72, 120, 136])
def test_tree_heads_of_odd_widths(torch_cuda, D, cache, rows):
    torch = torch_cuda
    pool = Pool(torch, [150, 31, 70], 6, 2, D, 12, cache, seed=D)
    pool.cache.reserve_tree(31)
    tree = Tree(torch, pool, [9, 31, 1], rows, seed=D)
    tree.run()
    pool.cache.check()
    tree.check()


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("length", [40, 3000])
@pytest.mark.parametrize("scale", [2.0 ** 27, 3e10, -7e15, 1e30])
def test_tree_logits_beyond_every_difference(torch_cuda, cache, rows, D, length, scale):
    """Logits so great that their last places are many units: the greatest ones, a few equal ones across the cache, share
    the output, and the others (1/64 of the greatest below it or more) have no part."""
    torch = torch_cuda
    dt = dtypes(torch)[cache]
    pool = Pool(torch, [length], 2, 1, D, 16, cache, seed=18)
    k = torch.zeros(1, length, D)
    k[0, :, 0] = 1.0 + torch.arange(length).remainder(32) / 64
    best = [3, length // 2, length - 7]
    k[0, best, 0] = 1.703125
    k = k.to(dt) * (1.0 if scale > 0 else -1.0)
    pool.put(0, k, pool.v[0], 0)
    pool.k[0] = k
    pool.cache.reserve_tree(4)
    tree = Tree(torch, pool, [4], rows, masks=[[list(range(i + 1)) for i in range(4)]])
    tree.q_cpu.zero_()
    tree.q_cpu[:, :, 0] = torch.tensor([1.37, 0.8125]).to(tree.q_cpu.dtype)
    tree.q.copy_(tree.q_cpu.reshape(4, -1))
    tree.run(scale=scale)
    pool.cache.check()
    out, lse = tree.out.reshape(4, 2, D).cpu().double(), tree.lse.cpu().double()
    v = pool.v[0][0][best].double()
    half = 0.0 if rows == "f32" else torch.finfo(dtypes(torch)[rows]).eps / 2
    # three equal weights, each within 2^-24 (fp32), 2^-11 (fp16) or 2^-8 (bf16) of itself; a division; the output's type
    tol = v.abs().mean(0) * (16 * EPS + 2 * UNIT[rows] + half) + 2.0 ** -25
    assert bool(((out - v.mean(0)).abs() <= tol).all())
    top = abs(float(np.float32(scale))) * 1.703125 * tree.q_cpu[:, :, 0].double()
    assert bool(((lse - top - math.log(3)).abs() <= 8 * EPS * top).all())


@gpu
@pytest.mark.parametrize("cache", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("q,scale", [(2e-38, 1e-9), (3e-38, -1e-30), (1e-30, 1e-38), (1.0, 1e-42)])
def test_tree_logits_next_to_nothing(torch_cuda, cache, q, scale):
    """Queries and scales whose product no float holds: every slot that is seen weighs the same."""
    torch = torch_cuda
    pool = Pool(torch, [90], 2, 1, 64, 16, cache, seed=19)
    pool.cache.reserve_tree(5)
    tree = Tree(torch, pool, [5], "f32")
    tree.q_cpu.mul_(q)
    tree.q.copy_(tree.q_cpu.reshape(5, -1))
    tree.run(scale=scale)
    pool.cache.check()
    tree.check(scale=scale)


@gpu
@pytest.mark.parametrize("cache", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [64, 128])
def test_tree_long_sums_have_no_drift(torch_cuda, cache, D):
    """fp32 rows, positive values, and over a hundred tiles to a block: rounding to nearest leaves errors of either sign, a
    sum that cuts off what it cannot hold is short by up to 2^-23 of itself every time.  Within a tile of 64 slots that
    happens 4 times for each of 3 terms of the weights; were it the whole way, a thousand times.  (Errors of the weights
    have either sign, and are in numerator and denominator.)"""
    torch = torch_cuda
    S, KV, L, ps, n = 10, 16, 16000, 16, 3
    dt, pages = dtypes(torch)[cache], S * (L // ps)
    g = torch.Generator(device="cuda").manual_seed(20)
    keys = torch.randn(pages, KV, ps, D, generator=g, device="cuda").to(dt)
    values = (1 + torch.rand(pages, KV, ps, D, generator=g, device="cuda")).to(dt)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").reshape(S, L // ps)
    lengths = torch.full((S,), L, dtype=torch.int32, device="cuda")
    pool = nb.PagedCache(keys.data_ptr(), values.data_ptr(), table.data_ptr(), lengths.data_ptr(), sequences=S, max_pages=L // ps,
                         n_pages=pages, page_size=ps, heads=KV, kv_heads=KV, head_dim=D, dtype=KINDS[cache])
    pool.reserve_tree(n)
    q = torch.randn(S * n, KV * D, generator=g, device="cuda")
    out = torch.empty_like(q)
    starts = torch.arange(S + 1, dtype=torch.int32, device="cuda") * n
    mask = torch.full((S * n, 1), 7, dtype=torch.int32, device="cuda")
    pool.tree_attention(q.data_ptr(), out.data_ptr(), starts.data_ptr(), mask.data_ptr(), S * n, n, 1, scale=0.125)
    pool.check()
    errors = []
    for s in range(S):
        k, v = (x[s * (L // ps):(s + 1) * (L // ps)].transpose(1, 2).reshape(L, KV, D).double() for x in (keys, values))
        z = 0.125 * torch.einsum("ihd,thd->iht", q[s * n:(s + 1) * n].reshape(n, KV, D).double(), k)
        want = torch.einsum("iht,thd->ihd", torch.softmax(z, -1), v)
        errors.append(out[s * n:(s + 1) * n].reshape(n, KV, D).double() / want - 1)
    assert abs(float(torch.stack(errors).mean())) <= 12 * 2.0 ** -23


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("length", [3, 15, 60, 2500])
def test_tree_lse_of_small_logits(torch_cuda, cache, rows, length):
    """Logits next to 0: the log-sum-exp is the logarithm of a count, to a few parts of its own last place."""
    torch = torch_cuda
    n = min(length, 28)
    pool = Pool(torch, [length], 8, 2, 40, 16, cache, seed=length)
    pool.cache.reserve_tree(n)
    tree = Tree(torch, pool, [n], rows, masks=[[list(range(i + 1)) for i in range(n)]])
    tree.run(scale=2.0 ** -20)
    pool.cache.check()
    # |logits| <= 2^-20 sqrt(40) 5^2 or so, known to (40 + 8) roundings; the sum rounded for every slot, a logarithm, a product
    for i in range(n):
        m = length - n + i + 1
        z = 2.0 ** -20 * torch.einsum("hgd,htd->hgt", tree.q_cpu[i].double().reshape(2, 4, 40), pool.k[0][:, :m].double())
        want = torch.logsumexp(z, -1).reshape(8)
        err = (tree.lse[i].cpu().double() - want).abs()
        tol = 48 * EPS * z.abs().amax(-1).reshape(8) + (4 + 2 * math.sqrt(m)) * EPS + 4 * EPS * want.abs()
        assert bool((err <= tol).all()), (i, float(err.max()))


@gpu
@pytest.mark.parametrize("cache,rows", [p for p in PAIRS if p[0] != "f32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("length", [40, 3000])
def test_tree_values_near_the_greatest(torch_cuda, cache, rows, D, length):
    """A mean of values near a 16-bit type's greatest is one of them: no sum on the way passes fp32's range."""
    torch = torch_cuda
    dt = dtypes(torch)[cache]
    pool = Pool(torch, [length], 4, 2, D, 16, cache, seed=1)
    v = torch.full((2, length, D), 0.9 * torch.finfo(dt).max).to(dt)
    v[:, :, 1::2] *= -1
    pool.put(0, pool.k[0], v, 0)
    pool.cache.reserve_tree(3)
    tree = Tree(torch, pool, [3], rows)
    tree.run()
    pool.cache.check()
    # weights and their sum as in the other tests, relative to the one value that there is
    tol = (2 * length + 64) * EPS + UNIT[rows] + (0.0 if rows == "f32" else torch.finfo(dt).eps / 2)
    error = tree.out.reshape(3, 2, 2, D).double().cpu() / v[None, :, None, 0].double() - 1
    assert bool((error.abs() <= tol).all())
