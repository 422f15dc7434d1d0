"""Decoding that branches on the paged KV cache: drafted trees
(nut_paged_append_at, nut_paged_tree_attention, nut_paged_compact), forked
pages (nut_pages_update, nut_paged_copy) and beam selection (nut_beam_select)
against plain implementations.

Whole numbers and moved bytes are compared bit for bit, attention with the
definition in 64 bits within the bounds of test_paged.py (fp32 arithmetic),
where rows of a 16-bit cache's type add what their weights' rounding may
cost: with every weight off by at most u of itself (2^-8 bf16, 2^-11 fp16),
  |d out| <= u sum_t w_t |v_t|;
fp16 weights end at 2^-25 beside a greatest of 2^8 or more: n 2^-33 max |v|.
"""
import ctypes as C
import math
import random

import numpy as np
import pytest

import nutllm_b200 as nb
from test_paged import EPS, KINDS, Pool, dtypes, head_reference

gpu = pytest.mark.gpu
UNIT = {"f32": 0.0, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


# ---------------------------------------------------------------------------
# trees


def ancestors(n, seed, most=6):
    """A random tree's masks, as lists of seen nodes."""
    r, seen = random.Random(seed), []
    for i in range(n):
        parent = i - 1 - r.randrange(min(i + 1, most))
        seen.append((seen[parent] if parent >= 0 else []) + [i])
    return seen


def words_of(torch, masks, words, noise=False):
    """Rows of 32-bit words; noise: bits behind a sequence's last token set too."""
    rows = []
    for seen, n in masks:
        bits = sum(1 << j for j in seen)
        if noise:
            bits |= ~((1 << n) - 1) & ((1 << 32 * words) - 1)
        rows.append([bits >> 32 * w & 0xffffffff for w in range(words)])
    got = np.array(rows, dtype=np.uint64).astype(np.uint32).view(np.int32).reshape(len(rows), words)
    return torch.from_numpy(got.copy()).cuda()


class Tree:
    """Queries, starts and masks of the newest nodes[s] slots of each sequence."""

    def __init__(self, torch, pool, nodes, kind, *, seed=1, masks=None, words=None, q_pad=0, out_pad=0, noise=False, spare=0):
        self.t, self.pool, self.nodes, self.kind = torch, pool, nodes, kind
        g = torch.Generator().manual_seed(seed)
        self.masks = masks or [ancestors(n, seed + 7 * s) for s, n in enumerate(nodes)]
        self.words = words or max(1, -(-max(nodes + [1]) // 32))
        self.rows = sum(nodes)
        flat = [(m, n) for ms, n in zip(self.masks, nodes) for m in ms]
        self.mask = words_of(torch, flat, self.words, noise) if flat else torch.zeros(1, self.words, dtype=torch.int32, device="cuda")
        starts = [0]
        for n in nodes:
            starts.append(starts[-1] + n)
        self.starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
        width = pool.heads * pool.D
        self.q_cpu = (1.5 * torch.randn(self.rows + spare, pool.heads, pool.D, generator=g)).to(dtypes(torch)[kind])
        self.q = torch.zeros(self.rows + spare, width + q_pad, dtype=dtypes(torch)[kind], device="cuda")
        self.q[:, :width] = self.q_cpu.reshape(-1, width).cuda()
        self.out = torch.full((self.rows + spare, width + out_pad), 77.0, dtype=dtypes(torch)[kind], device="cuda")
        self.lse = torch.full((self.rows + spare, pool.heads), 77.0, device="cuda")
        self.q_stride, self.out_stride = width + q_pad, width + out_pad

    def run(self, scale=0.0, rows=None, max_new=None, lse=True, stream=0):
        self.pool.cache.tree_attention(
            self.q.data_ptr(), self.out.data_ptr(), self.starts.data_ptr(), self.mask.data_ptr(),
            self.q.shape[0] if rows is None else rows, max(self.nodes + [1]) if max_new is None else max_new, self.words,
            dtype=KINDS[self.kind], scale=scale, q_stride=self.q_stride, out_stride=self.out_stride,
            lse=self.lse.data_ptr() if lse else 0, stream=stream)

    def check(self, scale=None, only=None):
        torch, p = self.t, self.pool
        scale = 1 / math.sqrt(p.D) if scale is None else scale
        G, r, u = p.heads // p.kv, 0, UNIT[self.kind]
        out = self.out[:, :p.heads * p.D].cpu().reshape(-1, p.heads, p.D)
        lse = self.lse.cpu()
        for s, (length, n) in enumerate(zip(p.lens, self.nodes)):
            for i in range(n):
                at = list(range(length - n)) + [length - n + j for j in self.masks[s][i]]
                for h in range(p.kv):
                    if only is not None and (s, i, h) not in only:
                        continue
                    of = slice(h * G, (h + 1) * G)
                    k, v = p.k[s][h][at], p.v[s][h][at]
                    o, l, w, dz, mass = head_reference(torch, self.q_cpu[r, of], k, v, scale)
                    got, m = out[r, of], len(at)
                    top = float(v.double().abs().max()) if m else 0.0
                    tol = (2 * dz + (2 * m + 64) * EPS) * mass + u * mass + 1e-30
                    if self.kind != "f32":
                        half = torch.finfo(dtypes(torch)[self.kind]).eps / 2
                        tol = tol * (1 + half) + o.abs() * half + (2.0 ** -25 + m * 2.0 ** -33 * top if self.kind == "f16" else 0.0)
                    err = (got.double() - o).abs()
                    assert bool((err <= tol).all()), (s, i, h, float(err.max()), float((err / tol).max()))
                    if m == 0:
                        assert bool((lse[r, of] == -math.inf).all())
                    else:
                        err = (lse[r, of].double() - l).abs()
                        tol = dz[:, 0] + (m + 8) * EPS + 4 * EPS * l.abs()
                        assert bool((err <= tol).all()), (s, i, h, float(err.max()))
                r += 1


TREES = [
    # lens (drafted tokens included), nodes, heads, kv, D, page, order
    ([45], [8], 8, 2, 64, 16, "contiguous"),
    ([1, 9, 300], [1, 9, 5], 4, 4, 32, 8, "contiguous"),  # nothing but a tree; one token
    ([130, 128, 129, 127], [3, 1, 2, 64], 8, 2, 128, 16, "slots first"),
    ([700, 33, 0, 257], [40, 33, 0, 0], 8, 1, 64, 24, "padded"),  # an idle place; a sequence without a draft
    ([515, 66], [65, 33], 4, 2, 80, 5, "contiguous"),  # pages of 5 slots
    ([260, 64], [17, 31], 6, 6, 48, 64, "padded"),
    ([333], [20], 4, 2, 256, 16, "contiguous"),
    ([200, 90], [7, 50], 16, 1, 96, 128, "contiguous"),
    ([600], [300], 4, 2, 64, 16, "contiguous"),  # more drafted tokens than a block of rows
]


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("shape", range(len(TREES)))
def test_tree_attention_against_64_bits(torch_cuda, shape, cache, rows):
    torch = torch_cuda
    lens, nodes, heads, kv, D, ps, order = TREES[shape]
    pool = Pool(torch, lens, heads, kv, D, ps, cache, seed=shape, order=order)
    pool.cache.reserve_tree(max(nodes))
    tree = Tree(torch, pool, nodes, rows, seed=shape + 3, q_pad=8 * (shape % 2), out_pad=8 * (shape % 3), noise=True)
    tree.run()
    pool.cache.check()
    tree.check()
    assert bool((tree.out[:, heads * D:] == 77).all())  # between rows


@pytest.fixture
def torch_cuda():
    return pytest.importorskip("torch")


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_tree_attention_splits_long_caches(torch_cuda, cache, rows):
    """Items that lie in many CTAs, with few and with many rows."""
    torch = torch_cuda
    for nodes, heads, kv in (([3, 2], 2, 1), ([40, 9], 8, 1)):
        pool = Pool(torch, [5000, 2111], heads, kv, 64, 16, cache, seed=5)
        pool.cache.reserve_tree(max(nodes))
        tree = Tree(torch, pool, nodes, rows)
        tree.run()
        first = tree.out.clone(), tree.lse.clone()
        tree.check(only={(0, 0, 0), (0, nodes[0] - 1, 0), (1, 1, 0)})
        for _ in range(3):
            tree.out.fill_(1.0)
            tree.run()
            assert torch.equal(tree.out, first[0]) and torch.equal(tree.lse, first[1])
        pool.cache.check()


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("D,ps", [(64, 1), (64, 8), (128, 5), (128, 8), (128, 16), (128, 64), (256, 16)])
def test_tree_long_runs_of_tiles(torch_cuda, D, ps, cache, rows):
    """Many tiles for each block, arriving in few or in many copies: equal keys, and values that name their slots, so
    that each output counts the slots of a class exactly."""
    torch = torch_cuda
    lens, heads, kv = [3000, 700, 3000, 1100, 2900, 64, 2300], 32, 8
    pool = Pool(torch, lens, heads, kv, D, ps, cache, seed=2, fill=False)
    classes = 40
    for s, n in enumerate(lens):
        v = torch.zeros(kv, n, D)
        t = torch.arange(n)
        v[:, t, (t // 64 + 7 * t) % classes] = 1.0  # by tile and by slot
        k = torch.zeros(kv, n, D).to(dtypes(torch)[cache])
        page = pool.table[s, (t // ps).cuda()].long()
        pool.keys[page, :, (t % ps).cuda()] = k.transpose(0, 1).cuda()
        pool.values[page, :, (t % ps).cuda()] = v.transpose(0, 1).to(pool.values.dtype).cuda()
    pool.cache.reserve_tree(3)
    nodes = [3, 1, 2, 3, 1, 2, 3]
    tree = Tree(torch, pool, nodes, rows, masks=[[list(range(i + 1)) for i in range(n)] for n in nodes])
    for _ in range(4):
        tree.out.fill_(5.0)
        tree.run()
        pool.cache.check()
        out, r = tree.out.reshape(-1, heads, D).float().cpu(), 0
        for n, m in zip(lens, nodes):
            for i in range(m):
                seen = n - m + i + 1
                t = torch.arange(seen)
                want = torch.bincount((t // 64 + 7 * t) % classes, minlength=D).double() / seen
                # equal weights: powers of two, their sum and the outputs are exact but for the division and the type
                tol = want * (4 * EPS + (0.0 if rows == "f32" else torch.finfo(dtypes(torch)[rows]).eps / 2)) + 2.0 ** -25
                assert bool(((out[r].double() - want).abs() <= tol).all()), (n, i)
                r += 1


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_tree_masks_that_are_no_trees(torch_cuda, cache, rows):
    """Rows that see nothing, only later tokens, or not themselves."""
    torch = torch_cuda
    n = 37
    masks = [[[] for _ in range(n)], [list(range(n)) for _ in range(n)], [[j for j in range(n) if j % 3 != i % 3] for i in range(n)]]
    pool = Pool(torch, [n, 80 + n, 128 + n], 4, 2, 64, 16, cache, seed=2)
    pool.cache.reserve_tree(n)
    tree = Tree(torch, pool, [n] * 3, rows, masks=masks, words=3, noise=True)
    tree.run()
    pool.cache.check()
    tree.check()
    assert bool((tree.out[:n, :256] == 0).all()) and bool((tree.lse[:n] == -math.inf).all())


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_tree_slots_that_a_row_does_not_see_take_no_part(torch_cuda, cache, rows, D):
    """Infinities and NaN among the keys and values of other branches."""
    torch = torch_cuda
    n, bad = 20, {3: float("nan"), 4: float("inf"), 9: -float("inf"), 15: torch.finfo(dtypes(torch)[cache]).min}
    masks = [[[j for j in range(i + 1) if j not in bad or j == i] for i in range(n)] for _ in range(2)]
    pool = Pool(torch, [n + 119, n], 4, 2, D, 16, cache, seed=4)
    for s in range(2):
        first = pool.lens[s] - n
        for j, value in bad.items():
            k, v = (torch.full((2, 1, D), value).to(dtypes(torch)[cache]) for _ in range(2))
            pool.put(s, k, v, first + j)
            pool.k[s][:, first + j], pool.v[s][:, first + j] = k[:, 0], v[:, 0]
    pool.cache.reserve_tree(n)
    tree = Tree(torch, pool, [n] * 2, rows, masks=masks)
    tree.run()
    pool.cache.check()
    good = [i for i in range(n) if i not in bad]
    tree.check(only={(s, i, h) for s in range(2) for i in good for h in range(2)})
    # a NaN that is seen is not hidden
    assert bool(tree.out[3].isnan().all()) and bool(tree.out[n + 3].isnan().all())


@gpu
@pytest.mark.parametrize("cache", ["f32", "f16", "bf16"])
def test_tree_infinite_values_that_are_seen(torch_cuda, cache):
    """An infinite value makes its dimension of the rows that see it infinite, and no others."""
    torch = torch_cuda
    n, D = 12, 64
    pool = Pool(torch, [n + 30], 4, 2, D, 16, cache, seed=6)
    v = pool.v[0][:, 30 + 5:30 + 6].clone()
    v[:, 0, 7], v[:, 0, 9] = math.inf, -math.inf
    pool.put(0, pool.k[0][:, 35:36], v, 35)
    pool.cache.reserve_tree(n)
    masks = [[[j for j in range(i + 1) if j != 5 or i % 2] for i in range(n)]]
    tree = Tree(torch, pool, [n], cache, masks=masks)
    tree.run()
    pool.cache.check()
    out = tree.out.reshape(n, 4, D).float().cpu()
    for i in range(n):
        sees = i >= 5 and i % 2
        assert bool((out[i, :, 7] == math.inf).all()) == bool(sees)
        assert bool((out[i, :, 9] == -math.inf).all()) == bool(sees)
        rest = [d for d in range(D) if d not in (7, 9)]
        assert bool(out[i][:, rest].isfinite().all())


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")])
def test_tree_rising_logits(torch_cuda, cache, rows):
    """Logits that rise and fall by many units along the cache, so that maxima change in every tile."""
    torch = torch_cuda
    L, n, D = 1500, 6, 64
    pool = Pool(torch, [L + n], 4, 1, D, 16, cache, seed=8)
    lift = torch.linspace(-8, 8, L)[None, :, None].to(dtypes(torch)[cache])
    k = pool.k[0].clone()
    k[:, :L] = torch.cat((lift.expand(1, L, 8), k[:, :L, 8:]), 2)
    pool.k[0] = k
    pool.put(0, k, pool.v[0], 0)
    pool.cache.reserve_tree(n)
    tree = Tree(torch, pool, [n], rows)
    for sign in (1.0, -1.0):
        tree.q_cpu[:, :, :8] = sign * 3.0
        tree.q.copy_(tree.q_cpu.reshape(n, -1))
        tree.run(scale=0.4)
        pool.cache.check()
        tree.check(scale=float(np.float32(0.4)))


PAIRS = [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")]


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("scale", [-0.25, 3.0, 1e-4])
def test_tree_scales(torch_cuda, cache, rows, scale):
    torch = torch_cuda
    pool = Pool(torch, [300, 40], 8, 2, 64, 16, cache, seed=12)
    pool.cache.reserve_tree(17)
    tree = Tree(torch, pool, [17, 5], rows)
    tree.run(scale=scale)
    pool.cache.check()
    tree.check(scale=float(np.float32(scale)))


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("power", [20, 24, 26])
def test_tree_logits_far_from_zero(torch_cuda, cache, rows, power):
    """Logits of 2^20 and more, all but a few of them equal: weights stay in their type's range, and the equal ones share
    the output."""
    torch = torch_cuda
    L, D = 700, 64
    pool = Pool(torch, [L + 1], 2, 1, D, 16, cache, seed=13)
    k = torch.zeros(1, L + 1, D)
    k[0, :, 0] = 2.0 ** 8
    k[0, 5::97, 0] = 2.0 ** 7
    v = torch.zeros(1, L + 1, D)
    v[0, torch.arange(L + 1), torch.arange(L + 1) % D] = 1.0
    k, v = k.to(dtypes(torch)[cache]), v.to(dtypes(torch)[cache])
    pool.put(0, k, v, 0)
    pool.k, pool.v = [k], [v]
    pool.cache.reserve_tree(1)
    tree = Tree(torch, pool, [1], rows)
    tree.q_cpu.zero_()
    tree.q_cpu[:, :, 0] = 2.0 ** 9
    tree.q.copy_(tree.q_cpu.reshape(1, -1))
    tree.run(scale=2.0 ** (power - 17))
    pool.cache.check()
    great = k[0, :, 0] == 2.0 ** 8
    want = (v[0].double() * great[:, None]).sum(0) / int(great.sum())
    err = (tree.out.reshape(2, D).cpu().double() - want).abs()
    assert bool((err <= want * (8 * EPS + torch.finfo(dtypes(torch)[rows]).eps / 2 + UNIT[rows]) + 2.0 ** -25).all())
    # log-sum-exp: the logit and the count, rounded a few times
    lse = 2.0 ** power + math.log(int(great.sum()))
    assert bool(((tree.lse.cpu().double() - lse).abs() <= 8 * EPS * lse).all())


@gpu
@pytest.mark.parametrize("cache,rows", PAIRS)
@pytest.mark.parametrize("D", [40, 128])
def test_tree_rows_at_any_element(torch_cuda, cache, rows, D):
    """q and out that begin and step at odd elements, and no lse."""
    torch = torch_cuda
    pool = Pool(torch, [600, 50], 6, 2, D, 16, cache, seed=14)
    pool.cache.reserve_tree(12)
    tree = Tree(torch, pool, [12, 7], rows, q_pad=3, out_pad=5)
    dt, n, width = dtypes(torch)[rows], tree.rows, 6 * D
    room = torch.full((n * tree.out_stride + 9,), 77.0, dtype=dt, device="cuda")
    q = torch.zeros(n * tree.q_stride + 9, dtype=dt, device="cuda")
    q[1:1 + n * tree.q_stride] = tree.q.reshape(-1)
    pool.cache.tree_attention(q[1:].data_ptr(), room[3:].data_ptr(), tree.starts.data_ptr(), tree.mask.data_ptr(), n, 12, tree.words,
                              dtype=KINDS[rows], q_stride=tree.q_stride, out_stride=tree.out_stride)
    pool.cache.check()
    tree.run()  # the same at even ones
    got = room[3:3 + n * tree.out_stride].view(n, tree.out_stride)
    assert torch.equal(got[:, :width], tree.out[:, :width]) and bool((got[:, width:] == 77).all())
    assert bool((room[:3] == 77).all()) and bool((room[3 + n * tree.out_stride:] == 77).all())
    tree.check()


@gpu
@pytest.mark.parametrize("D,cache,rows", [(40, "f32", "f32"), (128, "f32", "f32"), (256, "f32", "f32"), (256, "f16", "f32"),
                                          (256, "f16", "f16"), (256, "bf16", "f32"), (256, "bf16", "bf16"), (64, "f16", "f16")])
@pytest.mark.parametrize("most", [1, 6, 7, 16, 17, 45])
def test_tree_any_number_of_rows(torch_cuda, D, cache, rows, most):
    """8 query heads to a kv head: 8 to 360 rows of a sequence, in the items' every size and one beyond it."""
    torch = torch_cuda
    pool = Pool(torch, [260, most, 97], 8, 1, D, 16, cache, seed=17)
    pool.cache.reserve_tree(most)
    tree = Tree(torch, pool, [most, most, most // 2], rows)
    tree.run()
    pool.cache.check()
    tree.check()


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_tree_many_sequences_and_one_kv_head(torch_cuda, cache, rows):
    """More sequences than a block has threads; and a group of 48 heads, so that tokens lie across blocks of rows."""
    torch = torch_cuda
    r = random.Random(5)
    lens = [r.choice([0, 1, 5, 40, 90]) for _ in range(420)]
    nodes = [r.randrange(min(n, 4) + 1) for n in lens]
    pool = Pool(torch, lens, 2, 1, 32, 8, cache, seed=15)
    pool.cache.reserve_tree(4)
    tree = Tree(torch, pool, nodes, rows)
    tree.run()
    pool.cache.check()
    tree.check(only={(s, i, 0) for s in range(0, 420, 13) for i in range(4)})
    pool = Pool(torch, [333, 20], 48, 1, 64, 16, cache, seed=16)
    pool.cache.reserve_tree(9)
    tree = Tree(torch, pool, [9, 5], rows)
    tree.run()
    pool.cache.check()
    tree.check()


@gpu
def test_tree_many_small_weights_beside_a_great_one(torch_cuda):
    """2,047 weights 18 units below the greatest add up to a share of an fp32 row's output."""
    torch = torch_cuda
    D = 64
    for cache in ("f16", "bf16"):
        pool = Pool(torch, [2049], 1, 1, D, 16, cache, seed=9)
        k = torch.zeros(1, 2049, D)
        k[0, 0, 0] = 18.0
        v = torch.ones(1, 2049, D)
        v[0, 0] = 2.0 ** -14  # so that the small ones' share shows
        k, v = k.to(dtypes(torch)[cache]), v.to(dtypes(torch)[cache])
        pool.k, pool.v = [k], [v]
        pool.put(0, k, v, 0)
        pool.cache.reserve_tree(1)
        tree = Tree(torch, pool, [1], "f32")
        tree.q_cpu.zero_()
        tree.q_cpu[0, 0, 0] = 1.0
        tree.q.copy_(tree.q_cpu.reshape(1, -1))
        tree.run(scale=1.0)
        pool.cache.check()
        tree.check(scale=1.0)


@gpu
def test_tree_bad_tables_lengths_and_starts_are_reported(torch_cuda):
    torch = torch_cuda
    for cache in ("f32", "bf16"):
        pool = Pool(torch, [100, 60, 80], 4, 2, 64, 16, cache, seed=3)
        pool.cache.reserve_tree(8)
        tree = Tree(torch, pool, [5, 4, 6], cache, spare=2)
        # a page outside the pool: its slots are not seen
        page = int(pool.table[0, 2])
        pool.table[0, 2] = pool.n_pages
        tree.run()
        with pytest.raises(IndexError, match="page"):
            pool.cache.check()
        pool.table[0, 2] = page
        kept = [t for t in range(100) if not 32 <= t < 48]
        k, v = pool.k[0], pool.v[0]
        pool.k[0], pool.v[0], pool.lens[0] = k[:, kept], v[:, kept], 84
        tree.check()
        pool.k[0], pool.v[0], pool.lens[0] = k, v, 100
        assert bool((tree.out[15:] == 77).all()) and bool((tree.lse[15:] == 77).all())  # behind the last sequence
        # a length that the table cannot hold, and more drafted tokens than slots
        for length in (-1, pool.capacity + 1, 3):
            pool.lengths[1] = length
            tree.run()
            with pytest.raises(IndexError):
                pool.cache.check()
            assert bool((tree.out[5:9] == 0).all()) and bool((tree.lse[5:9] == -math.inf).all())
        pool.lengths[1] = 60
        # more than max_new
        tree.run(max_new=5)
        with pytest.raises(IndexError):
            pool.cache.check()
        assert bool((tree.out[9:15] == 0).all())
        # starts that do not ascend, or leave the rows
        for starts in ([0, 5, 4, 15], [0, 5, 9, 99], [-1, 5, 9, 15]):
            tree.starts.copy_(torch.tensor(starts, dtype=torch.int32))
            tree.out.fill_(77)
            tree.run()
            with pytest.raises(IndexError, match="starts"):
                pool.cache.check()
        tree.starts.copy_(torch.tensor([0, 5, 9, 15], dtype=torch.int32))
        tree.run()
        pool.cache.check()
        tree.check()


@gpu
def test_tree_captured_replayed_and_on_other_streams(torch_cuda):
    torch = torch_cuda
    pool = Pool(torch, [400, 77], 8, 2, 128, 16, "bf16", seed=11)
    pool.cache.reserve_tree(9)
    tree = Tree(torch, pool, [9, 4], "bf16")
    tree.run()
    torch.cuda.synchronize()
    want = tree.out.clone()
    tree.out.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tree.run(stream=torch.cuda.current_stream().cuda_stream)
    pool.cache.reserve_tree(300)  # a larger workspace: the graph keeps its own
    for _ in range(3):
        tree.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tree.out, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tree.out.zero_()
        tree.run(stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(tree.out, want)
    pool.cache.check()


@gpu
def test_tree_refusals(torch_cuda):
    torch = torch_cuda
    pool = Pool(torch, [50], 4, 2, 64, 16, "f16")
    tree = Tree(torch, pool, [5], "f16")
    with pytest.raises(nb.LengthError, match="reserved"):
        tree.run()
    for n in (0, -1):
        with pytest.raises(ValueError):
            pool.cache.reserve_tree(n)
    with pytest.raises(nb.LengthError):
        pool.cache.reserve_tree(1025)
    with pytest.raises(ValueError):
        pool.cache.reserve_tree(1 << 70)
    pool.cache.reserve_tree(40)
    pool.cache.reserve_tree(4)  # what is reserved stays
    at = dict(q=tree.q.data_ptr(), out=tree.out.data_ptr(), starts=tree.starts.data_ptr(), mask=tree.mask.data_ptr(), rows=5, max_new=5,
              mask_words=1, dtype=nb.F16)
    for more in (dict(q=0), dict(out=0), dict(starts=0), dict(mask=0), dict(rows=-1), dict(max_new=-1), dict(mask_words=0),
                 dict(max_new=33), dict(dtype=nb.BF16), dict(dtype=9), dict(scale=math.inf), dict(scale=math.nan), dict(q_stride=255),
                 dict(out_stride=-8), dict(rows=1 << 70)):
        with pytest.raises(ValueError):
            pool.cache.tree_attention(**(at | more))
    for more in (dict(max_new=41, mask_words=2), dict(rows=1 << 31)):
        with pytest.raises(nb.LengthError):
            pool.cache.tree_attention(**(at | more))
    pool.cache.tree_attention(**(at | dict(rows=0)))
    pool.cache.tree_attention(**(at | dict(max_new=0, mask_words=0)))
    torch.cuda.synchronize()
    assert bool((tree.out == 77).all())


# ---------------------------------------------------------------------------
# append with positions, compaction


def rotated(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    out = x.clone()
    out[..., 0::2] = a * cos - b * sin
    out[..., 1::2] = a * sin + b * cos
    return out


@gpu
@pytest.mark.parametrize("cache,rows", [("f32", "f32"), ("f16", "f32"), ("bf16", "bf16")])
def test_append_at_positions(torch_cuda, cache, rows):
    """Rows with positions of their own are stored as the appended row of that position is."""
    torch = torch_cuda
    news, D, heads, kv = [7, 1, 20], 64, 4, 2
    pools = [Pool(torch, [30, 1, 52], heads, kv, D, 16, cache, seed=1, fill=False) for _ in range(2)]
    g = torch.Generator().manual_seed(5)
    n = sum(news)
    q, k, v = ((torch.randn(n, h, D, generator=g)).to(dtypes(torch)[rows]).cuda() for h in (heads, kv, kv))
    angle = torch.arange(90, dtype=torch.float64)[:, None] / 100.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
    cos, sin = angle.cos().float().cuda(), angle.sin().float().cuda()
    position = torch.randint(0, 90, (n,), generator=g).int().cuda()
    starts = torch.tensor([0, 7, 8, 28], dtype=torch.int32, device="cuda")
    outs = torch.empty_like(q), torch.empty_like(q)
    places = [torch.full((3, kv, p.capacity), -1, dtype=torch.int32, device="cuda") for p in pools]
    weights = torch.ones(3, kv, pools[0].capacity, device="cuda")
    common = dict(dtype=KINDS[rows], cos=cos.data_ptr(), sin=sin.data_ptr(), rope_rows=90)
    pools[0].cache.append(q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), n, 20, q_out=outs[0].data_ptr(),
                          row_position=position.data_ptr(), positions=places[0].data_ptr(), weights=weights.data_ptr(), **common)
    pools[0].cache.check()
    # the same one row a call, `seen` saying the position
    for r in range(n):
        s = 0 if r < 7 else 1 if r < 8 else 2
        one = torch.zeros(4, dtype=torch.int32, device="cuda")
        one[s + 1:] = 1
        pools[1].lengths.copy_(torch.tensor([[30, 1, 52][i] if i != s else [30, 1, 52][s] - (starts[s + 1].item() - 1 - r)
                                             for i in range(3)], dtype=torch.int32))
        seen = torch.zeros(3, dtype=torch.int32, device="cuda") + position[r] + 1
        pools[1].cache.append(q[r].data_ptr(), k[r].data_ptr(), v[r].data_ptr(), one.data_ptr(), 1, 1, q_out=outs[1][r].data_ptr(),
                              seen=seen.data_ptr(), positions=places[1].data_ptr(), **common)
    pools[1].cache.check()
    assert torch.equal(outs[0], outs[1]) and torch.equal(places[0], places[1])
    for a, b in ((pools[0].keys, pools[1].keys), (pools[0].values, pools[1].values)):
        assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))
    assert int((weights == 0).sum()) == n * kv
    # a position without a rotation
    position[3] = 90
    pools[0].cache.append(q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), n, 20, q_out=outs[0].data_ptr(),
                          row_position=position.data_ptr(), **common)
    with pytest.raises(IndexError, match="position"):
        pools[0].cache.check()


def paths(torch, lists, width):
    return torch.tensor([x + [-1] * (width - len(x)) for x in lists], dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("cache,D,ps,order", [("f32", 64, 16, "contiguous"), ("f16", 80, 5, "padded"), ("bf16", 256, 8, "slots first"),
                                              ("bf16", 8, 64, "contiguous")])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(torch_cuda, cache, D, ps, order, in_place):
    torch = torch_cuda
    r = random.Random(D + ps)
    lens, nodes = [200, 64, 31, 90, 12, 700], [30, 64, 1, 0, 12, 600]
    pool = Pool(torch, lens, 4, 2, D, ps, cache, seed=7, order=order)
    width = 300
    lists = [sorted(r.sample(range(n), min(n, m))) for n, m in zip(nodes, (6, 64, 1, 0, 0, 300))]
    starts = torch.tensor(np.cumsum([0] + nodes), dtype=torch.int32, device="cuda")
    positions = torch.randint(0, 1000, (6, 2, pool.capacity), dtype=torch.int32, device="cuda")
    weights = torch.rand(6, 2, pool.capacity, device="cuda")
    before = positions.cpu(), weights.cpu()
    keys, values = pool.keys.clone(), pool.values.clone()
    left = pool.lengths if in_place else torch.zeros_like(pool.lengths)
    accepted = paths(torch, lists, width)
    pool.cache.compact(starts.data_ptr(), accepted.data_ptr(), width, new_lengths=left.data_ptr(), positions=positions.data_ptr(),
                       weights=weights.data_ptr())
    pool.cache.check()
    assert left.tolist() == [a - n + len(x) for a, n, x in zip(lens, nodes, lists)]
    changed = set()
    for s, path in enumerate(lists):
        first = lens[s] - nodes[s]
        want_k, want_v = pool.k[s].clone(), pool.v[s].clone()
        for i, j in enumerate(path):
            want_k[:, first + i], want_v[:, first + i] = pool.k[s][:, first + j], pool.v[s][:, first + j]
            before[0][s, :, first + i], before[1][s, :, first + i] = before[0][s, :, first + j], before[1][s, :, first + j]
            changed.add((s, first + i))
        assert torch.equal(pool.read(pool.keys, s, lens[s]), want_k)
        assert torch.equal(pool.read(pool.values, s, lens[s]), want_v)
    assert torch.equal(positions.cpu(), before[0]) and torch.equal(weights.cpu(), before[1])
    # nothing else in the pool
    for s, t in changed:
        page = int(pool.table_cpu[s, t // ps])
        keys[page, :, t % ps], values[page, :, t % ps] = pool.keys[page, :, t % ps], pool.values[page, :, t % ps]
    assert torch.equal(keys.nan_to_num(3.0), pool.keys.nan_to_num(3.0))
    assert torch.equal(values.nan_to_num(3.0), pool.values.nan_to_num(3.0))


@gpu
def test_compact_leaves_bad_sequences_as_they_are(torch_cuda):
    torch = torch_cuda
    pool = Pool(torch, [40, 40, 40, 40], 4, 2, 64, 16, "f16", seed=7)
    starts = torch.tensor([0, 8, 16, 24, 32], dtype=torch.int32, device="cuda")
    left = torch.zeros_like(pool.lengths)
    for bad, match in (([3, 2], "starts"), ([2, 2], "starts"), ([1, 8], "starts"), ([1, -2], "starts")):
        accepted = paths(torch, [[1, 2], bad, [], [0]], 2)
        keys = pool.keys.clone()
        pool.cache.compact(starts.data_ptr(), accepted.data_ptr(), 2, new_lengths=left.data_ptr())
        with pytest.raises(IndexError, match=match):
            pool.cache.check()
        assert left.tolist() == [34, 40, 32, 33]
        assert torch.equal(pool.read(pool.keys, 1, 40), pool.k[1])
        pool.keys.copy_(keys)
    accepted = paths(torch, [[1, 2], [4], [5], [6]], 2)
    pool.lengths[0], pool.lengths[1] = 4, pool.capacity + 1
    pool.table[2, 2] = -3
    pool.cache.compact(starts.data_ptr(), accepted.data_ptr(), 2, new_lengths=left.data_ptr())
    with pytest.raises(IndexError, match="page.*length.*starts"):
        pool.cache.check()
    assert left.tolist() == [4, pool.capacity + 1, 40, 33]
    assert torch.equal(pool.read(pool.keys, 2, 40), pool.k[2])
    at = dict(starts=starts.data_ptr(), accepted=accepted.data_ptr(), n_accepted=2, new_lengths=left.data_ptr())
    for more in (dict(starts=0), dict(accepted=0), dict(new_lengths=0), dict(n_accepted=-1)):
        with pytest.raises(ValueError):
            pool.cache.compact(**(at | more))
    with pytest.raises(nb.LengthError):
        pool.cache.compact(**(at | dict(n_accepted=1025)))
    pool.lengths.copy_(torch.tensor([40] * 4))
    pool.table.copy_(pool.table_cpu)
    pool.cache.compact(**(at | dict(n_accepted=0, accepted=0)))  # nothing accepted
    pool.cache.check()
    assert left.tolist() == [32] * 4


# ---------------------------------------------------------------------------
# pages


class Book:
    """A book of pages on the device beside the same one as lists."""

    def __init__(self, torch, sequences, max_pages, n_pages, ps, seed=0):
        self.t, self.S, self.M, self.P, self.ps = torch, sequences, max_pages, n_pages, ps
        order = list(range(n_pages))
        random.Random(seed).shuffle(order)
        self.table = [[-9] * max_pages for _ in range(sequences)]
        self.lengths, self.refs, self.free, self.count = [0] * sequences, [0] * n_pages, order, n_pages
        whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.dev = dict(table=whole(self.table), lengths=whole(self.lengths), refs=whole(self.refs), free=whole(self.free),
                        count=whole([self.count]))
        self.copies = torch.full((3, sequences), 55, dtype=torch.int32, device="cuda")
        self.book = nb.PageBook(*(self.dev[k].data_ptr() for k in ("table", "lengths", "refs", "free", "count")),
                                sequences=sequences, max_pages=max_pages, n_pages=n_pages, page_size=ps)

    def pages(self, n):
        return -(-n // self.ps)

    def plain(self, parent, keep, add):
        """The update on the lists; the copy lists, or None where it is refused."""
        S, ps = self.S, self.ps
        parent, add = parent or list(range(S)), add or [0] * S
        kept = [0 if p < 0 else self.lengths[p] for p in parent]
        kept = [min(k, w) for k, w in zip(kept, keep)] if keep else kept
        if any(k + a > self.M * ps for k, a in zip(kept, add)):
            return None
        refs, rows, writers = list(self.refs), [], {}
        for s in range(S):
            for p in self.table[s][:self.pages(self.lengths[s])]:
                refs[p] -= 1
        for s in range(S):
            rows.append(self.table[parent[s]][:self.pages(kept[s])] if kept[s] else [])
            for p in rows[s]:
                refs[p] += 1
            if add[s] and kept[s] % ps:
                writers.setdefault(rows[s][-1], []).append(s)
        split = set()
        for p, who in writers.items():
            if refs[p] > 1:
                split |= set(who[1:] if len(who) == refs[p] else who)
        free, count = list(self.free), self.count
        copies = [[-1] * S, [-1] * S, [0] * S]
        for s in range(S):
            new = ([1] if s in split else []) + [0] * (self.pages(kept[s] + add[s]) - self.pages(kept[s]))
            for is_copy in new:
                count -= 1
                if count < 0:
                    return None
                refs[free[count]] += 1
                if is_copy:
                    refs[rows[s][-1]] -= 1
                    copies[0][s], copies[1][s], copies[2][s] = rows[s][-1], free[count], kept[s] % ps
                    rows[s][-1] = free[count]
                else:
                    rows[s].append(free[count])
        for p in range(self.P):
            if self.refs[p] > 0 and refs[p] == 0:
                free[count] = p
                count += 1
        for s in range(S):
            self.table[s][:len(rows[s])] = rows[s]
        self.lengths, self.refs, self.free, self.count = [k + a for k, a in zip(kept, add)], refs, free, count
        return copies

    def update(self, parent=None, keep=None, add=None, stream=0):
        held = [self.t.tensor(x, dtype=self.t.int32, device="cuda") if x is not None else None for x in (parent, keep, add)]
        a, b, c = (x.data_ptr() if x is not None else 0 for x in held)
        self.book.update(parent=a, keep=b, add=c, copy_from=self.copies[0].data_ptr(), copy_to=self.copies[1].data_ptr(),
                         copy_slots=self.copies[2].data_ptr(), stream=stream)
        return held

    def same(self, copies):
        nothing = [[-1] * self.S, [-1] * self.S, [0] * self.S]
        assert self.copies.tolist() == (copies or nothing)
        assert self.dev["lengths"].tolist() == self.lengths
        assert self.dev["table"].tolist() == self.table
        assert self.dev["refs"].tolist() == self.refs
        assert self.dev["count"].tolist() == [self.count]
        assert self.dev["free"].tolist() == self.free


@gpu
@pytest.mark.parametrize("S,M,P,ps,seed", [(1, 4, 9, 4, 0), (8, 20, 120, 4, 1), (64, 9, 200, 16, 2), (700, 6, 3000, 5, 3),
                                           (1500, 3, 5000, 2, 4), (33, 300, 9000, 1, 5)])
def test_pages_follow_the_plain_book(torch_cuda, S, M, P, ps, seed):
    """Random forks, trims and extensions, some of them too large for the table or the pool."""
    torch = torch_cuda
    book, r = Book(torch, S, M, P, ps, seed), random.Random(seed)
    for step in range(25):
        kind = r.randrange(4)
        parent = None if kind == 0 else [r.randrange(-1 if kind == 1 else 0, S) for _ in range(S)]
        if kind == 2:  # beams of groups of 4
            parent = [s // 4 * 4 + r.randrange(min(4, S - s // 4 * 4)) for s in range(S)]
        keep = None if r.random() < 0.5 else [r.randrange(0, M * ps + 1) for _ in range(S)]
        add = None if r.random() < 0.2 else [r.choice([0, 1, 1, 2, ps, 2 * ps + 1]) if step % 5 else r.choice([0, 1]) for _ in range(S)]
        if step % 6 == 5:  # room again
            keep = [r.randrange(0, 2 * ps) for _ in range(S)]
        want = book.plain(parent, keep, add)
        book.update(parent, keep, add)
        book.same(want)
        if want is None:
            with pytest.raises((nb.LengthError, IndexError)):
                book.book.check()
        book.book.check()
    # every page is held as often as the table shows, or free
    held = [0] * P
    for s in range(S):
        for p in book.table[s][:book.pages(book.lengths[s])]:
            held[p] += 1
    assert held == book.refs and sorted(book.free[:book.count]) == [p for p in range(P) if not held[p]]


@gpu
def test_pages_held_by_the_caller_are_not_written(torch_cuda):
    """A prompt kept for later: its partly filled page is copied, and its pages outlive the sequences."""
    torch = torch_cuda
    book = Book(torch, 3, 8, 30, 4)
    want = book.plain(None, None, [10, 0, 0])
    book.update(None, None, [10, 0, 0])
    book.same(want)
    for p in book.table[0][:3]:
        book.refs[p] += 1
        book.dev["refs"][p] += 1
    want = book.plain([0, 0, 0], None, [1, 1, 0])
    book.update([0, 0, 0], None, [1, 1, 0])
    assert want[0][0] == want[0][1] == book.table[2][2] and want[2] == [2, 2, 0]
    book.same(want)
    want = book.plain([-1, -1, -1], None, None)
    book.update([-1, -1, -1])
    book.same(want)
    assert book.count == 27
    book.book.check()


@gpu
def test_pages_refuse_what_is_out_of_range(torch_cuda):
    torch = torch_cuda
    book = Book(torch, 4, 4, 12, 4)
    book.plain(None, None, [5, 6, 7, 8])
    book.update(None, None, [5, 6, 7, 8])
    for parent, keep, add, what in (([4, 0, 0, 0], None, None, IndexError), ([-2, 0, 0, 0], None, None, IndexError),
                                    (None, [-1, 3, 3, 3], None, IndexError), (None, None, [0, -1, 0, 0], IndexError),
                                    (None, None, [0, 0, 0, 9], IndexError), (None, None, [2 ** 31 - 1] * 4, IndexError),
                                    (None, None, [8, 8, 8, 8], nb.LengthError)):
        book.update(parent, keep, add)
        book.same(None)
        with pytest.raises(what):
            book.book.check()
    # a damaged book: lengths, a table entry, a free page that is in use, one listed twice
    for key, at, value in (("lengths", 1, -1), ("lengths", 2, 17), ("table", (0, 0), 12), ("free", 2, 99), ("free", 2, None),
                           ("free", 2, "twice"), ("count", 0, 13), ("count", 0, -1)):
        was = book.dev[key][at].clone()
        book.dev[key][at] = book.dev["table"][0, 0] if value is None else book.dev["free"][3] if value == "twice" else value
        book.copies.fill_(55)
        damaged = {k: v.clone() for k, v in book.dev.items()}
        book.update([1, 0, 2, 3], None, [4, 4, 4, 4])
        assert book.copies.tolist() == [[-1] * 4, [-1] * 4, [0] * 4], (key, value)
        assert all(torch.equal(v, damaged[k]) for k, v in book.dev.items()), (key, value)
        with pytest.raises(IndexError):
            book.book.check()
        book.dev[key][at] = was
    want = book.plain([1, 0, 2, 3], None, [1, 1, 1, 1])
    book.update([1, 0, 2, 3], None, [1, 1, 1, 1])
    book.same(want)
    book.book.check()
    with pytest.raises(ValueError):
        book.book.update(add=book.copies.data_ptr())
    with pytest.raises(ValueError):
        book.book.update(copy_from=book.copies.data_ptr())
    with pytest.raises(ValueError):
        book.book.update(parent=1 << 70)


@gpu
@pytest.mark.parametrize("cache,D,ps,order,bounds", [("f32", 64, 16, "contiguous", True), ("f16", 80, 5, "padded", False),
                                                     ("bf16", 256, 40, "slots first", True)])
def test_copy_pages(torch_cuda, cache, D, ps, order, bounds):
    torch = torch_cuda
    pool = Pool(torch, [ps * 6], 4, 2, D, ps, cache, order=order, spare=6, bounds=bounds)
    if bounds:
        pool.bounds.random_(-127, 128)
        pool.scales.uniform_()
    used = [int(p) for p in pool.table_cpu[0][:6]]
    free = [p for p in range(pool.n_pages) if p not in used]
    keys, values = pool.keys.clone(), pool.values.clone()
    pairs = [(used[0], free[0], ps), (-1, -1, 3), (used[1], free[1], 0), (used[0], free[2], 1), (used[3], free[3], ps - 1)]
    src, dst, slots = (torch.tensor([p[i] for p in pairs], dtype=torch.int32, device="cuda") for i in range(3))
    for with_slots in (True, False):
        b, c = (pool.bounds.clone(), pool.scales.clone()) if bounds else (None, None)
        pool.cache.copy_pages(src.data_ptr(), dst.data_ptr(), 5, slots=slots.data_ptr() if with_slots else 0)
        pool.cache.check()
        for a, t, n in pairs:
            if a >= 0:
                n = n if with_slots else ps
                keys[t, :, :n], values[t, :, :n] = keys[a, :, :n].clone(), values[a, :, :n].clone()
                if bounds:
                    b[t], c[t] = b[a], c[a]
        assert torch.equal(keys.nan_to_num(3.0), pool.keys.nan_to_num(3.0))
        assert torch.equal(values.nan_to_num(3.0), pool.values.nan_to_num(3.0))
        if bounds:
            assert torch.equal(b, pool.bounds) and torch.equal(c, pool.scales)
    # bad pages and counts are passed over
    for i, (a, t, n) in enumerate([(pool.n_pages, free[4], 1), (used[0], -1, 1), (-1, free[4], 1), (used[0], free[4], ps + 1),
                                   (used[0], free[4], -1)]):
        one = torch.tensor([[a], [t], [n]], dtype=torch.int32, device="cuda")
        pool.cache.copy_pages(one[0].data_ptr(), one[1].data_ptr(), 1, slots=one[2].data_ptr())
        with pytest.raises(IndexError):
            pool.cache.check()
    assert torch.equal(keys.nan_to_num(3.0), pool.keys.nan_to_num(3.0))
    pool.cache.copy_pages(0, 0, 0)
    for more in (dict(source=0), dict(target=0), dict(count=-1)):
        with pytest.raises(ValueError):
            pool.cache.copy_pages(**(dict(source=src.data_ptr(), target=dst.data_ptr(), count=5) | more))


# ---------------------------------------------------------------------------
# beams


def plain_beams(torch, logits, scores, finished, eos, n):
    """(score in 64 bits, row, token, finished) of each request's best, by the definition."""
    S, B = scores.shape
    V = logits.shape[-1]
    x = logits.double().reshape(S, B, V)
    x = x.masked_fill(x.isnan(), -math.inf).clamp(max=torch.finfo(torch.float32).max)
    got = []
    for s in range(S):
        cands = []
        for b in range(B):
            score = float(scores[s, b])
            score = -math.inf if math.isnan(score) else score
            if finished is not None and finished[s, b]:
                cands.append((-score, b, eos, 1))
                continue
            row = x[s, b]
            top = float(row.max())
            lse = top + math.log(float(torch.exp(row - top).sum())) if top > -math.inf else -math.inf
            t = score + (row - lse)
            t = t.masked_fill(t.isnan(), -math.inf).numpy()
            best = np.lexsort((np.arange(V), -t))[:n]
            cands += [(-t[i], b, int(i), int(i == eos)) for i in best]
        cands.sort(key=lambda c: c[:3])
        cands = [(-v, s * B + b, t, f) for v, b, t, f in cands[:n]]
        got.append(cands + [(-math.inf, -1, -1, 0)] * (n - len(cands)))
    return got


def run_beams(torch, logits, scores, n, finished=None, eos=-1, beam=None, vocab=None):
    S, B = scores.shape
    V = vocab or logits.shape[-1]
    beam = beam or nb.BeamSearch(S, B, V, n)
    kind = {torch.float32: nb.F32, torch.float16: nb.F16, torch.bfloat16: nb.BF16}[logits.dtype]
    out = [torch.full((S, n), 9, dtype=t, device="cuda") for t in (torch.float32, torch.int32, torch.int32, torch.uint8)]
    beam.select(logits.data_ptr(), scores.data_ptr(), *(o.data_ptr() for o in out[:3]), dtype=kind,
                logits_stride=logits.stride(-2), finished=finished.data_ptr() if finished is not None else 0, eos=eos,
                out_finished=out[3].data_ptr(), sequences=S)
    torch.cuda.synchronize()
    return [o.cpu() for o in out]


def same_beams(got, want):
    for s, row in enumerate(want):
        assert got[1][s].tolist() == [c[1] for c in row], s
        assert got[2][s].tolist() == [c[2] for c in row], s
        assert got[3][s].tolist() == [c[3] for c in row], s
        for g, c in zip(got[0][s].tolist(), row):
            # the sum of the exponentials is within 40 roundings of itself, the score rounded once
            assert g == c[0] or abs(g - c[0]) <= 40 * EPS + abs(c[0]) * EPS, (s, g, c)


BEAMS = [  # sequences, beams, vocab, out, kind, pad
    (1, 1, 1, 1, "f32", 0), (1, 1, 7, 7, "f16", 0), (2, 3, 40, 5, "bf16", 0), (3, 4, 32000, 8, "f32", 0), (2, 5, 50257, 10, "f16", 0),
    (1, 32, 8192, 64, "bf16", 3), (4, 2, 8193, 4, "f32", 1), (2, 7, 1000, 64, "bf16", 5), (1, 2, 160001, 33, "f16", 0),
    (5, 1, 3000, 1, "f32", 2), (1, 300, 129, 20, "f32", 0), (1, 2, 9300, 64, "bf16", 0),
]


@gpu
@pytest.mark.parametrize("shape", range(len(BEAMS)))
def test_beam_select_against_64_bits(torch_cuda, shape):
    torch = torch_cuda
    S, B, V, n, kind, pad = BEAMS[shape]
    g = torch.Generator().manual_seed(shape)
    room = (3 * torch.randn(S * B, V + pad, generator=g)).to(dtypes(torch)[kind])
    logits = room.cuda()[:, :V]
    scores = -10 * torch.rand(S, B, generator=g)
    eos = min(3, V - 1)
    for ended in (None, torch.rand(S, B, generator=g) < 0.4):
        done = ended.to(torch.uint8).cuda() if ended is not None else None
        got = run_beams(torch, logits, scores.cuda(), n, done, eos)
        same_beams(got, plain_beams(torch, room[:, :V], scores, ended, eos, n))


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [1, 2, 3, 7])
def test_beam_select_unaligned_rows(torch_cuda, kind, offset):
    torch = torch_cuda
    g = torch.Generator().manual_seed(offset)
    room = torch.randn(3 * 20011 + 8, generator=g).to(dtypes(torch)[kind]).cuda()
    logits = room[offset:offset + 3 * 20011].view(3, 20011)
    scores = torch.zeros(1, 3)
    same_beams(run_beams(torch, logits, scores.cuda(), 12), plain_beams(torch, logits.cpu(), scores, None, -1, 12))


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_beam_select_ties_and_what_is_not_finite(torch_cuda, kind):
    torch = torch_cuda
    B, V, n = 6, 20000, 40
    g = torch.Generator().manual_seed(1)
    dt = dtypes(torch)[kind]
    for case in ("constant", "few levels", "same rows", "masked", "all masked", "nan", "inf", "scores"):
        logits = torch.randn(B, V, generator=g)
        scores = -torch.rand(1, B, generator=g)
        if case == "constant":
            logits[:] = 2.0
        elif case == "few levels":
            logits = logits.round()
        elif case == "same rows":
            logits[:] = logits[0].clone()
            scores[:] = -1.0
        elif case == "masked":  # all but five tokens of each beam
            keep = torch.zeros(B, V, dtype=torch.bool)
            keep[:, [5, 77, 9000, 15000, 19999]] = True
            logits[~keep] = -math.inf
            logits[1, ~keep[1]] = torch.finfo(dt).min
        elif case == "all masked":
            logits[:] = -math.inf
            logits[2, 11] = 1.0
        elif case == "nan":
            logits[0, :] = math.nan
            logits[1, 5:9000] = math.nan
        elif case == "inf":
            logits[0, 100] = math.inf
            logits[1, 7], logits[1, 8] = math.inf, math.inf
            logits[2, :] = math.inf
        else:
            scores[0] = torch.tensor([0.0, -math.inf, math.nan, -math.inf, -1e30, -math.inf])
        logits = logits.to(dt)
        got = run_beams(torch, logits.cuda(), scores.cuda(), n)
        same_beams(got, plain_beams(torch, logits, scores, None, -1, n))


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [3, 700, 1025, 9001])
def test_beam_select_rows_of_the_lowest_value(torch_cuda, kind, V):
    """Rows of the type's lowest value, alone or but for a few logits: places outside the row count for nothing."""
    torch = torch_cuda
    dt = dtypes(torch)[kind]
    logits = torch.full((3, V), torch.finfo(dt).min, dtype=dt)
    logits[1, V // 2] = 1.0
    logits[2, :] = -math.inf
    logits[2, V - 1] = torch.finfo(dt).min
    scores = torch.tensor([[-1.0, -2.0, -0.5]])
    n = min(5, V)
    same_beams(run_beams(torch, logits.cuda(), scores.cuda(), n), plain_beams(torch, logits, scores, None, -1, n))


@gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [3, 40])
def test_beam_select_nan_among_ordinary_logits(torch_cuda, kind, n):
    """NaN counts as -infinity in the sums too, a logit here and there, and beside +infinity."""
    torch = torch_cuda
    g = torch.Generator().manual_seed(21)
    logits = (torch.randn(4, 5003, generator=g) * 3).to(dtypes(torch)[kind])
    logits[0, 5::97] = math.nan
    logits[1, 4099] = math.nan
    logits[2, 17], logits[2, 18], logits[2, 4999] = math.inf, math.nan, math.nan
    logits[3, :5000] = math.nan
    scores = torch.tensor([[-1.0, -1.5, -0.5, -2.0]])
    same_beams(run_beams(torch, logits.cuda(), scores.cuda(), n), plain_beams(torch, logits, scores, None, -1, n))


@gpu
def test_beam_select_finished_beams_and_too_few_candidates(torch_cuda):
    torch = torch_cuda
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(8, 6, generator=g)
    logits[1] = math.nan  # of a finished beam: not read
    scores = -torch.rand(2, 4, generator=g)
    ended = torch.tensor([[1, 1, 1, 1], [0, 1, 1, 1]])
    want = plain_beams(torch, logits, scores, ended, 2, 12)
    got = run_beams(torch, logits.cuda(), scores.cuda(), 12, ended.to(torch.uint8).cuda(), 2)
    same_beams(got, want)
    assert got[1][0].tolist() == sorted(range(4), key=lambda b: -float(scores[0, b])) + [-1] * 8
    assert got[1][1, 9:].tolist() == [-1] * 3


@gpu
def test_beam_select_in_place_fewer_sequences_and_captured(torch_cuda):
    torch = torch_cuda
    S, B, V = 5, 4, 1200
    g = torch.Generator().manual_seed(4)
    beam = nb.BeamSearch(S, B, V, B)
    logits = torch.randn(S * B, V, generator=g).cuda()
    start = -torch.rand(S, B, generator=g).cuda()
    want = plain_beams(torch, logits.cpu(), start.cpu(), torch.zeros(S, B), 7, B)
    scores, finished = start.clone(), torch.zeros(S, B, dtype=torch.uint8, device="cuda")
    rows, tokens = (torch.full((S, B), -7, dtype=torch.int32, device="cuda") for _ in range(2))

    def step(n):
        beam.select(logits.data_ptr(), scores.data_ptr(), scores.data_ptr(), rows.data_ptr(), tokens.data_ptr(),
                    finished=finished.data_ptr(), eos=7, out_finished=finished.data_ptr(), sequences=n,
                    stream=torch.cuda.current_stream().cuda_stream)

    step(3)
    torch.cuda.synchronize()
    same_beams([x.cpu()[:3] for x in (scores, rows, tokens, finished)], want[:3])
    assert bool((rows[3:] == -7).all()) and torch.equal(scores[3:], start[3:])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(S)
    for _ in range(2):
        scores.copy_(start)
        finished.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same_beams([x.cpu() for x in (scores, rows, tokens, finished)], want)


@gpu
def test_beam_select_refusals(torch_cuda):
    torch = torch_cuda
    beam = nb.BeamSearch(2, 2, 100, 4)
    buf = torch.zeros(4096, device="cuda")
    at = buf.data_ptr()
    good = dict(logits=at, scores=at, out_scores=at, out_rows=at, out_tokens=at)
    for more in (dict(logits=0), dict(scores=0), dict(out_scores=0), dict(out_rows=0), dict(out_tokens=0), dict(dtype=5),
                 dict(logits_stride=99), dict(sequences=-1), dict(eos=100), dict(eos=-2), dict(finished=at), dict(logits=at + 1),
                 dict(logits=at + 2), dict(logits_stride=1 << 70)):
        with pytest.raises(ValueError):
            beam.select(**(good | more))
    with pytest.raises(nb.LengthError):
        beam.select(**(good | dict(sequences=3)))
    beam.select(**(good | dict(sequences=0)))


@gpu
def test_arrays_in_the_wrong_place_are_refused(torch_cuda):
    """Between elements, or where a call would write what it still reads."""
    torch = torch_cuda
    buf = torch.zeros(8192, device="cuda")
    at = buf.data_ptr()
    pool = Pool(torch, [50], 4, 2, 64, 16, "f16")
    pool.cache.reserve_tree(8)
    tree = dict(q=at, out=at + 16384, starts=at, mask=at, rows=5, max_new=5, mask_words=1, dtype=nb.F16, lse=at + 8192)
    for more in (dict(q=at + 1), dict(out=at + 1), dict(starts=at + 2), dict(mask=at + 1), dict(lse=at + 2), dict(out=at),
                 dict(dtype=nb.F32, q=at + 2), dict(dtype=nb.F32, out=at + 2)):
        with pytest.raises(ValueError):
            pool.cache.tree_attention(**(tree | more))
    for name in ("source", "target", "slots"):
        with pytest.raises(ValueError, match="multiples"):
            pool.cache.copy_pages(count=1, **(dict(source=at, target=at) | {name: at + 2}))
    for name in ("starts", "accepted", "new_lengths", "positions", "weights"):
        with pytest.raises(ValueError, match="multiples"):
            pool.cache.compact(n_accepted=1, **(dict(starts=at, accepted=at, new_lengths=at) | {name: at + 2}))
    book = nb.PageBook(at, at + 4096, at + 8192, at + 12288, at + 16384, sequences=4, max_pages=8, n_pages=30, page_size=16)
    for name in ("parent", "keep", "add", "copy_from", "copy_to", "copy_slots"):
        with pytest.raises(ValueError, match="multiples"):
            book.update(**(dict(copy_from=at, copy_to=at, copy_slots=at) | {name: at + 2}))
    with pytest.raises(ValueError, match="multiples"):
        nb.PageBook(at + 2, at, at, at, at, sequences=4, max_pages=8, n_pages=30, page_size=16)
    beam = nb.BeamSearch(2, 2, 100, 4)
    good = dict(logits=at, scores=at, out_scores=at + 4096, out_rows=at + 8192, out_tokens=at + 12288)
    for more in (dict(scores=at + 2), dict(out_scores=at + 1), dict(out_rows=at + 2), dict(out_tokens=at + 3), dict(out_scores=at),
                 dict(finished=at, out_finished=at, eos=1)):
        with pytest.raises(ValueError):
            beam.select(**(good | more))
    torch.cuda.synchronize()
    assert not bool(buf.any())


# ---------------------------------------------------------------------------
# argument checks that need no GPU


def test_entry_points_refuse_null_handles():
    lib = nb.cuda_lib()
    for name in ("nut_paged_tree_attention", "nut_paged_compact", "nut_paged_copy", "nut_pages_update", "nut_beam_select"):
        assert getattr(lib, name)(None, None, None) == nb.NUT_INVALID_ARGUMENT
        assert b"null" in lib.nut_last_error()
    assert lib.nut_paged_reserve_tree(None, 4) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_append_at(None, None, None, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_append_at(None, None, 16, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_pages_error(None, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_pages_destroy(None) == 0 and lib.nut_beam_destroy(None) == 0
    assert lib.nut_beam_create(1, 1, 1, 1, 0, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_pages_create(None, 0, None) == nb.NUT_INVALID_ARGUMENT


def test_beams_and_books_of_impossible_sizes_are_refused():
    lib, h = nb.cuda_lib(), C.c_void_p()
    for sizes in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (-1, 1, 1, 1)):
        assert lib.nut_beam_create(*sizes, 0, C.byref(h)) == nb.NUT_INVALID_ARGUMENT
    for sizes in ((1, 1, 1, 65), (65536, 1, 10, 1), (1, 1025, 10, 1), (8192, 8, 10, 1), (1, 1, (1 << 28) + 1, 1),
                  (1, 1024, 1 << 28, 64)):
        assert lib.nut_beam_create(*sizes, 0, C.byref(h)) == nb.NUT_LENGTH_ERROR
    with pytest.raises(ValueError):
        nb.BeamSearch(1 << 70, 1, 1, 1)
    good = dict(sequences=4, max_pages=8, n_pages=30, page_size=16)
    for bad in (dict(sequences=0), dict(max_pages=0), dict(n_pages=-1), dict(page_size=0)):
        with pytest.raises(ValueError):
            nb.PageBook(16, 16, 16, 16, 16, **(good | bad))
    for k in range(5):
        with pytest.raises(ValueError, match="null"):
            nb.PageBook(*(0 if i == k else 16 for i in range(5)), **good)
    for bad in (dict(sequences=65536), dict(max_pages=1 << 25), dict(n_pages=1 << 31), dict(max_pages=1 << 20, page_size=1 << 12)):
        with pytest.raises(nb.LengthError):
            nb.PageBook(16, 16, 16, 16, 16, **(good | bad))
