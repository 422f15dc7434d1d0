"""The paged KV cache operators where a call is easily answered wrongly: rows
with one token far above the others, special values in used slots, wrong
numbers in device memory, and sizes at the ends of their ranges.  Tolerances
are those of test_paged.py, or derived beside the test."""
import math

import numpy as np
import pytest

import nutllm_b200 as nb
from tests.test_paged import EPS, KINDS, TYPES, Pool, check_bounds, close_out, dtypes, head_reference, run_select, select_reference

# ---------------------------------------------------------------------------
# attention


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("gap", [10.0, 14.0, 16.0, 18.0])
def test_tokens_far_below_the_greatest_keep_their_share(gpu, types, gap):
    """One token `gap` nats above all others has a value of 0, so that the output is what the others add up to.  512 rows of one
    sequence: an item then lies in one or two blocks, and its warps walk hundreds of slots.

    A weight is off by the logits' error (one product, its unit and the subtraction: 4 eps of the gap), by 2^-22 (16-bit caches:
    two terms; bf16: 2^-17 where the rows are bf16, whose weights have two terms of 8 bits) and, in fp16, by 2^-43 of the greatest
    weight.  The sums are chains of n / 64 products of 16 slots a warp, and the denominator's of n / 16."""
    import torch
    n, D, rows = 2048, 64, 512
    pool = Pool(torch, [n], 4, 1, D, 16, types[0], max_rows=rows, fill=False)
    dt = dtypes(torch)
    k = torch.zeros(1, n, D)
    k[0, 5, 0] = gap
    v = 500 + 1000 * torch.rand(1, n, D, generator=pool.g)
    v[0, 5] = 0.0
    k, v = k.to(dt[types[0]]), v.to(dt[types[0]])
    pool.put(0, k, v, 0)
    q = torch.zeros(rows, 4, D, dtype=dt[types[1]])
    q[:, :, 0] = 1.0
    q, seq = q.cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.zeros(rows, 4, device="cuda")
    pool.cache.attention(q.data_ptr(), out.data_ptr(), rows, dtype=KINDS[types[1]], scale=1.0, lse=lse.data_ptr(),
                         row_sequence=seq.data_ptr())
    pool.cache.check()
    want, want_lse, _, _, mass = head_reference(torch, q[0, :1].cpu(), k[0], v[0], 1.0)
    tol = 8 * EPS * gap + (n / 16 + 64) * EPS + 2.0 ** -22
    tol += {"f32": 0.0, "f16": 2.0 ** -43 * math.exp(gap), "bf16": 2.0 ** -17 if types[1] == "bf16" else 0.0}[types[0]]
    tol = tol * mass
    if types[1] != "f32":
        tol = tol + (want.abs() + tol) * torch.finfo(dt[types[1]]).eps / 2 + (2.0 ** -25 if types[1] == "f16" else 0.0)
    err = (out.cpu().double() - want).abs()
    assert bool((err <= tol).all()), f"error {float((err / want).max()):.2e} of the output, {float((err / tol).max()):.1f} of the bound"
    assert float((lse.cpu().double() - want_lse).abs().max()) <= 8 * EPS * gap + (n / 16 + 8) * EPS


@pytest.mark.gpu
@pytest.mark.parametrize("types", [t for t in TYPES if t[1] != "f16"], ids=lambda t: "-".join(t))
def test_infinite_values_reach_the_output(gpu, types):
    """An infinite value with a weight of its own makes its dimension infinite."""
    import torch
    pool = Pool(torch, [30], 2, 1, 64, 16, types[0])
    page = int(pool.table_cpu[0, 1])
    pool.values[page, 0, 3, 6], pool.values[page, 0, 4, 9] = float("inf"), -float("inf")
    q = torch.randn(1, 2, 64, generator=pool.g).to(dtypes(torch)[types[1]]).cuda()
    out = torch.zeros_like(q)
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 1, dtype=KINDS[types[1]])
    pool.cache.check()
    assert bool((out[0, :, 6] == math.inf).all()) and bool((out[0, :, 9] == -math.inf).all())
    assert bool(torch.isfinite(out[0, :, [d for d in range(64) if d not in (6, 9)]]).all())


@pytest.mark.gpu
def test_infinite_values_reach_fp16_rows(gpu):
    """Outputs are rounded to fp16, not saturated: infinities stay, and a mean of the largest finite values stays finite."""
    import torch
    pool = Pool(torch, [30], 2, 1, 64, 16, "f16")
    page = int(pool.table_cpu[0, 1])
    pool.values[page, 0, 3, 6], pool.values[page, 0, 4, 9] = float("inf"), -float("inf")
    for j in range(2):
        pool.values[int(pool.table_cpu[0, j]), 0, :, 11] = 65504.0
    q = torch.randn(1, 2, 64, generator=pool.g).half().cuda()
    out = torch.zeros_like(q)
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 1, dtype=KINDS["f16"])
    pool.cache.check()
    assert bool((out[0, :, 6] == math.inf).all()) and bool((out[0, :, 9] == -math.inf).all())
    assert bool((out[0, :, 11] == 65504.0).all())
    assert bool(torch.isfinite(out[0, :, [d for d in range(64) if d not in (6, 9)]]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_logits_that_are_all_minus_infinity_add_no_weight(gpu, types):
    """A row that gives every slot a weight of 0 is a row that sees nothing."""
    import torch
    lens = [40, 20]
    pool = Pool(torch, lens, 4, 2, 64, 16, types[0], track=True)
    for j in range(3):
        pool.keys[int(pool.table_cpu[0, j]), :, :, 2] = float("inf")
    q = torch.randn(2, 4, 64, generator=pool.g)
    q[0, :, 2] = -1.0
    q = q.to(dtypes(torch)[types[1]]).cuda()
    out, lse = torch.full_like(q, 7.0), torch.zeros(2, 4, device="cuda")
    w = torch.rand(2, 2, pool.capacity, generator=pool.g).cuda()
    before = w.clone()
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 2, dtype=KINDS[types[1]], lse=lse.data_ptr(), weights=w.data_ptr(),
                         weights_out=w.data_ptr())
    pool.cache.check()
    assert not bool(out[0].any()) and bool((lse[0] == -math.inf).all())
    assert torch.equal(w[0], before[0]) and torch.equal(w[1, :, 20:], before[1, :, 20:])
    assert bool(torch.isfinite(w[1]).all()) and abs(float((w[1] - before[1]).sum()) - 4) < 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("bad", ["one page", "every page"])
def test_slots_of_a_bad_page_receive_no_weight(gpu, types, bad):
    """Whatever an earlier call left in the workspace: what is not read adds nothing, and the other slots get the weights of an
    attention without it."""
    import torch
    n = 75
    pool = Pool(torch, [n], 4, 2, 64, 16, types[0], track=True)
    q = torch.randn(1, 4, 64, generator=pool.g).to(dtypes(torch)[types[1]]).cuda()
    out = torch.zeros_like(q)
    w = torch.zeros(1, 2, pool.capacity, device="cuda")

    def attend():
        pool.cache.attention(q.data_ptr(), out.data_ptr(), 1, dtype=KINDS[types[1]], weights=w.data_ptr(), weights_out=w.data_ptr())

    attend()  # leaves logits
    pool.cache.check()
    start = torch.rand(1, 2, pool.capacity, generator=pool.g)
    w.copy_(start)
    if bad == "one page":
        pool.table[0, 1] = pool.n_pages
        read = [t for t in range(n) if not 16 <= t < 32]
    else:
        pool.table[0, :5] = -1
        read = []
    attend()
    with pytest.raises(IndexError, match="page number"):
        pool.cache.check()
    got, want = w.cpu().double(), start.double()
    for h in range(2):
        _, _, x, dz, _ = head_reference(torch, q.cpu()[0, 2 * h:2 * h + 2], pool.k[0][h][read], pool.v[0][h][read], 1 / 8)
        want[0, h, read] += x.sum(0)
        tol = torch.zeros(pool.capacity, dtype=torch.float64)
        tol[read] = ((2 * dz + (n + 64) * EPS) * x).sum(0) + 6 * EPS * want[0, h, read]
        assert bool(((got[0, h] - want[0, h]).abs() <= tol).all())


@pytest.mark.gpu
def test_attention_leaves_room_behind_its_line_of_tiles(gpu):
    """42,966 rows over a table of 49,977 pages of 32 slots come to 2^31 - 2 places: the blocks' shares, rounded up, would pass
    32 bits."""
    import torch
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    cache = nb.PagedCache(p, p, p, p, sequences=1, max_pages=49977, n_pages=1, page_size=32, heads=1, kv_heads=1, head_dim=8,
                          max_rows=42966)
    with pytest.raises(nb.LengthError, match="split the call"):
        cache.attention(p, p, 42966, row_sequence=p)


@pytest.mark.gpu
def test_attention_refuses_lists_beyond_any_table(gpu):
    import torch
    pool = Pool(torch, [10, 20], 4, 2, 64, 16, "f16", bounds=True)
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    for n in (1 << 27, 1 << 60, (1 << 60) + 1, (1 << 63) - 1):
        with pytest.raises(nb.LengthError, match="paged: "):
            pool.cache.attention(p, p, 2, selected=p, n_selected=n)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("step", [2, 4, 8], ids=lambda s: f"+{s}")
@pytest.mark.parametrize("power", [23, 24, 25, 26, 27])
def test_logits_beyond_whole_numbers_stay_finite(gpu, types, power, step):
    """Logits of 2^23 and more, where fp32 counts in steps of 1 to 16: whatever the maximum in use rounds to, weights stay in
    their type's range.  The later half of the slots lies `step` (times log 2) higher, or the same where that is less than a
    step: outputs lie between the values of the two."""
    import torch
    n, rows, D = 256, 512, 64
    pool = Pool(torch, [n], 4, 1, D, 16, types[0], max_rows=rows, fill=False)
    k = torch.zeros(1, n, D)
    k[:, :, 0], k[:, n // 2:, 1] = 2.0 ** 14, step * 2.0 ** (14 - power)
    v = torch.ones(1, n, D)
    v[:, n // 2:] = 2.0
    pool.put(0, k.to(pool.keys.dtype), v.to(pool.keys.dtype), 0)
    q = torch.zeros(rows, 4, D)
    q[:, :, :2] = 1.0
    q, seq = q.to(dtypes(torch)[types[1]]).cuda(), torch.zeros(rows, dtype=torch.int32, device="cuda")
    out = torch.zeros_like(q)
    pool.cache.attention(q.data_ptr(), out.data_ptr(), rows, dtype=KINDS[types[1]], scale=2.0 ** (power - 14) * math.log(2.0),
                         row_sequence=seq.data_ptr())
    pool.cache.check()
    assert bool(((out >= 1.0) & (out <= 2.0)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_greatest_values_without_weight_add_nothing(gpu, types):
    """Tokens whose weight underflows (keys 200 nats below) may hold the greatest finite values."""
    import torch
    n = 60
    pool = Pool(torch, [n], 4, 1, 64, 16, types[0])
    most = torch.finfo(pool.values.dtype).max
    dead = [3, 17, 18, 40]
    for t in dead:
        page = int(pool.table_cpu[0, t // 16])
        pool.keys[page, 0, t % 16] = 0.0
        pool.keys[page, 0, t % 16, 5] = -1600.0
        pool.values[page, 0, t % 16] = most
    q = torch.randn(1, 4, 64, generator=pool.g)
    q[:, :, 5] = 1.0
    q = q.to(dtypes(torch)[types[1]]).cuda()
    out = torch.zeros_like(q)
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 1, dtype=KINDS[types[1]])
    pool.cache.check()
    keep = [t for t in range(n) if t not in dead]
    want, _, _, dz, mass = head_reference(torch, q.cpu()[0], pool.k[0][0][keep], pool.v[0][0][keep], 1 / 8)
    close_out(torch, out.cpu()[0], want, dz, mass, n, types[1])


# ---------------------------------------------------------------------------
# selection


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(5, 1, 136), (8, 1, 256), (16, 2, 160), (16, 1, 256), (32, 2, 200)], ids=str)
@pytest.mark.parametrize("page", [16, 1], ids=["block chooses", "scores in memory"])
def test_select_for_rows_of_wide_heads(gpu, shape, page):
    """Rows of given sequences, more than 4 query heads of more than 128 dims a kv head."""
    import torch
    H, KV, D = shape
    lens = [600, 130]
    pool = Pool(torch, lens, H, KV, D, page, "f16", bounds=True, max_rows=11)
    pool.cache.summarise()
    rows = [(0, 600), (0, 1), (0, 17), (1, 130), (1, 0), (0, 599), (0, 600), (1, 64), (0, 300), (0, 301), (1, 5)]
    q = torch.randn(len(rows), H, D, generator=pool.g).cuda()
    seq = torch.tensor([s for s, _ in rows], dtype=torch.int32, device="cuda")
    length = torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda")
    got = run_select(torch, pool, q, "f32", len(rows), 9, 1, 2, row_sequence=seq.data_ptr(), row_length=length.data_ptr())
    assert np.array_equal(got, select_reference(pool, q, rows, 9, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 1], ids=["block chooses", "scores in memory"])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_scores_beyond_fp32_stay_behind_the_pages_that_are_always_read(gpu, page, kind):
    """Infinite keys count as the largest finite float, whose products with a query pass fp32's range: such scores are equal to
    one another, below the sinks and the recent pages and above all others."""
    import torch
    pages = 40 if page == 16 else 700
    pool = Pool(torch, [pages * page], 4, 2, 64, page, kind, bounds=True)
    for j in (7, 9):
        pool.keys[int(pool.table_cpu[0, j]), :, 0, 3] = float("inf")
    pool.keys[int(pool.table_cpu[0, 11]), :, :, 5] = float("inf")  # every key of the page: no score above -inf
    pool.cache.summarise()
    q = torch.randn(1, 4, 64, generator=pool.g)
    q[:, :, 3], q[:, :, 5] = 3.0, -3.0
    q = q.cuda()
    for n, want in ((2, [0, pages - 1]), (3, [0, 7, pages - 1]), (4, [0, 7, 9, pages - 1])):
        got = run_select(torch, pool, q, "f32", 1, n, 1, 1)
        assert got.tolist() == [[want, want]]
    most = run_select(torch, pool, q, "f32", 1, pages - 1, 1, 1)
    assert most.tolist() == [[[j for j in range(pages) if j != 11]] * 2]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_bounds_hold_keys_far_below_the_unit(gpu, kind):
    """A key so small beside the page's greatest that it is no whole number of units: its bound is one unit, not none."""
    import torch
    pool = Pool(torch, [2], 1, 1, 16, 4, kind, bounds=True, fill=False)
    k = torch.zeros(2, 16)
    k[0, 3], k[1, 4] = 3e38, float("-inf")
    k[:, 5], k[:, 6] = 1e-30, -1e-30
    k[0, 7], k[1, 7], k[:, 8] = 1e-38, -1e-38, 1e-3
    k = k.to(dtypes(torch)[kind])
    pool.put(0, k[None], k[None], 0)
    pool.cache.summarise()
    pool.cache.check()
    check_bounds(pool, 0, 2)
    b = pool.bounds.cpu()[int(pool.table_cpu[0, 0]), 0]
    assert b[:, 5].tolist() == [1, 0] and b[:, 6].tolist() == [0, -1] and b[:, 7].tolist() == [1, -1]


# ---------------------------------------------------------------------------
# append


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_append_skips_rows_without_a_rotation(gpu, kind):
    """A position outside the table is reported, and its row stored nowhere; the other rows are."""
    import torch
    lens, H, KV, D = [6, 20, 9], 4, 2, 64
    pool = Pool(torch, lens, H, KV, D, 16, kind)
    q, k, v = (torch.randn(6, n, D, generator=pool.g).cuda() for n in (H, KV, KV))
    starts = torch.tensor([0, 2, 4, 6], dtype=torch.int32, device="cuda")
    seen = torch.tensor([1, 21, 9], dtype=torch.int32, device="cuda")  # positions -1, 0; 19, 20; 7, 8
    turn = torch.ones(20, D // 2, device="cuda"), torch.zeros(20, D // 2, device="cuda")
    q_out = torch.full_like(q, 7.0)
    w, at = torch.full((3, KV, pool.capacity), 5.0, device="cuda"), torch.full((3, KV, pool.capacity), -3, dtype=torch.int32, device="cuda")
    want = [x.clone() for x in (pool.keys, pool.values, q_out, w, at)]
    for row, (s, slot) in {1: (0, 5), 2: (1, 18), 4: (2, 7), 5: (2, 8)}.items():
        page = int(pool.table_cpu[s, slot // 16])
        want[0][page, :, slot % 16], want[1][page, :, slot % 16] = k[row].to(want[0].dtype), v[row].to(want[1].dtype)
        want[2][row], want[3][s, :, slot], want[4][s, :, slot] = q[row], 0.0, (0, 0, 19, 0, 7, 8)[row]
    want[4][0, :, 5] = 0
    pool.cache.append(q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), 6, 2, q_out=q_out.data_ptr(), cos=turn[0].data_ptr(),
                      sin=turn[1].data_ptr(), rope_rows=20, seen=seen.data_ptr(), positions=at.data_ptr(), weights=w.data_ptr())
    with pytest.raises(IndexError, match="rotation table"):
        pool.cache.check()
    for got, x in zip((pool.keys, pool.values, q_out, w, at), want):
        assert torch.equal(got.nan_to_num(77.0) if got.is_floating_point() else got, x.nan_to_num(77.0) if x.is_floating_point() else x)


@pytest.mark.gpu
def test_append_refuses_pages_whose_rows_it_cannot_count(gpu):
    """A page of 2^24 slots with 127 query heads a kv head has more rows than 32 bits count."""
    import torch
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()
    cache = nb.PagedCache(p, p, p, p, sequences=1, max_pages=1, n_pages=1, page_size=1 << 24, heads=127, kv_heads=1, head_dim=8)
    with pytest.raises(nb.LengthError, match="paged: "):
        cache.append(p, p, p, p, 1 << 24, 1 << 24, q_out=p)


# ---------------------------------------------------------------------------
# eviction


def eviction(torch, lens, max_pages=None, kv=2):
    pool = Pool(torch, lens, kv, kv, 64, 16, "f16", max_pages=max_pages)
    S, cap = len(lens), pool.capacity
    w = torch.rand(S, kv, cap, generator=pool.g)
    at = torch.arange(cap, dtype=torch.int32).expand(S, kv, cap).contiguous()
    return pool, w.cuda(), at.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("max_pages", [8, 600], ids=["a block", "a cluster"])
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("bad", ["length", "page"])
def test_evict_leaves_a_sequence_alone_that_it_cannot_serve(gpu, max_pages, in_place, bad):
    """A bad length or page number is reported, and nothing of its sequence changes; the other one is trimmed."""
    import torch
    pool, w, at = eviction(torch, [100, 90], max_pages)
    if bad == "length":
        pool.lengths[0] = pool.capacity + 1
    else:
        pool.table[0, 2] = -1
    seen = torch.tensor([100, 90], dtype=torch.int32, device="cuda")
    wo, po, left = (w, at, pool.lengths) if in_place else (torch.full_like(w, 9.0), torch.full_like(at, 9), torch.full_like(pool.lengths, 9))
    of = [x[0].clone() for x in (wo, po, left)]
    mine = pool.table_cpu[0, :7].long().cuda()
    before = pool.keys[mine].clone(), pool.values[mine].clone()
    want_w = w[1].cpu()
    pool.cache.evict(w.data_ptr(), at.data_ptr(), seen.data_ptr(), 50, sinks=2, recent=3, new_lengths=left.data_ptr(),
                     weights_out=wo.data_ptr(), positions_out=po.data_ptr())
    with pytest.raises(IndexError, match="length" if bad == "length" else "page number"):
        pool.cache.check()
    for got, x in zip((wo, po, left), of):
        assert torch.equal(got[0], x)
    assert torch.equal(pool.keys[mine].nan_to_num(7.0), before[0].nan_to_num(7.0))
    assert torch.equal(pool.values[mine].nan_to_num(7.0), before[1].nan_to_num(7.0))
    assert int(left[1]) == 50
    for h in range(2):
        key = want_w[h, :90].clone()
        key[:2], key[87:90] = 2.0, 2.0
        kept = key.sort(descending=True, stable=True).indices[:50]
        assert sorted(po.cpu()[1, h, :50].tolist()) == sorted(kept.tolist())
        assert bool((po.cpu()[1, h, 50:90] == -1).all())


# ---------------------------------------------------------------------------
# errors


@pytest.mark.gpu
def test_a_failed_call_leaves_no_error_for_the_next_one(gpu):
    """A workspace beyond the device's memory is refused, and the library's next call, which checks its launch, does not find
    that error."""
    import torch
    a, c = torch.ones(4096, device="cuda"), torch.zeros(16, 16, device="cuda")
    p = a.data_ptr()
    with pytest.raises(RuntimeError, match="workspace"):
        nb.PagedCache(p, p, p, p, sequences=65535, max_pages=1 << 20, n_pages=1, page_size=1 << 10, heads=64, kv_heads=1, head_dim=64,
                      track_weights=True)
    nb.matmul_f32_async(p, p, c.data_ptr(), 16, 64, 16, torch.cuda.current_stream().cuda_stream)
    assert bool((c == 64).all())


# ---------------------------------------------------------------------------
# the serving loop


@pytest.mark.gpu
def test_prompts_beyond_the_budget_keep_the_tokens_their_last_rows_attend_to(gpu):
    """The first trim, before any step: of each prompt's tokens those stay that its newest 32 rows give most weight (first
    layer, in 64 bits; a weight is a sum of 128 softmax weights in fp32, off by less than 1e-5 of the greatest)."""
    import torch
    from tests.test_paged_demo import D, HEADS, KV, LAYERS, setup as make
    lens, budget, sinks, recent = [100, 20, 70], 48, 2, 8
    demo, weights, prompts = make(torch, lens)
    session = demo.PagedSession(3, LAYERS, HEADS, KV, D, pages=20, max_pages=8, dtype=torch.float32, budget=budget, sinks=sinks,
                                recent=recent)
    demo.decode(session, weights, prompts, 1)
    session.check()
    assert session.length == [49, 21, 49]
    for s in (0, 2):
        n = lens[s]
        x = demo.norm(prompts[s].double()) @ weights[0][0].double()
        turn = torch.polar(torch.ones(n, 1, D // 2).double(), torch.arange(n)[:, None, None] * 10000.0 ** (
            -torch.arange(0, D, 2).double() / D)).cuda()
        qk = torch.view_as_real(torch.view_as_complex(x[:, :(HEADS + KV) * D].reshape(n, -1, D // 2, 2).contiguous()) * turn)
        qk = qk.reshape(n, HEADS + KV, D).transpose(0, 1)
        z = qk[:HEADS, n - 32:] @ qk[HEADS:].repeat_interleave(HEADS // KV, 0).transpose(1, 2) / D ** 0.5
        late = torch.arange(n, device="cuda") > torch.arange(n - 32, n, device="cuda")[:, None]
        w = torch.softmax(z.masked_fill(late, -math.inf), -1).sum(1).reshape(KV, -1, n).sum(1).cpu()
        for h in range(KV):
            kept = session.layers[0]["positions"][s, h, :budget].long().cpu()
            stays = torch.zeros(n, dtype=torch.bool)
            stays[kept] = True
            assert int(stays.sum()) == budget and bool(stays[:sinks].all()) and bool(stays[n - recent:].all())
            free = torch.ones(n, dtype=torch.bool)
            free[:sinks], free[n - recent:] = False, False
            assert float(w[h][stays & free].min()) >= float(w[h][~stays].max()) - 1e-5 * float(w[h].max())


@pytest.mark.gpu
def test_a_refused_extension_leaves_the_session_as_it_was(gpu):
    import torch
    from nutllm_b200 import paged_demo as demo
    session = demo.PagedSession(2, 1, 4, 2, 32, pages=6, max_pages=4)
    session.extend([20, 30])

    def state():
        return (list(session.length), list(session.seen), list(session.free), [list(p) for p in session.owned],
                session.table.tolist(), session.lengths.tolist())

    before = state()
    for news in ([20, 30], [0, 40], [65, 0]):  # more pages than are free, more than the table holds (two ways)
        with pytest.raises(RuntimeError, match="out of pages"):
            session.extend(news)
        assert state() == before
    assert session.extend([12, 1]).tolist() == [0, 12, 13] and session.lengths.tolist() == [32, 31]



def test_the_loop_refuses_empty_prompts():
    """Their first step would be fed another sequence's row."""
    import torch
    from nutllm_b200 import paged_demo as demo
    with pytest.raises(ValueError, match="empty prompt"):
        demo.decode(None, [], [torch.zeros(3, 8), torch.zeros(0, 8)], 1)


@pytest.mark.gpu
def test_numbers_that_do_not_fit_are_refused_like_others(gpu):
    """Arguments beyond the structures' fields raise ValueError from the call, as other wrong ones do."""
    import torch
    pool = Pool(torch, [10, 20], 4, 2, 64, 16, "f16", bounds=True)
    c, p = pool.cache, torch.zeros(4096, device="cuda").data_ptr()
    for call, args, more in ((c.attention, (p, p, 1 << 63), {}), (c.attention, (p, p, 2), dict(dtype=1 << 31)),
                             (c.attention, (p, p, 2), dict(scale=1e300)),
                             (c.select, (p, p, 2, 1 << 63), {}), (c.append, (0, p, p, p, 1 << 63, 1), {}),
                             (c.evict, (p, 0, 0, -1 << 64), dict(new_lengths=p, weights_out=p))):
        with pytest.raises(ValueError, match="paged: "):
            call(*args, **more)
