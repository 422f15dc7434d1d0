"""The paged KV cache (nut_paged_*): append, attention, page selection and
eviction against plain implementations.

What involves no rounding beyond a defined one (rotated and stored keys, key
bounds, chosen pages, evicted slots) is compared bit for bit.  Attention is
compared with the definition in 64 bits over the stored values, within
bounds that follow from fp32 arithmetic (eps = 2^-24):
  logit   |dz| <= (D + 8) eps scale sum_d |q_d k_d|  (D rounded sums, the
          scale, and operands split into terms that lose less than 8 eps)
  lse     |d| <= dz + (n + 8) eps + 4 eps |lse|       (n summed weights)
  out     |d| <= (2 dz + (2 n + 64) eps) sum_t w_t |v_t| + rounding to its type
  weight  |d| <= (2 dz + (n + 64) eps) w + 4 eps |total|
with dz the largest over the row's slots.
"""
import math

import numpy as np
import pytest

import nutllm_b200 as nb

EPS = 2.0 ** -24
KINDS = {"f32": nb.F32, "f16": nb.F16, "bf16": nb.BF16}


def dtypes(torch):
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


class Pool:
    """A pool of pages with its table; unused slots hold NaN and unused table
    entries numbers outside the pool."""

    def __init__(self, torch, lens, heads, kv, D, ps, kind, *, seed=0, order="contiguous", max_pages=None,
                 bounds=False, max_rows=0, track=False, spare=2, fill=True):
        self.t, self.lens, self.heads, self.kv, self.D, self.ps, self.kind = torch, list(lens), heads, kv, D, ps, kind
        g = torch.Generator().manual_seed(seed)
        self.g = g
        S = len(lens)
        per = [-(-n // ps) for n in lens]
        self.max_pages = max_pages or max(1, max(per) + 1)
        self.n_pages = sum(per) + spare
        perm = torch.randperm(self.n_pages, generator=g).tolist()
        table = torch.full((S, self.max_pages), 2 ** 31 - 7, dtype=torch.int32)
        table[:, -1] = -5
        k = 0
        for s, n in enumerate(per):
            for j in range(n):
                table[s, j] = perm[k]
                k += 1
        self.table_cpu = table
        dt = dtypes(torch)[kind]
        shape = (self.n_pages, kv, ps, D)
        if order == "contiguous":
            strides = None
        elif order == "slots first":  # [pages][slot][kv][D]
            strides = (ps * kv * D, D, kv * D)
        else:  # "padded": rows, heads and pages with room between
            pad = 16
            strides = ((D + pad) * (ps + 3) * kv + 32, (D + pad) * (ps + 3), D + pad)
        self.strides = strides

        def make():
            if strides is None:
                return torch.full(shape, float("nan"), dtype=dt, device="cuda")
            room = torch.full((strides[0] * self.n_pages + 64,), float("nan"), dtype=dt, device="cuda")
            return room.as_strided(shape, (strides[0], strides[1], strides[2], 1))

        self.keys, self.values = make(), make()
        self.k, self.v = [], []  # per sequence [kv][n][D], as stored
        for s, n in enumerate(lens):
            k = torch.randn(kv, n, D, generator=g).to(dt)
            v = torch.randn(kv, n, D, generator=g).to(dt)
            self.k.append(k)
            self.v.append(v)
            if fill and n:
                self.put(s, k, v, 0)
        self.table = table.cuda()
        self.lengths = torch.tensor(self.lens, dtype=torch.int32, device="cuda")
        self.bounds = torch.zeros(self.n_pages, kv, 2, D, dtype=torch.int8, device="cuda") if bounds else None
        self.scales = torch.zeros(self.n_pages, kv, device="cuda") if bounds else None
        s = strides or (0, 0, 0)
        self.cache = nb.PagedCache(
            self.keys.data_ptr(), self.values.data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(), sequences=S,
            max_pages=self.max_pages, n_pages=self.n_pages, page_size=ps, heads=heads, kv_heads=kv, head_dim=D,
            dtype=KINDS[kind], page_stride=s[0], head_stride=s[1], slot_stride=s[2],
            bounds=self.bounds.data_ptr() if bounds else 0, bound_scales=self.scales.data_ptr() if bounds else 0,
            max_rows=max_rows, track_weights=track)

    def put(self, s, k, v, first):
        for j in range(k.shape[1]):
            t = first + j
            page = int(self.table_cpu[s, t // self.ps])
            self.keys[page, :, t % self.ps] = k[:, j].cuda()
            self.values[page, :, t % self.ps] = v[:, j].cuda()

    def read(self, pool, s, n):
        """[kv][n][D] of a pool as it is now."""
        t = np.arange(n)
        pages = self.table_cpu[s].numpy()[t // self.ps]
        return pool.cpu()[pages, :, t % self.ps].permute(1, 0, 2)

    @property
    def capacity(self):
        return self.max_pages * self.ps


def head_reference(torch, q, k, v, scale):
    """64-bit attention of q [G][D] over k, v [n][D]: out, lse, w, and dz / sum w|v|."""
    q, k, v = q.double(), k.double(), v.double()
    n, D = k.shape
    if n == 0:
        return torch.zeros_like(q), torch.full((len(q),), -math.inf, dtype=torch.float64), torch.zeros(len(q), 0).double(), \
            torch.zeros(len(q), 1).double(), torch.zeros_like(q)
    z = q @ k.T * scale
    lse = torch.logsumexp(z, 1)
    w = torch.exp(z - lse[:, None])
    dz = ((D + 8) * EPS * abs(scale) * (q.abs() @ k.abs().T)).amax(1, keepdim=True)
    return w @ v, lse, w, dz, w @ v.abs()


def close_out(torch, got, want, dz, mass, n, kind):
    """`got` in its own type against 64 bits."""
    tol = (2 * dz + (2 * n + 64) * EPS) * mass + 1e-30
    if kind != "f32":  # half a unit in the last place, and of the smallest subnormal
        half = torch.finfo(dtypes(torch)[kind]).eps / 2
        tol = tol * (1 + half) + want.abs() * half + (2.0 ** -25 if kind == "f16" else 0.0)
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"error {float(err.max()):.3e}, worst over bound {float((err / tol).max()):.2f}"


def check_attention(torch, pool, q, out, lse, rows, scale, kind, listed=None):
    """rows: [(sequence, length)]; listed: [row][kv] page lists or None."""
    q, out = q.cpu(), out.cpu()
    lse = lse.cpu()
    G = pool.heads // pool.kv
    for r, (s, n) in enumerate(rows):
        for h in range(pool.kv):
            if listed is None:
                at = np.arange(n)
            else:
                at = np.concatenate([np.arange(j * pool.ps, min(n, (j + 1) * pool.ps)) for j in listed[r][h] if j >= 0]
                                    + [np.zeros(0, int)]).astype(int)
            sl = slice(h * G, (h + 1) * G)
            want, want_lse, _, dz, mass = head_reference(torch, q[r, sl], pool.k[s][h][at], pool.v[s][h][at], scale)
            close_out(torch, out[r, sl], want, dz, mass, len(at), kind)
            if len(at) == 0:
                assert bool((lse[r, sl] == -math.inf).all())
            else:
                tol = dz[:, 0] + (len(at) + 8) * EPS + 4 * EPS * want_lse.abs()
                assert bool(((lse[r, sl].double() - want_lse).abs() <= tol).all())


# ---------------------------------------------------------------------------
# append


def rotated(torch, x, pos, cos, sin):
    """fp32 rotation of neighbouring pairs with unfused products: x [heads][D]."""
    a, b = x[:, 0::2], x[:, 1::2]
    c, z = cos[pos], sin[pos]
    out = torch.empty_like(x)
    out[:, 0::2] = a * c - b * z
    out[:, 1::2] = a * z + b * c
    return out


def unit_of(top):
    if not top > 0:
        return 0.0
    u = 2.0 ** (math.frexp(top)[1] - 7)
    return max(2 * u if top > 127 * u else u, 2.0 ** -126)


def bounds_of(keys):
    """(int8 [2][D], unit) of one page's used keys [n][D]."""
    k = keys.double().numpy()
    k = np.where(np.isnan(k), 0.0, np.clip(k, -3.402823466e38, 3.402823466e38))
    most, least = k.max(0), k.min(0)
    u = unit_of(float(max(np.abs(most).max(), np.abs(least).max())))
    if u == 0:
        return np.zeros((2, k.shape[1]), np.int8), 0.0
    return np.stack([np.ceil(most / u), np.floor(least / u)]).astype(np.int8), u


def check_bounds(pool, s, n):
    for j in range(-(-n // pool.ps)):
        page = int(pool.table_cpu[s, j])
        k = pool.keys.cpu()[page, :, :min(pool.ps, n - j * pool.ps)]
        for h in range(pool.kv):
            want, u = bounds_of(k[h])
            assert np.array_equal(pool.bounds.cpu()[page, h].numpy(), want)
            assert float(pool.scales.cpu()[page, h]) == u


APPEND = [
    # lengths after, new rows, heads, kv, D, page, cache, rows, pool order
    ([1, 0, 17, 40], [1, 0, 1, 1], 4, 4, 32, 16, "f16", "f32", "contiguous"),
    ([37, 16, 33, 5], [20, 16, 1, 5], 8, 2, 64, 16, "bf16", "f32", "slots first"),
    ([100, 8], [100, 3], 6, 1, 48, 24, "f32", "f32", "padded"),
    ([70, 9], [9, 9], 12, 4, 80, 7, "f16", "f16", "padded"),
    ([65, 3, 0], [64, 2, 0], 2, 2, 256, 32, "bf16", "bf16", "contiguous"),
    ([600], [555], 16, 1, 8, 64, "f32", "f32", "slots first"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", APPEND, ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["rows", "packed"])
def test_append_is_exact(gpu, case, packed):
    import torch
    lens, news, H, KV, D, ps, kind, rkind, order = case
    pool = Pool(torch, [max(n, 1) for n in lens], H, KV, D, ps, kind, order=order, bounds=True, fill=False)
    pool.lens = lens
    pool.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    for s, (n, new) in enumerate(zip(lens, news)):
        if n > new:
            pool.put(s, pool.k[s][:, :n - new], pool.v[s][:, :n - new], 0)
    rdt, cdt = dtypes(torch)[rkind], dtypes(torch)[kind]
    rows, W = sum(news), (H + 2 * KV) * D
    x = torch.randn(rows, W, generator=pool.g).to(rdt)
    starts = torch.tensor([0] + np.cumsum(news).tolist(), dtype=torch.int32)
    offset = 11
    top = max(lens) + offset
    angle = torch.arange(top)[:, None].double() / 10000.0 ** (torch.arange(0, D, 2).double() / D)
    cos, sin = angle.cos().float(), angle.sin().float()
    if packed:
        dev = x.cuda()
        q, k, v = dev[:, :H * D], dev[:, H * D:(H + KV) * D], dev[:, (H + KV) * D:]
        strides = dict(q_stride=W, k_stride=W, v_stride=W, q_out_stride=W)
        q_out = q  # in place
    else:
        q, k, v = (t.contiguous().cuda() for t in (x[:, :H * D], x[:, H * D:(H + KV) * D], x[:, (H + KV) * D:]))
        strides, q_out = {}, torch.zeros_like(q)
    cap = pool.capacity
    positions = torch.full((len(lens), KV, cap), -3, dtype=torch.int32, device="cuda")
    weights = torch.full((len(lens), KV, cap), 5.0, device="cuda")
    before_k, before_v = pool.keys.cpu().clone(), pool.values.cpu().clone()
    dc, ds, dst = cos.cuda(), sin.cuda(), starts.cuda()
    seen = (pool.lengths + offset).to(torch.int32)
    pool.cache.append(q.data_ptr(), k.data_ptr(), v.data_ptr(), dst.data_ptr(), rows, max(news), dtype=KINDS[rkind],
                      cos=dc.data_ptr(), sin=ds.data_ptr(), rope_rows=top, seen=seen.data_ptr(), q_out=q_out.data_ptr(),
                      positions=positions.data_ptr(), weights=weights.data_ptr(), **strides)
    pool.cache.check()
    f = x.float().reshape(rows, H + 2 * KV, D)
    want_q = torch.empty(rows, H, D, dtype=rdt)
    want_pos, want_w = torch.full((len(lens), KV, cap), -3, dtype=torch.int32), torch.full((len(lens), KV, cap), 5.0)
    for s, (n, new) in enumerate(zip(lens, news)):
        for i in range(new):
            r, t = int(starts[s]) + i, n - new + i
            y = rotated(torch, f[r, :H + KV], t + offset, cos, sin)
            want_q[r] = y[:H].to(rdt)
            page = int(pool.table_cpu[s, t // ps])
            before_k[page, :, t % ps] = y[H:].to(cdt)
            before_v[page, :, t % ps] = f[r, H + KV:].to(cdt)
            want_pos[s, :, t] = t + offset
            want_w[s, :, t] = 0.0
    assert torch.equal(q_out.cpu().reshape(rows, H, D), want_q)
    assert torch.equal(before_k.nan_to_num(77.0), pool.keys.cpu().nan_to_num(77.0))
    assert torch.equal(before_v.nan_to_num(77.0), pool.values.cpu().nan_to_num(77.0))
    assert torch.equal(positions.cpu(), want_pos) and torch.equal(weights.cpu(), want_w)
    for s, n in enumerate(lens):
        if news[s]:
            # only the pages that received tokens are summarised
            first = (n - news[s]) // ps
            for j in range(first, -(-n // ps)):
                page = int(pool.table_cpu[s, j])
                for h in range(KV):
                    want, u = bounds_of(pool.keys.cpu()[page, h, :min(ps, n - j * ps)])
                    assert np.array_equal(pool.bounds.cpu()[page, h].numpy(), want)
                    assert float(pool.scales.cpu()[page, h]) == u
    pool.cache.summarise()
    pool.cache.check()
    for s, n in enumerate(lens):
        check_bounds(pool, s, n)


@pytest.mark.gpu
def test_append_keys_only_unrotated_and_extreme_values(gpu):
    """No queries, no table; fp16 saturates and keeps NaN; bounds of special keys."""
    import torch
    pool = Pool(torch, [3], 2, 1, 8, 4, "f16", bounds=True, fill=False)
    k = torch.tensor([[1e6, -1e6, float("nan"), 0.0, -0.0, 3e-8, float("inf"), 1.0],
                      [0.0] * 8, [127.0, -127.0, 2.0, 0.5, 1.0, 0.0, -float("inf"), 65504.0]], device="cuda")
    v = torch.ones(3, 8, device="cuda")
    starts = torch.tensor([0, 3], dtype=torch.int32, device="cuda")
    pool.cache.append(0, k.data_ptr(), v.data_ptr(), starts.data_ptr(), 3, 3)
    pool.cache.check()
    page = int(pool.table_cpu[0, 0])
    want = k.cpu().clamp(-65504, 65504).half()
    got = pool.keys.cpu()[page, 0, :3]
    assert torch.equal(got.nan_to_num(-9.0), want.nan_to_num(-9.0))
    check_bounds(pool, 0, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("top", [127.0, 127.5, 126.99, 64.0, 63.9, 1e-40, 2.0 ** -126, 3.4e38, 254.0, 255.0, 0.0])
def test_bounds_unit_is_the_least_power_of_two(gpu, top):
    import torch
    pool = Pool(torch, [2], 1, 1, 8, 4, "f32", bounds=True, fill=False)
    k = torch.zeros(2, 8)
    k[0, 3], k[1, 4], k[1, 5] = top, -top, top / 3
    pool.put(0, k[None], k[None], 0)
    pool.cache.summarise()
    pool.cache.check()
    check_bounds(pool, 0, 2)


# ---------------------------------------------------------------------------
# attention

TYPES = [("f32", "f32"), ("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")]
SHAPES = [(8, 1, 64, 16), (4, 4, 128, 16), (6, 6, 48, 24), (16, 1, 32, 8), (9, 3, 80, 5), (20, 2, 96, 64), (4, 2, 256, 32),
          (2, 2, 8, 1), (5, 1, 160, 3)]
LENGTHS = [0, 1, 2, 7, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 130, 257, 0]


def run_attention(torch, pool, rkind, rows, *, seed=3, gain=1.0, scale=0.0, stream=0, **more):
    """rows: how many; returns q, out, lse."""
    g = torch.Generator().manual_seed(seed)
    q = (gain * torch.randn(rows, pool.heads, pool.D, generator=g)).to(dtypes(torch)[rkind]).cuda()
    out = torch.full_like(q, float("nan"))
    lse = torch.full((rows, pool.heads), float("nan"), device="cuda")
    torch.cuda.synchronize()
    pool.cache.attention(q.data_ptr(), out.data_ptr(), rows, dtype=KINDS[rkind], lse=lse.data_ptr(), scale=scale,
                         stream=stream, **more)
    pool.cache.check(stream)
    return q, out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_of_ragged_lengths(gpu, types, shape):
    import torch
    H, KV, D, ps = shape
    pool = Pool(torch, LENGTHS, H, KV, D, ps, types[0], seed=D, order=["contiguous", "slots first", "padded"][D % 3])
    q, out, lse = run_attention(torch, pool, types[1], len(LENGTHS))
    check_attention(torch, pool, q, out, lse, list(enumerate(LENGTHS)), 1 / math.sqrt(D), types[1])


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("lens", [[9001], [3000, 1, 0, 4097], [5]], ids=str)
def test_attention_splits_long_sequences(gpu, types, lens):
    import torch
    pool = Pool(torch, lens, 8, 2, 64, 32, types[0])
    q, out, lse = run_attention(torch, pool, types[1], len(lens), gain=3.0)
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / 8, types[1])
    again = run_attention(torch, pool, types[1], len(lens), gain=3.0)
    assert torch.equal(again[1].cpu(), out.cpu()) and torch.equal(again[2].cpu(), lse.cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_attention_of_peaked_and_scaled_logits(gpu, types):
    """Logits of several hundred: the running maximum has to move; tiny queries; a given scale."""
    import torch
    lens = [200, 64, 3]
    for gain, scale in ((100.0, 0.5), (1e-3, 2.0), (1.0, -0.25)):
        pool = Pool(torch, lens, 4, 2, 64, 16, types[0])
        q, out, lse = run_attention(torch, pool, types[1], 3, gain=gain, scale=scale)
        check_attention(torch, pool, q, out, lse, list(enumerate(lens)), scale, types[1])


@pytest.mark.gpu
def test_attention_of_large_queries_keeps_its_precision(gpu):
    """fp32 queries beyond fp16's range on an fp16 cache."""
    import torch
    lens = [90, 33]
    pool = Pool(torch, lens, 4, 2, 64, 16, "f16")
    q, out, lse = run_attention(torch, pool, "f32", 2, gain=1e6, scale=1e-6)
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), float(np.float32(1e-6)), "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_attention_of_a_prompts_rows(gpu, types):
    """Rows that share a sequence, each with its own length, in any order; row strides."""
    import torch
    pool = Pool(torch, [77, 40], 6, 2, 64, 16, types[0], max_rows=64)
    rows = [(0, 77), (1, 13), (0, 1), (1, 40), (0, 0), (0, 16), (1, 17), (0, 50)]
    seq = torch.tensor([s for s, _ in rows], dtype=torch.int32, device="cuda")
    length = torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda")
    dt = dtypes(torch)[types[1]]
    W = 6 * 64
    wide = torch.randn(len(rows), W + 24, generator=pool.g).to(dt).cuda()
    out = torch.zeros(len(rows), W + 8, dtype=dt, device="cuda")
    lse = torch.zeros(len(rows), 6, device="cuda")
    pool.cache.attention(wide.data_ptr(), out.data_ptr(), len(rows), dtype=KINDS[types[1]], q_stride=W + 24,
                         out_stride=W + 8, lse=lse.data_ptr(), row_sequence=seq.data_ptr(), row_length=length.data_ptr())
    pool.cache.check()
    check_attention(torch, pool, wide[:, :W].reshape(-1, 6, 64), out[:, :W].reshape(-1, 6, 64), lse, rows, 1 / 8, types[1])
    assert not bool(out[:, W:].any())


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("shape", [(8, 2, 64, 16), (3, 3, 40, 5), (16, 1, 128, 32)], ids=str)
def test_attention_over_listed_pages(gpu, types, shape):
    """Any order, gaps, a last page half full, rows and heads that list nothing."""
    import torch
    H, KV, D, ps = shape
    lens = [ps * 9 + 3, ps * 4, 1, 0]
    pool = Pool(torch, lens, H, KV, D, ps, types[0], order="padded")
    n = 6
    rng = np.random.default_rng(5)
    listed = np.full((len(lens), KV, n), -1, np.int32)
    for r, L in enumerate(lens):
        pages = -(-L // ps)
        for h in range(KV):
            if (r + h) % 3 == 2:
                continue
            pick = rng.permutation(max(pages, 1))[:n]
            listed[r, h, rng.permutation(n)[:len(pick)]] = pick
    dev = torch.from_numpy(listed).cuda()
    q, out, lse = run_attention(torch, pool, types[1], len(lens), selected=dev.data_ptr(), n_selected=n)
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / math.sqrt(D), types[1], listed)


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
def test_attention_accumulates_weights(gpu, types, in_place):
    import torch
    lens = [300, 1, 0, 65]
    pool = Pool(torch, lens, 20, 2, 64, 16, types[0], track=True)
    cap = pool.capacity
    start = torch.rand(len(lens), 2, cap, generator=pool.g)
    weights = start.cuda()
    to = weights if in_place else torch.full_like(weights, 9.0)
    q, out, lse = run_attention(torch, pool, types[1], len(lens), weights=weights.data_ptr(), weights_out=to.data_ptr())
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / 8, types[1])
    got = to.cpu().double()
    for s, n in enumerate(lens):
        for h in range(2):
            _, _, w, dz, _ = head_reference(torch, q.cpu()[s, h * 10:(h + 1) * 10], pool.k[s][h], pool.v[s][h], 1 / 8)
            if n:
                want = start[s, h, :n].double() + w.sum(0)
                tol = ((2 * dz + (n + 64) * EPS) * w).sum(0) + 14 * EPS * want
                assert bool(((got[s, h, :n] - want).abs() <= tol).all())
            rest = start[s, h, n:] if in_place else torch.full((cap - n,), 9.0)
            assert torch.equal(to.cpu()[s, h, n:], rest)


@pytest.mark.gpu
def test_attention_passes_infinities_on(gpu):
    """A key that makes one logit -inf takes no weight; NaN in a used slot reaches its rows and no others."""
    import torch
    pool = Pool(torch, [20, 20], 2, 2, 16, 16, "f32")
    page = int(pool.table_cpu[0, 0])
    pool.keys[page, 0, 4, :] = 0.0
    pool.keys[page, 0, 4, 2] = float("inf")
    pool.k[0][0, 4] = pool.keys[page, 0, 4].cpu()
    page1 = int(pool.table_cpu[1, 1])
    pool.values[page1, 1, 1, 0] = float("nan")
    q = torch.randn(2, 2, 16, generator=pool.g).abs()
    q[0, 0, 2] = -1.0
    q = q.cuda()
    out, lse = torch.zeros_like(q), torch.zeros(2, 2, device="cuda")
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 2, lse=lse.data_ptr())
    pool.cache.check()
    keep = [t for t in range(20) if t != 4]
    want, want_lse, _, dz, mass = head_reference(torch, q.cpu()[0, :1], pool.k[0][0][keep], pool.v[0][0][keep], 0.25)
    close_out(torch, out.cpu()[0, :1], want, dz, mass, 19, "f32")
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(out[1, 0]).all())
    assert bool(torch.isnan(out[1, 1, 0])) and bool(torch.isfinite(out[1, 1, 1:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("types", [("f16", "f32"), ("f16", "f16"), ("bf16", "f32"), ("bf16", "bf16")], ids=lambda t: "-".join(t))
def test_infinite_keys_in_16_bits_keep_their_sign(gpu, types):
    """The lower terms of a split query do not turn an infinite logit into NaN: -inf takes no weight."""
    import torch
    pool = Pool(torch, [40], 4, 1, 64, 16, types[0])
    pool.keys[int(pool.table_cpu[0, 1]), 0, 3, 5] = float("inf")  # slot 19
    dt = dtypes(torch)[types[1]]
    q = torch.randn(1, 4, 64, generator=pool.g)
    q[:, :, 5] = -torch.rand(1, 4, generator=pool.g) - 0.1
    q = q.to(dt).cuda()
    out, lse = torch.zeros_like(q), torch.zeros(1, 4, device="cuda")
    pool.cache.attention(q.data_ptr(), out.data_ptr(), 1, dtype=KINDS[types[1]], lse=lse.data_ptr())
    pool.cache.check()
    keep = [t for t in range(40) if t != 19]
    want, want_lse, _, dz, mass = head_reference(torch, q.cpu()[0], pool.k[0][0][keep], pool.v[0][0][keep], 1 / 8)
    close_out(torch, out.cpu()[0], want, dz, mass, 39, types[1])
    assert bool(((lse.cpu()[0].double() - want_lse).abs() <= dz[:, 0] + 48 * EPS + 4 * EPS * want_lse.abs()).all())


@pytest.mark.gpu
def test_one_sequence_among_many_rows_and_places(gpu):
    """More rows than threads of a block, most of them idle, on a table far wider than the lengths."""
    import torch
    lens = [0] * 300
    for s, n in ((0, 1), (7, 33), (128, 70), (255, 16), (299, 129)):
        lens[s] = n
    pool = Pool(torch, lens, 4, 2, 64, 16, "bf16", max_pages=1000)
    q, out, lse = run_attention(torch, pool, "f32", 300)
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / 8, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f16", "f32"])
def test_offsets_pass_32_bits(gpu, kind):
    """A pool of more than 2^32 elements, the sequence in its first and last pages."""
    import torch
    D, KV, ps = 128, 4, 64
    per = KV * ps * D
    n_pages = 2 ** 32 // per + 5
    dt = dtypes(torch)[kind]
    keys, values = (torch.empty(n_pages, KV, ps, D, dtype=dt, device="cuda") for _ in range(2))
    n = 150
    table_cpu = torch.tensor([[n_pages - 1, 0, n_pages - 3]], dtype=torch.int32)
    table, lengths = table_cpu.cuda(), torch.tensor([n], dtype=torch.int32, device="cuda")
    cache = nb.PagedCache(keys.data_ptr(), values.data_ptr(), table.data_ptr(), lengths.data_ptr(), sequences=1, max_pages=3,
                          n_pages=n_pages, page_size=ps, heads=8, kv_heads=KV, head_dim=D, dtype=KINDS[kind])
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(n, KV, D, generator=g) for _ in range(2))
    starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    dk, dv = k.cuda(), v.cuda()
    cache.append(0, dk.data_ptr(), dv.data_ptr(), starts.data_ptr(), n, n)
    q = torch.randn(1, 8, D, generator=g)
    dq, out = q.cuda(), torch.zeros(1, 8, D, device="cuda")
    cache.attention(dq.data_ptr(), out.data_ptr(), 1)
    w_in = torch.arange(3 * ps, dtype=torch.float32, device="cuda").repeat(KV, 1)[None].contiguous()
    w_out, left = torch.zeros_like(w_in), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.check()
    for h in range(KV):
        want, _, _, dz, mass = head_reference(torch, q[0, 2 * h:2 * h + 2], k[:, h].to(dt), v[:, h].to(dt), 1 / math.sqrt(D))
        close_out(torch, out.cpu()[0, 2 * h:2 * h + 2], want, dz, mass, n, "f32")
    cache.evict(w_in.data_ptr(), 0, 0, 100, new_lengths=left.data_ptr(), weights_out=w_out.data_ptr())
    cache.check()
    # weights ascend: slots 50.. stay, and 0..49 take the tokens of 100..149
    assert torch.equal(keys[n_pages - 1, :, :50].cpu(), k[100:150].to(dt).permute(1, 0, 2))
    assert int(left) == 100


@pytest.mark.gpu
def test_calls_follow_their_stream_and_replay_in_graphs(gpu):
    import torch
    lens = [500, 90]
    pool = Pool(torch, lens, 8, 2, 64, 16, "f16", bounds=True)
    side = torch.cuda.Stream()
    q, out, lse = run_attention(torch, pool, "f32", 2, stream=side.cuda_stream)
    check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / 8, "f32")
    pool.cache.summarise()
    chosen = torch.zeros(2, 2, 5, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        pool.cache.select(q.data_ptr(), chosen.data_ptr(), 2, 5, stream=side.cuda_stream)
        pool.cache.attention(q.data_ptr(), out.data_ptr(), 2, lse=lse.data_ptr(), selected=chosen.data_ptr(), n_selected=5,
                             stream=side.cuda_stream)
    for seed in (7, 8):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(seed)))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        pool.cache.check()
        check_attention(torch, pool, q, out, lse, list(enumerate(lens)), 1 / 8, "f32", chosen.cpu().numpy())


@pytest.mark.gpu
def test_replays_read_what_has_changed_since(gpu):
    """A whole step as a graph, replayed while every input it reads is rewritten in place, and the same without a graph: each
    kernel starts while the one before it runs, and must not meet stale values."""
    import torch
    H, KV, D, ps, S, n = 8, 2, 64, 16, 3, 4
    pool = Pool(torch, [150, 60, 33], H, KV, D, ps, "f16", bounds=True, track=True, max_pages=20, spare=40)
    pool.cache.summarise()
    side = torch.cuda.Stream()
    dev = dict(device="cuda")
    k, v, q = torch.zeros(S, KV, D, **dev), torch.zeros(S, KV, D, **dev), torch.zeros(S, H, D, **dev)
    starts = torch.arange(S + 1, dtype=torch.int32, **dev)
    cos, sin = torch.zeros(400, D // 2, **dev), torch.zeros(400, D // 2, **dev)
    turned, out, sparse = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(q)
    chosen = torch.zeros(S, KV, n, dtype=torch.int32, **dev)
    w, w_out = torch.zeros(S, KV, pool.capacity, **dev), torch.zeros(S, KV, pool.capacity, **dev)
    c = pool.cache

    def step(stream, wait):
        def then(f, *a, **kw):
            f(*a, **kw)
            if wait:
                torch.cuda.synchronize()
        then(c.append, q.data_ptr(), k.data_ptr(), v.data_ptr(), starts.data_ptr(), S, 1, cos=cos.data_ptr(), sin=sin.data_ptr(),
             rope_rows=400, q_out=turned.data_ptr(), stream=stream)
        then(c.attention, turned.data_ptr(), out.data_ptr(), S, weights=w.data_ptr(), weights_out=w_out.data_ptr(), stream=stream)
        then(c.select, turned.data_ptr(), chosen.data_ptr(), S, n, stream=stream)
        then(c.attention, turned.data_ptr(), sparse.data_ptr(), S, selected=chosen.data_ptr(), n_selected=n, stream=stream)

    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(side.cuda_stream, False)
    results = (turned, out, sparse, chosen, w_out, pool.bounds, pool.scales)
    g = torch.Generator(device="cuda").manual_seed(4)
    for i in range(12):
        # new values in the same places; the table is shuffled and the lengths move on
        for x in (k, v, q, cos, sin, w):
            x.copy_(torch.randn(x.shape, generator=g, **dev))
        pool.keys.copy_(torch.randn(pool.keys.shape, generator=g, **dev))
        pool.values.copy_(torch.randn(pool.values.shape, generator=g, **dev))
        pool.table[:, :10] = torch.randperm(pool.n_pages, generator=g, **dev)[:30].int().reshape(3, 10)
        pool.lengths.copy_(torch.tensor([150 + i % 5, 61 - 7 * (i % 3), 33 + i], dtype=torch.int32))
        torch.cuda.synchronize()
        before = [x.clone() for x in (pool.keys, pool.values)]
        got = []
        for way in ("apart", "together", "graph"):
            pool.keys.copy_(before[0])
            pool.values.copy_(before[1])
            if way == "graph":
                graph.replay()
            else:
                step(torch.cuda.current_stream().cuda_stream, way == "apart")
            torch.cuda.synchronize()
            got.append([x.clone() for x in results])
        pool.cache.check()
        for way in (1, 2):
            assert all(torch.equal(a, b) for a, b in zip(got[0], got[way])), (i, way)


# ---------------------------------------------------------------------------
# selection


def select_reference(pool, q, rows, n, sinks, recent):
    """The definition, in Python's exact arithmetic over the stored bounds."""
    q = q.cpu().double().numpy()
    G = pool.heads // pool.kv
    out = np.full((len(rows), pool.kv, n), -1, np.int32)
    bounds, scales = pool.bounds.cpu().numpy().astype(np.int64), pool.scales.cpu().double().numpy()
    for r, (s, L) in enumerate(rows):
        P = -(-L // pool.ps)
        for h in range(pool.kv):
            score = []
            for j in range(P):
                if j < sinks or j >= P - recent:
                    score.append(math.inf)
                    continue
                page = int(pool.table_cpu[s, j])
                best = -math.inf
                for g in range(G):
                    x = q[r, h * G + g]
                    u = unit_of(float(np.abs(x).max()))
                    xi = np.rint(x / u).astype(np.int64) if u else np.zeros(pool.D, np.int64)
                    best = max(best, u * int(np.maximum(xi * bounds[page, h, 0], xi * bounds[page, h, 1]).sum()))
                score.append(best * scales[page, h])
            order = sorted(range(P), key=lambda j: (-score[j], j))[:n]
            out[r, h, :len(order)] = sorted(order)
    return out


SELECT = [
    # lengths, heads, kv, D, page, cache, rows, n, sinks, recent
    ([400, 33, 0, 1], 8, 2, 64, 16, "f16", "f32", 6, 1, 2),
    ([700], 4, 4, 128, 8, "bf16", "bf16", 20, 0, 1),
    ([300, 299], 6, 2, 48, 4, "f32", "f32", 64, 2, 0),
    ([129, 90], 16, 1, 256, 3, "f16", "f16", 7, 0, 0),
    ([64, 640], 3, 3, 40, 16, "bf16", "f32", 4, 9, 9),
    ([5000], 12, 4, 8, 2, "f16", "f32", 1200, 1, 1),
]


def run_select(torch, pool, q, rkind, rows, n, sinks, recent, **more):
    got = torch.full((rows, pool.kv, n), 99, dtype=torch.int32, device="cuda")
    pool.cache.select(q.data_ptr(), got.data_ptr(), rows, n, dtype=KINDS[rkind], sink_pages=sinks, recent_pages=recent, **more)
    pool.cache.check()
    return got.cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("case", SELECT, ids=str)
def test_select_is_exact(gpu, case):
    import torch
    lens, H, KV, D, ps, kind, rkind, n, sinks, recent = case
    pool = Pool(torch, lens, H, KV, D, ps, kind, bounds=True, order="slots first")
    pool.cache.summarise()
    q = torch.randn(len(lens), H, D, generator=pool.g).to(dtypes(torch)[rkind]).cuda()
    want = select_reference(pool, q, list(enumerate(lens)), n, sinks, recent)
    assert np.array_equal(run_select(torch, pool, q, rkind, len(lens), n, sinks, recent), want)


@pytest.mark.gpu
def test_select_breaks_ties_downwards_and_takes_rows_of_a_prompt(gpu):
    import torch
    lens = [16 * 40 + 1, 100]
    pool = Pool(torch, lens, 4, 2, 64, 16, "f16", bounds=True, max_rows=8)
    for j in range(5, 30):  # many pages with the same keys
        pool.keys[int(pool.table_cpu[0, j])] = pool.keys[int(pool.table_cpu[0, 4])]
    pool.cache.summarise()
    rows = [(0, 641), (1, 100), (0, 320), (0, 17), (1, 0), (0, 641)]
    q = torch.randn(len(rows), 4, 64, generator=pool.g)
    q[5] = 0.0  # every score 0: the lowest pages
    q = q.cuda()
    seq = torch.tensor([s for s, _ in rows], dtype=torch.int32, device="cuda")
    length = torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda")
    got = run_select(torch, pool, q, "f32", len(rows), 12, 1, 1, row_sequence=seq.data_ptr(), row_length=length.data_ptr())
    want = select_reference(pool, q, rows, 12, 1, 1)
    assert np.array_equal(got, want)
    assert got[5, 0].tolist() == list(range(11)) + [40]


@pytest.mark.gpu
def test_select_scores_bound_the_logits(gpu):
    """With all pages' bounds, a page outside the choice has no logit above its score, up to the queries' rounding."""
    import torch
    pool = Pool(torch, [600], 8, 2, 64, 16, "f16", bounds=True)
    pool.cache.summarise()
    q = torch.randn(1, 8, 64, generator=pool.g)
    for h in range(2):
        for g in range(4):
            x = q[0, 4 * h + g].double()
            u = unit_of(float(x.abs().max()))
            xi = torch.round(x / u)
            for j in range(38):
                page = int(pool.table_cpu[0, j])
                b = pool.bounds.cpu()[page, h].double()
                score = u * float(pool.scales[page, h]) * float(torch.maximum(xi * b[0], xi * b[1]).sum())
                k = pool.k[0][h][16 * j:16 * j + 16].double()
                slack = float((0.5 * u * k.abs().sum(1)).max())
                assert float((k @ x).max()) <= score + slack + 1e-9


# ---------------------------------------------------------------------------
# eviction


def evict_reference(pool, weights, positions, seen, budget, sinks, recent):
    """(kept source slot of each new slot, new lengths) by sorting."""
    out, left = {}, []
    for s, n in enumerate(pool.lens):
        m = min(n, budget)
        left.append(m)
        for h in range(pool.kv):
            def key(t):
                p = int(positions[s, h, t]) if positions is not None else 0
                if (sinks and p < sinks) or (recent and p >= int(seen[s]) - recent):
                    return math.inf
                w = float(weights[s, h, t])
                return -math.inf if math.isnan(w) else w
            nan_last = sorted(range(n), key=lambda t: (-key(t), math.isnan(float(weights[s, h, t])) and key(t) == -math.inf, t))
            kept = sorted(nan_last[:m])
            source = list(range(m))
            tail = [t for t in kept if t >= m]
            low = set(kept)
            for t in range(m):
                if t not in low:
                    source[t] = tail.pop(0)
            out[s, h] = source
    return out, left


EVICT = [
    # lengths, kv, D, page, cache, budget, sinks, recent
    ([50, 20, 0, 33], 2, 64, 16, "f16", 32, 2, 5),
    ([200], 4, 128, 16, "bf16", 199, 0, 1),
    ([777, 64, 65], 1, 48, 24, "f32", 64, 0, 0),
    ([40, 41], 3, 8, 5, "f16", 10, 4, 20),
    ([30, 1], 2, 32, 8, "f32", 0, 1, 1),
    ([3000, 2500], 2, 16, 32, "bf16", 1024, 4, 128),
    ([10], 2, 256, 4, "f32", 100, 4, 4),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", EVICT, ids=str)
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
@pytest.mark.parametrize("tied", [False, True], ids=["distinct", "ties"])
def test_evict_is_exact(gpu, case, in_place, tied):
    import torch
    lens, KV, D, ps, kind, budget, sinks, recent = case
    pool = Pool(torch, lens, KV, KV, D, ps, kind, order="padded", bounds=True)
    cap, S = pool.capacity, len(lens)
    g = pool.g
    w = torch.randint(0, 3, (S, KV, cap), generator=g).float() if tied else torch.randn(S, KV, cap, generator=g).exp()
    if not tied and max(lens) > 30:
        w[0, 0, 3], w[0, 0, 7], w[0, -1, 9] = float("nan"), float("inf"), -1.0
    pos = torch.rand(S, KV, cap + 50, generator=g).argsort(-1)[..., :cap].int().contiguous()
    seen = torch.tensor([cap + 50 - s for s in range(S)], dtype=torch.int32)
    protects = bool(sinks or recent)
    dw, dp, dseen = w.cuda(), pos.cuda(), seen.cuda()
    wo = dw if in_place else torch.full_like(dw, 7.0)
    po = dp if in_place else torch.full_like(dp, 7)
    left = pool.lengths if in_place else torch.zeros(S, dtype=torch.int32, device="cuda")
    source, want_left = evict_reference(pool, w, pos if protects else None, seen, budget, sinks, recent)
    before_k, before_v = pool.keys.cpu().clone(), pool.values.cpu().clone()
    pool.cache.evict(dw.data_ptr(), dp.data_ptr() if protects else 0, dseen.data_ptr() if recent else 0, budget, sinks=sinks,
                     recent=recent, new_lengths=left.data_ptr(), weights_out=wo.data_ptr(),
                     positions_out=po.data_ptr() if protects else 0)
    pool.cache.check()
    assert left.cpu().tolist() == want_left
    want_w = w.clone() if in_place else torch.full_like(w, 7.0)
    want_p = pos.clone() if in_place else torch.full_like(pos, 7)
    for s, n in enumerate(lens):
        for h in range(KV):
            src, m = source[s, h], want_left[s]
            assert torch.equal(pool.read(pool.keys, s, m)[h], pool.k[s][h][src])
            assert torch.equal(pool.read(pool.values, s, m)[h], pool.v[s][h][src])
            want_w[s, h, :m], want_w[s, h, m:n] = w[s, h][src], 0.0
            want_p[s, h, :m], want_p[s, h, m:n] = pos[s, h][src], -1
            # the slots given up keep what they held
            for t in range(m, n):
                page = int(pool.table_cpu[s, t // ps])
                assert torch.equal(pool.keys[page, h, t % ps].cpu(), before_k[page, h, t % ps])
                assert torch.equal(pool.values[page, h, t % ps].cpu(), before_v[page, h, t % ps])
    assert torch.equal(wo.cpu().nan_to_num(-5.0), want_w.nan_to_num(-5.0))
    if protects:
        assert torch.equal(po.cpu(), want_p)
    if in_place:
        pool.cache.summarise()
        pool.cache.check()
        for s, m in enumerate(want_left):
            check_bounds(pool, s, m)


@pytest.mark.gpu
def test_eviction_leaves_the_attention_to_the_kept_tokens(gpu):
    """Weights from the attention, eviction, and the attention over what is left."""
    import torch
    lens, budget = [300, 120], 100
    pool = Pool(torch, lens, 8, 2, 64, 16, "f16", track=True)
    w = torch.zeros(2, 2, pool.capacity, device="cuda")
    pos = torch.arange(pool.capacity, dtype=torch.int32, device="cuda").expand(2, 2, -1).contiguous()
    seen = pool.lengths.clone()
    for seed in (1, 2):
        run_attention(torch, pool, "f32", 2, seed=seed, weights=w.data_ptr(), weights_out=w.data_ptr())
    source, _ = evict_reference(pool, w.cpu(), pos.cpu(), seen.cpu(), budget, 4, 32)
    pool.cache.evict(w.data_ptr(), pos.data_ptr(), seen.data_ptr(), budget, sinks=4, recent=32,
                     new_lengths=pool.lengths.data_ptr(), weights_out=w.data_ptr(), positions_out=pos.data_ptr())
    q, out, lse = run_attention(torch, pool, "f32", 2, seed=9)
    pool.k = [torch.stack([pool.k[s][h][source[s, h]] for h in range(2)]) for s in range(2)]
    pool.v = [torch.stack([pool.v[s][h][source[s, h]] for h in range(2)]) for s in range(2)]
    check_attention(torch, pool, q, out, lse, [(0, 100), (1, 100)], 1 / 8, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("lens,page,n", [([10001], 2, 700), ([9000, 300, 8193 * 2], 2, 5000)], ids=str)
def test_select_among_thousands_of_pages(gpu, lens, page, n):
    import torch
    pool = Pool(torch, lens, 4, 1, 8, page, "f16", bounds=True, fill=False)
    for s in range(len(lens)):
        t = torch.arange(lens[s])
        pages = pool.table_cpu[s].long()[t // page].cuda()
        pool.keys[pages, :, (t % page).cuda()] = pool.k[s].permute(1, 0, 2).cuda()
    pool.cache.summarise()
    q = torch.randn(len(lens), 4, 8, generator=pool.g).cuda()
    want = select_reference(pool, q, list(enumerate(lens)), n, 1, 2)
    assert np.array_equal(run_select(torch, pool, q, "f32", len(lens), n, 1, 2), want)


@pytest.mark.gpu
@pytest.mark.parametrize("tied", [False, True], ids=["distinct", "ties"])
@pytest.mark.parametrize("lens,budget", [([40001, 9000, 0, 5], 3000), ([33000], 32999), ([8200, 8193], 8192)], ids=str)
def test_evict_from_long_caches(gpu, lens, budget, tied):
    """Capacities beyond what one block holds."""
    import torch
    KV, D, ps = 2, 8, 64
    pool = Pool(torch, lens, KV, KV, D, ps, "f16", fill=False)
    for s, n in enumerate(lens):
        t = torch.arange(n)
        pages = pool.table_cpu[s].long()[t // ps].cuda()
        pool.keys[pages, :, (t % ps).cuda()] = pool.k[s].permute(1, 0, 2).cuda()
        pool.values[pages, :, (t % ps).cuda()] = pool.v[s].permute(1, 0, 2).cuda()
    S, cap, g = len(lens), pool.capacity, pool.g
    w = torch.randint(0, 3, (S, KV, cap), generator=g).float() if tied else torch.randn(S, KV, cap, generator=g).exp()
    pos = torch.rand(S, KV, cap, generator=g).argsort(-1).int()
    seen = torch.full((S,), cap, dtype=torch.int32)
    dw, dp, dseen = w.cuda(), pos.cuda(), seen.cuda()
    pool.cache.evict(dw.data_ptr(), dp.data_ptr(), dseen.data_ptr(), budget, sinks=4, recent=100,
                     new_lengths=pool.lengths.data_ptr(), weights_out=dw.data_ptr(), positions_out=dp.data_ptr())
    pool.cache.check()
    source, left = evict_reference(pool, w, pos, seen, budget, 4, 100)
    assert pool.lengths.cpu().tolist() == left
    for s, n in enumerate(lens):
        m = left[s]
        for h in range(KV):
            src = source[s, h]
            assert torch.equal(pool.read(pool.keys, s, m)[h], pool.k[s][h][src])
            assert torch.equal(pool.read(pool.values, s, m)[h], pool.v[s][h][src])
            assert torch.equal(dw.cpu()[s, h, :m], w[s, h][src]) and not bool(dw.cpu()[s, h, m:n].any())
            assert torch.equal(dp.cpu()[s, h, :m], pos[s, h][src]) and bool((dp.cpu()[s, h, m:n] == -1).all())


# ---------------------------------------------------------------------------
# refusals


def view(**change):
    v = dict(keys=256, values=256, table=256, lengths=256, sequences=1, max_pages=1, n_pages=1, page_size=16, heads=4,
             kv_heads=2, head_dim=64)
    v.update(change)
    return v


@pytest.mark.parametrize("change,error", [
    (dict(keys=0), ValueError), (dict(values=0), ValueError), (dict(table=0), ValueError), (dict(lengths=0), ValueError),
    (dict(keys=8), ValueError), (dict(values=264), ValueError), (dict(sequences=0), ValueError), (dict(page_size=0), ValueError),
    (dict(heads=3), ValueError), (dict(head_dim=12), ValueError), (dict(head_dim=264), ValueError), (dict(head_dim=0), ValueError),
    (dict(dtype=3), ValueError), (dict(dtype=-1), ValueError), (dict(bounds=256), ValueError), (dict(bound_scales=256), ValueError),
    (dict(page_stride=4096), ValueError), (dict(page_stride=4096, head_stride=1024, slot_stride=66), ValueError),
    (dict(page_stride=-4096, head_stride=1024, slot_stride=64), ValueError), (dict(max_rows=-1), ValueError),
    (dict(max_pages=1 << 25), nb.LengthError), (dict(max_pages=1 << 20, page_size=1 << 11), nb.LengthError),
    (dict(sequences=70000), nb.LengthError), (dict(n_pages=1 << 31), nb.LengthError),
], ids=str)
def test_create_refuses_before_any_device_work(change, error):
    with pytest.raises(error, match="paged: "):
        nb.PagedCache(**view(**change))


def test_null_handles_are_refused():
    lib = nb.cuda_lib()
    for name, kind in (("append", nb.PagedAppendArgs), ("attention", nb.PagedAttentionArgs), ("select", nb.PagedSelectArgs),
                       ("evict", nb.PagedEvictArgs)):
        assert getattr(lib, f"nut_paged_{name}")(None, kind(), None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_summarise(None, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_error(None, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_create(None, 0, None) == nb.NUT_INVALID_ARGUMENT
    assert lib.nut_paged_destroy(None) == nb.NUT_OK


@pytest.mark.gpu
def test_calls_refuse_wrong_arguments(gpu):
    import torch
    pool = Pool(torch, [10, 20], 4, 2, 64, 16, "f16")
    c = pool.cache
    x = torch.zeros(4096, device="cuda")
    p = x.data_ptr()

    def refuse(error, call, *a, **k):
        with pytest.raises(error, match="paged: "):
            call(*a, **k)

    refuse(ValueError, c.attention, 0, p, 2)
    refuse(ValueError, c.attention, p, 0, 2)
    refuse(ValueError, c.attention, p, p, -1)
    refuse(nb.LengthError, c.attention, p, p, 3)
    refuse(ValueError, c.attention, p, p, 2, dtype=nb.BF16)
    refuse(ValueError, c.attention, p, p, 2, q_stride=255)
    refuse(ValueError, c.attention, p, p, 2, out_stride=-256)
    refuse(ValueError, c.attention, p, p, 2, scale=float("nan"))
    refuse(ValueError, c.attention, p, p, 2, selected=p, n_selected=0)
    refuse(ValueError, c.attention, p, p, 2, weights=p)
    refuse(ValueError, c.attention, p, p, 2, weights=p, weights_out=p)  # not tracked
    refuse(ValueError, c.select, p, p, 2, 1)  # no bounds
    refuse(ValueError, c.summarise)
    refuse(ValueError, c.append, p, p, p, p, 1, 1)  # q without q_out
    refuse(ValueError, c.append, 0, 0, p, p, 1, 1)
    refuse(ValueError, c.append, 0, p, p, 0, 1, 1)
    refuse(ValueError, c.append, 0, p, p, p, -1, 1)
    refuse(ValueError, c.append, 0, p, p, p, 1, 1, cos=p)
    refuse(ValueError, c.append, 0, p, p, p, 1, 1, cos=p, sin=p)  # empty table
    refuse(ValueError, c.append, 0, p, p, p, 1, 1, k_stride=127)
    refuse(nb.LengthError, c.append, 0, p, p, p, 1, 1000)
    refuse(ValueError, c.evict, 0, 0, 0, 4, new_lengths=p, weights_out=p)
    refuse(ValueError, c.evict, p, 0, 0, -1, new_lengths=p, weights_out=p)
    refuse(ValueError, c.evict, p, p, 0, 4, new_lengths=p, weights_out=p)  # positions alone
    refuse(ValueError, c.evict, p, 0, 0, 4, new_lengths=p, weights_out=p, sinks=1)
    refuse(ValueError, c.evict, p, p, 0, 4, new_lengths=p, weights_out=p, positions_out=p, recent=1)
    tracked = Pool(torch, [10, 20], 4, 2, 64, 16, "f16", track=True, bounds=True)
    refuse(ValueError, tracked.cache.attention, p, p, 2, weights=p, weights_out=p, selected=p, n_selected=1)
    refuse(ValueError, tracked.cache.attention, p, p, 2, weights=p, weights_out=p, row_sequence=p)
    refuse(ValueError, tracked.cache.select, p, p, 2, 0)
    refuse(ValueError, tracked.cache.select, p, p, 2, 1, sink_pages=-1)
    c.attention(p, p, 0)  # nothing to do
    c.append(0, p, p, p, 0, 0)
    torch.cuda.synchronize()
    c.check()


@pytest.mark.gpu
def test_the_device_reports_what_it_cannot_serve(gpu):
    """Wrong numbers in device memory are met by the kernels' own checks: the work is skipped and reported once."""
    import torch
    lens = [40, 33]
    pool = Pool(torch, lens, 4, 2, 64, 16, "f16", max_rows=4)
    good = pool.table.clone()
    q = torch.randn(2, 4, 64, generator=pool.g).cuda()
    out, lse = torch.zeros_like(q), torch.zeros(2, 4, device="cuda")

    def attend(**more):
        pool.cache.attention(q.data_ptr(), out.data_ptr(), 2, lse=lse.data_ptr(), **more)

    def reported(text):
        with pytest.raises(IndexError, match=text):
            pool.cache.check()
        pool.cache.check()  # cleared

    for bad in (-1, pool.n_pages, 2 ** 31 - 1):
        pool.table[0, 1] = bad
        attend()
        reported("page number")
    pool.table.copy_(good)
    for bad in (-1, pool.capacity + 1):
        pool.lengths[0] = bad
        attend()
        assert bool((lse[0] == -math.inf).all()) and not bool(out[0].any())
        reported("length")
    pool.lengths[0] = 40
    seq = torch.tensor([2, 1], dtype=torch.int32, device="cuda")
    attend(row_sequence=seq.data_ptr())
    reported("sequence")
    k = torch.randn(3, 2, 64, device="cuda")
    for bad in ([0, 4, 5], [0, 2, 1], [0, 3, 3]):  # beyond the rows, descending, more than max_new
        starts = torch.tensor(bad, dtype=torch.int32, device="cuda")
        pool.cache.append(0, k.data_ptr(), k.data_ptr(), starts.data_ptr(), 3, 2)
        reported("starts")
    cos = torch.ones(4, 32, device="cuda")
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    pool.cache.append(0, k.data_ptr(), k.data_ptr(), starts.data_ptr(), 2, 1, cos=cos.data_ptr(), sin=cos.data_ptr(), rope_rows=4)
    reported("rotation table")
    attend()
    pool.cache.check()


# groups of every width share products between rows, or do not
PACKED = [(1, 1), (2, 1), (6, 2), (8, 2), (10, 2), (7, 1), (16, 2), (18, 2)]


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 1], ids=["block chooses", "scores in memory"])
@pytest.mark.parametrize("heads,kv", PACKED)
def test_select_for_rows_of_mixed_sequences(gpu, heads, kv, page):
    """Neighbouring rows of one sequence and of others, of unequal lengths, in blocks of whole and of ragged size."""
    import torch
    lens = [600, 130, 0]
    pool = Pool(torch, lens, heads, kv, 32, page, "f16", bounds=True, max_rows=21)
    pool.cache.summarise()
    rows = [(0, 600), (0, 1), (0, 17), (1, 130), (1, 0), (0, 599), (0, 600), (1, 64),
            (2, 0), (1, 130), (0, 300), (0, 301), (0, 302), (0, 303), (1, 5), (1, 6),
            (1, 129), (0, 33), (0, 600), (0, 16), (1, 100)]
    q = torch.randn(len(rows), heads, 32, generator=pool.g).cuda()
    seq = torch.tensor([s for s, _ in rows], dtype=torch.int32, device="cuda")
    length = torch.tensor([n for _, n in rows], dtype=torch.int32, device="cuda")
    got = run_select(torch, pool, q, "f32", len(rows), 9, 1, 2, row_sequence=seq.data_ptr(), row_length=length.data_ptr())
    assert np.array_equal(got, select_reference(pool, q, rows, 9, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("length", [300, 700, 9000])
def test_select_writes_distinct_pages_whatever_the_scores(gpu, length, scale):
    """Scales that no summary writes: the choice is arbitrary, but of n pages of the row, in order, and no more."""
    import torch
    pool = Pool(torch, [length], 4, 2, 8, 1, "f16", bounds=True)
    pool.cache.summarise()
    pool.scales[::3] = scale
    if math.isnan(scale):
        pool.scales.view(torch.int32)[::6] = 0x7fffffff
    q = torch.randn(1, 4, 8, generator=pool.g).cuda()
    for n in (1, 40, length - 1):
        got = torch.full((1, 2, n + 8), 99999, dtype=torch.int32, device="cuda")
        pool.cache.select(q.data_ptr(), got.data_ptr(), 1, n, dtype=KINDS["f32"], sink_pages=1, recent_pages=1)
        pool.cache.check()
        flat = got.cpu().numpy().reshape(-1)
        assert (flat[2 * n:] == 99999).all()
        for chosen in flat[:2 * n].reshape(2, n):
            assert (np.diff(chosen) > 0).all() and chosen[0] >= 0 and chosen[-1] < length
