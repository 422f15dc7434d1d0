"""The paged key/value cache and the operators that work on it, case by case.

A serving loop keeps the keys and values of many sequences in one pool of
fixed-size pages.  Four operators work on that pool: `append` (rotate new
queries and keys, store keys and values, refresh the pages' key bounds),
`attend` (one new token per sequence over its pages, with the attention
weight each cached token received where the caller tracks it), `sparse`
(score pages by their key bounds, keep the best for each query and kv head,
attend to those only) and `evict` (drop the tokens that received least
weight, filling their slots from the cache's tail).

`run` computes a case in plain torch operations, or with the framework's
operators where `own` is true.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---------------------------------------------------------------------------
# cases


def listed():
    return [
        # One token of one chat: every layer of every step makes this call,
        # so its latency is what counts.
        dict(name="append token", op="append", sequences=1, length=37, new=1, heads=32, kv_heads=4,
             head_dim=64, page=16, cache="f16", rows="f32", bounds=False, track=False, offset=0),
        # A decode step of a full batch whose caches lost tokens to eviction
        # (positions run ahead of the slots).
        dict(name="append batch", op="append", sequences=64, length=1024, new=1, heads=32, kv_heads=32,
             head_dim=128, page=16, cache="bf16", rows="bf16", bounds=False, track=True, offset=100),
        # A prefill batch of prompts of unequal lengths behind cached prefixes.
        dict(name="append prompts", op="append", sequences=12, length=1003, new=1000, heads=32, kv_heads=8,
             head_dim=128, page=16, cache="f16", rows="f32", bounds=True, track=False, offset=0),
        # The first steps of one chat.
        dict(name="attend short", op="attend", sequences=1, length=37, heads=32, kv_heads=4,
             head_dim=64, page=16, cache="f16", rows="f32", idle=0, weights=False),
        # A serving batch at ragged lengths, two of its places idle.
        dict(name="attend batch", op="attend", sequences=64, length=4096, heads=32, kv_heads=8,
             head_dim=128, page=16, cache="bf16", rows="bf16", idle=2, weights=False),
        # One long document; the weights feed a later eviction.
        dict(name="attend long", op="attend", sequences=1, length=131071, heads=32, kv_heads=8,
             head_dim=128, page=64, cache="f16", rows="f32", idle=0, weights=True),
        # A small model on an fp32 cache, pages that are no power of two.
        dict(name="attend f32", op="attend", sequences=6, length=1536, heads=6, kv_heads=6,
             head_dim=48, page=24, cache="f32", rows="f32", idle=1, weights=True),
        # Sparse decode where the context has only just outgrown the budget.
        dict(name="sparse short", op="sparse", sequences=1, queries=1, length=2043, heads=32, kv_heads=4,
             head_dim=64, page=16, cache="f16", rows="f32", budget=32, sinks=1, recent=2),
        # Sparse decode of a batch of long contexts.
        dict(name="sparse batch", op="sparse", sequences=32, queries=1, length=32768, heads=32, kv_heads=8,
             head_dim=128, page=32, cache="bf16", rows="bf16", budget=64, sinks=1, recent=4),
        # The last chunk of a prompt, every token choosing its own pages.
        dict(name="sparse prompt", op="sparse", sequences=1, queries=256, length=8190, heads=32, kv_heads=8,
             head_dim=128, page=16, cache="f16", rows="f32", budget=64, sinks=1, recent=2),
        # One chat that reached its budget.
        dict(name="evict one", op="evict", sequences=1, length=768, heads=32, kv_heads=4,
             head_dim=64, page=16, cache="f16", budget=512, sinks=4, recent=128),
        # A batch trimmed back to its budget; the shorter ones keep all they have.
        dict(name="evict batch", op="evict", sequences=64, length=5000, heads=32, kv_heads=8,
             head_dim=128, page=16, cache="bf16", budget=2048, sinks=4, recent=512),
    ]


SHAPES = [(32, 4, 64), (32, 32, 128), (32, 8, 128), (6, 6, 48), (16, 2, 80), (24, 8, 96),
          (16, 1, 128), (8, 4, 256), (12, 4, 32)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges, no dearer than the dearest listed one of its operator."""
    op = rng.choice(["append", "attend", "sparse", "evict"])
    caps = [_cost(c) for c in listed() if c["op"] == op]
    cap = max(caps)
    while True:
        heads, kv_heads, head_dim = rng.choice(SHAPES)
        cache = rng.choice(["f32", "f16", "bf16"])
        c = dict(op=op, sequences=_log(rng, 1, 64), length=_log(rng, 1, 60000), heads=heads, kv_heads=kv_heads,
                 head_dim=head_dim, page=rng.choice([8, 16, 24, 32, 64]), cache=cache)
        if op != "evict":
            c["rows"] = rng.choice(["f32", cache])
        if op == "append":
            c.update(new=_log(rng, 1, 1024), bounds=rng.random() < 0.5, track=rng.random() < 0.5, offset=rng.choice([0, 100]))
            c["length"] = max(c["length"], c["new"])
        elif op == "attend":
            c.update(idle=min(rng.randrange(3), c["sequences"] - 1), weights=rng.random() < 0.5)
        elif op == "sparse":
            c.update(queries=_log(rng, 1, 256) if c["sequences"] == 1 else 1, budget=_log(rng, 2, 256), sinks=rng.randrange(2),
                     recent=rng.randrange(1, 5))
        else:
            c.update(budget=_log(rng, 16, 4096), sinks=rng.choice([0, 4]), recent=_log(rng, 1, 512))
        if _cost(c) <= cap:
            return c


# ---------------------------------------------------------------------------
# what a case has to move and compute


def _lengths(c):
    """The lengths of a case's sequences, in no particular order."""
    n, top = c["sequences"], c["length"]
    low = c.get("new", 1) if c["op"] == "append" else 1
    got = [max(low, (top * (i + 1)) // n) for i in range(n)]
    for i in range(c.get("idle", 0)):
        got[i] = 0
    return got


def _news(c):
    """How many tokens an append brings to each sequence."""
    n, top = c["sequences"], c["new"]
    return [max(1, (top * (i + 1)) // n) for i in range(n)]


def _pages_of(length, page):
    return -(-length // page)


def work(c):
    e, D, H, KV, ps = BYTES[c["cache"]], c["head_dim"], c["heads"], c["kv_heads"], c["page"]
    r = BYTES[c.get("rows", "f32")]
    lens = _lengths(c)
    if c["op"] == "append":
        rows = sum(_news(c))
        # rows in, rotated queries out, keys and values stored, one cos/sin row a token
        b = rows * ((2 * H + 2 * KV) * D * r + 2 * KV * D * e + D * 4)
        if c["bounds"]:
            b += sum(-(-n // ps) for n in _news(c)) * KV * (2 * D + 4)
        if c["track"]:
            b += rows * KV * 8
        return {"bytes": b, "flops": rows * (H + KV) * D * 3}
    if c["op"] == "attend":
        b = sum(lens) * KV * D * 2 * e + 2 * c["sequences"] * H * D * r + c["sequences"] * H * 4
        b += sum(_pages_of(n, ps) for n in lens) * 4
        if c["weights"]:
            b += sum(lens) * KV * 8
        return {"bytes": b, "flops": sum(lens) * H * D * 4}
    if c["op"] == "sparse":
        q = c["queries"]
        pages = [_pages_of(n, ps) for n in lens]
        kept = [min(c["budget"], p) for p in pages]
        # each sequence's bounds once, each query's chosen pages (a prompt's queries share
        # one cache: no more than the cache itself)
        b = sum(pages) * KV * (2 * D + 4)
        b += sum(min(k * q, p) * ps for k, p in zip(kept, pages)) * KV * D * 2 * e
        b += c["sequences"] * q * (2 * H * D * r + H * 4 + KV * c["budget"] * 4)
        return {"bytes": b, "flops": q * (sum(pages) * H * D * 4 + sum(kept) * ps * H * D * 4)}
    moved = sum((n - c["budget"]) * c["budget"] // n for n in lens if n > c["budget"])
    # weights and positions read and written, keys and values of the kept tail moved
    return {"bytes": KV * (sum(lens) * 16 + moved * 4 * D * e), "flops": KV * sum(lens)}


def _cost(c):
    w = work(c)
    cost = max(w["bytes"], w["flops"] / 50)
    if c["op"] == "sparse":  # the plain form holds every query's pages at once
        cost = max(cost, c["sequences"] * c["queries"] * min(c["budget"], _pages_of(c["length"], c["page"])) * c["page"]
                   * c["kv_heads"] * c["head_dim"] / 4)
    if c["op"] in ("append", "evict", "sparse"):  # the pool that has to be made
        cost = max(cost, sum(_lengths(c)) * c["kv_heads"] * c["head_dim"] * BYTES[c["cache"]] / 16)
    if c["op"] in ("attend", "evict"):  # padded forms
        cost = max(cost, c["sequences"] * c["length"] * c["kv_heads"] * c["head_dim"])
    return cost


# ---------------------------------------------------------------------------
# inputs


def _pool(c, s, g):
    """A pool of pages holding every sequence's cache in shuffled pages, the table and the lengths."""
    dev, ps, KV, D = "cuda", c["page"], c["kv_heads"], c["head_dim"]
    lens = torch.tensor(_lengths(c), dtype=torch.int32, device=dev)
    lens = lens[torch.randperm(c["sequences"], generator=g, device=dev)] if c["op"] != "append" else lens
    per = max(1, _pages_of(c["length"], ps))
    pages = [max(1, _pages_of(n, ps)) for n in lens.tolist()]
    total = sum(pages) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    first = torch.tensor([0] + pages, device=dev).cumsum(0)[:-1]
    at = first[:, None] + torch.arange(per, device=dev)
    used = torch.arange(per, device=dev) < torch.tensor(pages, device=dev)[:, None]
    # places behind a sequence's last page hold its first page's number: they are not read
    s["table"] = order[torch.where(used, at, first[:, None])].contiguous()
    s["lengths"] = lens
    dt = DTYPES[c["cache"]]
    s["keys"] = torch.randn(total, KV, ps, D, generator=g, device=dev, dtype=dt)
    s["values"] = torch.randn(total, KV, ps, D, generator=g, device=dev, dtype=dt)


def _page_fill(s):
    """How many slots of each page of the pool are filled."""
    ps = s["keys"].shape[2]
    per = s["table"].shape[1]
    fill = (s["lengths"].long()[:, None] - ps * torch.arange(per, device="cuda")).clamp(0, ps)
    got = torch.zeros(s["keys"].shape[0], dtype=torch.long, device="cuda")
    return got.scatter_reduce_(0, s["table"].long().reshape(-1), fill.reshape(-1), "amax")


def _two_to(power):
    """2 to a whole power in 32 bits, exactly."""
    return ((power + 127) << 23).to(torch.int32).view(torch.float32)


def _bounds(keys, fill):
    """For pages [n, kv, slots, D]: each dimension's least and greatest key over the filled slots, in 8 bits with
    one power of two for each page and kv head, the least rounded down and the greatest up."""
    inside = (torch.arange(keys.shape[2], device=keys.device) < fill[:, None])[:, None, :, None]
    least = torch.where(inside, keys, torch.inf).amin(2).float()
    most = torch.where(inside, keys, -torch.inf).amax(2).float()
    empty = (fill == 0)[:, None, None]
    least, most = least.masked_fill(empty, 0), most.masked_fill(empty, 0)
    top = torch.maximum(least.abs(), most.abs()).amax(-1)
    part, power = torch.frexp(top)
    power = torch.where(part > 127 / 128, power - 6, power - 7)
    scale = torch.where(top > 0, _two_to(power.clamp(min=-126)), 0.0)
    inv = torch.where(top > 0, 1 / scale, 0.0)[..., None]
    return torch.stack((torch.ceil(most * inv), torch.floor(least * inv)), 2).to(torch.int8), scale


def _handle(c, s, rows):
    """The framework's handle on the pool, as its user makes it once."""
    import nutllm_b200 as nb
    p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    return nb.PagedCache(p["keys"], p["values"], p["table"], p["lengths"], sequences=c["sequences"],
                         max_pages=s["table"].shape[1], n_pages=s["keys"].shape[0], page_size=c["page"], heads=c["heads"],
                         kv_heads=c["kv_heads"], head_dim=c["head_dim"], dtype=_code(nb, c["cache"]),
                         bounds=p.get("bounds", 0), bound_scales=p.get("bound_scales", 0), max_rows=rows,
                         track_weights=bool(c.get("weights")))


def _code(nb, name):
    return {"f32": nb.F32, "f16": nb.F16, "bf16": nb.BF16}[name]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dev, H, KV, D = "cuda", c["heads"], c["kv_heads"], c["head_dim"]
    s = {"case": c}
    _pool(c, s, g)
    rows = c["sequences"]
    if c["op"] == "append":
        news = torch.tensor(_news(c), device=dev)
        s["starts"] = torch.cat((news.new_zeros(1), news.cumsum(0))).to(torch.int32)
        rows = sum(_news(c))
        # the rows of one [q; k; v] projection
        s["qkv"] = torch.randn(rows, (H + 2 * KV) * D, generator=g, device=dev).to(DTYPES[c["rows"]])
        s["seen"] = s["lengths"] + c["offset"]
        angle = torch.arange(c["length"] + c["offset"], device=dev, dtype=torch.float64)[:, None] / 10000.0 ** (
            torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
        s["cos"], s["sin"] = angle.cos().float().contiguous(), angle.sin().float().contiguous()
        s["q_out"] = torch.empty(rows, H, D, device=dev, dtype=DTYPES[c["rows"]])
        if c["track"]:
            cap = s["table"].shape[1] * c["page"]
            s["positions"] = torch.full((c["sequences"], KV, cap), -1, device=dev, dtype=torch.int32)
            s["weights"] = torch.rand(c["sequences"], KV, cap, generator=g, device=dev)
        if c["bounds"]:
            s["bounds"] = torch.zeros(s["keys"].shape[0], KV, 2, D, device=dev, dtype=torch.int8)
            s["bound_scales"] = torch.zeros(s["keys"].shape[0], KV, device=dev)
    elif c["op"] in ("attend", "sparse"):
        if c["op"] == "sparse":
            rows = c["sequences"] * c["queries"]
            s["bounds"], s["bound_scales"] = _bounds(s["keys"], _page_fill(s))
            s["selected"] = torch.empty(rows, KV, c["budget"], device=dev, dtype=torch.int32)
            if c["queries"] > 1:  # the last tokens of one prompt, each seeing itself and what precedes it
                s["row_sequence"] = torch.zeros(rows, device=dev, dtype=torch.int32)
                s["row_length"] = (s["lengths"] - rows + 1 + torch.arange(rows, device=dev, dtype=torch.int32)).clamp(min=0)
        s["q"] = (2 * torch.randn(rows, H, D, generator=g, device=dev)).to(DTYPES[c["rows"]])
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, H, device=dev)
        if c.get("weights"):
            cap = s["table"].shape[1] * c["page"]
            s["weights"] = torch.rand(c["sequences"], KV, cap, generator=g, device=dev)
            s["weights_out"] = torch.zeros_like(s["weights"])
    else:
        cap = s["table"].shape[1] * c["page"]
        # weight collected over many steps has a long tail; positions are those of the tokens that
        # earlier evictions left, in the order in which those filled the slots
        s["weights"] = torch.exp(2 * torch.randn(c["sequences"], KV, cap, generator=g, device=dev))
        s["positions"] = torch.rand(c["sequences"], KV, cap + 100, generator=g, device=dev).argsort(-1)[..., :cap].to(torch.int32)
        s["seen"] = torch.full((c["sequences"],), cap + 100, device=dev, dtype=torch.int32)
        s["weights_out"] = torch.zeros_like(s["weights"])
        s["positions_out"] = torch.zeros_like(s["positions"])
        s["lengths_out"] = torch.zeros_like(s["lengths"])
    s["rows"] = rows
    s["handle"] = _handle(c, s, rows) if own else None
    return s


# ---------------------------------------------------------------------------
# one pass


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["op"]](s)


def _rotate(x, cos, sin):
    """Rotation of neighbouring pairs: x [rows, heads, D] in 32 bits."""
    a, b = x[..., 0::2], x[..., 1::2]
    cos, sin = cos[:, None], sin[:, None]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).reshape(x.shape)


def _plain_append(s):
    c = s["case"]
    H, KV, D, ps, n = c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["rows"]
    qkv = s["qkv"].float().reshape(n, H + 2 * KV, D)
    row = torch.arange(n, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(s["starts"][1:].contiguous(), row, right=True)
    slot = s["lengths"][seq] - s["starts"][seq + 1] + row
    at = (slot + (s["seen"] - s["lengths"])[seq]).long()
    cos, sin = s["cos"][at], s["sin"][at]
    s["q_out"].copy_(_rotate(qkv[:, :H], cos, sin))
    page, inside = s["table"][seq, (slot // ps).long()].long(), (slot % ps).long()
    s["keys"][page, :, inside] = _rotate(qkv[:, H:H + KV], cos, sin).to(s["keys"].dtype)
    s["values"][page, :, inside] = qkv[:, H + KV:].to(s["values"].dtype)
    got = {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}
    if c["track"]:
        s["positions"][seq, :, slot.long()] = at.to(torch.int32)[:, None]
        s["weights"][seq, :, slot.long()] = 0.0
        got.update(positions=s["positions"], weights=s["weights"])
    if c["bounds"]:
        touched = page.unique()
        s["bounds"][touched], s["bound_scales"][touched] = _bounds(s["keys"][touched], _page_fill(s)[touched])
        got["bounds"] = s["bounds"] * s["bound_scales"][..., None, None]
    return got


def _softmax(logits, valid):
    """(weights, log-sum-exp), with zeros and -inf for a row that sees nothing."""
    logits = torch.where(valid, logits, -torch.inf)
    top = logits.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    e = torch.exp(logits - top)
    total = e.sum(-1, keepdim=True)
    return torch.where(total > 0, e / total, 0.0), (top + torch.log(total)).squeeze(-1)


def _plain_attend(s):
    c = s["case"]
    H, KV, D, n = c["heads"], c["kv_heads"], c["head_dim"], s["rows"]
    table = s["table"].long()
    cap = table.shape[1] * c["page"]
    keys = s["keys"][table].transpose(1, 2).reshape(n, KV, cap, D).float()
    q = s["q"].float().reshape(n, KV, H // KV, D)
    valid = (torch.arange(cap, device="cuda") < s["lengths"][:, None])[:, None, None]
    w, lse = _softmax(torch.matmul(q, keys.transpose(-1, -2)) / math.sqrt(D), valid)
    del keys
    values = s["values"][table].transpose(1, 2).reshape(n, KV, cap, D).float()
    out = torch.matmul(w, values).reshape(n, H, D)
    s["out"].copy_(out)
    s["lse"].copy_(lse.reshape(n, H))
    got = {"out": s["out"], "lse": s["lse"]}
    if c["weights"]:
        s["weights_out"].copy_(torch.where(valid[:, :, 0], s["weights"] + w.sum(2), 0.0))
        got["weights"] = s["weights_out"]
    return got


def _plain_sparse(s):
    c = s["case"]
    H, KV, D, ps, n, k = c["heads"], c["kv_heads"], c["head_dim"], c["page"], s["rows"], c["budget"]
    many = c["queries"] > 1
    length = (s["row_length"] if many else s["lengths"]).long()
    table = s["table"].long()
    P = table.shape[1]
    q = s["q"].float().reshape(n, KV, H // KV, D)
    # queries in 8 bits, one power of two a head
    top = q.abs().amax(-1, keepdim=True)
    part, power = torch.frexp(top)
    power = torch.where(part > 127 / 128, power - 6, power - 7)
    scale = torch.where(top > 0, _two_to(power.clamp(min=-126)), 0.0)
    whole = torch.round(q * torch.where(top > 0, 1 / scale, 0.0))
    # the greatest that a head's logit can be on a page, of the group's heads the greatest
    b = s["bounds"][table].float().permute(0, 2, 3, 4, 1)  # [sequences, kv, 2, D, pages]
    score = torch.matmul(whole.clamp(min=0), b[:, :, 0]) + torch.matmul(whole.clamp(max=0), b[:, :, 1])
    score = (score * scale).amax(2) * s["bound_scales"][table].transpose(1, 2)
    pages = (length + ps - 1) // ps
    j = torch.arange(P, device="cuda")
    forced = (j < c["sinks"]) | (j >= pages[:, None] - c["recent"])
    score = torch.where(forced[:, None], torch.inf, score)
    score = torch.where((j < pages[:, None])[:, None], score, -torch.inf)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :k]
    best = torch.where(best < pages[:, None, None], best, P).sort(-1).values
    s["selected"].fill_(-1)
    s["selected"][..., :best.shape[-1]] = torch.where(best < P, best, -1)
    # attention over the chosen pages
    seq = torch.zeros_like(length) if many else torch.arange(n, device="cuda")
    real = best.clamp(max=P - 1)
    page = table[seq[:, None, None], real]
    head = torch.arange(KV, device="cuda")[:, None]
    T = best.shape[-1] * ps
    keys = s["keys"][page, head].reshape(n, KV, T, D).float()
    place = (best[..., None] * ps + torch.arange(ps, device="cuda")).reshape(n, KV, 1, T)
    w, lse = _softmax(torch.matmul(q, keys.transpose(-1, -2)) / math.sqrt(D), place < length[:, None, None, None])
    del keys
    out = torch.matmul(w, s["values"][page, head].reshape(n, KV, T, D).float())
    s["out"].copy_(out.reshape(n, H, D))
    s["lse"].copy_(lse.reshape(n, H))
    return {"selected": s["selected"], "out": s["out"], "lse": s["lse"]}


def _plain_evict(s):
    c = s["case"]
    ps, n, KV = c["page"], c["sequences"], c["kv_heads"]
    slot = torch.arange(s["weights"].shape[-1], device="cuda")
    there = slot < s["lengths"][:, None, None]
    place = s["positions"]
    safe = (place < c["sinks"]) | (place >= (s["seen"] - c["recent"])[:, None, None])
    key = torch.where(safe, torch.inf, s["weights"])
    key = torch.where(there, key, -torch.inf)
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    left = s["lengths"].clamp(max=c["budget"])
    keep = torch.zeros_like(there.expand_as(key)).scatter_(-1, order, (slot < left[:, None, None]).expand_as(key))
    low = slot < left[:, None, None]
    # the hole of each rank takes the kept tail token of that rank
    a, h, to = torch.nonzero(low & ~keep, as_tuple=True)
    _, _, of = torch.nonzero(~low & keep, as_tuple=True)
    table = s["table"].long()
    pt, it, po, io = table[a, to // ps], to % ps, table[a, of // ps], of % ps
    s["keys"][pt, h, it] = s["keys"][po, h, io]
    s["values"][pt, h, it] = s["values"][po, h, io]
    # dropped slots become empty; behind the old length nothing is written
    s["weights_out"].copy_(torch.where(low, s["weights"], torch.where(there, 0.0, s["weights_out"])))
    s["weights_out"][a, h, to] = s["weights"][a, h, of]
    s["positions_out"].copy_(torch.where(low, place, torch.where(there, -1, s["positions_out"])))
    s["positions_out"][a, h, to] = place[a, h, of]
    s["lengths_out"].copy_(left)
    return _evicted(s)


def _evicted(s):
    return {"keys": s["keys"], "values": s["values"], "weights": s["weights_out"], "positions": s["positions_out"],
            "lengths": s["lengths_out"]}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_append(s):
    import nutllm_b200 as nb
    c = s["case"]
    H, KV, D = c["heads"], c["kv_heads"], c["head_dim"]
    at, e, width = s["qkv"].data_ptr(), s["qkv"].element_size() * D, (H + 2 * KV) * D
    s["handle"].append(at, at + H * e, at + (H + KV) * e, s["starts"].data_ptr(), s["rows"], c["new"],
                       dtype=_code(nb, c["rows"]), q_stride=width, k_stride=width, v_stride=width,
                       cos=s["cos"].data_ptr(), sin=s["sin"].data_ptr(), rope_rows=s["cos"].shape[0],
                       seen=s["seen"].data_ptr(), q_out=s["q_out"].data_ptr(),
                       positions=s["positions"].data_ptr() if c["track"] else 0,
                       weights=s["weights"].data_ptr() if c["track"] else 0, stream=_stream())
    got = {"q": s["q_out"], "keys": s["keys"], "values": s["values"]}
    if c["track"]:
        got.update(positions=s["positions"], weights=s["weights"])
    if c["bounds"]:
        got["bounds"] = s["bounds"] * s["bound_scales"][..., None, None]
    return got


def _own_attend(s):
    import nutllm_b200 as nb
    c = s["case"]
    tracked = c["weights"]
    s["handle"].attention(s["q"].data_ptr(), s["out"].data_ptr(), s["rows"], dtype=_code(nb, c["rows"]), lse=s["lse"].data_ptr(),
                          weights=s["weights"].data_ptr() if tracked else 0, weights_out=s["weights_out"].data_ptr() if tracked else 0,
                          stream=_stream())
    got = {"out": s["out"], "lse": s["lse"]}
    if tracked:
        got["weights"] = s["weights_out"]
    return got


def _own_sparse(s):
    import nutllm_b200 as nb
    c = s["case"]
    kind, stream, many = _code(nb, c["rows"]), _stream(), c["queries"] > 1
    rows = dict(row_sequence=s["row_sequence"].data_ptr(), row_length=s["row_length"].data_ptr()) if many else {}
    q, selected = s["q"].data_ptr(), s["selected"].data_ptr()
    s["handle"].select(q, selected, s["rows"], c["budget"], dtype=kind, sink_pages=c["sinks"], recent_pages=c["recent"], stream=stream,
                       **rows)
    s["handle"].attention(q, s["out"].data_ptr(), s["rows"], dtype=kind, lse=s["lse"].data_ptr(), selected=selected,
                          n_selected=c["budget"], stream=stream, **rows)
    return {"selected": s["selected"], "out": s["out"], "lse": s["lse"]}


def _own_evict(s):
    c = s["case"]
    s["handle"].evict(s["weights"].data_ptr(), s["positions"].data_ptr(), s["seen"].data_ptr(), c["budget"], sinks=c["sinks"],
                      recent=c["recent"], new_lengths=s["lengths_out"].data_ptr(), weights_out=s["weights_out"].data_ptr(),
                      positions_out=s["positions_out"].data_ptr(), stream=_stream())
    return _evicted(s)


_PLAIN = {"append": _plain_append, "attend": _plain_attend, "sparse": _plain_sparse, "evict": _plain_evict}
_OWN = {"append": _own_append, "attend": _own_attend, "sparse": _own_sparse, "evict": _own_evict}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"append": _exact_append, "attend": _exact_attend, "sparse": _exact_sparse, "evict": _exact_evict}[c["op"]](c, s)


def _line(c, s, pool, a, h, upto):
    """The first `upto` rows of sequence a, kv head h, in 64 bits."""
    pages = s["table"][a, :_pages_of(upto, c["page"])].long()
    return pool[pages, h].reshape(-1, c["head_dim"])[:upto].double()


def _exact_append(c, s):
    H, KV, D, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    x = s["qkv"].double().reshape(s["rows"], H + 2 * KV, D)
    lens, starts = s["lengths"].tolist(), s["starts"].tolist()
    place = torch.cat([torch.arange(n - (b - a), n, device="cuda") for n, a, b in zip(lens, starts, starts[1:])])
    seq = torch.cat([torch.full((b - a,), i, device="cuda") for i, (a, b) in enumerate(zip(starts, starts[1:]))])
    turn = torch.complex(s["cos"].double(), s["sin"].double())[place + c["offset"]][:, None]
    qk = torch.view_as_real(torch.view_as_complex(x[:, :H + KV].reshape(s["rows"], H + KV, D // 2, 2).contiguous()) * turn).reshape(
        s["rows"], H + KV, D)
    page, slot = s["table"].long()[seq, place // ps], place % ps
    keys, values = s["keys"].double(), s["values"].double()
    keys[page, :, slot] = qk[:, H:]
    values[page, :, slot] = x[:, H + KV:]
    got = {"q": qk[:, :H], "keys": keys, "values": values}
    if c["track"]:
        got |= {"positions": s["positions"].clone(), "weights": s["weights"].double()}
        got["positions"][seq, :, place] = (place + c["offset"]).int()[:, None]
        got["weights"][seq, :, place] = 0.0
    # the bounds are those of the stored keys, which are rounded: they have no value in 64 bits
    return got | ({"bounds": None} if c["bounds"] else {})


def _head(q, keys, values):
    """Attention of q [G, D] over the rows of keys and values."""
    if not len(keys):
        return torch.zeros_like(q), torch.full((len(q),), -math.inf, device="cuda", dtype=torch.float64), torch.zeros(len(q), 0, device="cuda")
    z = q @ keys.T / math.sqrt(q.shape[1])
    lse = torch.logsumexp(z, 1)
    w = torch.exp(z - lse[:, None])
    return w @ values, lse, w


def _exact_attend(c, s):
    KV, G = c["kv_heads"], c["heads"] // c["kv_heads"]
    q, out, lse = s["q"].double(), torch.zeros_like(s["q"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
    weights = torch.zeros_like(s["weights"], dtype=torch.float64) if c["weights"] else None
    for a, n in enumerate(s["lengths"].tolist()):
        for h in range(KV):
            of = slice(h * G, (h + 1) * G)
            out[a, of], lse[a, of], w = _head(q[a, of], _line(c, s, s["keys"], a, h, n), _line(c, s, s["values"], a, h, n))
            if c["weights"] and n:
                weights[a, h, :n] = s["weights"][a, h, :n].double() + w.sum(0)
    return {"out": out, "lse": lse} | ({"weights": weights} if c["weights"] else {})


def _exact_sparse(c, s):
    KV, G, D, ps, k = c["kv_heads"], c["heads"] // c["kv_heads"], c["head_dim"], c["page"], c["budget"]
    if s["rows"] * KV > 3000:
        return None
    q, out, lse = s["q"].double(), torch.zeros_like(s["q"], dtype=torch.float64), torch.zeros_like(s["lse"], dtype=torch.float64)
    chosen = torch.full_like(s["selected"], -1)
    lens = (s["row_length"] if c["queries"] > 1 else s["lengths"]).tolist()
    step = torch.arange(ps, device="cuda")
    for r, n in enumerate(lens):
        a = 0 if c["queries"] > 1 else r
        P = _pages_of(n, ps)
        if not P:
            lse[r] = -math.inf
            continue
        pages = s["table"][a, :P].long()
        for h in range(KV):
            of = slice(h * G, (h + 1) * G)
            x = q[r, of]
            top = x.abs().amax(1, keepdim=True)
            least = torch.ceil(torch.log2(top / 127) - 1e-12).long()
            unit = ((least + 1023) << 52).view(torch.float64)  # the least power of two under which all fit 127
            x = torch.round(x / unit)
            b = s["bounds"][pages, h].double() * s["bound_scales"][pages, h].double()[:, None, None]
            score = (torch.maximum(x[:, None] * b[:, 0], x[:, None] * b[:, 1]).sum(-1) * unit).amax(0)
            score[:c["sinks"]] = math.inf
            score[max(0, P - c["recent"]):] = math.inf
            best = torch.argsort(score, descending=True, stable=True)[:k].sort().values
            chosen[r, h, :len(best)] = best.int()
            at = (best[:, None] * ps + step).reshape(-1)
            at = at[at < n]
            keys = s["keys"][pages[at // ps], h, at % ps].double()
            out[r, of], lse[r, of], _ = _head(q[r, of], keys, s["values"][pages[at // ps], h, at % ps].double())
    return {"selected": chosen, "out": out, "lse": lse}


def _exact_evict(c, s):
    ps, m = c["page"], c["budget"]
    keys, values = s["keys"].double(), s["values"].double()
    weights, places = torch.zeros_like(s["weights"], dtype=torch.float64), s["positions_out"].clone()
    lens = s["lengths"].tolist()
    for a, n in enumerate(lens):
        left = min(n, m)
        for h in range(c["kv_heads"]):
            w, p = s["weights"][a, h, :n].double(), s["positions"][a, h, :n]
            rank = w.masked_fill((p < c["sinks"]) | (p >= int(s["seen"][a]) - c["recent"]), math.inf)
            kept = torch.argsort(rank, descending=True, stable=True)[:left].sort().values
            stays = torch.zeros(n, dtype=torch.bool, device="cuda")
            stays[kept] = True
            source = torch.arange(left, device="cuda")
            source[~stays[:left]] = kept[kept >= left]
            weights[a, h, :left], places[a, h, :left], places[a, h, left:n] = w[source], p[source], -1
            pages = s["table"][a].long()
            to = torch.arange(left, device="cuda")
            for pool in (keys, values):
                pool[pages[to // ps], h, to % ps] = pool[pages[source // ps], h, source % ps]
    return {"keys": keys, "values": values, "weights": weights, "positions": places,
            "lengths": torch.tensor([min(n, m) for n in lens], device="cuda", dtype=torch.int32)}
