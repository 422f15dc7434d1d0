"""Decoding that branches, on the paged key/value cache, case by case.

A serving loop may follow several continuations of one sequence: a tree of
drafted tokens that one pass over the cache verifies, or the beams of a beam
search.  Four operators carry that: `tree` (attention of all drafted tokens of
each sequence over its cache and over their own ancestors), `compact` (keep the
accepted tokens of each tree, next to one another), `beam` (the best
continuations of all beams over the vocabulary) and `pages` (every sequence
continues another one: whole pages are shared, a page that two would write is
copied, new pages are taken, pages without a holder are given back).

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
        # A first guess at one chat's next tokens: every layer makes this call.
        dict(name="tree chat", op="tree", sequences=1, prefix=37, nodes=8, heads=32, kv_heads=4, head_dim=64, page=16,
             cache="f16", rows="f32"),
        # One chat some way in, an odd tree.
        dict(name="tree step", op="tree", sequences=1, prefix=1999, nodes=25, heads=32, kv_heads=8, head_dim=128, page=16,
             cache="bf16", rows="bf16"),
        # A batch of unequal caches, small trees.
        dict(name="tree batch", op="tree", sequences=32, prefix=4096, nodes=16, heads=32, kv_heads=8, head_dim=128, page=16,
             cache="bf16", rows="bf16"),
        # Wide trees, eight query heads to a kv head: 512 rows share the keys.
        dict(name="tree wide", op="tree", sequences=16, prefix=2048, nodes=64, heads=32, kv_heads=4, head_dim=128, page=64,
             cache="f16", rows="f16"),
        # Long documents, few sequences: the cache has to be split.
        dict(name="tree long", op="tree", sequences=2, prefix=60000, nodes=33, heads=32, kv_heads=8, head_dim=128, page=16,
             cache="bf16", rows="bf16"),
        # A cache in 32 bits, every head with its own keys.
        dict(name="tree f32", op="tree", sequences=4, prefix=1000, nodes=12, heads=32, kv_heads=32, head_dim=128, page=16,
             cache="f32", rows="f32"),
        # The beams of one request.
        dict(name="beam one", op="beam", sequences=1, beams=4, vocab=32000, out=8, logits="f32", finished=0),
        # A batch of requests, some of whose beams have ended.
        dict(name="beam batch", op="beam", sequences=32, beams=8, vocab=32000, out=16, logits="bf16", finished=2),
        # Many beams over a large vocabulary.
        dict(name="beam large", op="beam", sequences=16, beams=16, vocab=128000, out=16, logits="f32", finished=1),
        # One step of a beam search: the survivors' pages, then the pages that two of them would write.
        dict(name="pages beams", op="pages", groups=16, beams=4, length=1003, add=1, pool=6000, heads=32, kv_heads=8, head_dim=128,
             page=16, cache="bf16"),
        # A step of many long requests: the table is large.
        dict(name="pages many", op="pages", groups=64, beams=8, length=16000, add=1, pool=120000, heads=4, kv_heads=1, head_dim=64,
             page=16, cache="f16"),
        # After a batch of trees was verified.
        dict(name="compact batch", op="compact", sequences=64, prefix=2048, nodes=64, accept=9, heads=32, kv_heads=8, head_dim=128,
             page=16, cache="bf16"),
    ]


SHAPES = [(32, 4, 64), (32, 32, 128), (32, 8, 128), (6, 6, 48), (16, 2, 80), (24, 8, 96),
          (16, 1, 128), (8, 4, 256), (12, 4, 32)]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the same ranges, no dearer than the dearest listed one of its operator."""
    op = rng.choice(["tree", "tree", "beam", "pages", "compact"])
    cap = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        if op == "beam":
            c = dict(op=op, sequences=_log(rng, 1, 64), beams=_log(rng, 1, 32), vocab=_log(rng, 40, 160000),
                     out=_log(rng, 1, 64), logits=rng.choice(["f32", "f16", "bf16"]), finished=rng.randrange(3))
            c["out"], c["finished"] = min(c["out"], c["vocab"]), min(c["finished"], c["beams"] - 1)
        else:
            heads, kv_heads, head_dim = rng.choice(SHAPES)
            c = dict(op=op, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([8, 16, 24, 32, 64]),
                     cache=rng.choice(["f32", "f16", "bf16"]))
            if op == "pages":
                c.update(groups=_log(rng, 1, 64), beams=_log(rng, 1, 16), length=_log(rng, 1, 16000), add=rng.choice([1, 1, 1, 7]))
                each = _pages_of(c["length"], c["page"]) + 6 * c["beams"]
                c["pool"] = c["groups"] * each + rng.randrange(1000)
            else:
                c.update(sequences=_log(rng, 1, 64), prefix=_log(rng, 1, 60000), nodes=_log(rng, 1, 128))
                if op == "tree":
                    c["rows"] = rng.choice(["f32", c["cache"]])
                else:
                    c["accept"] = rng.randrange(1, min(c["nodes"], 16) + 1)
        if _cost(c) <= cap:
            return c


# ---------------------------------------------------------------------------
# what a case has to move and compute


def _spread(top, n, low):
    """n sizes from low to top."""
    return [max(low, (top * (i + 1)) // n) for i in range(n)]


def _pages_of(length, page):
    return -(-length // page)


def _prefixes(c):
    return _spread(c["prefix"], c["sequences"], 0)


def _nodes(c):
    """Drafted tokens of each sequence, the longest caches' first."""
    return _spread(c["nodes"], c["sequences"], 1)[::-1]


def work(c):
    if c["op"] == "beam":
        rows = c["sequences"] * (c["beams"] - c["finished"])
        b = rows * c["vocab"] * BYTES[c["logits"]] + c["sequences"] * (c["beams"] * 5 + c["out"] * 13)
        return {"bytes": b, "flops": rows * c["vocab"] * 4}
    e, D, H, KV, ps = BYTES[c["cache"]], c["head_dim"], c["heads"], c["kv_heads"], c["page"]
    if c["op"] == "tree":
        r, words = BYTES[c["rows"]], -(-c["nodes"] // 32)
        lens = [p + n for p, n in zip(_prefixes(c), _nodes(c))]
        b = sum(lens) * KV * D * 2 * e + sum(_pages_of(n, ps) for n in lens) * 4
        b += sum(_nodes(c)) * (2 * H * D * r + 4 * H + 4 * words)
        return {"bytes": b, "flops": sum(n * m for n, m in zip(lens, _nodes(c))) * H * D * 4}
    if c["op"] == "compact":
        moved = c["sequences"] * max(0, c["accept"] - 1)
        return {"bytes": moved * KV * D * 4 * e + c["sequences"] * (c["accept"] * 4 + 12), "flops": moved * KV * D}
    S = c["groups"] * c["beams"]
    # the tables read and written, the pages' counts, the copied part of a page of about half the sequences
    copied = S // 2 * (c["length"] % ps) * KV * D * 4 * e
    return {"bytes": S * _pages_of(c["length"], ps) * 8 + c["pool"] * 4 + S * 24 + copied, "flops": S * _pages_of(c["length"], ps)}


def _cost(c):
    w = work(c)
    cost = max(w["bytes"], w["flops"] / 50)
    if c["op"] in ("tree", "compact"):  # the pool that has to be made, and the plain form's padded logits
        cost = max(cost, (sum(_prefixes(c)) + sum(_nodes(c))) * c["kv_heads"] * c["head_dim"] * BYTES[c["cache"]] / 16)
    if c["op"] == "tree":
        cap = c["prefix"] + c["nodes"]
        cost = max(cost, c["sequences"] * c["heads"] * c["nodes"] * cap, c["sequences"] * c["kv_heads"] * c["head_dim"] * cap)
    if c["op"] == "pages":
        cost = max(cost, c["pool"] * c["page"] * c["kv_heads"] * c["head_dim"] * BYTES[c["cache"]] / 16)
    return cost


# ---------------------------------------------------------------------------
# inputs


def _pool(c, s, g, lens):
    """A pool of shuffled pages that holds sequences of these lengths, their table and lengths."""
    dev, ps, KV, D = "cuda", c["page"], c["kv_heads"], c["head_dim"]
    per = max(1, max(_pages_of(n, ps) for n in lens))
    pages = torch.tensor([max(1, _pages_of(n, ps)) for n in lens], device=dev)
    total = int(pages.sum()) + 3
    order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    first = pages.cumsum(0) - pages
    at = torch.arange(per, device=dev)
    # places behind a sequence's last page hold its first page's number: they are not read
    s["table"] = order[first[:, None] + torch.where(at < pages[:, None], at, 0)].contiguous()
    s["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["keys"] = torch.randn(total, KV, ps, D, generator=g, device=dev, dtype=DTYPES[c["cache"]])
    s["values"] = torch.randn(total, KV, ps, D, generator=g, device=dev, dtype=DTYPES[c["cache"]])


def _handle(c, s, sequences):
    """The framework's handle on the pool, as its user makes it once."""
    import nutllm_b200 as nb
    return nb.PagedCache(s["keys"].data_ptr(), s["values"].data_ptr(), s["table"].data_ptr(), s["lengths"].data_ptr(),
                         sequences=sequences, max_pages=s["table"].shape[1], n_pages=s["keys"].shape[0], page_size=c["page"],
                         heads=c["heads"], kv_heads=c["kv_heads"], head_dim=c["head_dim"], dtype=_code(nb, c["cache"]))


def _code(nb, name):
    return {"f32": nb.F32, "f16": nb.F16, "bf16": nb.BF16}[name]


def _starts(counts):
    n = torch.tensor([0] + list(counts), device="cuda")
    return n.cumsum(0).to(torch.int32)


def _trees(c, g):
    """Masks of random trees: a node sees itself and its ancestors."""
    words = -(-c["nodes"] // 32)
    pick = torch.rand(sum(_nodes(c)), generator=g, device="cuda").tolist()
    rows = []
    for n in _nodes(c):
        seen = []
        for i in range(n):
            # drafts are deeper than they are wide: a parent among the last few, or the prefix
            parent = i - 1 - int(pick[len(rows)] * min(i + 1, 6))
            seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
            rows.append([seen[i] >> 32 * w & 0xffffffff for w in range(words)])
    bits = torch.tensor(rows, dtype=torch.int64)
    return torch.where(bits < 1 << 31, bits, bits - (1 << 32)).to(torch.int32).cuda()


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    {"tree": _prepare_tree, "compact": _prepare_compact, "beam": _prepare_beam, "pages": _prepare_pages}[c["op"]](c, s, g)
    return s


def _prepare_tree(c, s, g):
    H, D = c["heads"], c["head_dim"]
    _pool(c, s, g, [p + n for p, n in zip(_prefixes(c), _nodes(c))])
    rows = sum(_nodes(c))
    s["starts"], s["mask"] = _starts(_nodes(c)), _trees(c, g)
    s["q"] = (2 * torch.randn(rows, H, D, generator=g, device="cuda")).to(DTYPES[c["rows"]])
    s["out"], s["lse"] = torch.empty_like(s["q"]), torch.empty(rows, H, device="cuda")
    if own:
        s["handle"] = _handle(c, s, c["sequences"])
        s["handle"].reserve_tree(c["nodes"])


def _prepare_compact(c, s, g):
    nodes = _nodes(c)
    _pool(c, s, g, [p + n for p, n in zip(_prefixes(c), nodes)])
    s["starts"] = _starts(nodes)
    # a path through each tree: its first node, then some of the others, ascending; -1 behind it
    least = torch.rand(c["sequences"], c["nodes"], generator=g, device="cuda")
    least[:, 0] = -1.0
    n = torch.tensor(nodes, device="cuda")[:, None]
    least = torch.where(torch.arange(c["nodes"], device="cuda") < n, least, 2.0)
    path = least.argsort(-1)[:, :c["accept"]]
    path = torch.where(torch.arange(c["accept"], device="cuda") < n, path, c["nodes"]).sort(-1).values
    s["accepted"] = torch.where(path < c["nodes"], path, -1).to(torch.int32).contiguous()
    s["lengths_out"] = torch.zeros_like(s["lengths"])
    if own:
        s["handle"] = _handle(c, s, c["sequences"])


def _prepare_beam(c, s, g):
    S, B, V, n = c["sequences"], c["beams"], c["vocab"], c["out"]
    s["logits"] = (3 * torch.randn(S * B, V, generator=g, device="cuda")).to(DTYPES[c["logits"]])
    s["scores"] = -20 * torch.rand(S, B, generator=g, device="cuda")
    ended = torch.rand(S, B, generator=g, device="cuda").argsort(-1) < c["finished"]
    s["finished"] = ended.to(torch.uint8)
    s["eos"] = 2 % V
    s["out_scores"] = torch.empty(S, n, device="cuda")
    s["out_rows"] = torch.empty(S, n, device="cuda", dtype=torch.int32)
    s["out_tokens"] = torch.empty(S, n, device="cuda", dtype=torch.int32)
    s["out_finished"] = torch.empty(S, n, device="cuda", dtype=torch.uint8)
    if own:
        import nutllm_b200 as nb
        s["handle"] = nb.BeamSearch(S, B, V, n)


def _prepare_pages(c, s, g):
    """Groups of beams that split lately: they share their first pages and have a few of their own."""
    dev, ps, B, S, P = "cuda", c["page"], c["beams"], c["groups"] * c["beams"], c["pool"]
    used = _pages_of(c["length"], ps)
    per = _pages_of(c["length"] + c["add"], ps) + 1
    own_pages = min(used, 3)
    shared = used - own_pages
    order = torch.randperm(P, generator=g, device=dev).to(torch.int32)
    group, beam = torch.arange(S, device=dev) // B, torch.arange(S, device=dev) % B
    at = torch.arange(per, device=dev)
    each = shared + own_pages * B
    where = torch.where(at < shared, at, shared + beam[:, None] * own_pages + at - shared) + (group * each)[:, None]
    table = torch.where(at < used, order[where.clamp(max=P - 1)], 0).to(torch.int32)
    taken = c["groups"] * each
    refs = torch.zeros(P, dtype=torch.int32, device=dev)
    flat = table[:, :used].reshape(-1).long()
    refs.scatter_add_(0, flat, torch.ones_like(flat, dtype=torch.int32))
    lengths = torch.full((S,), c["length"], dtype=torch.int32, device=dev)
    # free pages in no particular order; places behind their number hold pages that are in use
    free = torch.cat((order[taken:], order[:taken]))
    s["start"] = torch.cat((table.reshape(-1), lengths, refs, free, torch.tensor([P - taken], dtype=torch.int32, device=dev)))
    s["book"] = s["start"].clone()
    cuts = [0, S * per, S * per + S, S * per + S + P, S * per + S + 2 * P]
    s["table"] = s["book"][:cuts[1]].view(S, per)
    s["lengths"], s["refs"], s["free"], s["count"] = (s["book"][a:b] for a, b in zip(cuts[1:], cuts[2:] + [cuts[4] + 1]))
    # survivors: beams drawn with repetition, some of them twice and some gone
    s["parent"] = (group * B + torch.randint(0, B, (S,), generator=g, device=dev)).to(torch.int32)
    s["add"] = torch.full((S,), c["add"], dtype=torch.int32, device=dev)
    s["copies"] = torch.empty(3, S, dtype=torch.int32, device=dev)
    shape = (P, c["kv_heads"], ps, c["head_dim"])
    s["keys"] = torch.randn(shape, generator=g, device=dev, dtype=DTYPES[c["cache"]])
    s["values"] = torch.randn(shape, generator=g, device=dev, dtype=DTYPES[c["cache"]])
    if own:
        import nutllm_b200 as nb
        s["handle"] = _handle(c, s, S)
        s["pages"] = nb.PageBook(s["table"].data_ptr(), s["lengths"].data_ptr(), s["refs"].data_ptr(), s["free"].data_ptr(),
                                 s["count"].data_ptr(), sequences=S, max_pages=per, n_pages=P, page_size=ps)


# ---------------------------------------------------------------------------
# one pass


def run(s):
    return (_OWN if own else _PLAIN)[s["case"]["op"]](s)


def _bits(mask, n):
    """The first n bits of each row, as truth values."""
    j = torch.arange(n, device=mask.device)
    return (mask[:, j // 32] >> (j % 32).to(torch.int32)) & 1 != 0


def _plain_tree(s):
    c = s["case"]
    S, H, KV, D, n = c["sequences"], c["heads"], c["kv_heads"], c["head_dim"], c["nodes"]
    starts, table = s["starts"].long(), s["table"].long()
    counts = starts[1:] - starts[:-1]
    cap = table.shape[1] * c["page"]
    # rows padded to the same number for each sequence
    rows = s["q"].shape[0]
    at = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), at, right=True)
    node = at - starts[seq]
    q = torch.zeros(S, n, H, D, device="cuda")
    q[seq, node] = s["q"].float()
    q = q.reshape(S, n, KV, H // KV, D).permute(0, 2, 3, 1, 4).reshape(S, KV, -1, D)
    sees = torch.zeros(S, n, n, dtype=torch.bool, device="cuda")
    sees[seq, node] = _bits(s["mask"], n)
    place = torch.arange(cap, device="cuda") - (s["lengths"].long() - counts)[:, None]  # below 0: the prefix
    drafted = (place >= 0) & (place < counts[:, None])
    valid = torch.gather(sees, 2, place.clamp(0, n - 1)[:, None].expand(S, n, cap))
    valid = (place < 0)[:, None] | drafted[:, None] & valid
    valid = valid[:, None, None].expand(S, 1, H // KV, n, cap).reshape(S, 1, -1, cap)
    keys = s["keys"][table].transpose(1, 2).reshape(S, KV, cap, D).float()
    z = torch.matmul(q, keys.transpose(-1, -2)) / math.sqrt(D)
    del keys
    z = torch.where(valid, z, -torch.inf)
    top = z.amax(-1, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    z = torch.exp(z - top)
    total = z.sum(-1, keepdim=True)
    values = s["values"][table].transpose(1, 2).reshape(S, KV, cap, D).float()
    out = torch.matmul(z, values) / torch.where(total > 0, total, 1.0)
    lse = (top + torch.log(total)).squeeze(-1)
    out = out.reshape(S, KV, H // KV, n, D).permute(0, 3, 1, 2, 4).reshape(S, n, H, D)
    lse = lse.reshape(S, KV, H // KV, n).permute(0, 3, 1, 2).reshape(S, n, H)
    s["out"].copy_(out[seq, node])
    s["lse"].copy_(lse[seq, node])
    return {"out": s["out"], "lse": s["lse"]}


def _plain_compact(s):
    c = s["case"]
    ps, table, path = c["page"], s["table"].long(), s["accepted"].long()
    starts = s["starts"].long()
    prefix = s["lengths"].long() - (starts[1:] - starts[:-1])
    there = path >= 0
    seq = torch.arange(c["sequences"], device="cuda")[:, None]
    to = prefix[:, None] + torch.arange(c["accept"], device="cuda")
    of = torch.where(there, prefix[:, None] + path, to)  # places behind the path stay as they are
    to, of = (torch.where(there, x, prefix[:, None]) for x in (to, of))
    # the first node is always accepted and does not move: places behind the path stand for it
    pt, it, po, io = table[seq, to // ps], to % ps, table[seq, of // ps], of % ps
    s["keys"][pt, :, it] = s["keys"][po, :, io]
    s["values"][pt, :, it] = s["values"][po, :, io]
    s["lengths_out"].copy_(prefix + there.sum(-1))
    return {"keys": s["keys"], "values": s["values"], "lengths": s["lengths_out"]}


def _plain_beam(s):
    c = s["case"]
    S, B, V, n = c["sequences"], c["beams"], c["vocab"], c["out"]
    # in 64 bits: neighbouring candidates may be closer than 32 bits' rounding of a sum
    x = s["logits"].double().reshape(S, B, V)
    top = x.amax(-1, keepdim=True)
    lse = top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    score = s["scores"].double()[..., None]
    done = (s["finished"] != 0)[..., None]
    token = torch.arange(V, device="cuda")
    total = torch.where(done, torch.where(token == s["eos"], score, -torch.inf), score + (x - lse))
    best, at = torch.sort(total.reshape(S, B * V), dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    beam, token = at // V, at % V
    s["out_scores"].copy_(best)
    s["out_rows"].copy_(beam + B * torch.arange(S, device="cuda")[:, None])
    s["out_tokens"].copy_(token)
    s["out_finished"].copy_(torch.gather(s["finished"], 1, beam) | (token == s["eos"]))
    return _selected(s)


def _selected(s):
    return {k: s["out_" + k] for k in ("scores", "rows", "tokens", "finished")}


def _plain_pages(s):
    c = s["case"]
    ps, S, P = c["page"], s["table"].shape[0], c["pool"]
    s["book"].copy_(s["start"])  # so that every pass forks the same sequences
    table, parent, add = s["table"], s["parent"].long(), s["add"].long()
    lengths = s["lengths"].long()
    i = torch.arange(table.shape[1], device="cuda")
    had = (lengths + ps - 1) // ps
    kept = lengths[parent]
    pages = (kept + ps - 1) // ps
    more = (kept + add + ps - 1) // ps
    new = table[parent]

    def holders(at, where):
        """How many of the places `where` hold each page."""
        n = torch.zeros(P + 1, dtype=torch.int32, device="cuda")
        return n.scatter_add_(0, torch.where(where, at, P).reshape(-1).long(), where.reshape(-1).int())[:P]

    refs = s["refs"] + holders(new, i < pages[:, None]) - holders(table, i < had[:, None])
    # a partly filled page that is to be written: the first of its writers keeps it if none else holds it
    tail = new.gather(1, (kept // ps)[:, None])[:, 0].long()
    writes = (add > 0) & (kept % ps != 0)
    tail = torch.where(writes, tail, P)
    writers = holders(tail, writes)
    seq = torch.arange(S, device="cuda")
    first = torch.full((P + 1,), S, device="cuda").scatter_reduce_(0, tail, seq, "amin")
    at = tail.clamp(max=P - 1)
    copies = writes & (refs[at] > 1) & ~((writers[at] == refs[at]) & (first[at] == seq))
    refs = refs - holders(tail, copies)
    need = copies.long() + more - pages
    before = need.cumsum(0) - need
    count = s["count"].long()
    # taken from the end of the free list: a copy's page first, then the new ones
    take = lambda k: s["free"][(count - 1 - k).clamp(0, P - 1)]  # noqa: E731
    fresh = take(before)
    new = torch.where(copies[:, None] & (i == (kept // ps)[:, None]), fresh[:, None], new)
    beyond = (i >= pages[:, None]) & (i < more[:, None])
    new = torch.where(beyond, take((before + copies.long())[:, None] + i - pages[:, None]), new)
    s["copies"][0] = torch.where(copies, tail, -1)
    s["copies"][1] = torch.where(copies, fresh, -1)
    s["copies"][2] = torch.where(copies, kept % ps, 0)
    freed = (refs == 0) & (s["refs"] > 0)
    taken = need.sum()
    refs = refs + holders(new, beyond | copies[:, None] & (i == (kept // ps)[:, None]))
    left = torch.where(i < more[:, None], new, table)
    rank = freed.long().cumsum(0) - 1
    free = torch.cat((s["free"], s["free"][:1]))
    free = free.scatter(0, torch.where(freed, count - taken + rank, P), torch.arange(P, device="cuda", dtype=torch.int32))[:P]
    s["table"].copy_(left)
    s["lengths"].copy_(kept + add)
    s["refs"].copy_(refs)
    s["free"].copy_(free)
    s["count"].copy_(count - taken + freed.sum())
    # the pages' slots
    of, to = (torch.where(copies, x.long(), new[:, 0].long()) for x in (tail, fresh))
    inside = (torch.arange(ps, device="cuda") < (kept % ps)[:, None]) & copies[:, None]
    for pool in (s["keys"], s["values"]):
        # a sequence without a copy writes its first page as it is
        pool[to] = torch.where(inside[:, None, :, None], pool[of], pool[to])
    return _booked(s)


def _booked(s):
    return {k: s[k] for k in ("table", "lengths", "refs", "free", "count", "copies", "keys", "values")}


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _own_tree(s):
    import nutllm_b200 as nb
    c = s["case"]
    s["handle"].tree_attention(s["q"].data_ptr(), s["out"].data_ptr(), s["starts"].data_ptr(), s["mask"].data_ptr(),
                               s["q"].shape[0], c["nodes"], s["mask"].shape[1], dtype=_code(nb, c["rows"]), lse=s["lse"].data_ptr(),
                               stream=_stream())
    return {"out": s["out"], "lse": s["lse"]}


def _own_compact(s):
    s["handle"].compact(s["starts"].data_ptr(), s["accepted"].data_ptr(), s["case"]["accept"],
                        new_lengths=s["lengths_out"].data_ptr(), stream=_stream())
    return {"keys": s["keys"], "values": s["values"], "lengths": s["lengths_out"]}


def _own_beam(s):
    import nutllm_b200 as nb
    s["handle"].select(s["logits"].data_ptr(), s["scores"].data_ptr(), s["out_scores"].data_ptr(), s["out_rows"].data_ptr(),
                       s["out_tokens"].data_ptr(), dtype=_code(nb, s["case"]["logits"]), finished=s["finished"].data_ptr(),
                       eos=s["eos"], out_finished=s["out_finished"].data_ptr(), stream=_stream())
    return _selected(s)


def _own_pages(s):
    s["book"].copy_(s["start"])
    at = [row.data_ptr() for row in s["copies"]]
    s["pages"].update(parent=s["parent"].data_ptr(), add=s["add"].data_ptr(), copy_from=at[0], copy_to=at[1], copy_slots=at[2],
                      stream=_stream())
    s["handle"].copy_pages(at[0], at[1], s["table"].shape[0], slots=at[2], stream=_stream())
    return _booked(s)


_PLAIN = {"tree": _plain_tree, "compact": _plain_compact, "beam": _plain_beam, "pages": _plain_pages}
_OWN = {"tree": _own_tree, "compact": _own_compact, "beam": _own_beam, "pages": _own_pages}


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits


def exact(c, seed):
    s = prepare(c, seed)
    with torch.no_grad():
        return {"tree": _exact_tree, "compact": _exact_compact, "beam": _exact_beam, "pages": _exact_pages}[c["op"]](c, s)


def _exact_tree(c, s):
    H, KV, D, ps = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    G = H // KV
    q = s["q"].double()
    out, lse = torch.zeros_like(q), torch.zeros_like(s["lse"], dtype=torch.float64)
    words = s["mask"].cpu().tolist()
    starts, lens = s["starts"].tolist(), s["lengths"].tolist()
    for a, length in enumerate(lens):
        lo, hi = starts[a], starts[a + 1]
        n = hi - lo
        pages = s["table"][a, :_pages_of(length, ps)].long()
        blocked = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            for j in range(n):
                blocked[i, length - n + j] = not words[lo + i][j // 32] >> j % 32 & 1
        blocked = blocked.cuda().repeat(G, 1)  # rows by head, then node
        for h in range(KV):
            keys = s["keys"][pages, h].reshape(-1, D)[:length].double()
            values = s["values"][pages, h].reshape(-1, D)[:length].double()
            x = q[lo:hi, h * G:(h + 1) * G].transpose(0, 1).reshape(-1, D)
            z = (x @ keys.T / math.sqrt(D)).masked_fill(blocked, -math.inf)
            l = torch.logsumexp(z, 1)
            out[lo:hi, h * G:(h + 1) * G] = (torch.exp(z - l[:, None]) @ values).reshape(G, n, D).transpose(0, 1)
            lse[lo:hi, h * G:(h + 1) * G] = l.reshape(G, n).T
    return {"out": out, "lse": lse}


def _exact_compact(c, s):
    ps = c["page"]
    keys, values = s["keys"].double(), s["values"].double()
    starts, lens = s["starts"].tolist(), s["lengths"].tolist()
    left = []
    for a, path in enumerate(s["accepted"].tolist()):
        prefix, table = lens[a] - (starts[a + 1] - starts[a]), s["table"][a].tolist()
        path = [j for j in path if j >= 0]
        for k, j in enumerate(path):
            to, of = prefix + k, prefix + j
            for pool in (keys, values):
                pool[table[to // ps], :, to % ps] = pool[table[of // ps], :, of % ps]
        left.append(prefix + len(path))
    return {"keys": keys, "values": values, "lengths": torch.tensor(left, dtype=torch.int32, device="cuda")}


def _exact_beam(c, s):
    S, B, V, n = c["sequences"], c["beams"], c["vocab"], c["out"]
    got = {"scores": [], "rows": [], "tokens": [], "finished": []}
    for a in range(S):
        candidates = []
        for b in range(B):
            score, ended = s["scores"][a, b].double(), bool(s["finished"][a, b])
            if ended:
                candidates.append((float(score), b * V + s["eos"], True))
                continue
            p = torch.log_softmax(s["logits"][a * B + b].double(), 0) + score
            few = min(V, n + 8)
            edge = torch.topk(p, few).values[-1]
            at = torch.nonzero(p >= edge)[:, 0]
            candidates += [(v, b * V + t, t == s["eos"]) for v, t in zip(p[at].tolist(), at.tolist())]
        candidates.sort(key=lambda x: (-x[0], x[1]))
        if len(candidates) < n:
            return None
        got["scores"].append([x[0] for x in candidates[:n]])
        got["rows"].append([a * B + x[1] // V for x in candidates[:n]])
        got["tokens"].append([x[1] % V for x in candidates[:n]])
        got["finished"].append([int(x[2]) for x in candidates[:n]])
    kinds = dict(scores=torch.float64, rows=torch.int32, tokens=torch.int32, finished=torch.uint8)
    return {k: torch.tensor(v, dtype=kinds[k], device="cuda") for k, v in got.items()}


def _exact_pages(c, s):
    ps, P = c["page"], c["pool"]
    table, lengths = s["table"].tolist(), s["lengths"].tolist()
    refs, free, count = s["refs"].tolist(), s["free"].tolist(), int(s["count"])
    parent, add = s["parent"].tolist(), s["add"].tolist()
    S = len(parent)
    new, wants = [], {}
    before = list(refs)
    for a in range(S):
        for p in table[a][:_pages_of(lengths[a], ps)]:
            refs[p] -= 1
    for a in range(S):
        k = lengths[parent[a]]
        new.append(table[parent[a]][:_pages_of(k, ps)])
        for p in new[a]:
            refs[p] += 1
        if add[a] and k % ps:
            wants.setdefault(new[a][-1], []).append(a)
    copied = set()
    for p, who in wants.items():
        if refs[p] > 1:
            copied |= set(who[1:] if len(who) == refs[p] else who)
    copies = [[-1] * S, [-1] * S, [0] * S]
    keys, values = s["keys"].double(), s["values"].double()
    for a in range(S):
        k = lengths[parent[a]]
        if a in copied:
            of, count = new[a][-1], count - 1
            to = free[count]
            refs[of] -= 1
            refs[to] += 1
            new[a][-1] = to
            copies[0][a], copies[1][a], copies[2][a] = of, to, k % ps
            for pool in (keys, values):
                pool[to, :, :k % ps] = pool[of, :, :k % ps]
        while len(new[a]) < _pages_of(k + add[a], ps):
            count -= 1
            new[a].append(free[count])
            refs[free[count]] += 1
    for p in range(P):
        if before[p] > 0 and refs[p] == 0:
            free[count] = p
            count += 1
    after = [lengths[parent[a]] + add[a] for a in range(S)]
    for a in range(S):
        table[a][:len(new[a])] = new[a]
    whole = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return {"table": whole(table), "lengths": whole(after), "refs": whole(refs), "free": whole(free), "count": whole([count]),
            "copies": whole(copies), "keys": keys, "values": values}
