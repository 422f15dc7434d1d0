"""Decoding that branches, on the paged KV cache: beam search, and greedy
decoding with drafted trees.

    python -m nutllm_b200.branch_demo --prompts 300,45,120 --steps 32 --beams 4

The model is a stack of attention layers with random weights between an
embedding and a head (there is no checkpoint to load); what it shows is how the
operators go together.

  a beam step   update (each beam continues the one that was chosen for it:
                whole pages are shared), copy_pages (a partly filled page that
                two beams would write), append, attention, select
  a tree step   update (what was accepted stays, room for the next tree),
                append with positions by depth, tree_attention (all drafted
                tokens in one pass over the cache), compact (the accepted ones)

A prompt is a tree without branches.  Tables, lengths and the book of pages
stay on the device; every tensor is the caller's (torch).
"""
from __future__ import annotations

import argparse
import time

import torch

import nutllm_b200 as nb

TYPES = {torch.float32: nb.F32, torch.float16: nb.F16, torch.bfloat16: nb.BF16}


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def masks(parents: list) -> torch.Tensor:
    """Mask words of a forest: a node sees itself and its ancestors (parents[i] < i, -1: the cache)."""
    seen = []
    for i, parent in enumerate(parents):
        seen.append((seen[parent] if parent >= 0 else 0) | 1 << i)
    words = max(1, -(-len(parents) // 32))
    rows = [[s >> 32 * w & 0xffffffff for w in range(words)] for s in seen]
    return torch.tensor(rows, dtype=torch.int64).reshape(-1, words)


def mask_tensor(rows: list) -> torch.Tensor:
    """The masks of several sequences' trees, one behind the other, in words of 32 bits on the device."""
    words = max(r.shape[1] for r in rows)
    bits = torch.cat([torch.nn.functional.pad(r, (0, words - r.shape[1])) for r in rows])
    return torch.where(bits < 1 << 31, bits, bits - (1 << 32)).to(torch.int32).cuda()


def depths(parents: list) -> list:
    got = []
    for parent in parents:
        got.append(got[parent] + 1 if parent >= 0 else 0)
    return got


def _check_prompts(prompts: list) -> None:
    """A prompt's last row gives the first token: there has to be one."""
    if not all(len(p) > 0 for p in prompts):
        raise ValueError("branch session: empty prompt")


class Model:
    """Embedding, attention layers and a head, with random weights."""

    def __init__(self, vocab: int, layers: int, heads: int, kv_heads: int, head_dim: int, seed: int = 1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        dim = heads * head_dim
        draw = lambda a, b: torch.randn(a, b, generator=g, device="cuda") / a ** 0.5  # noqa: E731
        self.vocab, self.heads, self.kv_heads, self.head_dim = vocab, heads, kv_heads, head_dim
        self.embedding = torch.randn(vocab, dim, generator=g, device="cuda")
        self.head = 3 * draw(dim, vocab)
        # (layers that add little: what the draft says without them is often right)
        self.layers = [(draw(dim, (heads + 2 * kv_heads) * head_dim), 0.4 * draw(dim, dim)) for _ in range(layers)]

    def logits(self, x: torch.Tensor) -> torch.Tensor:
        return norm(x) @ self.head


def norm(x: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


class BranchSession:
    """`sequences` caches of a model's layers over pools of `pages` pages, whose book is kept on the device."""

    def __init__(self, model: Model, sequences: int, pages: int, max_pages: int, most: int, page_size: int = 16,
                 dtype: torch.dtype = torch.float16, max_positions: int = 4096):
        self.model, self.sequences = model, sequences
        heads, kv, D = model.heads, model.kv_heads, model.head_dim
        dev = torch.device("cuda")
        self.table = torch.zeros(sequences, max_pages, dtype=torch.int32, device=dev)
        self.lengths, self.refs = _ints([0] * sequences), _ints([0] * pages)
        self.free, self.count = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device=dev), _ints([pages])
        self.copies = torch.empty(3, sequences, dtype=torch.int32, device=dev)
        self.book = nb.PageBook(self.table.data_ptr(), self.lengths.data_ptr(), self.refs.data_ptr(), self.free.data_ptr(),
                                self.count.data_ptr(), sequences=sequences, max_pages=max_pages, n_pages=pages, page_size=page_size)
        angle = torch.arange(max_positions, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(0, D, 2, dtype=torch.float64) / D)
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        self.pools, self.caches = [], []
        for _ in model.layers:
            pool = torch.zeros(2, pages, kv, page_size, D, dtype=dtype, device=dev)
            cache = nb.PagedCache(pool[0].data_ptr(), pool[1].data_ptr(), self.table.data_ptr(), self.lengths.data_ptr(),
                                  sequences=sequences, max_pages=max_pages, n_pages=pages, page_size=page_size, heads=heads,
                                  kv_heads=kv, head_dim=D, dtype=TYPES[dtype])
            cache.reserve_tree(most)
            self.pools.append(pool)
            self.caches.append(cache)

    def update(self, parent: torch.Tensor = None, keep: torch.Tensor = None, add: torch.Tensor = None) -> None:
        """Every sequence continues parent[s], keeps keep[s] slots and gets add[s] more; split pages are copied."""
        at = [x.data_ptr() if x is not None else 0 for x in (parent, keep, add)]
        lists = [row.data_ptr() for row in self.copies]
        self.book.update(parent=at[0], keep=at[1], add=at[2], copy_from=lists[0], copy_to=lists[1], copy_slots=lists[2],
                         stream=_stream())
        for cache in self.caches:
            cache.copy_pages(lists[0], lists[1], self.sequences, slots=lists[2], stream=_stream())

    def forward(self, tokens: torch.Tensor, starts: torch.Tensor, most: int, mask: torch.Tensor = None,
                position: torch.Tensor = None) -> torch.Tensor:
        """Hidden rows of the tokens in the sequences' newest slots; without a mask one token of each."""
        m, x = self.model, self.model.embedding[tokens.long()]
        H, KV, D, rows = m.heads, m.kv_heads, m.head_dim, tokens.shape[0]
        for (qkv_weight, out_weight), cache in zip(m.layers, self.caches):
            qkv = norm(x) @ qkv_weight
            q, out = torch.empty(2, rows, H * D, device="cuda").unbind()
            at, width = qkv.data_ptr(), qkv.shape[1]
            cache.append(at, at + H * D * 4, at + (H + KV) * D * 4, starts.data_ptr(), rows, most, q_stride=width, k_stride=width,
                         v_stride=width, q_out=q.data_ptr(), cos=self.cos.data_ptr(), sin=self.sin.data_ptr(),
                         rope_rows=self.cos.shape[0], row_position=position.data_ptr() if position is not None else 0,
                         stream=_stream())
            if mask is None:
                cache.attention(q.data_ptr(), out.data_ptr(), rows, stream=_stream())
            else:
                cache.tree_attention(q.data_ptr(), out.data_ptr(), starts.data_ptr(), mask.data_ptr(), rows, most, mask.shape[1],
                                     stream=_stream())
            x = x + out @ out_weight
        return x

    def prompts(self, prompts: list) -> torch.Tensor:
        """Fills the caches with prompts (token lists, empty for a sequence without one); the hidden rows."""
        news = [len(p) for p in prompts]
        self.update(add=_ints(news))
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        mask = mask_tensor([masks(list(range(-1, n - 1))) for n in news if n])
        return self.forward(_ints([t for p in prompts for t in p]), _ints(starts), max(news), mask)

    def check(self) -> None:
        self.book.check(_stream())
        for cache in self.caches:
            cache.check(_stream())


def beam_search(model: Model, prompts: list, steps: int, beams: int, eos: int, dtype: torch.dtype = torch.float16,
                page_size: int = 16) -> list:
    """The `beams` best continuations of each prompt as (score, tokens), best first.  The loop over the steps never waits
    for the device."""
    _check_prompts(prompts)
    requests = len(prompts)
    most, S = max(map(len, prompts)), requests * beams
    max_pages = -(-(most + steps) // page_size)
    # every beam may come to own the pages behind its prompt, and a page while it is split
    pages = requests * -(-most // page_size) + S * (-(-steps // page_size) + 2)
    s = BranchSession(model, S, pages, max_pages, most, page_size, dtype, most + steps)
    search = nb.BeamSearch(requests, beams, model.vocab, beams)
    x = s.prompts([prompts[i // beams] if i % beams == 0 else [] for i in range(S)])
    last = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
    logits = torch.zeros(S, model.vocab, device="cuda")
    logits[::beams] = model.logits(x[last.cuda()])
    # at first there is one beam
    scores = torch.full((requests, beams), -torch.inf, device="cuda")
    scores[:, 0] = 0.0
    finished = torch.zeros(requests, beams, dtype=torch.uint8, device="cuda")
    rows, tokens = (torch.empty(steps, S, dtype=torch.int32, device="cuda") for _ in range(2))
    starts, one = torch.arange(S + 1, dtype=torch.int32, device="cuda"), _ints([1] * S)
    for i in range(steps):
        search.select(logits.data_ptr(), scores.data_ptr(), scores.data_ptr(), rows[i].data_ptr(), tokens[i].data_ptr(),
                      finished=finished.data_ptr(), eos=eos, out_finished=finished.data_ptr(), stream=_stream())
        if i + 1 < steps:
            # (with fewer candidates than beams a row is -1: nothing is kept, and its score stays -infinity)
            s.update(parent=rows[i], add=one)
            logits = model.logits(s.forward(tokens[i].clamp(min=0), starts, 1))
    s.check()
    rows, tokens, scores = rows.tolist(), tokens.tolist(), scores.tolist()
    got = []
    for r in range(requests):
        best = []
        for b in range(beams):
            path, at = [], r * beams + b
            for i in reversed(range(steps)):
                if at < 0:
                    break
                path.append(tokens[i][at])
                at = rows[i][at]
            path.reverse()
            best.append((scores[r][b], path[:path.index(eos) + 1] if eos in path else path))
        got.append(best)
    return got


def draft(model: Model, root: int, widths: list) -> tuple:
    """A tree of guesses behind token `root`: (tokens, parents), the root first.  A guess is what the model says without
    its layers; widths[d] of them at depth d + 1."""
    tokens, parents, level = [root], [-1], [0]
    for width in widths:
        said = model.logits(model.embedding[torch.tensor([tokens[i] for i in level], device="cuda")])
        below = []
        for i, guesses in zip(level, said.topk(width).indices.tolist()):
            for t in guesses:
                below.append(len(tokens))
                tokens.append(t)
                parents.append(i)
        level = below
    return tokens, parents


def tree_greedy(model: Model, prompts: list, steps: int, widths: list, dtype: torch.dtype = torch.float16,
                page_size: int = 16) -> tuple:
    """Greedy continuations of `steps` tokens, verified a drafted tree at a time (widths []: a token at a time), and the
    number of passes over the caches."""
    _check_prompts(prompts)
    S, size = len(prompts), 1
    for w in reversed(widths):
        size = 1 + w * size
    most = max(map(len, prompts))
    max_pages = -(-(most + steps + 2 * size) // page_size)
    s = BranchSession(model, S, S * max_pages, max_pages, max(most, size), page_size, dtype, most + steps + 2 * size)
    x = s.prompts(prompts)
    last = torch.tensor([len(p) for p in prompts]).cumsum(0) - 1
    pending = model.logits(x[last.cuda()]).argmax(-1).tolist()  # known, not in the cache yet
    lengths = [len(p) for p in prompts]
    got, passes = [[] for _ in prompts], 0
    left = s.lengths.clone()
    while min(map(len, got)) < steps:
        trees = [draft(model, t, widths) for t in pending]
        tokens = [t for tree in trees for t in tree[0]]
        n = len(trees[0][0])
        starts = _ints([n * i for i in range(S + 1)])
        s.update(keep=left, add=_ints([n] * S))
        position = _ints([lengths[i] + d for i, tree in enumerate(trees) for d in depths(tree[1])])
        x = s.forward(_ints(tokens), starts, n, mask_tensor([masks(tree[1]) for tree in trees]), position)
        passes += 1
        said = model.logits(x).argmax(-1).tolist()
        accepted = []
        for i, (drafted, parents) in enumerate(trees):
            path = [0]
            while True:
                follows = said[i * n + path[-1]]
                below = [j for j in range(len(drafted)) if parents[j] == path[-1] and drafted[j] == follows]
                if not below:
                    break
                path.append(below[0])
            got[i] += [drafted[j] for j in path]
            pending[i] = said[i * n + path[-1]]
            lengths[i] += len(path)
            accepted.append(path + [-1] * (len(widths) + 1 - len(path)))
        accepted = _ints(accepted)
        for cache in s.caches:
            cache.compact(starts.data_ptr(), accepted.data_ptr(), accepted.shape[1], new_lengths=left.data_ptr(), stream=_stream())
        # a sequence that is ahead waits for the others with what it has
        for i in range(S):
            if len(got[i]) >= steps + size and min(map(len, got)) < steps:
                back = len(got[i]) - steps
                pending[i] = got[i][steps]
                got[i], lengths[i] = got[i][:steps], lengths[i] - back
                left[i] -= back
    s.check()
    return [g[:steps] for g in got], passes


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", default="300,45,120", help="prompt lengths, up to 1024")
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--head-dim", type=int, default=64)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--beams", type=int, default=4)
    ap.add_argument("--widths", default="4,2,1", help="branches at each depth of a drafted tree")
    a = ap.parse_args()
    model = Model(a.vocab, a.layers, a.heads, a.kv_heads, a.head_dim)
    g = torch.Generator().manual_seed(7)
    prompts = [torch.randint(0, a.vocab, (int(n),), generator=g).tolist() for n in a.prompts.split(",")]
    torch.cuda.synchronize()

    def timed(what, f):
        began = time.perf_counter()
        got = f()
        torch.cuda.synchronize()
        print(f"{what:24s} {(time.perf_counter() - began) * 1e3:8.1f} ms", end="  ")
        return got

    best = timed(f"beam search, {a.beams} beams", lambda: beam_search(model, prompts, a.steps, a.beams, eos=2))
    print("best scores", [round(b[0][0], 2) for b in best])
    plain, passes = timed("greedy, token by token", lambda: tree_greedy(model, prompts, a.steps, []))
    print(passes, "passes")
    tree, fewer = timed("greedy, drafted trees", lambda: tree_greedy(model, prompts, a.steps, [int(w) for w in a.widths.split(",")]))
    print(f"{fewer} passes; tokens as before: {sum(p == t for p, t in zip(plain, tree))} of {len(plain)} sequences")


if __name__ == "__main__":
    main()
