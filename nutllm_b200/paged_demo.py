"""A small serving loop on the paged KV cache: sequences of unequal lengths
decoded together, with eviction to a budget and sparse attention.

    python -m nutllm_b200.paged_demo --prompts 700,90,300 --steps 64 --budget 512 --sparse-pages 24

The model is a stack of attention layers with random weights (there is no
checkpoint to load); what it shows is how the operators go together:

  append     a layer's new queries, keys and values out of one [q; k; v]
             product; rotated, stored, key bounds and positions kept
  attention  over each sequence's own pages; with a budget it also collects
             the attention weight each cached token received
  select + attention  the same over the pages whose keys can match best
             (a prompt's tokens receive that of its newest rows, attended to
             a second time, one row of every sequence a call)
  evict      once a sequence outgrows its budget by a page or more, then its
             pages behind the budget go back to the pool

Every tensor is the caller's (torch); the library allocates its workspace
once per layer.
"""
from __future__ import annotations

import argparse
import time

import torch

import nutllm_b200 as nb

PROMPT_ROWS = 512  # prompt rows of one attention call
PROMPT_WINDOW = 32  # newest prompt rows whose attention ranks a prompt's tokens for eviction
TYPES = {torch.float32: nb.F32, torch.float16: nb.F16, torch.bfloat16: nb.BF16}


class PagedSession:
    """`sequences` caches of `layers` layers over one pool of `pages` pages."""

    def __init__(self, sequences: int, layers: int, heads: int, kv_heads: int, head_dim: int, pages: int,
                 max_pages: int, page_size: int = 16, dtype: torch.dtype = torch.float16, budget: int = 0,
                 sinks: int = 4, recent: int = 64, sparse_pages: int = 0, max_positions: int = 8192):
        if budget and sparse_pages:
            raise ValueError("paged session: weights are collected by attention over all pages only")
        if budget and budget < sinks + recent:
            raise ValueError("paged session: the budget must hold the sinks and the recent tokens")
        dev = torch.device("cuda")
        self.heads, self.kv_heads, self.head_dim, self.page_size = heads, kv_heads, head_dim, page_size
        self.budget, self.sinks, self.recent, self.sparse_pages = budget, sinks, recent, sparse_pages
        self.free = list(range(pages))
        self.owned = [[] for _ in range(sequences)]
        self.length, self.seen = [0] * sequences, [0] * sequences
        self.table = torch.zeros(sequences, max_pages, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device=dev)
        self.seen_dev = torch.zeros_like(self.lengths)
        angle = torch.arange(max_positions, dtype=torch.float64)[:, None] / 10000.0 ** (
            torch.arange(0, head_dim, 2, dtype=torch.float64) / head_dim)
        self.cos, self.sin = angle.cos().float().to(dev), angle.sin().float().to(dev)
        shape, slots = (pages, kv_heads, page_size, head_dim), (sequences, kv_heads, max_pages * page_size)
        self.layers = []
        for _ in range(layers):
            t = dict(keys=torch.zeros(shape, dtype=dtype, device=dev), values=torch.zeros(shape, dtype=dtype, device=dev))
            if sparse_pages:
                t.update(bounds=torch.zeros(pages, kv_heads, 2, head_dim, dtype=torch.int8, device=dev),
                         bound_scales=torch.zeros(pages, kv_heads, device=dev))
            if budget:
                t.update(weights=torch.zeros(slots, device=dev), positions=torch.full(slots, -1, dtype=torch.int32, device=dev))
            at = {k: v.data_ptr() for k, v in t.items()}
            t["cache"] = nb.PagedCache(
                at["keys"], at["values"], self.table.data_ptr(), self.lengths.data_ptr(), sequences=sequences,
                max_pages=max_pages, n_pages=pages, page_size=page_size, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=TYPES[dtype], bounds=at.get("bounds", 0), bound_scales=at.get("bound_scales", 0),
                max_rows=max(sequences, PROMPT_ROWS), track_weights=bool(budget))
            self.layers.append(t)

    def extend(self, news: list) -> torch.Tensor:
        """Makes room for news[s] more tokens of each sequence; the rows' `starts`."""
        pages = [-(-(self.length[s] + n) // self.page_size) for s, n in enumerate(news)]
        if max(pages) > self.table.shape[1] or sum(pages) - sum(map(len, self.owned)) > len(self.free):
            raise RuntimeError("paged session: out of pages")
        for s, n in enumerate(news):
            self.length[s] += n
            self.seen[s] += n
            while len(self.owned[s]) < pages[s]:
                page = self.free.pop()
                self.table[s, len(self.owned[s])] = page
                self.owned[s].append(page)
        self._publish()
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        return torch.tensor(starts, dtype=torch.int32, device="cuda")

    def _publish(self) -> None:
        self.lengths.copy_(torch.tensor(self.length, dtype=torch.int32))
        self.seen_dev.copy_(torch.tensor(self.seen, dtype=torch.int32))

    def append(self, layer: int, qkv: torch.Tensor, starts: torch.Tensor, most: int) -> torch.Tensor:
        """Stores a layer's new rows qkv [rows][(heads + 2 kv_heads) head_dim]; the rotated queries."""
        t, width, step = self.layers[layer], qkv.shape[1], self.head_dim * qkv.element_size()
        q = torch.empty(qkv.shape[0], self.heads * self.head_dim, dtype=qkv.dtype, device=qkv.device)
        at = qkv.data_ptr()
        t["cache"].append(
            at, at + self.heads * step, at + (self.heads + self.kv_heads) * step, starts.data_ptr(), qkv.shape[0], most,
            dtype=TYPES[qkv.dtype], q_stride=width, k_stride=width, v_stride=width, q_out=q.data_ptr(),
            cos=self.cos.data_ptr(), sin=self.sin.data_ptr(), rope_rows=self.cos.shape[0], seen=self.seen_dev.data_ptr(),
            positions=t["positions"].data_ptr() if self.budget else 0, weights=t["weights"].data_ptr() if self.budget else 0,
            stream=torch.cuda.current_stream().cuda_stream)
        return q

    def attend(self, layer: int, q: torch.Tensor) -> torch.Tensor:
        """The newest token of each sequence (q [sequences][heads head_dim]) over its cache."""
        t, kind, stream = self.layers[layer], TYPES[q.dtype], torch.cuda.current_stream().cuda_stream
        out, rows, more = torch.empty_like(q), q.shape[0], {}
        if self.sparse_pages:
            chosen = torch.empty(rows, self.kv_heads, self.sparse_pages, dtype=torch.int32, device=q.device)
            t["cache"].select(q.data_ptr(), chosen.data_ptr(), rows, self.sparse_pages, dtype=kind, sink_pages=1,
                              recent_pages=2, stream=stream)
            more = dict(selected=chosen.data_ptr(), n_selected=self.sparse_pages)
        elif self.budget:
            more = dict(weights=t["weights"].data_ptr(), weights_out=t["weights"].data_ptr())
        t["cache"].attention(q.data_ptr(), out.data_ptr(), rows, dtype=kind, stream=stream, **more)
        return out

    def attend_prompt(self, layer: int, q: torch.Tensor, sequence: torch.Tensor, length: torch.Tensor) -> torch.Tensor:
        """Prompt rows, each over the first length[r] slots of its sequence."""
        out = torch.empty_like(q)
        for i in range(0, q.shape[0], PROMPT_ROWS):
            n = min(PROMPT_ROWS, q.shape[0] - i)
            self.layers[layer]["cache"].attention(
                q[i:].data_ptr(), out[i:].data_ptr(), n, dtype=TYPES[q.dtype], row_sequence=sequence[i:].data_ptr(),
                row_length=length[i:].data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
        return out

    def weigh_prompt(self, layer: int, q: torch.Tensor, starts: torch.Tensor, news: list) -> None:
        """Collects the attention weight that the newest rows of each sequence's prompt (q, as append() gave it) give to
        its tokens: weights are collected from one row per sequence, so a call for each place from the end."""
        t, new = self.layers[layer], starts[1:] - starts[:-1]
        weights = t["weights"].data_ptr()
        for back in range(min(PROMPT_WINDOW, max(news))):
            rows = q[(starts[1:].long() - 1 - back).clamp(min=0)]
            length = torch.where(new > back, self.lengths - back, 0).int()  # 0: sees nothing, adds nothing
            out = torch.empty_like(rows)
            t["cache"].attention(rows.data_ptr(), out.data_ptr(), rows.shape[0], dtype=TYPES[q.dtype], row_length=length.data_ptr(),
                                 weights=weights, weights_out=weights, stream=torch.cuda.current_stream().cuda_stream)

    def trim(self) -> bool:
        """Evicts down to the budget where a sequence is a page or more beyond it; whether it did."""
        if not self.budget or max(self.length) < self.budget + self.page_size:
            return False
        left = torch.empty_like(self.lengths)
        for t in self.layers:
            t["cache"].evict(t["weights"].data_ptr(), t["positions"].data_ptr(), self.seen_dev.data_ptr(), self.budget,
                             sinks=self.sinks, recent=self.recent, new_lengths=left.data_ptr(),
                             weights_out=t["weights"].data_ptr(), positions_out=t["positions"].data_ptr(),
                             stream=torch.cuda.current_stream().cuda_stream)
        for s, n in enumerate(self.length):
            self.length[s] = min(n, self.budget)
            while (len(self.owned[s]) - 1) * self.page_size >= self.length[s]:
                self.free.append(self.owned[s].pop())
        self._publish()
        return True

    def check(self) -> None:
        for t in self.layers:
            t["cache"].check(torch.cuda.current_stream().cuda_stream)


def random_weights(layers: int, heads: int, kv_heads: int, head_dim: int, seed: int = 1) -> list:
    """[q; k; v] and output projections of each layer, as [in][out]."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dim = heads * head_dim
    draw = lambda a, b: torch.randn(a, b, generator=g, device="cuda") / a ** 0.5  # noqa: E731
    return [(draw(dim, (heads + 2 * kv_heads) * head_dim), draw(dim, dim)) for _ in range(layers)]


def norm(x: torch.Tensor) -> torch.Tensor:
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5)


def decode(session: PagedSession, weights: list, prompts: list, steps: int) -> torch.Tensor:
    """Prompts (hidden rows [n][dim] of each sequence), then `steps` tokens of every sequence, each fed the hidden
    row before it; the last hidden rows of all steps [steps][sequences][dim]."""
    news = [len(p) for p in prompts]
    if not all(news):
        raise ValueError("paged session: empty prompt")
    starts = session.extend(news)
    x = torch.cat(prompts)
    seq = torch.repeat_interleave(torch.arange(len(news)), torch.tensor(news)).int().cuda()
    upto = torch.cat([torch.arange(1, n + 1) for n in news]).int().cuda()
    for i, (qkv, out) in enumerate(weights):
        q = session.append(i, norm(x) @ qkv, starts, max(news))
        if session.budget:
            session.weigh_prompt(i, q, starts, news)
        x = x + session.attend_prompt(i, q, seq, upto) @ out
    h, got = norm(x[starts[1:].long() - 1]), []
    for _ in range(steps):
        session.trim()
        starts, x = session.extend([1] * len(news)), h
        for i, (qkv, out) in enumerate(weights):
            x = x + session.attend(i, session.append(i, norm(x) @ qkv, starts, 1)) @ out
        h = norm(x)
        got.append(h)
    return torch.stack(got)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--prompts", default="700,90,300", help="prompt lengths")
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=4)
    ap.add_argument("--head-dim", type=int, default=64)
    ap.add_argument("--budget", type=int, default=512, help="slots a sequence keeps in the run with eviction")
    ap.add_argument("--sparse-pages", type=int, default=24, help="pages a token attends to in the sparse run")
    a = ap.parse_args()
    lens = [int(n) for n in a.prompts.split(",")]
    dim, most = a.heads * a.head_dim, max(lens) + a.steps
    weights = random_weights(a.layers, a.heads, a.kv_heads, a.head_dim)
    g = torch.Generator(device="cuda").manual_seed(7)
    prompts = [torch.randn(n, dim, generator=g, device="cuda") for n in lens]
    per = -(-most // 16)
    full = None
    for name, more in (("all pages", {}), ("evicting to %d" % a.budget, dict(budget=a.budget)),
                       ("%d pages" % a.sparse_pages, dict(sparse_pages=a.sparse_pages))):
        session = PagedSession(len(lens), a.layers, a.heads, a.kv_heads, a.head_dim, pages=len(lens) * per, max_pages=per, **more)
        torch.cuda.synchronize()
        began = time.perf_counter()
        h = decode(session, weights, prompts, a.steps)
        session.check()
        took = time.perf_counter() - began
        full = h if full is None else full
        like = torch.nn.functional.cosine_similarity(h, full, dim=-1).mean().item()
        print(f"{name:18s} {took * 1e3:8.1f} ms for {sum(lens)} prompt rows and {a.steps} steps of {len(lens)}; "
              f"slots in use {session.length}; cosine to all pages {like:.4f}")


if __name__ == "__main__":
    main()
