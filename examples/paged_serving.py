"""Continuous batching on the paged 4-bit cache: sequences of unlike lengths join and leave, share a prefix, and branch.

    python examples/paged_serving.py [--layers 4] [--rows 32] [--prefix 2048] [--requests 96] [--new-tokens 128]

A stack of attention layers with random projections stands in for a model.  A common prefix is written once and forked into every request's row (pages are
shared, only the 16-bit window is copied); requests bring prompts of their own, decode until they are done, and make room for the next ones; one
in eight branches into two continuations half way.  A decode step (extend, then append and attend per layer) is captured once in a CUDA graph:
lengths and pages live on the device.  The first sequence that ends, the first branch that does and the prefix are checked in every layer: their attention against dense
attention over what their pages hold, and of the first one what its pages hold against the keys that were written.
"""
from __future__ import annotations

import argparse
import os
import random
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from muzero_b200 import MuZeroPagedCache  # noqa: E402


class Layer:
    """Random projections of an attention layer and its share of the cache."""

    def __init__(self, index: int, hidden: int, heads: int, kv_heads: int, dim: int, gen: torch.Generator):
        def weight(n, m):
            return (torch.randn(n, m, device="cuda", generator=gen) * n ** -0.5).bfloat16()
        self.index, self.heads, self.kv_heads, self.dim = index, heads, kv_heads, dim
        self.q, self.kv, self.o = weight(hidden, heads * dim), weight(hidden, 2 * kv_heads * dim), weight(heads * dim, hidden)

    def project(self, x: torch.Tensor):
        kv = (x @ self.kv).view(-1, 2, self.kv_heads, self.dim)
        return (x @ self.q).view(-1, self.heads, self.dim), kv[:, 0], kv[:, 1]

    def decode(self, cache: MuZeroPagedCache, x: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
        q, k, v = self.project(x)
        cache.append(self.index, k, v, rows=rows)
        return x + cache.attend(self.index, q, rows=rows).flatten(1) @ self.o


def prefill(cache: MuZeroPagedCache, layers: list, x: torch.Tensor, rows: torch.Tensor, lengths: list) -> None:
    """Writes prompts (entry after entry in ``x``).  Their own attention is a model's prefill and not the point here; layers see the embeddings."""
    offsets = torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    cache.extend(rows=rows, offsets=offsets)
    for layer in layers:
        _, k, v = layer.project(x)
        cache.append(layer.index, k, v, rows=rows, offsets=offsets, max_new=max(lengths))


def main(argv=None) -> dict:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--rows", type=int, default=32)
    ap.add_argument("--prefix", type=int, default=2048)
    ap.add_argument("--requests", type=int, default=96)
    ap.add_argument("--new-tokens", type=int, default=128)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args(argv)
    heads, kv_heads, dim, hidden, residual = 32, 8, 128, 1024, 128
    rng, gen = random.Random(a.seed), torch.Generator(device="cuda").manual_seed(a.seed)
    layers = [Layer(i, hidden, heads, kv_heads, dim, gen) for i in range(a.layers)]
    longest = a.prefix + 512 + a.new_tokens
    # the prefix's pages once, each row's own pages, and the row that holds the prefix (the last one)
    pages = longest // 64 + (a.rows + 1) * ((512 + a.new_tokens + residual) // 64 + 2)
    cache = MuZeroPagedCache.allocate(layers=a.layers, kv_heads=kv_heads, head_dim=dim, pages=pages, rows=a.rows + 1, max_length=longest, residual_length=residual)
    home = a.rows
    index = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    history = [torch.randn(a.prefix, hidden, device="cuda", generator=gen).bfloat16()]      # what the first request's row is given, in the end
    prefill(cache, layers, history[0], index(home), [a.prefix])

    left = [0] * a.rows                                   # tokens that a row still has to decode; 0: the row is free
    x = torch.zeros(a.rows, hidden, device="cuda", dtype=torch.bfloat16)
    rows = torch.arange(a.rows, dtype=torch.int32, device="cuda")

    def admit(waiting: int) -> int:
        """Starts requests in free rows: fork the prefix, write the prompts."""
        new = [r for r in range(a.rows) if left[r] == 0][:waiting]
        if new:
            cache.fork(index(*[home] * len(new)), index(*new))
            lengths = [rng.randint(1, 512) for _ in new]
            prompts = torch.randn(sum(lengths), hidden, device="cuda", generator=gen).bfloat16()
            prefill(cache, layers, prompts, index(*new), lengths)
            if len(history) == 1:
                history.append(prompts[:lengths[0]])      # the first request has row 0
            for r in new:
                left[r] = a.new_tokens - rng.randint(0, a.new_tokens // 2)
        return len(new)

    def step() -> torch.Tensor:
        cache.extend(rows=rows)
        y = x
        for layer in layers:
            y = layer.decode(cache, y, rows)
        return y

    waiting = a.requests - admit(a.requests)
    # All rows take part in a captured step; a free row is a sequence that nobody reads, emptied again when its place is given away
    for r in range(a.rows):
        if left[r] == 0:
            cache.fork(index(home), index(r))
    cache.check()
    # warm up on a copy of the tables (the graph's first run must not be the second write of a token): the steps' effects are put back
    state = [t.clone() for t in (cache.block_table, cache.lengths, cache.page_refs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip((cache.block_table, cache.lengths, cache.page_refs), state):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = step()

    def dense_error(row: int) -> float:
        """The largest error, over the layers, of a row's attention against dense attention over what its pages and ring hold."""
        q, worst = torch.randn(1, heads, dim, device="cuda", generator=gen).bfloat16(), 0.0
        for layer in range(a.layers):
            got = cache.attend(layer, q, rows=index(row)).float()
            k, v = read_row(cache, layer, row)
            s = torch.einsum("hd,thd->ht", q[0].float(), k.repeat_interleave(heads // kv_heads, 1)) * dim ** -0.5
            want = torch.einsum("ht,thd->hd", torch.softmax(s, -1), v.repeat_interleave(heads // kv_heads, 1))
            worst = max(worst, float((got[0] - want).norm() / want.norm()))
        return worst

    errors, branches, held = {}, [], None
    done = branched = decoded = moved = 0
    torch.cuda.synchronize()
    began = time.perf_counter()
    while any(left):
        if held is None:
            history.append(x[:1].clone())
        graph.replay()
        x.copy_(torch.nn.functional.normalize(y.float(), dim=-1).mul_(hidden ** 0.5))      # the next token's embedding
        ended = []
        for r in range(a.rows):
            if left[r] > 0:
                left[r] -= 1
                decoded += 1
                if left[r] == 0:
                    ended.append(r)
        if ended:
            done += len(ended)
            first, branch = held is None and 0 in ended, "branch" not in errors and set(branches) & set(ended)
            if first or branch:
                torch.cuda.synchronize()
                paused = time.perf_counter()
                if first:
                    errors["first"] = dense_error(0)
                    _, key, _ = layers[0].project(torch.cat(history))
                    held = float((read_row(cache, 0, 0)[0] - key.float()).norm() / key.float().norm())
                if branch:
                    errors["branch"] = dense_error(min(branch))
                began += time.perf_counter() - paused
            branches = [r for r in branches if r not in ended]
            cache.free(index(*ended))
            waiting -= admit(waiting)
            idle = [r for r in range(a.rows) if left[r] == 0]
            if idle:                                      # rows for which nobody waits: a branch of a running sequence, or the prefix again
                running = [r for r in range(a.rows) if left[r] > a.new_tokens // 2]
                if running and rng.random() < 0.125:
                    cache.fork(index(running[0]), index(idle[0]))
                    x[idle[0]] = x[running[0]] + 0.1 * torch.randn(hidden, device="cuda", generator=gen).bfloat16()
                    left[idle[0]] = left[running[0]]
                    branches.append(idle[0])
                    branched += 1
                    idle = idle[1:]
                if idle:
                    cache.fork(index(*[home] * len(idle)), index(*idle))
            if done % 16 == 0:
                cache.compact()
                moved += 1
    torch.cuda.synchronize()
    seconds = time.perf_counter() - began
    cache.check()

    errors["prefix"] = dense_error(home)
    out = {"requests": done, "branches": branched, "compactions": moved, "tokens": decoded, "seconds": round(seconds, 3),
           "tokens_per_s": round(decoded / seconds, 1), "free_pages": cache.free_pages(), "pages": pages,
           "error": max(errors.values()), "errors": errors, "held": held}
    print(out)
    return out


def read_row(cache: MuZeroPagedCache, layer: int, row: int):
    """A row's keys and values as they stand in its pages and ring, [tokens, kv_heads, head_dim] in fp32."""
    import ctypes
    book = (ctypes.c_ubyte * 2048)()
    cache._lib.mz_paged_books(book, (ctypes.c_ubyte * 16384)())
    book = torch.tensor(list(book), device=cache.device).view(128, 16)
    n, d, h = int(cache.lengths[row]), cache.head_dim, cache.kv_heads
    np_ = max(0, n - cache.residual_length) // 64
    raw = cache.store[layer, cache.block_table[row, :np_].long()]

    def side(codes, words):
        w = words.contiguous().view(torch.int32)
        t, field = (w & 0xFFFF).short().view(torch.float16).float(), (w >> 16) & 0xFFFF
        off = (field & 0x7FFF) >= 128
        anchor = torch.where(off, field.short().view(torch.float16).float(), torch.zeros_like(t))
        z = torch.where(off, torch.where(anchor < 0, 127, 0), field).long()
        e = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
        return anchor[..., None] + t[..., None] * (book[z[..., None], e] - z[..., None]) / 32

    kc, kw, vc, vw = raw.split([32 * d, 4 * d, 32 * d, 4 * d], -1)
    k = side(kc.reshape(np_, h, d, 32), kw).permute(0, 3, 1, 2).reshape(np_ * 64, h, d)
    v = side(vc.reshape(np_, h, 64 * d // 64, 32), vw).reshape(np_, h, 64, d).transpose(1, 2).reshape(np_ * 64, h, d)
    at = torch.arange(np_ * 64, n, device=cache.device) % cache.tail.shape[4]
    ring = cache.tail[layer, row][:, :, at].float().transpose(1, 2)
    return torch.cat([k, ring[0]]), torch.cat([v, ring[1]])


if __name__ == "__main__":
    main()
