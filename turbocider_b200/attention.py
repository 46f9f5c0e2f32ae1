"""An attention block on quantised weights and a paged cache: the q / k / v
projection (qlinear), the heads' norm and rotation on the way into the cache
(kv_append), attention over it (paged_attention) and the output projection.

    python -m turbocider_b200.attention [--requests N] [--prompt T] [--steps K]

runs prompts and single-token steps of synthetic requests through a block and
prints what they take.
"""
from __future__ import annotations

from . import cuda as tcc


class PagePool:
    """Which page of a cache holds which tokens of which request (host side).
    Pages are taken as requests grow and given back by release()."""

    def __init__(self, n_pages: int, page_size: int):
        self.page_size = page_size
        self._free = list(range(n_pages - 1, -1, -1))
        self._pages: dict = {}
        self._length: dict = {}

    def length(self, request) -> int:
        return self._length.get(request, 0)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def grow(self, request, tokens: int) -> int:
        """Room for `tokens` more of the request; its new length.  Takes
        nothing when the pool has too few pages left."""
        if tokens < 0:
            raise ValueError("a request cannot shrink")
        length = self.length(request) + tokens
        pages = self._pages.get(request, [])
        missing = -(-length // self.page_size) - len(pages)
        if missing > len(self._free):
            raise MemoryError(f"the cache has {len(self._free)} free pages, {missing} are needed")
        self._pages[request] = pages + [self._free.pop() for _ in range(missing)]
        self._length[request] = length
        return length

    def release(self, request) -> None:
        self._free.extend(reversed(self._pages.pop(request, [])))
        self._length.pop(request, None)

    def table(self, requests) -> list[list[int]]:
        """Rows of page numbers, padded with -1 to the longest."""
        rows = [self._pages.get(r, []) for r in requests]
        width = max([len(r) for r in rows] + [1])
        return [r + [-1] * (width - len(r)) for r in rows]

    def step(self, requests, new, device):
        """Grows each request by its new tokens; the PagedBatch of the step.
        A step that fails changes nothing."""
        import torch
        requests, new = list(requests), list(new)
        if len(requests) != len(new):
            raise ValueError(f"{len(requests)} requests, new tokens of {len(new)}")
        if not requests:
            raise ValueError("a step needs a request")

        def ints(v):
            return torch.tensor(v, dtype=torch.int32, device=device)
        lengths, offsets, before = [], [0], []
        try:
            for r, n in zip(requests, new):
                pages, length = self._pages.get(r), self._length.get(r)
                lengths.append(self.grow(r, n))
                before.append((r, pages, length))
                offsets.append(offsets[-1] + n)
            return tcc.PagedBatch(ints(offsets), ints(lengths), ints(self.table(requests)), max(new), max(lengths))
        except BaseException:
            for r, pages, length in reversed(before):
                self._free.extend(reversed(self._pages[r][len(pages or []):]))
                if pages is None:
                    del self._pages[r], self._length[r]
                else:
                    self._pages[r], self._length[r] = pages, length
            raise


class AttentionBlock:
    """Causal attention of one layer in bf16.  qkv: a Weight of (n_heads + 2 n_kv) head_dim
    rows (queries' heads, keys', values'); out: a Weight of n_heads head_dim
    columns.  q_norm / k_norm: f32 [head_dim], or None for no norm.  freq: the
    rotation's frequencies (cuda.rope_freqs), positions being the tokens' places
    in the cache."""

    def __init__(self, ctx: tcc.Context, qkv: tcc.Weight, out: tcc.Weight, cache: tcc.PagedCache, n_heads: int,
                 q_norm=None, k_norm=None, eps: float = 1e-6, freq=None, layout: str = "half", amplitude: float = 1.0,
                 window: int = 0):
        dim, n_kv = cache.head_dim, cache.n_heads
        if qkv.n != (n_heads + 2 * n_kv) * dim or out.k != n_heads * dim:
            raise ValueError("the projections do not fit the heads of the cache")
        if (q_norm is None) != (k_norm is None):
            raise ValueError("a norm of the queries and one of the keys, or neither")
        self.ctx, self.qkv, self.out, self.cache = ctx, qkv, out, cache
        self.n_heads, self.n_kv, self.dim = n_heads, n_kv, dim
        self.q_norm, self.k_norm, self.eps = q_norm, k_norm, None if q_norm is None else eps
        self.rope = None if freq is None else tcc.Rope(freq, layout=layout, amplitude=amplitude)
        self.window = window

    def __call__(self, x, batch: tcc.PagedBatch, stream=None):
        """x: contiguous bf16 [tokens, hidden] of the step's new tokens; returns
        the block's output [tokens, out.n] (bf16).  The cache must be bf16.
        With a stream that is not the current one the block runs there, after
        what the current stream holds, on memory of that stream; the caller
        has to order what reads the result after it."""
        import torch
        # (the projection takes its rows at their address, whatever they are)
        if x.dtype is not torch.bfloat16 or x.dim() != 2 or x.shape[1] != self.qkv.k or not x.is_contiguous():
            raise tcc.BackendError(f"x must be a contiguous bf16 tensor [tokens, {self.qkv.k}]")
        if x.get_device() != self.ctx.device:
            raise tcc.BackendError("x must be on the context's device")
        if not x.shape[0]:
            return x.new_empty((0, self.out.n))
        caller = torch.cuda.current_stream(self.ctx.device)
        if stream is None:
            return self._run(x, batch, caller)
        if not isinstance(stream, torch.cuda.Stream):   # an address, as the other calls take it
            stream = torch.cuda.ExternalStream(stream, self.ctx.device) if stream else \
                torch.cuda.default_stream(self.ctx.device)
        if stream == caller:
            return self._run(x, batch, caller)
        stream.wait_stream(caller)
        with torch.cuda.stream(stream):
            y = self._run(x, batch, stream)
        # freed, these go back to their streams' memory only once both are through with them
        for t in (x, *batch.tensors):
            t.record_stream(stream)
        y.record_stream(caller)
        return y

    def _run(self, x, batch, stream):
        """The block on `stream`, which is the current one of the context's device."""
        row = tcc.qlinear(self.ctx, self.qkv, x, stream=stream)
        heads = row.view(x.shape[0], self.n_heads + 2 * self.n_kv, self.dim)
        q, k, v = heads.split((self.n_heads, self.n_kv, self.n_kv), 1)
        q = tcc.kv_append(self.ctx, self.cache, batch, k, v, self.rope, q=q, q_weight=self.q_norm,
                          k_weight=self.k_norm, eps=self.eps, stream=stream)
        y = tcc.paged_attention(self.ctx, self.cache, batch, q, window=self.window, stream=stream)
        return tcc.qlinear(self.ctx, self.out, y.view(x.shape[0], -1), stream=stream)


def _demo(n_requests: int, prompt: int, steps: int, hidden: int = 2560, n_heads: int = 32, n_kv: int = 8,
          dim: int = 128, page: int = 16) -> None:
    import numpy as np
    import torch
    rng = np.random.default_rng(0)
    ctx = tcc.Context(0)

    def weight(n, k):
        w = rng.standard_normal((n, k), dtype=np.float32) * 0.02
        return tcc.Weight.upload(ctx, tcc.Q4_K, n, k, tcc.quantize(tcc.Q4_K, w))
    pages = n_requests * (-(-(prompt + steps) // page))
    k, v = (torch.zeros((pages, n_kv, page, dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    freq, amplitude = tcc.rope_freqs(dim, 1e6, device="cuda")
    ones = torch.ones(dim, device="cuda")
    block = AttentionBlock(ctx, weight((n_heads + 2 * n_kv) * dim, hidden), weight(hidden, n_heads * dim),
                           tcc.PagedCache(k, v), n_heads, ones, ones, freq=freq, amplitude=amplitude)
    pool, requests = PagePool(pages, page), list(range(n_requests))

    def timed(new):
        batch = pool.step(requests, [new] * n_requests, "cuda")
        x = torch.randn((new * n_requests, hidden), device="cuda").bfloat16()
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        block(x, batch)
        end.record()
        torch.cuda.synchronize()
        return begin.elapsed_time(end) * 1e3
    timed(prompt)                      # first use: modules and workspaces
    for r in requests:
        pool.release(r)
    first = timed(prompt)
    each = sorted(timed(1) for _ in range(steps))
    print(f"{n_requests} prompts of {prompt} tokens: {first:.0f} us; a token for each: {each[len(each) // 2]:.1f} us "
          f"(median of {steps} steps)")
    if ctx.status():
        raise SystemExit("a kernel reported an error")


if __name__ == "__main__":
    import argparse
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--steps", type=int, default=20)
    a = ap.parse_args()
    _demo(a.requests, a.prompt, a.steps)
