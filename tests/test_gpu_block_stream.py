"""The attention block on a stream that is not the current one."""
from __future__ import annotations

import pytest
import torch

import test_gpu_attention_block as tb

pytestmark = pytest.mark.gpu

TOKENS = 150
LATE = 200_000_000   # cycles, about a tenth of a second


def _shapes(block):
    return [(TOKENS, block.qkv.n), (TOKENS, tb.HEADS, tb.DIM), (TOKENS, block.out.n)]


def _setup(ctx):
    block, pool, _, _ = tb.build(ctx, 20)
    step = pool.step(["a", "b"], [TOKENS - 20, 20], "cuda")
    x = torch.randn((TOKENS, tb.HIDDEN), device="cuda").bfloat16()
    want = block(x, step).clone()    # the same step again writes the same cache
    torch.cuda.synchronize()
    return block, step, x, want


def test_later_work_of_the_current_stream_keeps_its_memory(ctx):
    block, step, x, want = _setup(ctx)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(LATE)
    y = block(x, step, stream=side)
    mine = [torch.full(s, 3.0, dtype=torch.bfloat16, device="cuda") for s in _shapes(block) * 3]
    torch.cuda.synchronize()
    assert all(bool((t == 3).all()) for t in mine)
    assert torch.equal(y, want) and ctx.status() == 0


def test_earlier_work_of_the_current_stream_spares_the_result(ctx):
    block, step, x, want = _setup(ctx)
    side = torch.cuda.Stream()
    before = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in _shapes(block) * 3]
    torch.cuda._sleep(LATE)
    for t in before:
        t.fill_(float("nan"))
    del before, t
    y = block(x, step, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and ctx.status() == 0


def test_inputs_made_on_the_current_stream_are_waited_for(ctx):
    block, step, x, want = _setup(ctx)
    side, late = torch.cuda.Stream(), torch.zeros_like(x)
    torch.cuda._sleep(LATE)
    late.copy_(x)
    y = block(late, step, stream=side)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@pytest.mark.parametrize("form", ["stream", "address"])
def test_a_freed_result_is_not_overwritten_while_it_is_read(ctx, form):
    block, step, x, want = _setup(ctx)
    side = torch.cuda.Stream()
    y = block(x, step, stream=side if form == "stream" else side.cuda_stream)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda._sleep(LATE)
    read = y.clone()                      # runs after the sleep
    del y
    with torch.cuda.stream(side):
        other = [torch.full(s, 3.0, dtype=torch.bfloat16, device="cuda") for s in _shapes(block) * 3]
    torch.cuda.synchronize()
    assert torch.equal(read, want) and len(other) == 9
