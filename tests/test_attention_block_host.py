"""What the attention block takes as its input (no GPU: the projection that
would read it is a stand-in)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from turbocider_b200 import cuda as tcc
from turbocider_b200.attention import AttentionBlock

HIDDEN, HEADS, KV, DIM = 64, 4, 2, 16


@pytest.fixture
def block(monkeypatch):
    def reached(*a, **kw):
        pytest.fail("the projection was reached")
    monkeypatch.setattr(tcc, "qlinear", reached)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: SimpleNamespace(cuda_stream=0))
    qkv, out = SimpleNamespace(n=(HEADS + 2 * KV) * DIM, k=HIDDEN), SimpleNamespace(n=HIDDEN, k=HEADS * DIM)
    return AttentionBlock(SimpleNamespace(device=0), qkv, out, SimpleNamespace(head_dim=DIM, n_heads=KV), HEADS)


X = torch.zeros((5, HIDDEN), dtype=torch.bfloat16)


@pytest.mark.parametrize("x", [X.half(), X.float(), X[:, :-1], X[:, :32], X[None], X[0],
                               torch.zeros((5, 2 * HIDDEN), dtype=torch.bfloat16)[:, :HIDDEN],
                               torch.zeros((HIDDEN, 5), dtype=torch.bfloat16).T, torch.zeros((1, HIDDEN)).bfloat16().expand(5, -1)],
                         ids=["f16", "f32", "narrow", "half", "batched", "vector", "slice", "transposed", "broadcast"])
def test_inputs_that_the_projection_would_misread_are_refused(block, x):
    with pytest.raises(tcc.BackendError, match="contiguous bf16"):
        block(x, None)


def test_an_input_elsewhere_is_refused(block):
    with pytest.raises(tcc.BackendError, match="context's device"):
        block(X, None)


def test_a_step_without_tokens_is_empty(block):
    block.ctx.device = -1   # where X is
    y = block(X[:0], None)
    assert y.shape == (0, HIDDEN) and y.dtype == torch.bfloat16
