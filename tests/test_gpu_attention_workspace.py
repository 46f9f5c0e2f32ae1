"""Paged attention where the GPU has no room for its partial results."""
from __future__ import annotations

import pytest
import torch

import attn_cases as ac

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,new,length,group,heads", [(1, 1536, 31537, 4, 8), (64, 1, 8000, 16, 8)])
def test_a_full_gpu_costs_shares_not_the_call(n, new, length, group, heads):
    """Many rows take one share, few rows go in smaller launches."""
    from turbocider_b200 import cuda as tcc
    g = ac.gen(71)
    k, v, table, ks, vs = ac.paged([(new, length)], 64, heads, 128, torch.bfloat16, g)
    offsets = torch.arange(n + 1, dtype=torch.int32, device="cuda") * new
    lengths = torch.full((n,), length, dtype=torch.int32, device="cuda")
    q = ac.normal(g, (n * new, heads * group, 128), torch.bfloat16)
    args = tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table.expand(n, -1).contiguous(), new, length), q
    roomy, tight = tcc.Context(0), tcc.Context(0)
    need = tcc.attention_plan(heads * group, heads, 128, n, n * new, new, length, page_size=64).workspace_bytes
    assert need > 32 << 20
    out = torch.empty_like(q)
    want = tcc.paged_attention(roomy, *args)      # modules are loaded, and here is room
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = torch.empty(torch.cuda.mem_get_info()[0] - need + (8 << 20), dtype=torch.uint8, device="cuda")
    try:
        for _ in range(2):
            tcc.paged_attention(tight, *args, out=out)
            torch.cuda.synchronize()
        assert tight.status() == 0
    finally:
        del taken
        torch.cuda.empty_cache()
    # the same sums in another order: as far apart as two roundings of the probabilities and results
    scale = vs[0].abs().max()
    assert float((out.double() - want.double()).abs().max()) <= 4 * 2.0 ** -8 * float(scale)
    tcc.paged_attention(tight, *args, out=out)    # room again
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    roomy.close()
    tight.close()


@pytest.mark.parametrize("new,length", [(1536, 31537), (1, 9000)])
def test_a_capture_that_would_have_to_grow_it_is_refused(new, length):
    """With the reason (memory cannot be had in a capture), not by what the spoilt
    capture does to the launch."""
    from turbocider_b200 import cuda as tcc
    rt = pytest.importorskip("cuda.bindings.runtime")
    g = ac.gen(72)
    k, v, table, ks, vs = ac.paged([(new, length)], 64, 2, 128, torch.bfloat16, g)
    offsets, lengths = ac.offsets_of([(new, length)])
    q = ac.normal(g, (new, 8, 128), torch.bfloat16)
    args = tcc.PagedCache(k, v), tcc.PagedBatch(offsets, lengths, table, new, length), q
    out, fresh, side = torch.empty_like(q), tcc.Context(0), torch.cuda.Stream()
    torch.cuda.synchronize()
    err, = rt.cudaStreamBeginCapture(side.cuda_stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeGlobal)
    assert err == rt.cudaError_t.cudaSuccess
    try:
        with pytest.raises(tcc.BackendError, match="attention workspace allocation.*captur"):
            tcc.paged_attention(fresh, *args, out=out, stream=side)
    finally:
        rt.cudaStreamEndCapture(side.cuda_stream)
        rt.cudaGetLastError()
    tcc.paged_attention(fresh, *args, out=out, stream=side)   # outside it grows
    torch.cuda.synchronize()
    want, _, tol, _ = ac.attention_ref(q, [(new, length)], ks, vs, 128 ** -0.5, True, 0)
    ac.close(out, want, tol)
    assert fresh.status() == 0
    fresh.close()
