"""Attention over cache pages on the CPU: what lies at keys that a row does not see."""
import pytest
import torch

from llmss_b200 import ops
from pages_oracle import attend64, make_batch, make_pages


@pytest.mark.parametrize("kind", [None, torch.int8])
@pytest.mark.parametrize("filler", [float("nan"), float("inf")])
def test_rows_before_a_token_do_not_see_its_values(kind, filler):
    new, ctx, hq, hkv, d, page = [9, 4], [20, 16], 4, 2, 32, 16
    batch, seen = make_batch(new, ctx, page, [([0, 1], 16)], "cpu", seed=1)
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, torch.float32, "cpu", seed=i) for i in range(2))
    q = torch.randn(13, hq * d, generator=torch.Generator().manual_seed(2))
    want = attend64(q, k, v, batch, seen, hq, hkv, d, 0.2)
    at, tok, column = ctx[0] + 5, 5, 7
    if kind is None:
        v[seen.tables[0][at // page], 1, at % page, column] = filler
    else:
        v.scale[seen.tables[0][at // page], 1, at % page] = filler
    out = ops.attention(q, torch.zeros_like(q), batch, k, v, hq, hkv, d, 0.2, 0, 0, 0)
    sees = torch.zeros(13, hq, d, dtype=torch.bool)
    sees[tok:9, 2:, column if kind is None else slice(None)] = True
    sees = sees.view(13, -1)
    assert ((out.double() - want).abs()[~sees] < 1e-5).all() and not torch.isfinite(out[sees]).any()
