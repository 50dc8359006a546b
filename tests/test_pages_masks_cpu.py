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


def test_buffers_longer_than_the_batch_and_rows_of_no_sequence():
    """A step's buffers hold more sequences than it has; rows in front of the first sequence and behind the last stay as they are."""
    hq, hkv, d, page = 4, 2, 32, 16
    batch, seen = make_batch([3, 1, 2], [20, 40, 33], page, [([0, 1], 16)], "cpu", seed=1)
    k, v = (make_pages(seen.blocks, hkv, page, d, torch.int8, torch.float32, "cpu", seed=i) for i in range(2))
    q = torch.randn(9, hq * d, generator=torch.Generator().manual_seed(2))
    want = attend64(q[2:8], k, v, batch, seen, hq, hkv, d, 0.2)
    batch.cu_q = torch.cat([batch.cu_q + 2, torch.tensor([99, 0], dtype=torch.int32)])
    batch.seq_lens = torch.cat([batch.seq_lens, torch.tensor([7, 7], dtype=torch.int32)])
    batch.block_tables = torch.cat([batch.block_tables, batch.block_tables[:2]])
    out = ops.attention(q, torch.full_like(q, 7.0), batch, k, v, hq, hkv, d, 0.2, 0, 0, 0)
    assert (out[2:8].double() - want).abs().max() < 1e-5 and (out[:2] == 7).all() and (out[8:] == 7).all()
