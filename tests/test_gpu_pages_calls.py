"""8-bit cache pages and shared prefixes on the GPU: calls that are refused before anything is launched, and counts of what is."""
import pytest
import torch

from llmss_b200 import ops
from llmss_b200.ops._lib import KernelError
from llmss_b200.ops.pages import QuantPages
from pages_oracle import make_batch, make_pages

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
I8 = torch.int8


def test_write_refuses_columns_behind_a_views_rows():
    """The stride of a view may be longer than its rows: what follows the last one is not the caller's."""
    hq, hkv, d = 4, 2, 64
    whole = torch.zeros(3, 1024, dtype=BF, device="cuda")
    k, v = (QuantPages(torch.zeros(2, hkv, 16, d, dtype=I8, device="cuda"), torch.zeros(2, hkv, 16, device="cuda")) for _ in range(2))
    pos = torch.arange(3, dtype=torch.int32, device="cuda")
    ops.rope_kv_write(whole[:, 512:], pos, pos, k, v, hq, hkv, d, 0, ops.ROPE_NONE, 1e4, 0, 256, 384)
    for offsets in ((0, 256, 448), (320, 0, 128), (0, 464, 256)):
        with pytest.raises(KernelError, match="column ranges"):
            ops.rope_kv_write(whole[:, 512:], pos, pos, k, v, hq, hkv, d, 0, ops.ROPE_NONE, 1e4, *offsets)
    with pytest.raises(ValueError, match="QuantPages both"):
        ops.rope_kv_write(whole, pos, pos, k, v.data, hq, hkv, d, 0, ops.ROPE_NONE, 1e4, 0, 256, 384)


@pytest.mark.parametrize("kind", [None, I8])
@pytest.mark.parametrize("new", [[1, 1, 1], [30, 2, 41]])
def test_a_negative_length_shares_nothing(kind, new):
    """Lengths lie in device memory, where no call can look at them: a wrong one is a wrong result at most."""
    hq, hkv, d = 8, 2, 128
    batch, seen = make_batch(new, [90, 70, 64], 64, [([0, 1], 64)], "cuda", seed=1)
    k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i) for i in range(2))
    q = torch.randn(sum(new), hq * d, device="cuda").to(BF)
    outs = []
    for n in (0, -64, -5):
        batch.prefix.lens[0] = n
        outs.append(ops.attention(q, torch.empty_like(q), batch, k, v, hq, hkv, d, 0.1, 0, 0, 0))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2]) and torch.isfinite(outs[0].float()).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [30, 2, 41]])
def test_an_output_that_overlaps_the_queries_is_refused(new):
    """Lists of keys are worked on at once, so that one would write what another still reads.  The queries' own columns and columns beside them are fine."""
    hq, hkv, d = 8, 2, 64
    batch, seen = make_batch(new, [90, 70, 64], 64, [], "cuda", seed=1)
    k, v = (make_pages(seen.blocks, hkv, 64, d, I8, BF, "cuda", seed=i) for i in range(2))
    T, w = sum(new), hq * d
    x = torch.randn(T + 4, 3 * w, device="cuda").to(BF)
    call = lambda q, out, q_off, out_off: ops.attention(q, out, batch, k, v, hq, hkv, d, 0.1, q_off, 0, 0, out_off=out_off)
    want = call(x.clone()[:T], torch.empty(T, w, dtype=BF, device="cuda"), w, 0)
    for out_off in (w - 64, w + 8, 2 * w - 8):
        with pytest.raises(ValueError, match="overlaps"):
            call(x[:T], x[:T], w, out_off)
    with pytest.raises(ValueError, match="overlaps"):
        call(x[:T], x[1:T + 1], w, w)                                       # a row further
    with pytest.raises(ValueError, match="overlaps"):
        call(x[:T], x.view(-1)[w:].as_strided((T, w), (w, 1)), w, 0)        # rows of another stride
    for out_off in (0, 2 * w, w):
        y = x.clone()
        got = call(y[:T], y[:T], w, out_off)
        assert torch.equal(got[:, out_off:out_off + w], want)
    y = x.clone()
    assert torch.equal(call(y[:T, w:], y[:T, :w], 0, 0), want)               # views of one tensor, side by side
