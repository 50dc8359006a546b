"""Attention over cache pages on the GPU within bounds that count each rounding: a result of zeros, or one without 16 of its keys, is outside of them."""
import pytest
import torch

from llmss_b200 import ops
from pages_bounds import expected
from pages_oracle import make_batch, make_pages

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
I8, E4 = torch.int8, torch.float8_e4m3fn

CASES = {
    # name: query lengths, context before them, page, prefix groups, heads
    "single_tokens": ([1] * 5, [63, 64, 2000, 17, 131], 64, [], (32, 8, 128)),
    "single_tokens_of_many_heads": ([1] * 4, [300, 900, 31, 64], 16, [], (48, 1, 128)),
    "wide_heads": ([1] * 6, [700, 64, 1040, 90, 333, 20], 64, [], (16, 16, 256)),
    "some_tokens": ([2, 1, 4], [200, 700, 61], 32, [], (4, 4, 128)),
    "portions": ([64, 130, 1, 7], [0, 100, 1300, 64], 64, [], (8, 2, 128)),
    "long_portions": ([200, 333], [500, 40], 64, [], (16, 2, 128)),
    "small_heads": ([150, 40], [0, 600], 16, [], (16, 16, 64)),
    "other_head_sizes": ([1, 30, 2], [200, 100, 0], 16, [], (6, 3, 96)),
    "step_behind_a_prefix": ([1] * 40, [1024 + 7 * i % 90 for i in range(40)], 64, [(list(range(40)), 1024)], (32, 8, 128)),
    "step_of_many_heads_behind_a_prefix": ([1] * 9, [640 + 5 * i for i in range(9)], 64, [(list(range(9)), 640)], (48, 1, 128)),
    "own_keys_longer_than_the_prefix": ([1] * 17, [256 + (700 + 13 * i) % 701 for i in range(17)], 64, [(list(range(17)), 256)], (32, 8, 128)),
    "two_prefixes": ([1] * 7, [130, 140, 129, 64, 65, 400, 20], 16, [([0, 1, 2], 128), ([3, 4], 64)], (8, 2, 128)),
    "questions_behind_a_prefix": ([33, 20, 9], [1000, 960, 970], 64, [([0, 1, 2], 960)], (16, 16, 64)),
    "prefix_that_ends_inside_a_page": ([3, 2], [100, 120], 32, [([0, 1], 100)], (4, 4, 128)),
}


@pytest.mark.parametrize("q_scale", [0.05, 1.0, 30.0])
@pytest.mark.parametrize("dtype,kind", [(BF, None), (HF, None), (BF, I8), (HF, I8), (BF, E4), (HF, E4)])
@pytest.mark.parametrize("case", sorted(CASES))
def test_results_within_their_roundings(case, dtype, kind, q_scale):
    new, ctx, page, groups, (hq, hkv, d) = CASES[case]
    if kind is None and not groups:
        pytest.skip("16-bit pages without a prefix are another kernel's")
    batch, seen = make_batch(new, ctx, page, groups, "cuda", seed=len(case))
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, dtype, "cuda", seed=7 + i) for i in range(2))
    g = torch.Generator(device="cuda").manual_seed(1)
    q = (torch.randn(sum(new), hq * d, generator=g, device="cuda") * q_scale).to(dtype)
    scale = d ** -0.5
    want, tol, less = expected(q, k, v, batch, seen, hq, hkv, d, scale)
    # what the bounds are worth
    assert (want.abs() > tol).double().mean() > 0.9
    assert ((less - want).abs() > tol).double().mean() > (0.1 if q_scale <= 1 else 0.01)      # (sharp: a few keys of each row alone count)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, scale, 0, 0, 0).double()
    off = (got - want).abs()
    assert (off <= tol).all(), f"off by {float(off.max()):.3g}; up to {float((off / tol).max()):.3g} times the bound, {int((off > tol).sum())} of {off.numel()}"


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [150, 40, 1]])
@pytest.mark.parametrize("page", [48, 80, 112, 144, 256, 5, 24])
def test_pages_of_any_size(page, new, kind):
    hq, hkv, d = 8, 2, 128
    ctx = [700, page, 2 * page + 7]
    batch, seen = make_batch(new, ctx, page, [([1, 2], page)] if kind is None or page % 3 else [], "cuda", seed=page)
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, BF, "cuda", seed=i) for i in range(2))
    q = torch.randn(sum(new), hq * d, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0).double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", [None, I8])
@pytest.mark.parametrize("tokens", [1, 20])
def test_more_sequences_than_a_block_keeps_lengths_of(kind, tokens):
    n, hq, hkv, d = 2500, 4, 2, 64
    new = [tokens] * 3 + [1] * (n - 3)
    groups = [(list(range(2 * i, 2 * i + 2)), 16) for i in range(n // 2)] if kind is None else []
    batch, seen = make_batch(new, [16 + i * 7 % 50 for i in range(n)], 16, groups, "cuda", seed=1)
    k, v = (make_pages(seen.blocks, hkv, 16, d, kind, BF, "cuda", seed=i) for i in range(2))
    q = torch.randn(sum(new), hq * d, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0).double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new", [[1], [7], [200]])
def test_a_context_of_300000_tokens(new, kind):
    """The bounds hold over the whole length: nothing is left out at its ends or between."""
    hq, hkv, d = 6, 1, 64
    groups = [([0], 64)] if kind is None else []
    batch, seen = make_batch(new, [300000], 64, groups, "cuda", seed=1)
    k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i) for i in range(2))
    q = torch.randn(sum(new), hq * d, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0).double()
    assert ((got - want).abs() <= tol).all()
    marked = torch.zeros(300000 + new[0])
    marked[[0, 63, 64, 4095, 150001, 262144, 299999]] = 1.0        # large values of single keys are seen with their weight
    for p in marked.nonzero().flatten().tolist():
        table = seen.fronts[0] if groups and p < 64 else seen.tables[0]
        if kind is None:
            v[table[p // 64], 0, p % 64] = 1000.0
        else:
            v.scale[table[p // 64], 0, p % 64] *= 1000.0
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0).double()
    assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("new", [[1, 1], [70, 3], [300, 40]])
@pytest.mark.parametrize("sizes", [(None, 80), (80, None), (-60, 60), (100, -60), (-75, -75), (118, 118), (0, 40)])
def test_pages_whose_values_differ_by_many_orders(sizes, new, kind):
    """All values of a sequence's first page against all of the others: 2^this, or zeros.  Keys weigh what their scores say, whatever their values are."""
    hq, hkv, d = 8, 2, 128
    batch, seen = make_batch(new, [700, 350], 64, [], "cuda", seed=2)
    k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i) for i in range(2))
    for table in seen.tables:
        for n, b in enumerate(table):
            size = sizes[0 if n == 0 else 1]
            v.scale[b] *= 0.0 if size is None else 2.0 ** size
            if size is None:
                v.data.view(torch.int8)[b] = 0
    q = torch.randn(sum(new), hq * d, generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    got = ops.attention(q, torch.full_like(q, float("nan")), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0).double()
    assert ((got - want).abs() <= tol).all()
