"""Attention over cache pages on the GPU: rows that see nothing, and what lies at keys that a row does not see."""
import pytest
import torch

from llmss_b200 import ops
from llmss_b200.engine.batch import SharedPrefix
from llmss_b200.ops.pages import QuantPages
from pages_bounds import expected
from pages_oracle import make_batch, make_pages

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
I8, E4 = torch.int8, torch.float8_e4m3fn
INF, NAN = float("inf"), float("nan")


def nothing_shared(sequences):
    """A prefix of no tokens: pages of 16 bits go to these kernels too, without groups."""
    i32 = dict(dtype=torch.int32, device="cuda")
    return SharedPrefix(block_tables=torch.zeros(1, 1, **i32), lens=torch.zeros(1, **i32), first=torch.tensor([0, sequences], **i32), num_groups=1, max_len=0,
                        max_rows=0)


def queries(rows, width, dtype, seed=2):
    return torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


# ----------------------------------------------------------------------------- rows without a key
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 64), (16, 2, 128), (8, 2, 256), (4, 4, 128), (6, 3, 96)])
@pytest.mark.parametrize("new", [[40, 1, 9], [200, 3, 130], [3, 1, 2]])
def test_rows_in_front_of_a_sequence_are_zero(new, hq, hkv, d, kind, dtype):
    """One to many tiles of rows, written by the kernel itself or by the merge; values far below and far above 1."""
    batch, seen = make_batch(new, [20, 30, 64], 16, [], "cuda", seed=3)
    batch.seq_lens[0] = 2
    if kind is None:
        batch.prefix = nothing_shared(3)
    q = queries(sum(new), hq * d, dtype)
    for size in ((1.0,) if kind is None else (2.0 ** -12, 1.0, 2.0 ** 9, 2.0 ** 30)):
        if dtype == HF and size > 2.0 ** 9:
            continue                                            # results beyond f16
        k, v = (make_pages(seen.blocks, hkv, 16, d, kind, dtype, "cuda", seed=i) for i in range(2))
        if kind is not None:
            v.scale *= size
        out = ops.attention(q, torch.full_like(q, NAN), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
        assert not out[:new[0] - 2].any()
        want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new", [[30, 41], [2, 1], [170, 90]])
def test_rows_in_front_of_a_sequence_behind_a_prefix_are_zero(new, kind):
    """More rows than tokens, some of them shared: parts of several kernels are joined."""
    hq, hkv, d = 16, 2, 128
    batch, seen = make_batch(new, [64, 70], 64, [([0, 1], 64)], "cuda", seed=4)
    for length in (1, 20, 64, 65):
        if length > new[0]:
            continue
        batch.seq_lens[0] = length
        k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i) for i in range(2))
        q = queries(sum(new), hq * d, BF)
        out = ops.attention(q, torch.full_like(q, NAN), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
        assert not out[:new[0] - length].any()
        want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
        assert ((out.double() - want).abs() <= tol).all()


# ----------------------------------------------------------------------------- keys that a row does not see
# query lengths, context, page, groups, (sequence, one of its new tokens)
HIDDEN = {
    "few_rows": ([4, 1, 3], [70, 10, 64], 64, [], (0, 2)),
    "one_tile": ([40, 3], [70, 10], 16, [], (0, 33)),
    "many_tiles": ([300, 20], [100, 64], 64, [], (0, 170)),
    "first_row": ([200, 20], [0, 64], 64, [], (0, 1)),
    "many_portions": ([150, 150, 7], [900, 33, 5], 32, [], (1, 149)),
    "few_rows_behind_a_prefix": ([3, 1], [70, 80], 64, [([0, 1], 64)], (0, 1)),
    "portions_behind_a_prefix": ([70, 21], [70, 80], 64, [([0, 1], 64)], (0, 30)),
}


def _spoil(pages, table, page, pos, head, column, filler):
    """Token ``pos`` of one key head is ``filler`` at one column (16-bit pages), or its scale is."""
    b, o = table[pos // page], pos % page
    if isinstance(pages, QuantPages):
        pages.scale[b, head, o] = filler
    else:
        pages[b, head, o, column] = filler


@pytest.mark.parametrize("kind,dtype", [(None, BF), (None, HF), (I8, BF), (E4, HF)])
@pytest.mark.parametrize("filler", [NAN, INF])
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 128), (12, 2, 256), (6, 2, 96)])
@pytest.mark.parametrize("case", sorted(HIDDEN))
def test_rows_before_a_token_do_not_see_its_values(case, hq, hkv, d, filler, kind, dtype):
    new, ctx, page, groups, (seq, tok) = HIDDEN[case]
    batch, seen = make_batch(new, ctx, page, groups, "cuda", seed=5)
    if kind is None and not groups:
        batch.prefix = nothing_shared(len(new))
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, dtype, "cuda", seed=i) for i in range(2))
    q = queries(sum(new), hq * d, dtype)
    want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    column = d // 2 + 3
    for pages in (v, k):
        _spoil(pages, seen.tables[seq], page, ctx[seq] + tok, 1, column, filler)
        out = ops.attention(q, torch.full_like(q, 7.0), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
        over = q.clone()                                        # and over its own queries
        ops.attention(over, over, batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
        assert ((over == out) | (torch.isnan(over) & torch.isnan(out))).all()
        row = sum(new[:seq]) + tok                              # the first row that sees the token
        after = slice(row, sum(new[:seq + 1]))
        sees = torch.zeros(sum(new), hq, d, dtype=torch.bool, device="cuda")
        if pages is k or kind is not None:
            sees[after, hq // 2:] = True                        # a score, or every value of the token
        else:
            sees[after, hq // 2:, column] = True
        sees = sees.view(sum(new), -1)
        off = (out.double() - want).abs()
        assert (off <= tol)[~sees].all(), f"{int((~(off <= tol))[~sees].sum())} results that do not see it changed"
        got = out.float()[sees]
        if filler != filler:
            assert torch.isnan(got).all()
        elif pages is v:                                        # a code of 0 times infinity is NaN
            assert (got == INF).all() if kind is None else not torch.isfinite(got).any()
        if pages is v:
            _spoil(v, seen.tables[seq], page, ctx[seq] + tok, 1, column, 0.5)
            want, tol, _ = expected(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)


@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 128), (12, 2, 256)])
@pytest.mark.parametrize("case", sorted(HIDDEN))
def test_rows_before_a_token_do_not_see_its_largest_values(case, hq, hkv, d):
    """The largest numbers of the type at keys that most rows do not see: not one bit of those rows changes."""
    new, ctx, page, groups, (seq, tok) = HIDDEN[case]
    batch, seen = make_batch(new, ctx, page, groups, "cuda", seed=5)
    if not groups:
        batch.prefix = nothing_shared(len(new))
    k, v = (make_pages(seen.blocks, hkv, page, d, None, BF, "cuda", seed=i) for i in range(2))
    q = queries(sum(new), hq * d, BF)
    first = ops.attention(q, torch.full_like(q, 7.0), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
    for p in range(ctx[seq] + tok, ctx[seq] + new[seq]):
        v[seen.tables[seq][p // page], :, p % page] = 3e38
    out = ops.attention(q, torch.full_like(q, 7.0), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
    row = sum(new[:seq]) + tok
    assert torch.equal(out[:row], first[:row]) and torch.equal(out[sum(new[:seq + 1]):], first[sum(new[:seq + 1]):])


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("new,ctx,groups", [([1, 1, 1], [90, 64, 130], [([0, 1, 2], 64)]), ([40, 9, 1], [90, 64, 130], [([0, 1, 2], 64)]), ([60, 2, 1], [90, 30, 5], []),
                                            ([3, 2, 1], [90, 30, 5], [])])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 64)])
def test_keys_that_are_infinite(hq, hkv, d, new, ctx, groups, dtype):
    """A score of plus infinity makes its row NaN, one of minus infinity takes the key out; a row whose scores all are minus infinity is NaN."""
    batch, seen = make_batch(new, ctx, 64, groups, "cuda", seed=8)
    if not groups:
        batch.prefix = nothing_shared(len(new))
    k, v = (make_pages(seen.blocks, hkv, 64, d, None, dtype, "cuda", seed=i) for i in range(2))
    q = queries(sum(new), hq * d, dtype)
    a = new[0]
    for at in (0, 1, 2, 3, 5, 66, 89):                          # of the first sequence: every row of it sees these
        kk, table = k.clone(), seen.fronts[0] if groups and at < 64 else seen.tables[0]
        kk[table[at // 64], 1, at % 64, 5] = INF
        out = ops.attention(q, torch.empty_like(q), batch, kk, v, hq, hkv, d, d ** -0.5, 0, 0, 0).float().view(-1, hq, d)[:a, hq // 2:]
        up = (q.view(-1, hq, d)[:a, hq // 2:, 5] > 0)
        assert torch.isnan(out[up]).all() and torch.isfinite(out[~up]).all()
    kk = k.clone()
    for p in range(ctx[0] + a):
        kk[(seen.fronts[0] if groups and p < 64 else seen.tables[0])[p // 64], 1, p % 64, 5] = INF
    out = ops.attention(q, torch.empty_like(q), batch, kk, v, hq, hkv, d, d ** -0.5, 0, 0, 0).float().view(-1, hq, d)
    assert torch.isnan(out[:a, hq // 2:]).all() and torch.isfinite(out[:a, :hq // 2]).all()


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [40, 1, 30]])
def test_buffers_longer_than_the_batch_and_rows_of_no_sequence(new, kind):
    """As the plain form on the CPU has it."""
    hq, hkv, d = 8, 2, 128
    batch, seen = make_batch(new, [90, 70, 64], 64, [([0, 1], 64)], "cuda", seed=1)
    k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i) for i in range(2))
    T = sum(new)
    q = queries(T + 5, hq * d, BF)
    want, tol, _ = expected(q[2:2 + T], k, v, batch, seen, hq, hkv, d, d ** -0.5)
    i32 = dict(dtype=torch.int32, device="cuda")
    batch.cu_q = torch.cat([batch.cu_q + 2, torch.tensor([T + 4, 0], **i32)])
    batch.seq_lens = torch.cat([batch.seq_lens, torch.tensor([7, 7], **i32)])
    batch.block_tables = torch.cat([batch.block_tables, batch.block_tables[:2]])
    out = ops.attention(q, torch.full_like(q, 7.0), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
    assert ((out[2:2 + T].double() - want).abs() <= tol).all() and (out[:2] == 7).all() and (out[2 + T:] == 7).all()
