"""8-bit cache pages and shared prefixes on the GPU: the kernels against the definitions in 64 bits."""
import pytest
import torch

from llmss_b200 import ops
from llmss_b200.ops import reference as R
from llmss_b200.ops.pages import QMAX, QuantPages
from pages_oracle import attend64, make_batch, make_pages, values64

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
I8, E4 = torch.int8, torch.float8_e4m3fn
UNIT = {BF: 2.0 ** -8, HF: 2.0 ** -11}          # half a step, relative


# ----------------------------------------------------------------------------- write
def _write(T, hq, hkv, d, rotary, style, page, kind, dtype, seed, wide=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    W = (hq + 2 * hkv) * d
    qkv = (torch.randn(T, W + wide, generator=g, device="cuda") * torch.exp(torch.randn(T, 1, generator=g, device="cuda"))).to(dtype)
    pos = torch.randint(0, 100000, (T,), generator=g, device="cuda", dtype=torch.int32)
    blocks = -(-2 * T // page) + 1
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:T].int()
    k, v = (QuantPages(torch.zeros(blocks, hkv, page, d, device="cuda").to(kind), torch.zeros(blocks, hkv, page, device="cuda")) for _ in range(2))
    return qkv, pos, slots, k, v


def _turned(x, pos, rotary, style):
    """Rotation in 64 bits of x [T, heads, d]."""
    if style == ops.ROPE_NONE:
        return x
    ang = pos.double()[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=x.device) / rotary)
    return R.apply_rope(x, ang.cos(), ang.sin(), rotary, style)


WRITES = [
    # tokens, query heads, key heads, head size, rotated columns, style, page
    (1, 4, 4, 64, 0, ops.ROPE_NONE, 16), (64, 16, 16, 256, 64, ops.ROPE_GPTJ, 64), (37, 32, 8, 128, 128, ops.ROPE_NEOX, 64),
    (5, 48, 1, 128, 0, ops.ROPE_NONE, 16), (3, 5, 5, 80, 32, ops.ROPE_NEOX, 16), (9, 3, 1, 96, 96, ops.ROPE_GPTJ, 32),
    (1500, 8, 2, 64, 64, ops.ROPE_NEOX, 64), (2, 7, 7, 8, 0, ops.ROPE_NONE, 1), (21, 6, 3, 256, 256, ops.ROPE_NEOX, 48), (4, 2, 2, 16, 16, ops.ROPE_NEOX, 5),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("case", range(len(WRITES)))
def test_write(case, kind, dtype):
    T, hq, hkv, d, rotary, style, page = WRITES[case]
    qkv, pos, slots, k, v = _write(T, hq, hkv, d, rotary, style, page, kind, dtype, case, wide=16)
    if T > 4:
        slots[2], slots[4] = -1, k.shape[0] * page + 3          # not written: told so, or beyond the pages
    qkv[0, :hkv * d] *= 1e-30                                   # small numbers, down to scales that are not normal ones
    qkv[0, hkv * d:2 * hkv * d] *= 1e-38 if dtype == BF else 1e-5
    before = qkv.clone()
    # the columns in another order than q, k, v, as the fused block has them
    k_off, v_off, q_off = 0, hkv * d, 2 * hkv * d
    ops.rope_kv_write(qkv, pos, slots, k, v, hq, hkv, d, rotary, style, 10000.0, q_off, k_off, v_off)
    x = before.double()
    q = _turned(x[:, q_off:q_off + hq * d].reshape(T, hq, d), pos, rotary, style).reshape(T, -1)
    # q: half a step of the result, and 32-bit products of it before (3 roundings of values up to sqrt(2) times the pair's larger one)
    top = x.abs().amax(1, keepdim=True)
    assert ((qkv[:, q_off:q_off + hq * d].double() - q).abs() <= UNIT[dtype] * q.abs() + 8 * 2.0 ** -24 * top).all()
    assert torch.equal(qkv[:, :q_off], before[:, :q_off]) and torch.equal(qkv[:, q_off + hq * d:], before[:, q_off + hq * d:])
    ok = (slots >= 0) & (slots < k.shape[0] * page)
    at = slots[ok].long()
    for pages, rows in ((k, _turned(x[:, k_off:k_off + hkv * d].reshape(T, hkv, d), pos, rotary, style)), (v, x[:, v_off:v_off + hkv * d].reshape(T, hkv, d))):
        rows = rows[ok]
        scale = pages.scale[at // page, :, at % page].double()
        codes = pages.data.view(torch.int8)[at // page, :, at % page].view(kind).double()
        amax = rows.abs().amax(-1)
        # below 2^-126 a 32-bit number has a step of 2^-149
        assert ((scale - amax / QMAX[kind]).abs() <= 10 * 2.0 ** -24 * amax / QMAX[kind] + 2.0 ** -149).all()
        step = amax[..., None] / 254 if kind == I8 else torch.maximum(rows.abs(), amax[..., None] * 2.0 ** -6 / 448) * 2.0 ** -4
        assert ((codes * scale[..., None] - rows).abs() <= step + 16 * 2.0 ** -24 * amax[..., None] + QMAX[kind] * 2.0 ** -149).all()
        assert int((pages.scale != 0).sum()) == int((amax > 0).sum())     # nothing else was touched
    # values are not rotated: their codes are those of the plain form, bit for bit
    codes, scale = R.quantise(before[:, v_off:v_off + hkv * d].reshape(T, hkv, d)[ok], kind)
    assert torch.equal(v.data.view(torch.int8)[at // page, :, at % page], codes.view(torch.int8)) and torch.equal(v.scale[at // page, :, at % page], scale)


@pytest.mark.parametrize("kind", [I8, E4])
def test_write_of_rows_that_are_not_finite_or_all_zero(kind):
    qkv, pos, slots, k, v = _write(4, 2, 2, 64, 64, ops.ROPE_NEOX, 16, kind, BF, 3)
    qkv[0, 128:192] = 0
    qkv[1, 130] = float("inf")
    qkv[2, 256 + 70] = float("nan")
    ops.rope_kv_write(qkv, pos, slots, k, v, 2, 2, 64, 64, ops.ROPE_NEOX, 10000.0, 0, 128, 256)
    s = [int(x) for x in slots]
    ks, vs = (p.scale.permute(0, 2, 1).reshape(-1, 2)[s] for p in (k, v))
    assert ks[0, 0] == 0 and torch.isnan(ks[1, 0]) and torch.isfinite(ks[1, 1]) and torch.isnan(vs[2, 1]) and torch.isfinite(vs[2, 0])
    assert not values64(k).permute(0, 2, 1, 3).reshape(-1, 2, 64)[s[0], 0].any()


# ----------------------------------------------------------------------------- attention
def _bound(q, k, v, batch, seen, hq, hkv, d, scale, dtype):
    """How far an output may be off: its own rounding, and those of the operands on the way.  Keys, values and probabilities may each be rounded to the
    16-bit type (u): a score moves by at most u scale sum |q k|, probabilities by twice the largest of those, and what is summed is p |v|; scores and
    sums in 32 bits add 2^-18 of the same (a few hundred roundings of 2^-24)."""
    u = UNIT[dtype]
    ka, va = values64(k).abs(), values64(v).abs()
    mass = attend64_abs(q, k, v, batch, seen, hq, hkv, d, scale)
    big = _largest(q.double().abs(), ka, batch, seen, hq, hkv, d) * scale
    return mass * (2 * u + 2 * (u + 2.0 ** -18) * big + 2.0 ** -18)


def attend64_abs(q, k, v, batch, seen, hq, hkv, d, scale):
    """sum_k p_k |v_k|"""
    return attend64(q, values64(k), values64(v).abs(), batch, seen, hq, hkv, d, scale)


def _largest(qa, ka, batch, seen, hq, hkv, d):
    """max_k sum_i |q_i| |k_i| of every query row and head, spread over the head's columns"""
    out, at = [], 0
    for i, (a, L) in enumerate(zip(seen.new, batch.seq_lens.tolist())):
        j, n = seen.front_of.get(i, (0, 0))
        block = torch.tensor([(seen.fronts[j] if p < n else seen.tables[i])[p // seen.page] for p in range(L)], dtype=torch.long, device=ka.device)
        rows = qa[at:at + a].view(a, hkv, hq // hkv, d)
        z = torch.einsum("ahgd,lhd->ahgl", rows, ka[block, :, torch.arange(L, device=ka.device) % seen.page])
        z = z.amax(-1) if L else torch.zeros(rows.shape[:3], dtype=torch.float64, device=ka.device)
        out.append(z[..., None].expand(a, hkv, hq // hkv, d).reshape(a, hq * d))
        at += a
    return torch.cat(out)


def _check(new, ctx, page, groups, hq, hkv, d, kind, dtype, seed=0, max_kv=None, q_scale=1.0, alias=False):
    batch, seen = make_batch(new, ctx, page, groups, "cuda", seed=seed, max_kv=max_kv)
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, dtype, "cuda", seed=3 * seed + i) for i in range(2))
    T = sum(new)
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(T + 2, hq * d + 24, generator=g, device="cuda") * q_scale).to(dtype)
    scale = d ** -0.5
    want = attend64(q[:T, 8:8 + hq * d], k, v, batch, seen, hq, hkv, d, scale)
    tol = _bound(q[:T, 8:8 + hq * d], k, v, batch, seen, hq, hkv, d, scale, dtype) + UNIT[dtype] * want.abs()
    out = q if alias else torch.full((T + 2, hq * d + 16), 7.0, dtype=dtype, device="cuda")
    before = q.clone()
    if alias:
        ops.attention(q, q, batch, k, v, hq, hkv, d, scale, 8, 0, 0, out_off=8)
    else:
        ops.attention(q, out, batch, k, v, hq, hkv, d, scale, 8, 0, 0, out_off=8)
        assert torch.equal(q, before) and (out[T:] == 7).all() and (out[:, :8] == 7).all() and (out[:, 8 + hq * d:] == 7).all()
    got = out[:T, 8:8 + hq * d].double()
    assert torch.isfinite(got).all()
    off = (got - want).abs() - tol
    assert (off <= 0).all(), f"off by {(got - want).abs().max():.3g}, {float(off.max()):.3g} over the bound; {int((off > 0).sum())} of {off.numel()}"
    return batch, k, v, q, want


LAYOUTS = [(16, 16, 64), (4, 4, 128), (4, 4, 256), (8, 2, 128), (12, 2, 64), (10, 2, 256), (16, 2, 128), (24, 2, 128), (32, 2, 64), (48, 1, 128), (71, 1, 64), (130, 1, 128),
           (5, 5, 80), (6, 3, 96), (20, 1, 256)]
STEPS = [
    ([1], [0], []), ([1], [15], []), ([1, 1, 1, 1, 1], [63, 64, 200, 0, 131], []), ([1, 1], [1500, 3], []),
    ([1, 1, 1], [300, 290, 257], [([0, 1, 2], 256)]), ([1] * 7, [130, 140, 129, 64, 65, 400, 2], [([0, 1, 2], 128), ([3, 4], 64)]),
]
PORTIONS = [
    ([2, 1, 3], [20, 0, 61], []), ([150], [0], []), ([64, 130, 1, 7], [0, 100, 300, 64], []), ([33, 20], [192, 210], [([0, 1], 192)]),
    ([5, 9, 1], [70, 64, 90], [([0, 1, 2], 64)]), ([3, 2], [100, 120], [([0, 1], 100)]),
]


@pytest.mark.parametrize("dtype,kind", [(BF, I8), (HF, E4)])
@pytest.mark.parametrize("case", range(len(STEPS)))
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_single_tokens(layout, case, dtype, kind):
    new, ctx, groups = STEPS[case]
    _check(new, ctx, (16, 32, 64)[(layout + case) % 3], groups, *LAYOUTS[layout], kind, dtype, seed=layout * 10 + case)


@pytest.mark.parametrize("dtype,kind", [(HF, I8), (BF, E4)])
@pytest.mark.parametrize("case", range(len(PORTIONS)))
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_portions(layout, case, dtype, kind):
    new, ctx, groups = PORTIONS[case]
    _check(new, ctx, (64, 16, 32)[(layout + case) % 3], groups, *LAYOUTS[layout], kind, dtype, seed=layout * 10 + case)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("layout", range(len(LAYOUTS)))
def test_shared_prefix_of_16_bit_pages(layout, dtype):
    for case, (new, ctx, groups) in enumerate([c for c in STEPS + PORTIONS if c[2]]):
        _check(new, ctx, (64, 32, 16)[(layout + case) % 3], groups, *LAYOUTS[layout], None, dtype, seed=layout * 10 + case)


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 16, 256), (48, 1, 128)])
def test_many_sequences_behind_a_long_prefix(kind, hq, hkv, d):
    new = [1] * 40
    _check(new, [1024 + 7 * i % 90 for i in range(40)], 64, [(list(range(40)), 1024)], hq, hkv, d, kind, BF, seed=1)


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (48, 1, 128)])
def test_one_long_sequence_among_short_ones(kind, hq, hkv, d):
    """Its list is cut into far more parts than a warp has lanes; the others are a part each."""
    for groups in ([], [(list(range(40)), 64)]):
        if kind is None and not groups:
            continue                     # 16-bit pages without a prefix are another kernel's
        _check([1] * 40, [20000] + [64 + i for i in range(39)], 64, groups, hq, hkv, d, kind, BF, seed=6)


@pytest.mark.parametrize("kind", [None, I8])
@pytest.mark.parametrize("seqs,own,prefix", [(3, 4000, 64), (60, 3, 6400), (100, 40, 640), (17, 700, 2560)])
def test_prefix_and_own_keys_of_very_different_size(kind, seqs, own, prefix):
    """Whatever share of the machine either part gets."""
    _check([1] * seqs, [prefix + (own + 13 * i) % (own + 1) for i in range(seqs)], 64, [(list(range(seqs)), prefix)], 32, 8, 128, kind, BF, seed=7)


@pytest.mark.parametrize("kind", [I8, E4])
def test_output_over_the_queries_columns(kind):
    """The fused block writes the context over its queries."""
    for new, ctx, groups in (([1] * 5, [40, 700, 64, 3, 129], []), ([40, 3], [10, 200], []), ([1, 1], [130, 140], [([0, 1], 128)])):
        _check(new, ctx, 64, groups, 8, 2, 128, kind, BF, seed=4, alias=True)


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new,ctx,groups", [([1, 1, 1], [128, 64, 90], [([0, 1, 2], 64)]), ([9, 30], [128, 64], [([0, 1], 64)]), ([1, 1], [5, 130], [([1], 128)])])
def test_lengths_far_below_their_bounds(kind, new, ctx, groups):
    """A captured step knows the largest lengths alone."""
    _check(new, ctx, 64, groups, 8, 2, 128, kind, BF, seed=2, max_kv=16384)


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (48, 1, 128), (4, 4, 256), (5, 5, 80)])
def test_rows_without_a_key_are_zero(kind, hq, hkv, d):
    for groups in ([], [([0, 1, 2], 64)]):
        batch, seen = make_batch([1, 1, 1], [100, 80, 70], 16, groups, "cuda", seed=5)
        batch.seq_lens[1] = 0
        k, v = (make_pages(seen.blocks, hkv, 16, d, kind, BF, "cuda", seed=i) for i in range(2))
        out = torch.full((3, hq * d), float("nan"), dtype=BF, device="cuda")
        ops.attention(torch.randn(3, hq * d, device="cuda").to(BF), out, batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)
        assert not out[1].any() and torch.isfinite(out.float()).all() and out[0].any() and out[2].any()


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (48, 1, 128), (4, 4, 256), (5, 5, 80), (16, 16, 64)])
@pytest.mark.parametrize("new,ctx", [([1, 1], [83, 130]), ([21, 3], [83, 130])])
def test_what_lies_behind_the_last_key_is_not_seen(kind, hq, hkv, d, new, ctx):
    """NaN and infinities in the unused places of the last page, and in pages of nobody."""
    groups = [([0, 1], 64)] if kind is None else []
    batch, seen = make_batch(new, ctx, 32, groups, "cuda", seed=6)
    k, v = (make_pages(seen.blocks, hkv, 32, d, kind, BF, "cuda", seed=i) for i in range(2))
    q = torch.randn(sum(new), hq * d, device="cuda").to(BF)
    outs = [torch.empty_like(q) for _ in range(2)]
    ops.attention(q, outs[0], batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)
    used = torch.zeros(seen.blocks, 32, dtype=torch.bool)
    for i, L in enumerate(batch.seq_lens.tolist()):
        for p in range(L):
            used[seen.tables[i][p // 32], p % 32] = True
    for j, f in enumerate(seen.fronts):
        used[f] = True
    bad = (~used).nonzero()
    for n, (pages, filler) in enumerate(((k, float("nan")), (v, float("inf")))):
        if kind is None:
            pages[bad[:, 0], :, bad[:, 1]] = filler
        else:
            pages.scale[bad[:, 0], :, bad[:, 1]] = filler
            pages.data.view(torch.int8)[bad[:, 0], :, bad[:, 1]] = 127        # NaN in e4m3
    ops.attention(q, outs[1], batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)
    assert torch.equal(outs[0], outs[1]) and torch.isfinite(outs[1].float()).all()


@pytest.mark.parametrize("kind", [I8, E4])
@pytest.mark.parametrize("new", [[1, 1], [40, 3]])
@pytest.mark.parametrize("which", [0, 1, 2, 3, 66, 89])
def test_a_key_that_is_not_finite_reaches_its_own_sequence_alone(which, kind, new):
    batch, seen = make_batch(new, [90, 200], 64, [], "cuda", seed=7)
    k, v = (make_pages(seen.blocks, 2, 64, 128, kind, BF, "cuda", seed=i) for i in range(2))
    k.scale[seen.tables[0][which // 64], 1, which % 64] = float("nan")
    out = torch.empty(sum(new), 1024, dtype=BF, device="cuda")
    ops.attention(torch.randn(sum(new), 1024, device="cuda").to(BF), out, batch, k, v, 8, 2, 128, 0.1, 0, 0, 0)
    o = out.float().view(-1, 2, 512)
    assert torch.isnan(o[:new[0], 1]).all() and torch.isfinite(o[:new[0], 0]).all() and torch.isfinite(o[new[0]:]).all()


@pytest.mark.parametrize("kind", [None, I8, E4])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 64, 1]])
def test_sharp_and_flat_softmax(kind, new):
    """Scores hundreds apart, and keys whose scales and values differ by many orders."""
    groups = [([0, 1, 2], 128)]
    for q_scale in (1e-3, 30.0):
        _check(new, [300, 129, 260], 64, groups, 8, 2, 128, kind, BF, seed=8, q_scale=q_scale)


@pytest.mark.parametrize("new", [[1, 1], [70, 3]])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("kind", [I8, E4])
def test_values_of_very_different_size(kind, dtype, new):
    batch, seen = make_batch(new, [200, 150], 64, [], "cuda", seed=9)
    g = torch.Generator().manual_seed(1)
    k = make_pages(seen.blocks, 2, 64, 128, kind, dtype, "cuda", seed=1)
    v = make_pages(seen.blocks, 2, 64, 128, kind, dtype, "cuda", seed=2)
    v.scale *= torch.exp2(torch.randint(-12, 8, v.scale.shape, generator=g).float()).cuda()
    q = torch.randn(sum(new), 1024, generator=g).to(dtype).cuda()
    out = torch.empty_like(q)
    ops.attention(q, out, batch, k, v, 8, 2, 128, 0.1, 0, 0, 0)
    want = attend64(q, k, v, batch, seen, 8, 2, 128, 0.1)
    tol = _bound(q, k, v, batch, seen, 8, 2, 128, 0.1, dtype) + UNIT[dtype] * want.abs()
    # f16 has a step of 2^-24 below 2^-14: half of it, 2^-25 absolute, where the relative bounds above count less.  Operands of 8-bit pages are f16:
    # values stand relative to a power of two below twice the largest scale of their 64 keys, s, so they are off by 2^-24 s each, and their weights add up to
    # 1; a probability stands times 2^7 relative to a reference not above the row's maximum, and times the ratio of its keys' power of two to the largest
    # one: off by 2^-32 (largest / own), on a value of at most qmax own, so 2^-31 qmax s for every key.  A result in f16 is off by 2^-25
    at = 0
    for i, (a, L) in enumerate(zip(new, batch.seq_lens.tolist())):
        block = torch.tensor([seen.tables[i][p // 64] for p in range(L)], device="cuda")
        top = v.scale.double()[block, :, torch.arange(L, device="cuda") % 64].amax(0)                               # [key heads]
        tol[at:at + a] += (top * (2.0 ** -24 + L * QMAX[kind] * 2.0 ** -31))[:, None].expand(2, 512).reshape(1, -1)
        at += a
    if dtype == HF:
        tol += 2.0 ** -25
    assert ((out.double() - want).abs() <= tol).all()


def test_pages_beyond_32_bit_offsets():
    hkv, page, d = 4, 64, 128
    blocks = (1 << 31) // (hkv * page * d) + 40
    k, v = (QuantPages(torch.zeros(blocks, hkv, page, d, dtype=I8, device="cuda"), torch.zeros(blocks, hkv, page, device="cuda")) for _ in range(2))
    for new, groups in (([1, 1], []), ([30, 2], []), ([1, 1], [([0, 1], 64)])):
        batch, seen = make_batch(new, [100, 150], page, groups, "cuda", seed=10)
        small = [make_pages(seen.blocks, hkv, page, d, I8, BF, "cuda", seed=i) for i in range(2)]
        shift = blocks - seen.blocks
        for big, s in zip((k, v), small):
            big.data[shift:], big.scale[shift:] = s.data, s.scale
        q = torch.randn(sum(new), 8 * d, device="cuda").to(BF)
        outs = [torch.empty_like(q) for _ in range(2)]
        ops.attention(q, outs[0], batch, *small, 8, hkv, d, 0.1, 0, 0, 0)
        batch.block_tables += shift
        if batch.prefix is not None:
            batch.prefix.block_tables += shift
        ops.attention(q, outs[1], batch, k, v, 8, hkv, d, 0.1, 0, 0, 0)
        assert torch.equal(outs[0], outs[1])
    # and written there
    qkv = torch.randn(2, 16 * d, device="cuda").to(BF)
    slots = torch.tensor([blocks * page - 1, blocks * page - 70], dtype=torch.int32, device="cuda")
    ops.rope_kv_write(qkv, slots, slots, k, v, 8, hkv, d, 0, ops.ROPE_NONE, 1e4, 0, 8 * d, 12 * d)
    codes, scale = R.quantise(qkv[:, 12 * d:].reshape(2, hkv, d), I8)
    assert torch.equal(v.data[-1, :, page - 1], codes[0]) and torch.equal(v.scale[-2, :, page - 6], scale[1])


@pytest.mark.parametrize("groups", [[], [([0, 1, 2, 3], 192)]])
@pytest.mark.parametrize("kind", [I8, None])
def test_replayed_steps_follow_their_inputs(kind, groups):
    """Two captured steps in flight on two streams, lengths changed between replays: the results of eager calls."""
    if kind is None and not groups:
        pytest.skip("16-bit pages without a prefix are another kernel's")
    hq, hkv, d = 8, 2, 128
    runs = []
    for n in range(2):
        batch, seen = make_batch([1] * 4, [500 + 40 * n, 300, 200, 260], 64, groups, "cuda", seed=11 + n, max_kv=1024)
        k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=i + n) for i in range(2))
        q = torch.randn(4, hq * d, device="cuda").to(BF)
        out = torch.empty_like(q)
        ops.attention(q, out, batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            ops.attention(q, out, batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)
        runs.append((g, batch, k, v, q, out, torch.cuda.Stream()))
    for lens in ([501, 301, 201, 261], [193, 250, 194, 200], [520, 0, 201, 193]):
        want = []
        for g, batch, k, v, q, out, stream in runs:
            batch.seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            want.append(ops.attention(q, torch.empty_like(q), batch, k, v, hq, hkv, d, 0.1, 0, 0, 0))
        torch.cuda.synchronize()
        for _ in range(20):
            for g, *_, stream in runs:
                with torch.cuda.stream(stream):
                    g.replay()
        torch.cuda.synchronize()
        for (_, _, _, _, _, out, _), w in zip(runs, want):
            assert torch.equal(out, w)


@pytest.mark.parametrize("kind,groups", [(I8, []), (E4, [(list(range(9)), 192)]), (None, [(list(range(9)), 192)])])
@pytest.mark.parametrize("new", [1, 30, 200])
def test_calls_on_two_streams_at_once(kind, groups, new):
    """Each has a scratch of its own, and a call's result has the same bits every time."""
    hq, hkv, d = 16, 2, 128
    calls = []
    for seed in (11, 12):
        batch, seen = make_batch([new] * 9, [200 + 40 * i for i in range(9)], 64, groups, "cuda", seed=seed)
        k, v = (make_pages(seen.blocks, hkv, 64, d, kind, BF, "cuda", seed=2 * seed + i) for i in range(2))
        q = torch.randn(9 * new, hq * d, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(BF)
        calls.append((q, batch, k, v))
    run = lambda c, out: ops.attention(c[0], out, c[1], c[2], c[3], hq, hkv, d, d ** -0.5, 0, 0, 0)
    want = [run(c, torch.empty_like(c[0])).clone() for c in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    got = [[torch.empty_like(c[0]) for _ in range(12)] for c in calls]
    torch.cuda.synchronize()
    for n in range(12):
        for c, s, outs in zip(calls, streams, got):
            with torch.cuda.stream(s):
                run(c, outs[n])
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(o, w) for o in outs)


def test_more_rows_than_cached_tokens():
    """Rows before a sequence's first position see nothing."""
    for new, hq, hkv in (([5, 1, 3], 4, 4), ([40, 1, 9], 16, 2)):
        batch, seen = make_batch(new, [20, 30, 64], 16, [], "cuda", seed=3)
        batch.seq_lens[0] = 3
        for kind in (I8, E4):
            k, v = (make_pages(seen.blocks, hkv, 16, 128, kind, BF, "cuda", seed=i) for i in range(2))
            out = torch.full((sum(new), hq * 128), float("nan"), dtype=BF, device="cuda")
            ops.attention(torch.randn(sum(new), hq * 128, device="cuda").to(BF), out, batch, k, v, hq, hkv, 128, 0.1, 0, 0, 0)
            assert not out[:new[0] - 3].any() and torch.isfinite(out.float()).all() and out[new[0] - 3:].any(-1).all()


def test_write_and_attention_together():
    """A layer's step as a model runs it: a prompt in portions and then single tokens behind a shared prefix, cache in 8 bits."""
    hq, hkv, d, page = 8, 2, 128, 64
    W = (hq + 2 * hkv) * d
    g = torch.Generator(device="cuda").manual_seed(12)
    prompt = torch.randn(256, W, generator=g, device="cuda").to(BF)
    for kind in (I8, E4):
        k, v = (QuantPages(torch.zeros(20, hkv, page, d, device="cuda").to(kind), torch.zeros(20, hkv, page, device="cuda")) for _ in range(2))
        tables = [[3, 1, 7, 2, 5], [3, 1, 7, 2, 9], [3, 1, 7, 2, 4]]
        outs = []
        for lo, hi in ((0, 256), (0, 100), (100, 256)):         # at once, and in two portions: the same cache, the same result
            from llmss_b200.engine.batch import BatchInput

            batch = BatchInput.build([[0] * (hi - lo)], [lo], tables[:1], page, "cuda")
            qkv = prompt[lo:hi].clone()
            ops.rope_kv_write(qkv, batch.positions, batch.slot_mapping, k, v, hq, hkv, d, d, ops.ROPE_NEOX, 1e4, 0, hq * d, (hq + hkv) * d)
            out = torch.zeros(hi - lo, hq * d, dtype=BF, device="cuda")
            outs.append(ops.attention(qkv, out, batch, k, v, hq, hkv, d, d ** -0.5, 0, hq * d, (hq + hkv) * d))
        u = UNIT[BF]
        assert ((torch.cat(outs[1:]) - outs[0]).abs().float() <= 4 * u * outs[0].abs().float() + 8 * u * values64(v).abs().max().float()).all()
        for step in range(3):
            batch, seen = make_batch([1] * 3, [256 + step] * 3, page, [([0, 1, 2], 256)], "cuda")
            batch.block_tables = torch.tensor(tables, dtype=torch.int32, device="cuda")
            batch.prefix.block_tables = batch.block_tables[:1, :4].contiguous()
            batch.slot_mapping = batch.block_tables[:, 4] * page + step
            seen.tables, seen.fronts = tables, [tables[0][:4]]
            qkv = torch.randn(3, W, generator=g, device="cuda").to(BF)
            ops.rope_kv_write(qkv, batch.positions, batch.slot_mapping, k, v, hq, hkv, d, d, ops.ROPE_NEOX, 1e4, 0, hq * d, (hq + hkv) * d)
            out = ops.attention(qkv, torch.zeros(3, hq * d, dtype=BF, device="cuda"), batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
            want = attend64(qkv[:, :hq * d], k, v, batch, seen, hq, hkv, d, d ** -0.5)
            tol = _bound(qkv[:, :hq * d], k, v, batch, seen, hq, hkv, d, d ** -0.5, BF) + u * want.abs()
            assert ((out.double() - want).abs() <= tol).all()


# ----------------------------------------------------------------------------- refusals
def test_calls_that_are_refused():
    from llmss_b200.ops._lib import KernelError

    batch, seen = make_batch([1, 1], [20, 30], 16, [], "cuda")
    k, v = (make_pages(seen.blocks, 2, 16, 64, I8, BF, "cuda", seed=i) for i in range(2))
    q = torch.zeros(2, 256, dtype=BF, device="cuda")

    def call(q=q, out=None, batch=batch, k=k, v=v, hq=4, hkv=2, d=64):
        return ops.attention(q, torch.empty_like(q) if out is None else out, batch, k, v, hq, hkv, d, 0.1, 0, 0, 0)

    call()
    with pytest.raises(ValueError, match="pages"):
        call(hkv=4)
    with pytest.raises(ValueError, match="pages"):
        call(v=v.data)
    with pytest.raises(ValueError, match="pages"):
        call(v=make_pages(seen.blocks, 2, 16, 64, E4, BF, "cuda"))
    with pytest.raises(TypeError, match="queries"):
        call(q=q.float())
    with pytest.raises(TypeError, match="queries"):
        call(out=torch.empty(2, 256, dtype=HF, device="cuda"))
    with pytest.raises(ValueError, match="block_tables"):
        batch2, _ = make_batch([1, 1], [20, 30], 16, [], "cuda")
        batch2.block_tables = batch2.block_tables.long()
        call(batch=batch2)
    with pytest.raises(ValueError, match="seq_lens"):
        batch2, _ = make_batch([1, 1], [20, 30], 16, [], "cuda")
        batch2.seq_lens = batch2.seq_lens[:1]
        call(batch=batch2)
    with pytest.raises(KernelError, match="grouping"):
        call(hq=3, q=torch.zeros(2, 256, dtype=BF, device="cuda"))
    big = QuantPages(torch.zeros(2, 2, 16, 264, dtype=I8, device="cuda"), torch.zeros(2, 2, 16, device="cuda"))
    with pytest.raises(KernelError, match="head_dim"):
        call(q=torch.zeros(2, 4 * 264, dtype=BF, device="cuda"), k=big, v=big, d=264)
    pos = torch.zeros(2, dtype=torch.int32, device="cuda")
    qkv = torch.zeros(2, 8 * 64, dtype=BF, device="cuda")
    args = (4, 2, 64, 64, ops.ROPE_NEOX, 1e4, 0, 256, 384)
    ops.rope_kv_write(qkv, pos, pos - 1, k, v, *args)
    with pytest.raises(ValueError, match="positions"):
        ops.rope_kv_write(qkv, pos.long(), pos, k, v, *args)
    with pytest.raises(TypeError, match="float16 or bfloat16"):
        ops.rope_kv_write(qkv.float(), pos, pos, k, v, *args)
    with pytest.raises(KernelError, match="rotary_dim"):
        ops.rope_kv_write(qkv, pos, pos - 1, k, v, 4, 2, 64, 24, ops.ROPE_NEOX, 1e4, 0, 256, 384)
    with pytest.raises(KernelError, match="column ranges"):
        ops.rope_kv_write(qkv, pos, pos - 1, k, v, 4, 2, 64, 64, ops.ROPE_NEOX, 1e4, 0, 256, 392)


# ----------------------------------------------------------------------------- the engine
@pytest.mark.parametrize("family", ["gptj", "llama", "gpt_bigcode", "opt"])
@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_engine_on_8_bit_pages(tmp_path, family, kind):
    """Logits of prompts and of steps over what they left, on the kernels and on the plain forms with the same pages' kind."""
    from llmss_b200.engine.engine import Engine
    from llmss_b200.engine.runner import SamplingParams
    from tiny import make_tiny

    make_tiny(family, tmp_path, hidden=256)
    path = str(tmp_path)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(1, 128, (n,), generator=g).tolist() for n in (5, 44, 33, 1)]
    kw = dict(max_batch=4, max_seq_len=64, kv_cache_dtype=kind)
    gpu, cpu = Engine.from_pretrained(path, dtype=HF, device="cuda", **kw), Engine.from_pretrained(path, device="cpu", **kw)
    for step in range(3):
        toks = prompts if step == 0 else [[7 + step], [9], [11 + step], [2]]
        a, b = (e.feed([(i, t, [len(t) - 1]) for i, t in enumerate(toks)]) for e in (gpu, cpu))
        # activations in f16 against 32 bits: codes near a half step may fall to either side, a step of 1 / 127 or 1 / 16 of a value among dozens
        assert (a.float().cpu() - b).abs().max() < (0.03 if kind == "int8" else 0.06) * b.abs().max()
    sp = SamplingParams(max_new_tokens=10, is_greedy=True)
    graph, eager = (Engine.from_pretrained(path, dtype=HF, device="cuda", use_cuda_graph=u, **kw) for u in (True, False))
    assert graph.generate(prompts, sp) == eager.generate(prompts, sp) and graph.runner.stats["graph_replays"] > 0


@pytest.mark.parametrize("kind", [None, "int8"])
def test_engine_reads_a_shared_prefix_once(tmp_path, monkeypatch, kind):
    from llmss_b200.engine import runner as R2
    from llmss_b200.engine.batch import BatchInput
    from llmss_b200.engine.engine import Engine
    from llmss_b200.engine.runner import SamplingParams
    from llmss_b200.utils.checkpoint import write_random_checkpoint

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    path = str(write_random_checkpoint(tmp_path, "gptj-tiny", dtype=torch.float32, device="cpu", std=0.08))
    g = torch.Generator().manual_seed(4)
    draw = lambda n: torch.randint(1, 400, (n,), generator=g).tolist()
    a, b = draw(70), draw(40)
    prompts = [a + draw(5), b + draw(3), draw(9), a + draw(11), b + draw(8), a + draw(1)]
    eng = Engine.from_pretrained(path, dtype=HF, device="cuda", max_batch=8, max_seq_len=128, block_size=16, prefix_cache=True, shared_prefix=True,
                                 kv_cache_dtype=kind)
    eng.generate([a + [3], b + [4]], SamplingParams(max_new_tokens=2, is_greedy=True))
    for p in prompts:
        eng.add_request(p, SamplingParams(max_new_tokens=20, is_greedy=True))
    for _ in range(4):
        eng.step()
    r = eng.runner
    assert r._prefix is not None and r.stats["graph_replays"] >= 3
    # the step's logits with and without the groups: the same numbers, up to roundings of 16-bit activations
    r._fill_step_inputs()
    r.d_in.copy_(r.h_in)
    tok, pos, slot, slen, bt, _ = r._dev_views(8)
    logits = []
    for prefix in (None, r._step_prefix(8)):
        batch = BatchInput(tokens=tok, positions=pos, slot_mapping=slot, block_tables=bt, seq_lens=slen, cu_q=r.d_cu[:9], last_idx=r.d_last_idx[:8], num_seqs=8,
                           max_q=1, max_kv=r.max_seq_len, is_decode=True, is_fresh_prefill=False, prefix=prefix)
        logits.append(r.core.forward(batch, r.kv, last_only=False)[:6].float())
    assert (logits[0] - logits[1]).abs().max() < 0.01 * logits[0].abs().max()
    while eng.has_work():
        eng.step()
    assert r.alloc.num_free == r.alloc.num_blocks - 1


def test_with_early_launches():
    """LLMSS_PDL=1 lets every kernel start before the one in front of it has ended; the variable is read once per process."""
    import os
    import subprocess
    import sys

    which = "write_and_attention_together or replayed_steps or two_streams or very_different_size"
    r = subprocess.run([sys.executable, "-m", "pytest", __file__, "-x", "-q", "-m", "gpu", "-k", which, "-p", "no:cacheprovider"],
                       env={**os.environ, "LLMSS_PDL": "1"}, capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout[-2000:]
