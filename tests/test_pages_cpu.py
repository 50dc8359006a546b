"""8-bit cache pages and shared prefixes on the CPU: the plain forms against the definitions in 64 bits, and what the calls refuse."""
import math

import pytest
import torch

from llmss_b200 import ops
from llmss_b200.engine.batch import BatchInput, SharedPrefix
from llmss_b200.ops import reference as R
from llmss_b200.ops.pages import QMAX, QuantPages, quantise
from pages_oracle import attend64, make_batch, make_pages

KINDS = [torch.int8, torch.float8_e4m3fn]
HALF_STEP = {torch.int8: 0.5 / 127, torch.float8_e4m3fn: 2.0 ** -4}


@pytest.mark.parametrize("kind", KINDS)
def test_quantised_rows_are_off_by_half_a_step(kind):
    x = torch.randn(7, 5, 96, generator=torch.Generator().manual_seed(1)) * torch.logspace(-6, 4, 7)[:, None, None]
    codes, scale = quantise(x, kind)
    back = codes.double() * scale.double()[..., None]
    top = x.double().abs().amax(-1, keepdim=True)
    # half a step of the largest value (integers) or of each value, below 2^-6 of qmax of the smallest normal one (e4m3); the scale's own rounding is 2^-24
    step = top * HALF_STEP[kind] if kind == torch.int8 else torch.maximum(x.double().abs(), top * 2.0 ** -6 / 448) * HALF_STEP[kind]
    assert ((back - x.double()).abs() <= step * (1 + 2.0 ** -20)).all()
    assert torch.equal(codes.float().abs().amax(-1), torch.full(scale.shape, QMAX[kind]))


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_zeros_and_rows_that_are_not_finite(kind):
    x = torch.zeros(4, 16)
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    x[3] = 1e-44
    codes, scale = quantise(x, kind)
    assert scale[0] == 0 and torch.isnan(scale[1]) and torch.isnan(scale[2])
    assert not codes[:3].float().any() and codes[3].float().abs().max() <= QMAX[kind]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("style,rotary", [(ops.ROPE_NONE, 0), (ops.ROPE_GPTJ, 32), (ops.ROPE_NEOX, 64)])
def test_write_matches_the_definition(kind, style, rotary):
    g = torch.Generator().manual_seed(5)
    hq, hkv, d, page, T = 4, 2, 64, 16, 9
    qkv = torch.randn(T, (hq + 2 * hkv) * d, generator=g)
    before = qkv.clone()
    pos = torch.tensor([0, 1, 2, 5000, 31999, 7, 8, 100000, 3], dtype=torch.int32)
    slots = torch.tensor([17, 16, -1, 40, 47, 33, 5 * 16, 2, 10 ** 6], dtype=torch.int32)      # one skipped, one beyond the pages
    k, v = (QuantPages(torch.zeros(6, hkv, page, d).to(kind), torch.zeros(6, hkv, page)) for _ in range(2))
    ops.rope_kv_write(qkv, pos, slots, k, v, hq, hkv, d, rotary, style, 10000.0, 0, hq * d, (hq + hkv) * d)
    assert torch.equal(qkv[:, hq * d:], before[:, hq * d:])
    x = before.double().view(T, hq + 2 * hkv, d)
    if style != ops.ROPE_NONE:
        ang = pos.double()[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
        rot = x[:, :hq + hkv, :rotary].clone()
        a, b = (rot[..., 0::2], rot[..., 1::2]) if style == ops.ROPE_GPTJ else (rot[..., :rotary // 2], rot[..., rotary // 2:])
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        y = torch.stack((a * c - b * s, b * c + a * s), -1 if style == ops.ROPE_GPTJ else -2).flatten(-2)
        x[:, :hq + hkv, :rotary] = y
    assert (qkv[:, :hq * d].double() - x[:, :hq].reshape(T, -1)).abs().max() < 2e-6
    written = 0
    for t, slot in enumerate(slots.tolist()):
        if not 0 <= slot < 6 * page:
            continue
        written += 1
        for pages, rows in ((k, x[t, hq:hq + hkv]), (v, x[t, hq + hkv:])):
            top = rows.abs().amax(-1)
            assert torch.allclose(pages.scale[slot // page, :, slot % page].double(), top / QMAX[kind], rtol=1e-6)
            step = HALF_STEP[kind] * (top[:, None] if kind == torch.int8 else torch.maximum(rows.abs(), top[:, None] * 2.0 ** -6 / 448))
            assert ((pages.values()[slot // page, :, slot % page].double() - rows).abs() <= step + 1e-5 * top[:, None]).all()
    assert int((k.scale != 0).sum()) == written * hkv == int((v.scale != 0).sum())


CASES = [
    # query lengths, context before them, page, prefix groups (sequences, shared tokens)
    ([1], [0], 16, []),
    ([1, 1, 1], [5, 0, 40], 16, []),
    ([3, 1, 17], [0, 33, 15], 16, []),
    ([1, 1, 1, 1], [40, 33, 70, 32], 16, [([0, 1, 2, 3], 32)]),
    ([2, 5, 1, 1], [48, 50, 20, 3], 16, [([0, 1], 48), ([2], 16)]),
    ([4, 1], [37, 40], 16, [([0, 1], 37)]),                    # a prefix that ends inside a page
    ([1, 1], [64, 80], 16, [([0, 1], 0)]),
]


@pytest.mark.parametrize("kind", [None] + KINDS)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_matches_64_bits(kind, case):
    new, ctx, page, groups = CASES[case]
    hq, hkv, d = 4, 2, 32
    batch, seen = make_batch(new, ctx, page, groups, "cpu", seed=case)
    k, v = (make_pages(seen.blocks, hkv, page, d, kind, torch.float32, "cpu", seed=case * 2 + i) for i in range(2))
    q = torch.randn(sum(new), hq * d, generator=torch.Generator().manual_seed(9))
    out = torch.full((sum(new) + 2, hq * d), 7.0)
    q = torch.cat([q, torch.ones(2, hq * d)])
    ops.attention(q, out, batch, k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)
    want = attend64(q, k, v, batch, seen, hq, hkv, d, d ** -0.5)
    assert (out[:sum(new)].double() - want).abs().max() < 1e-5
    if kind is not None or batch.prefix is not None:
        assert (out[sum(new):] == 7.0).all()                   # rows behind the last sequence


def test_a_row_that_sees_nothing_is_zero():
    batch, seen = make_batch([1, 1], [20, 3], 16, [([0, 1], 16)], "cpu", seed=3)
    batch.seq_lens[1] = 0
    k, v = (make_pages(seen.blocks, 2, 16, 32, torch.int8, torch.float32, "cpu", seed=i) for i in range(2))
    out = torch.full((2, 128), 7.0)
    ops.attention(torch.randn(2, 128), out, batch, k, v, 4, 2, 32, 0.2, 0, 0, 0)
    assert not out[1].any() and out[0].any()


def test_pages_refuse_what_they_do_not_hold():
    with pytest.raises(TypeError, match="int8 or float8"):
        QuantPages(torch.zeros(1, 1, 16, 8), torch.zeros(1, 1, 16))
    with pytest.raises(ValueError, match="32-bit scales"):
        QuantPages(torch.zeros(1, 1, 16, 8, dtype=torch.int8), torch.zeros(1, 1, 8))
    with pytest.raises(ValueError, match="32-bit scales"):
        QuantPages(torch.zeros(1, 1, 16, 8, dtype=torch.int8), torch.zeros(1, 1, 16, dtype=torch.float16))
    with pytest.raises(ValueError, match="contiguous"):
        QuantPages(torch.zeros(1, 1, 16, 16, dtype=torch.int8)[..., :8], torch.zeros(1, 1, 16))


def test_prefix_groups_are_consecutive():
    assert SharedPrefix.build([], [], [0], [1], "cpu") is None
    assert SharedPrefix.build([[0, 1]], [[]], [0], [1, 1], "cpu") is None
    with pytest.raises(ValueError, match="consecutive"):
        SharedPrefix.build([[0, 2]], [[3]], [16], [1, 1, 1], "cpu")
    p = SharedPrefix.build([[1, 2], [3]], [[3, 4], [5]], [32, 16], [1, 2, 3, 4], "cpu")
    assert p.first.tolist() == [1, 3, 4] and p.max_rows == 5 and p.max_len == 32 and p.block_tables.tolist() == [[3, 4], [5, 0]]


def test_merge_of_two_parts_is_the_softmax_over_both():
    """The identity that the shared form rests on, at scores far apart."""
    s = torch.tensor([3.0, -700.0, 650.0, 650.5], dtype=torch.float64)
    v = torch.randn(4, 3, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    parts = [(x.max(), torch.exp(x - x.max()).sum(), torch.exp(x - x.max()) @ w) for x, w in ((s[:2], v[:2]), (s[2:], v[2:]))]
    m = max(p[0] for p in parts)
    w = [math.exp(p[0] - m) for p in parts]
    o = sum(a * p[2] for a, p in zip(w, parts)) / sum(a * p[1] for a, p in zip(w, parts))
    assert torch.allclose(o, torch.softmax(s, 0) @ v)


# ----------------------------------------------------------------------------- the engine
def _tiny(tmp_path, preset="gptj-tiny"):
    from llmss_b200.utils.checkpoint import write_random_checkpoint

    return str(write_random_checkpoint(tmp_path, preset, dtype=torch.float32, device="cpu", std=0.08))


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_engine_on_8_bit_pages(tmp_path, kind):
    from llmss_b200.engine.engine import Engine
    from llmss_b200.engine.runner import SamplingParams

    path = _tiny(tmp_path)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(1, 500, (n,), generator=g).tolist() for n in (5, 37, 20, 1)]
    kw = dict(device="cpu", max_seq_len=128, block_size=16)
    full, eng = Engine.from_pretrained(path, max_batch=4, **kw), Engine.from_pretrained(path, max_batch=4, kv_cache_dtype=kind, **kw)
    assert eng.runner.kv.data.element_size() == 1
    want, got = (e.feed([(i, p, range(len(p))) for i, p in enumerate(prompts)]) for e in (full, eng))
    # what quantising keys and values does to the logits of this model: a few steps of the largest of a row
    assert (got - want).abs().max() < (0.05 if kind == "int8" else 0.25) * want.abs().max() and not torch.equal(got, want)
    # a prompt cut into portions reads the same pages: the same logits, up to the order of 32-bit sums
    cut = Engine.from_pretrained(path, max_batch=4, kv_cache_dtype=kind, **kw)
    parts = [cut.feed([(1, prompts[1][a:b], range(b - a))]) for a, b in ((0, 16), (16, 17), (17, 37))]
    assert torch.allclose(torch.cat(parts), got[5:42], atol=1e-4)
    eng2, chunked = (Engine.from_pretrained(path, max_batch=2, kv_cache_dtype=kind, prefill_chunk=c, **kw) for c in (None, 7))
    sp = SamplingParams(max_new_tokens=8, is_greedy=True)
    assert eng2.generate(prompts, sp) == chunked.generate(prompts, sp)
    assert eng2.runner.alloc.num_free == eng2.runner.alloc.num_blocks - 1


def test_engine_refuses_what_has_no_such_pages(tmp_path):
    from llmss_b200.engine.engine import Engine

    path = _tiny(tmp_path / "a")
    with pytest.raises(ValueError, match="'fp8' or 'int8'"):
        Engine.from_pretrained(path, device="cpu", max_batch=2, max_seq_len=64, kv_cache_dtype="int4")
    with pytest.raises(ValueError, match="prefix_cache"):
        Engine.from_pretrained(path, device="cpu", max_batch=2, max_seq_len=64, shared_prefix=True)
    with pytest.raises(ValueError, match="sliding"):
        Engine.from_pretrained(path, device="cpu", max_batch=2, max_seq_len=64, shared_prefix=True, prefix_cache=True, sliding_window=True)
    native = _tiny(tmp_path / "b", "bedovik-tiny")
    with pytest.raises(ValueError, match="kind of cache"):
        Engine.from_pretrained(native, device="cpu", max_batch=2, max_seq_len=64, kv_cache_dtype="int8")


def test_quant_cache_copies_blocks():
    from llmss_b200.engine.kv_cache import QuantKVCache

    a, b = (QuantKVCache(2, 4, 16, 2, 8, "fp8", "cpu") for _ in range(2))
    a.data.view(torch.int8).random_(0, 100)
    a.scale.uniform_()
    b.copy_blocks_from(a, 1, 2, 2)
    assert torch.equal(b.k(1).values()[2:4], a.k(1).values()[1:3]) and torch.equal(b.v(0).values()[2:4], a.v(0).values()[1:3])
    assert not b.scale[:, :, :2].any()
    assert QuantKVCache.bytes_per_block(2, 16, 2, 8) == 2 * 2 * 16 * 2 * 12


@pytest.mark.parametrize("kind", [None, "int8"])
def test_engine_reads_a_shared_prefix_once(tmp_path, monkeypatch, kind):
    """Two system prompts and a request of its own, decoded together: the tokens of an engine without sharing, and the groups that the step had."""
    from llmss_b200.engine import runner as R2
    from llmss_b200.engine.engine import Engine
    from llmss_b200.engine.runner import SamplingParams

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    path = _tiny(tmp_path)
    g = torch.Generator().manual_seed(4)
    draw = lambda n: torch.randint(1, 500, (n,), generator=g).tolist()
    a, b = draw(40), draw(20)
    prompts = [a + draw(5), b + draw(3), draw(9), a + draw(11), b + draw(8), a + draw(1)]
    sp = [SamplingParams(max_new_tokens=n, is_greedy=True) for n in (9, 12, 7, 4, 12, 10)]
    kw = dict(device="cpu", max_batch=6, max_seq_len=128, block_size=16, prefix_cache=True, kv_cache_dtype=kind)
    plain, eng = Engine.from_pretrained(path, **kw), Engine.from_pretrained(path, shared_prefix=True, **kw)
    seen = []
    bind = eng.runner._bind_prefix

    def watch(seqs):
        bind(seqs)
        seen.append(eng.runner.prefix_groups(seqs))

    eng.runner._bind_prefix = watch
    for e in (plain, eng):                      # a first wave registers the prefixes
        e.generate([a + [3], b + [4]], SamplingParams(max_new_tokens=2, is_greedy=True))
    assert eng.generate(prompts, sp) == plain.generate(prompts, sp)
    sizes = [sorted((n, len(c)) for _, n, c in s) for s in seen]
    assert [(2, 1), (3, 2)] in sizes            # b's one block for two, a's two blocks for three
    assert eng.runner._prefix is None or eng.runner._prefix[0] >= 1
    assert eng.runner.alloc.num_free == eng.runner.alloc.num_blocks - 1


def test_groups_and_the_rows_between_them(tmp_path, monkeypatch):
    from types import SimpleNamespace

    from llmss_b200.engine import runner as R2
    from llmss_b200.engine.engine import Engine

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    r = Engine.from_pretrained(_tiny(tmp_path), device="cpu", max_batch=40, max_seq_len=128, block_size=16, prefix_cache=True, shared_prefix=True).runner
    seq = lambda blocks, length: SimpleNamespace(blocks=blocks, length=length)
    seqs = [seq([9, 1], 20), seq([2, 3, 4], 40), seq([2, 3, 5], 40), seq([7], 16), seq([8, 6], 17), seq([8, 10], 17), seq([11], 3)]
    assert r.prefix_groups(seqs) == [(1, 2, [2, 3]), (4, 2, [8])]
    r._bind_prefix(seqs)
    p = r._step_prefix(8)
    assert p.num_groups == 4 and p.first[:5].tolist() == [1, 3, 4, 6, 6] and p.lens[:4].tolist() == [32, 0, 16, 0]
    assert p.block_tables[0, :2].tolist() == [2, 3] and p.block_tables[2, 0] == 8 and p.max_len == 32
    # a block that is not full yet is nobody else's
    assert r.prefix_groups([seq([2], 15), seq([2], 15)]) == []
    # more groups than a step takes: those that save most, still in order
    many = [seq([100 + i // 2, 200 + i], 20) for i in range(24)]
    assert [f for f, _, _ in r.prefix_groups(many)] == list(range(0, 16, 2))
    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 1 << 30)
    assert r.prefix_groups(seqs) == []
    r._bind_prefix(seqs)
    assert r._step_prefix(8) is None
