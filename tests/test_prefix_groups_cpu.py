"""Which neighbours of a decode batch read a common front once."""
import random
from types import SimpleNamespace

import pytest

from llmss_b200.engine import runner as R2
from llmss_b200.engine.runner import ModelRunner


def groups_of(seqs, hkv=8, d=128, page=64, hq=None, quantised=False):
    r = SimpleNamespace(core=SimpleNamespace(hq=hq or hkv, hkv=hkv, d=d), quantised=quantised, block_size=page)
    return ModelRunner.prefix_groups(r, seqs)


def seq(blocks, page=64):
    return SimpleNamespace(blocks=blocks, length=len(blocks) * page + 1)


def test_documents_behind_one_common_block_keep_their_fronts():
    ids = iter(range(10 ** 6))
    head = [next(ids)]
    docs = [[next(ids) for _ in range(64)] for _ in range(2)]
    plain = groups_of([seq(doc + [next(ids)]) for doc in docs for _ in range(32)])
    assert [(i, n, len(c)) for i, n, c in plain] == [(0, 32, 64), (32, 32, 64)]
    behind = groups_of([seq(head + doc + [next(ids)]) for doc in docs for _ in range(32)])
    assert [(i, n, len(c)) for i, n, c in behind] == [(0, 32, 65), (32, 32, 65)] and behind[1][2] == head + docs[1]


@pytest.mark.parametrize("where", ["front", "back"])
def test_one_sequence_that_shares_a_block_does_not_cut_the_others_front(where):
    ids = iter(range(10 ** 6))
    doc = [next(ids) for _ in range(129)]
    seqs = [seq(doc + [next(ids)]) for _ in range(16)]
    other = seq(doc[:1] + [next(ids)])
    got = groups_of([other] + seqs if where == "front" else seqs + [other])
    assert got == [(1 if where == "front" else 0, 16, doc)]


def test_the_choice_saves_most(monkeypatch):
    """Against every choice of up to three groups of up to seven rows."""
    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    monkeypatch.setattr(R2, "_MAX_GROUPS", 3)
    rng = random.Random(1)

    def front(a, b):
        n = 0
        while n < min(len(a), len(b)) and a[n] == b[n]:
            n += 1
        return n

    def saved(seqs, runs):
        return sum((j - i - 1) * min(front(seqs[i].blocks, s.blocks) for s in seqs[i:j]) for i, j in runs)

    def choices(n, i, g):
        yield []
        if g:
            for a in range(i, n):
                for b in range(a + 2, n + 1):
                    for rest in choices(n, b, g - 1):
                        yield [(a, b)] + rest

    for _ in range(60):
        n = rng.randint(0, 7)
        seqs = sorted((seq([rng.randint(0, 1) * 10 ** k + k for k in range(rng.randint(0, 5))]) for _ in range(n)), key=lambda s: s.blocks)
        got = groups_of(seqs)
        at = 0
        for i, rows, common in got:
            assert i >= at and rows > 1 and common and all(s.blocks[:len(common)] == common for s in seqs[i:i + rows])
            at = i + rows
        best = max(saved(seqs, c) for c in choices(n, 0, 3))
        assert len(got) <= 3 and sum((rows - 1) * len(common) for _, rows, common in got) == best


def test_a_full_batch_is_looked_at_quickly():
    import time

    seqs = [seq([1] + [2 + i // 64 for _ in range(100)] + [1000 + i]) for i in range(256)]
    groups_of(seqs)
    t = time.perf_counter()
    got = groups_of(seqs)
    assert [(i, n, len(c)) for i, n, c in got] == [(64 * k, 64, 101) for k in range(4)]
    assert time.perf_counter() - t < 1.0          # 10 ms


@pytest.mark.parametrize("sizes,hq,hkv,quantised,shared", [
    ((16,), 32, 8, False, True), ((8,), 32, 8, False, False),                  # one prefix of 18 and 17 blocks: 71 and 31 MB
    ((8,) * 8, 32, 8, True, False), ((8,) * 2, 32, 32, True, True),            # 8 bits, nine blocks: 68 MB each, eight groups and two
    ((64,), 48, 1, False, False), ((64,), 48, 1, True, False),                 # 46 blocks and more than 16 query heads a key head: 95 and 49 MB
])
def test_sharing_has_to_pay_for_its_kernels(sizes, hq, hkv, quantised, shared):
    ids = iter(range(10 ** 6))
    blocks = {16: 18, 8: 17 if not quantised else 9, 64: 46}
    seqs = []
    for n in sizes:
        doc = [next(ids) for _ in range(blocks[n])]
        seqs += [seq(doc + [next(ids)]) for _ in range(n)]
    got = groups_of(seqs, hkv=hkv, hq=hq, quantised=quantised)
    assert [n for _, n, _ in got] == (list(sizes) if shared else [])


def test_sequences_that_share_nothing_stand_behind_the_groups():
    r = SimpleNamespace(shared_prefix=True)
    order = ModelRunner.by_prefix(r, [seq([9, 1]), seq([3]), seq([2, 5]), seq([9, 4]), seq([]), seq([2, 6]), seq([7])])
    assert [s.blocks for s in order] == [[2, 5], [2, 6], [9, 1], [9, 4], [], [3], [7]]
    assert ModelRunner.by_prefix(SimpleNamespace(shared_prefix=False), order[::-1]) == order[::-1]


def test_bounds_lie_close_to_the_groups(tmp_path, monkeypatch):
    from llmss_b200.engine.engine import Engine
    from llmss_b200.utils.checkpoint import write_random_checkpoint

    import torch

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    path = str(write_random_checkpoint(tmp_path, "gptj-tiny", dtype=torch.float32, device="cpu", std=0.08))
    r = Engine.from_pretrained(path, device="cpu", max_batch=64, max_seq_len=128, block_size=1, prefix_cache=True, shared_prefix=True).runner
    for rows, blocks, want in ((3, 1, (1, 4)), (5, 8, (8, 8)), (9, 9, (10, 16)), (17, 33, (40, 24)), (40, 64, (64, 48)), (2, 65, (80, 2)), (2, 127, (128, 2))):
        seqs = [seq(list(range(blocks)) + [1000 + i], page=1) for i in range(rows)] + [seq([500 + i], page=1) for i in range(20)]
        r._bind_prefix(seqs)
        p = r._step_prefix(64)
        assert (p.max_len, p.max_rows) == want and p.num_groups == 1
        assert max(p.lens.tolist()) <= p.max_len and rows <= p.max_rows
    assert r._step_prefix(1).max_rows == 1
