"""Captured decode steps with shared prefixes: how many are kept, and what is counted of them."""
import pytest
import torch

from llmss_b200.engine import runner as R2
from llmss_b200.engine.engine import Engine
from llmss_b200.engine.runner import SamplingParams

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [None, "int8"])
def test_captured_steps_with_prefixes_are_few_and_counted_apart(tmp_path, monkeypatch, kind):
    from llmss_b200.utils.checkpoint import write_random_checkpoint

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    monkeypatch.setattr(R2, "_MAX_PREFIX_GRAPHS", 2)
    path = str(write_random_checkpoint(tmp_path, "gptj-tiny", dtype=torch.float32, device="cpu", std=0.08))
    g = torch.Generator().manual_seed(4)
    draw = lambda n: torch.randint(1, 400, (n,), generator=g).tolist()
    eng = Engine.from_pretrained(path, dtype=torch.float16, device="cuda", max_batch=4, max_seq_len=256, block_size=16, prefix_cache=True, shared_prefix=True,
                                 kv_cache_dtype=kind)
    r, sp = eng.runner, SamplingParams(max_new_tokens=4, is_greedy=True)
    eng.generate([draw(9), draw(12)], sp)                      # two requests that share nothing
    alone = dict(r.launches_per_graph)
    fronts = [draw(n) for n in (17, 40, 70, 140)]              # bounds of 16, 32, 64 and 128 tokens
    waves = [[f + draw(3), f + draw(5)] for f in fronts]
    for f in fronts:
        eng.generate([f + [1]], SamplingParams(max_new_tokens=2, is_greedy=True))
    first = [eng.generate(w, sp) for w in waves]
    kept = [k for k in r.graphs if k[2] is not None]
    assert [k[2][1] for k in kept] == [64, 128]
    assert eng.generate(waves[2], sp) == first[2]              # used again, and so the last to go
    assert [eng.generate(w, sp) for w in waves[:2]] == first[:2]
    assert [k[2][1] for k in r.graphs if k[2] is not None] == [16, 32]
    assert {k: v for k, v in r.launches_per_graph.items() if not isinstance(k, tuple)}.items() >= alone.items()
    assert {k for k in r.launches_per_graph if isinstance(k, tuple)} == {(k[0], k[2]) for k in r.graphs if k[2] is not None}
    assert r.alloc.num_free == r.alloc.num_blocks - 1
