"""What the attention of a decode step is told about fronts that its sequences share."""
import pytest
import torch

from llmss_b200.engine import runner as R2
from llmss_b200.engine.engine import Engine
from llmss_b200.engine.runner import SamplingParams


@pytest.mark.parametrize("kind", [None, "int8"])
def test_the_attention_of_a_step_gets_the_groups(tmp_path, monkeypatch, kind):
    from llmss_b200 import ops
    from llmss_b200.utils.checkpoint import write_random_checkpoint

    monkeypatch.setattr(R2, "_SHARE_MIN_BYTES", 0)
    path = str(write_random_checkpoint(tmp_path, "gptj-tiny", dtype=torch.float32, device="cpu", std=0.08))
    g = torch.Generator().manual_seed(4)
    draw = lambda n: torch.randint(1, 500, (n,), generator=g).tolist()
    a, b = draw(40), draw(20)
    prompts = [a + draw(5), b + draw(3), draw(9), a + draw(11), b + draw(8), a + draw(1)]
    eng = Engine.from_pretrained(path, device="cpu", max_batch=6, max_seq_len=128, block_size=16, prefix_cache=True, shared_prefix=True, kv_cache_dtype=kind)
    eng.generate([a + [3], b + [4]], SamplingParams(max_new_tokens=2, is_greedy=True))
    given, real = [], ops.attention

    def watch(qkv, out, batch, *rest, **kw):
        p = batch.prefix
        given.append((batch.is_decode, None if p is None else (p.lens[:p.num_groups].tolist(), p.first[:p.num_groups + 1].tolist(),
                                                               [p.block_tables[j, :n // 16].tolist() for j, n in enumerate(p.lens[:p.num_groups].tolist())])))
        return real(qkv, out, batch, *rest, **kw)

    monkeypatch.setattr(ops, "attention", watch)
    for p, n in zip(prompts, (9, 12, 7, 4, 6, 10)):
        eng.add_request(p, SamplingParams(max_new_tokens=n, is_greedy=True))
    shared = alone = 0
    while eng.has_work():
        given.clear()
        eng.step()
        live = list(eng.runner.batch_seqs)
        for decode, p in given:
            if not decode:
                assert p is None
                continue
            want = [(i, n, c) for i, n, c in eng.runner.prefix_groups(live)] if all(s.blocks for s in live) else None
            if want is None:
                continue                                   # a request ended in this step: its blocks are gone
            if not want:
                assert p is None
                alone += 1
                continue
            lens, first, tables = p
            assert [(first[j], first[j + 1] - first[j], tables[j]) for j in range(len(lens)) if lens[j]] == want
            assert all(lens[j] == 16 * len(tables[j]) for j in range(len(lens)))
            shared += 1
    assert shared > 4 and alone > 0
    assert eng.runner._prefix is None
