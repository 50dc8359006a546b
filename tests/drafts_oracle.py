"""Trees of drafted tokens: batches of them, what their rows see, and attention over them in 64 bits."""
import random
from unittest import mock

import torch

import pages_bounds
from llmss_b200.engine.batch import BatchInput, DraftTree, SharedPrefix
from pages_oracle import values64


def random_parents(n, rng, shape="any"):
    """``shape``: chain, star, forest (several first tokens), any."""
    if n == 0:
        return []
    if shape == "chain":
        return [j - 1 for j in range(n)]
    if shape == "star":
        return [-1] + [0] * (n - 1)
    if shape == "forest":
        return [-1 if rng.random() < 0.3 else rng.randrange(j) if j else -1 for j in range(n)]
    return [-1] + [j - 1 if rng.random() < 0.4 else rng.randrange(j) for j in range(1, n)]


def ancestors(parents):
    """Sets of places that each token sees."""
    out = []
    for j, p in enumerate(parents):
        out.append((out[p] if 0 <= p < j else set()) | {j})
    return out


def words_of(sets, words):
    rows = [[sum(1 << x % 32 for x in s if x // 32 == w) for w in range(words)] for s in sets]
    return torch.tensor([[x - (1 << 32) if x >> 31 else x for x in r] for r in rows], dtype=torch.int32).reshape(len(sets), words)


def set_masks(batch, seen, sets, words=None):
    """A batch whose rows see exactly ``sets`` of their sequence's new tokens."""
    words = words or max(1, -(-batch.max_q // 32))
    dev = batch.cu_q.device
    batch.tree = DraftTree(parents=torch.full((batch.tokens.numel(),), -1, dtype=torch.int32, device=dev), masks=words_of(sets, words).to(dev))
    seen.sets = sets
    return batch


def sequences(q, k, v, batch, seen, hq, hkv, d, scale):
    """As pages_bounds.sequences, of rows that see all cached tokens and ``seen.sets`` of the new ones."""
    keys, values, at = values64(k), values64(v), 0
    for i, (a, L) in enumerate(zip(seen.new, batch.seq_lens.tolist())):
        j, n = seen.front_of.get(i, (0, 0))
        block = torch.tensor([(seen.fronts[j] if p < n else seen.tables[i])[p // seen.page] for p in range(L)], dtype=torch.long, device=keys.device)
        off = torch.arange(L, device=keys.device) % seen.page
        kk, vv = (x[block, :, off].transpose(0, 1) for x in (keys, values))
        rows = q[at:at + a].double().view(a, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        z = (rows @ kk[:, None].transpose(-1, -2)) * scale
        hidden = torch.tensor([[p - (L - a) >= 0 and p - (L - a) not in s for p in range(L)] for s in seen.sets[at:at + a]], dtype=torch.bool).reshape(a, L)
        yield at, z.masked_fill(hidden.to(z.device), float("-inf")), rows, kk, vv
        at += a


def expected(q, k, v, batch, seen, hq, hkv, d, scale):
    """(result, how far an output may be off, results without 16 keys): the bounds count the same roundings as those of attention over pages."""
    with mock.patch.object(pages_bounds, "sequences", sequences):
        return pages_bounds.expected(q, k, v, batch, seen, hq, hkv, d, scale)


def path_of(parents, tokens, sampled):
    path = [0] if parents else []
    while path:
        step = [c for c in range(path[-1] + 1, len(parents)) if parents[c] == path[-1] and tokens[c] == sampled[path[-1]]]
        if not step:
            break
        path.append(step[0])
    return path
