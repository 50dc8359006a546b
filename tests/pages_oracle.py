"""Batches over scattered (and shared) pages, and attention over them in 64 bits."""
import random
from types import SimpleNamespace

import torch

from llmss_b200.engine.batch import BatchInput, SharedPrefix
from llmss_b200.ops.pages import QuantPages, quantise


def make_batch(new, ctx, page, groups, device, seed=0, max_kv=None):
    """``groups``: [(consecutive sequences, shared tokens)].  A prefix that ends inside a page has that page for itself: the sequences' own tables name
    another one there, whose first tokens are not looked at."""
    rng = random.Random(seed)
    need = [-(-(a + c) // page) for a, c in zip(new, ctx)]
    shared = [-(-n // page) for _, n in groups]
    ids = list(range(1, 1 + sum(need) + sum(shared)))
    rng.shuffle(ids)
    take = iter(ids)
    fronts = [[next(take) for _ in range(n)] for n in shared]
    tables = [[next(take) for _ in range(n)] for n in need]
    front_of = {i: (j, n) for j, (g, n) in enumerate(groups) for i in g}
    for i, (j, n) in front_of.items():
        tables[i][:n // page] = fronts[j][:n // page]
    batch = BatchInput.build([[0] * a for a in new], ctx, tables, page, device)
    if max_kv is not None:
        batch.max_kv = max_kv
    if groups:
        batch.prefix = SharedPrefix.build([g for g, _ in groups], fronts, [n for _, n in groups], new, device)
    return batch, SimpleNamespace(blocks=1 + len(ids), new=new, ctx=ctx, tables=tables, fronts=fronts, front_of=front_of, page=page)


def make_pages(blocks, hkv, page, d, kind, dtype, device, seed=0):
    x = torch.randn(blocks, hkv, page, d, generator=torch.Generator().manual_seed(seed)) * (1 + seed % 3)
    if kind is None:
        return x.to(dtype).to(device)
    codes, scale = quantise(x, kind)
    return QuantPages(codes.to(device), scale.to(device))


def values64(pages):
    return pages.data.double() * pages.scale.double()[..., None] if isinstance(pages, QuantPages) else pages.double()


def attend64(q, k, v, batch, seen, hq, hkv, d, scale):
    """[sum(new), hq * d] in 64 bits, a token's key and value looked up one by one."""
    k, v = values64(k), values64(v)
    out, at = [], 0
    for i, (a, L) in enumerate(zip(seen.new, batch.seq_lens.tolist())):
        j, n = seen.front_of.get(i, (0, 0))
        block = torch.tensor([(seen.fronts[j] if p < n else seen.tables[i])[p // seen.page] for p in range(L)], dtype=torch.long, device=k.device)
        off = torch.arange(L, device=k.device) % seen.page
        rows = q[at:at + a].double().view(a, hkv, hq // hkv, d)
        z = torch.einsum("ahgd,lhd->hgal", rows, k[block, :, off]) * scale
        z = z.masked_fill(torch.arange(L, device=k.device) > torch.arange(L - a, L, device=k.device)[:, None], float("-inf"))
        o = torch.einsum("hgal,lhd->ahgd", torch.softmax(z, -1), v[block, :, off]).reshape(a, hq * d)
        o[:max(0, a - L)] = 0
        out.append(o)
        at += a
    return torch.cat(out)
