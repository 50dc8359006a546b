"""Steps that check drafted tokens, as cases whose speed and results can be measured.

Three operators, each a call of ``llmss_b200.ops``: ``step_layout`` (block tables, cache slots, positions and tree masks from request lengths),
``attention`` for trees of drafted tokens over 16-bit or 8-bit pages (``batch.tree``), and ``accept_drafts`` (the path of a tree that agrees with what was
sampled, and its cache rows moved behind one another).  The ranges: 1 to 256 sequences of unequal lengths, 1 to 65536 rows, trees of 1 to 256
tokens, contexts up to 36000 tokens, the head layouts of the models that this framework serves, pages of 16 to 64 tokens in scattered order.

``own`` False: plain torch, attention in 32 bits.  ``own`` True: the framework's calls.
"""
import math
import random

import torch

own = False

F32, F64, I32 = torch.float32, torch.float64, torch.int32
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
PAGE_TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "fp8": 448.0}
# query heads, key / value heads, head size
HEADS = {"gptj": (16, 16, 256), "llama": (32, 32, 128), "grouped": (32, 8, 128), "multi_query": (48, 1, 128), "small": (16, 16, 64)}
VOCAB = 50400


def listed():
    return [
        # a decode step's metadata: the smallest launch, where latency counts
        {"name": "layout_step", "kind": "layout", "seqs": 64, "tokens": 1, "context": 1040, "page": 64, "tree": False},
        # a step that checks a tree of guesses for every request of a batch
        {"name": "layout_trees", "kind": "layout", "seqs": 64, "tokens": 24, "context": 1040, "page": 64, "tree": True},
        # a full round of prompts
        {"name": "layout_prompts", "kind": "layout", "seqs": 64, "tokens": 1000, "context": 0, "page": 16, "tree": False},
        # one request alone, a dozen guesses
        {"name": "tree_one", "kind": "attend", "heads": "grouped", "seqs": 1, "tokens": 12, "context": 611, "page": 64, "pages": "16", "dtype": "bfloat16"},
        # a batch of a GPT-J-6B shape, a few guesses each: one query head a key head
        {"name": "tree_step", "kind": "attend", "heads": "gptj", "seqs": 64, "tokens": 10, "context": 1040, "page": 64, "pages": "16", "dtype": "bfloat16"},
        # grouped heads, larger trees, 8-bit cache
        {"name": "tree_step_int8", "kind": "attend", "heads": "grouped", "seqs": 48, "tokens": 24, "context": 1500, "page": 64, "pages": "int8",
         "dtype": "bfloat16"},
        # all query heads on one key head
        {"name": "tree_step_multi_query", "kind": "attend", "heads": "multi_query", "seqs": 24, "tokens": 8, "context": 2000, "page": 16, "pages": "16",
         "dtype": "float16"},
        # a few requests with long contexts: the cache is nearly all that is read
        {"name": "tree_long", "kind": "attend", "heads": "grouped", "seqs": 6, "tokens": 40, "context": 24000, "page": 64, "pages": "16", "dtype": "bfloat16"},
        # few requests, wide trees, small heads, 8-bit cache
        {"name": "tree_wide", "kind": "attend", "heads": "small", "seqs": 8, "tokens": 170, "context": 3000, "page": 32, "pages": "fp8", "dtype": "float16"},
        # one request, a cache of few layers
        {"name": "accept_one", "kind": "accept", "heads": "grouped", "layers": 16, "seqs": 1, "tokens": 12, "context": 611, "page": 64, "pages": "16",
         "dtype": "bfloat16"},
        # a batch, 12 layers of a GPT-J-6B shape
        {"name": "accept_step", "kind": "accept", "heads": "gptj", "layers": 12, "seqs": 64, "tokens": 12, "context": 20, "page": 16, "pages": "16",
         "dtype": "bfloat16"},
        # the same in 8 bits with larger trees
        {"name": "accept_step_fp8", "kind": "accept", "heads": "grouped", "layers": 16, "seqs": 48, "tokens": 60, "context": 24, "page": 16, "pages": "fp8",
         "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["layout", "attend", "attend", "attend", "accept"])
    case = {"kind": kind, "page": rng.choice([16, 32, 64, 64])}
    if kind == "layout":
        tree = rng.random() < 0.5
        seqs = _log(rng, 1, 256)
        case.update(seqs=seqs, tokens=_log(rng, 1, 160 if tree else min(8000, 40000 // seqs)), context=_log(rng, 8, 8000), tree=tree)
        return case
    heads = rng.choice(sorted(HEADS))
    hq, hkv, d = HEADS[heads]
    case.update(heads=heads, dtype=rng.choice(["bfloat16", "bfloat16", "float16"]))
    if kind == "accept":
        # the whole cache comes back: a few hundred megabytes of it
        layers = _log(rng, 2, 32)
        seqs = _log(rng, 1, 64)
        rows = 128 * 1024 * 1024 // (layers * 2 * hkv * d)
        tokens = _log(rng, 1, min(128, max(2, rows // seqs // 4)))
        case.update(layers=layers, seqs=seqs, tokens=tokens, context=_log(rng, 1, max(2, min(600, rows // seqs // 2))), pages=rng.choice(["16", "16", "fp8"]))
        return case
    case["pages"] = rng.choice(["16", "16", "int8", "fp8"])
    seqs = _log(rng, 1, 64)
    tokens = _log(rng, 1, min(170, max(1, 5000 * 4096 // (hq * d) // seqs)))
    most = 24000 * 6 * 1024 // (hkv * d)          # cached tokens of all sequences
    case.update(seqs=seqs, tokens=tokens, context=_log(rng, 16, min(24000, most // seqs // 2, 24000 * 240 * 32 // (seqs * tokens * hq))))
    return case


# ----------------------------------------------------------------------------- lengths, trees and pages of a case
def _spread(mean, n):
    """n unequal lengths between half and one and a half times the mean (a function of the case alone, so its work is known)."""
    if mean <= 1:
        return [mean] * n
    return [max(1, round(mean * (0.5 + ((7 * i + 3) % n + 0.5) / n))) for i in range(n)]


def _lengths(case):
    """(new tokens, cached tokens before them) of every sequence."""
    return list(zip(_spread(case["tokens"], case["seqs"]), _spread(case["context"], case["seqs"])))


def _tree(rng, n):
    """Parents of a tree of guesses: a trunk of the likeliest ones, branches off any earlier token, parents before children."""
    trunk = max(1, n // 4)
    return [-1] + [j - 1 if j <= trunk else rng.randrange(j) for j in range(1, n)]


def _layout(case, seed):
    """Scattered pages and trees: lists for the device, and the same for ``exact``."""
    page, lens = case["page"], _lengths(case)
    rng = random.Random(seed)
    need = [-(-(a + c) // page) for a, c in lens]
    ids = list(range(1, 1 + sum(need)))
    rng.shuffle(ids)
    tables, at = [], 0
    for k in need:
        tables.append(ids[at:at + k])
        at += k
    trees = [_tree(rng, a) for a, _ in lens] if case.get("tree", True) else None
    return lens, tables, trees, 1 + sum(need)


def _words(case):
    return -(-max(a for a, _ in _lengths(case)) // 32)


def _visible(trees):
    """Sets of a sequence's own tokens that each of them sees: itself and its ancestors."""
    out = []
    for parents in trees:
        seen = []
        for j, p in enumerate(parents):
            seen.append((seen[p] if p >= 0 else 0) | 1 << j)
        out.append(seen)
    return out


def _signed(x):
    return x - (1 << 32) if x >= 1 << 31 else x


def _mask_words(trees, words):
    return [[_signed(m >> 32 * w & 0xFFFFFFFF) for w in range(words)] for seen in _visible(trees) for m in seen]


def _ints(v):
    return torch.tensor(v, dtype=I32).cuda()


def _pages(gen, shape, kind, dtype, channels):
    """Pages as a layer leaves them: keys with some strong channels, values without."""
    x = torch.randn(shape, generator=gen, device="cuda", dtype=F32)
    if channels:
        x *= torch.exp(0.5 * torch.randn(shape[-3], 1, shape[-1], generator=gen, device="cuda"))
    if kind == "16":
        return x.to(dtype), None
    scale = x.abs().amax(-1) / QMAX[kind]
    x /= scale[..., None]
    return (x.round_().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)), scale


def _drafts(case, seed, trees):
    """Tokens of the trees, and what was sampled at every one of them: along a path of some length what the tree guessed, elsewhere anything."""
    rng = random.Random(seed + 1)
    tokens, sampled = [], []
    for parents in trees:
        n = len(parents)
        tok = [rng.randrange(VOCAB) for _ in range(n)]
        for j in range(1, n):                       # now and then two guesses for a place are the same token
            if rng.random() < 0.1:
                tok[j] = tok[rng.randrange(1, n)]
        got = [rng.randrange(VOCAB) for _ in range(n)]
        node = 0
        while rng.random() < 0.8:
            children = [j for j in range(node + 1, n) if parents[j] == node]
            if not children:
                break
            child = rng.choice(children)
            got[node] = tok[child]
            node = next(j for j in children if tok[j] == tok[child])
        tokens += tok
        sampled += got
    return tokens, sampled


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, tables, trees, blocks = _layout(case, seed)
    T, width = sum(a for a, _ in lens), max(len(t) for t in tables)
    s = {"case": dict(case), "rows": T, "width": width, "max_new": max(a for a, _ in lens), "max_kv": max(a + c for a, c in lens),
         "new": _ints([a for a, _ in lens]), "context": _ints([c for _, c in lens])}
    s["parents"] = None if trees is None else _ints([p for t in trees for p in t])
    if case["kind"] == "layout":
        s["pages"], s["counts"] = _ints([b for t in tables for b in t]), _ints([len(t) for t in tables])
        return s
    hq, hkv, d = HEADS[case["heads"]]
    dt = DTYPES[case["dtype"]]
    cu = [0]
    for a, _ in lens:
        cu.append(cu[-1] + a)
    s.update(tables=_ints([t + [0] * (width - len(t)) for t in tables]), seq_lens=_ints([a + c for a, c in lens]), cu=_ints(cu),
             masks=_ints(_mask_words(trees, _words(case))))
    if case["kind"] == "attend":
        s["q"] = torch.randn(T, hq * d, generator=gen, device="cuda", dtype=F32).to(dt)
        for n in ("k", "v"):
            s[n], s[n + "_scale"] = _pages(gen, (blocks, hkv, case["page"], d), case["pages"], dt, n == "k")
        return s
    s["data"], s["scale"] = _pages(gen, (case["layers"], 2, blocks, hkv, case["page"], d), case["pages"], dt, False)
    tokens, sampled = _drafts(case, seed, trees)
    s["tokens"], s["sampled"] = _ints(tokens), _ints(sampled)
    return s


# ----------------------------------------------------------------------------- the plain forms
def _padded(x, cu, width, fill):
    """Rows of a packed tensor as [sequences, width], ``fill`` behind a sequence's last."""
    row = torch.arange(width, device="cuda")
    at = cu[:-1, None] + row
    live = at < cu[1:, None]
    return torch.where(live, x[at.clamp(max=x.numel() - 1)], fill), live


def _layout_plain(s):
    case, T = s["case"], s["rows"]
    page = case["page"]
    new, ctx = s["new"].long(), s["context"].long()
    B, zero = new.numel(), torch.zeros(1, dtype=torch.long, device="cuda")
    cu = torch.cat([zero, new.cumsum(0)])
    first = torch.cat([zero, s["counts"].long().cumsum(0)])
    col = torch.arange(s["width"], device="cuda")
    at = first[:-1, None] + col
    tables = torch.where(at < first[1:, None], s["pages"][at.clamp(max=s["pages"].numel() - 1)], 0)
    row = torch.arange(T, device="cuda")
    seq = (row[:, None] >= cu[1:]).sum(1)                  # the sequence that a row belongs to
    j = row - cu[seq]
    place = ctx[seq] + j
    slots = tables[seq, place // page].long() * page + place % page
    out = {"seq_lens": ctx + new, "cu_q": cu, "last": cu[1:] - 1, "slots": slots, "block_tables": tables, "positions": place}
    if case["tree"]:
        words = -(-s["max_new"] // 32)
        bits = torch.zeros(T, 32 * words, dtype=torch.long, device="cuda")
        up, depth = j.clone(), torch.full_like(j, -1)
        parents = s["parents"].long()
        for _ in range(s["max_new"]):                      # no path is longer
            live = up >= 0
            bits[row, up.clamp(min=0)] |= live.long()
            depth += live
            up = torch.where(live, parents[cu[seq] + up.clamp(min=0)], -1)
        out["positions"] = ctx[seq] + depth
        out["masks"] = (bits.view(T, words, 32) << torch.arange(32, device="cuda")).sum(-1)
    return {n: x if n == "last" else x.to(I32) for n, x in out.items()}


def _gathered(s, n):
    """Keys or values of every sequence as numbers, [B, heads, tokens of all its table's pages, d]."""
    t = s["tables"].long()
    x = s[n][t].float()
    if s[n + "_scale"] is not None:
        x = x * s[n + "_scale"][t][..., None]
    B, nb, hkv, page, d = x.shape
    return x.transpose(1, 2).reshape(B, hkv, nb * page, d)


def _attend_plain(s):
    hq, hkv, d = HEADS[s["case"]["heads"]]
    T, cu, mq = s["rows"], s["cu"].long(), s["max_new"]
    k, v = _gathered(s, "k"), _gathered(s, "v")
    B, L = k.shape[0], k.shape[2]
    row = torch.arange(mq, device="cuda")
    at = (cu[:-1, None] + row).clamp_(max=T - 1)                                       # [B, mq]; rows behind a sequence's last go nowhere
    ctx = s["context"].long()
    bits = (s["masks"].long()[:, :, None] >> torch.arange(32, device="cuda") & 1).view(T, -1)
    own_key = torch.arange(L, device="cuda") - ctx[:, None]                            # [B, L]: which of the new tokens a key is
    inside = (own_key >= 0) & (own_key < bits.shape[1])
    seen = bits[at[:, :, None], own_key.clamp(0, bits.shape[1] - 1)[:, None, :]] > 0   # [B, mq, L]
    seen = (own_key < 0)[:, None] | (inside[:, None] & seen)
    q = s["q"].view(T, hkv, hq // hkv, d).float()[at].permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    scores = (q @ k.transpose(-1, -2)).view(B, hkv, hq // hkv, mq, L) * d ** -0.5
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, hkv, -1, L) @ v).view(B, hkv, hq // hkv, mq, d).permute(0, 3, 1, 2, 4).reshape(B, mq, hq * d)
    return o[row < s["new"].long()[:, None]].to(s["q"].dtype)                          # packed again


def _accept_plain(s):
    cu, n, page = s["cu"].long(), s["max_new"], s["case"]["page"]
    B = cu.numel() - 1
    tokens, live = _padded(s["tokens"].long(), cu, n, -1)
    parents, _ = _padded(s["parents"].long(), cu, n, -2)
    sampled, _ = _padded(s["sampled"].long(), cu, n, -1)
    col, seq = torch.arange(n, device="cuda"), torch.arange(B, device="cuda")
    node, alive = torch.zeros(B, dtype=torch.long, device="cuda"), live[:, 0]
    path, got, counts = [], [], torch.zeros(B, dtype=torch.long, device="cuda")
    for _ in range(n):
        path.append(torch.where(alive, node, -1))
        got.append(torch.where(alive, sampled[seq, node], -1))
        counts += alive
        hit = live & (parents == node[:, None]) & (tokens == sampled[seq, node][:, None]) & alive[:, None]
        child = torch.where(hit, col, n).amin(1)
        alive = child < n
        node = torch.where(alive, child, 0)
    path = torch.stack(path, 1)
    k, i = torch.arange(n, device="cuda").expand(B, n), seq[:, None].expand(B, n)
    moved = (path >= 0) & (path != k)
    base = (s["seq_lens"] - s["new"]).long()[:, None].expand(B, n)[moved]
    src, dst, i, table = base + path[moved], base + k[moved], i[moved], s["tables"].long()
    for x in (s["data"].view(torch.int8) if s["data"].dtype == torch.float8_e4m3fn else s["data"], s["scale"]):
        if x is not None:
            x[:, :, table[i, dst // page], :, dst % page] = x[:, :, table[i, src // page], :, src % page]
    return {"tokens": torch.stack(got, 1).to(I32), "counts": counts.to(I32), "path": path.to(I32), "data": s["data"], "scale": s["scale"]}


# ----------------------------------------------------------------------------- the framework's calls
def _layout_own(s):
    from llmss_b200 import ops

    got = ops.step_layout(s["context"], s["new"], s["pages"], s["case"]["page"], s["rows"], s["max_new"], page_counts=s["counts"], max_blocks=s["width"],
                          parents=s["parents"])
    out = {"seq_lens": got.seq_lens, "cu_q": got.cu_q, "last": got.last_idx, "slots": got.slot_mapping, "block_tables": got.block_tables,
           "positions": got.positions}
    if s["case"]["tree"]:
        out["masks"] = got.masks
    return out


def _batch(s):
    from llmss_b200.engine.batch import BatchInput, DraftTree

    tokens = s.get("tokens", s["parents"])
    return BatchInput(tokens=tokens, positions=tokens, slot_mapping=tokens, block_tables=s["tables"], seq_lens=s["seq_lens"], cu_q=s["cu"], last_idx=s["cu"],
                      num_seqs=s["new"].numel(), max_q=s["max_new"], max_kv=s["max_kv"], is_decode=False, is_fresh_prefill=False,
                      tree=DraftTree(parents=s["parents"], masks=s["masks"]))


def _attend_own(s):
    from llmss_b200 import ops

    hq, hkv, d = HEADS[s["case"]["heads"]]
    k, v = (s["k"], s["v"]) if s["k_scale"] is None else (ops.QuantPages(s["k"], s["k_scale"]), ops.QuantPages(s["v"], s["v_scale"]))
    out = torch.empty_like(s["q"])
    return ops.attention(s["q"], out, _batch(s), k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)


def _accept_own(s):
    from llmss_b200 import ops

    got = ops.accept_drafts(s["sampled"], _batch(s), [s["data"]] if s["scale"] is None else [s["data"], s["scale"]])
    return {"tokens": got.tokens, "counts": got.counts, "path": got.path, "data": s["data"], "scale": s["scale"]}


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"layout": _layout_own, "attend": _attend_own, "accept": _accept_own}[kind](state)
    return {"layout": _layout_plain, "attend": _attend_plain, "accept": _accept_plain}[kind](state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    lens = _lengths(case)
    T, B = sum(a for a, _ in lens), len(lens)
    if case["kind"] == "layout":
        used = [-(-(a + c) // case["page"]) for a, c in lens]
        words = _words(case) + 1 if case["tree"] else 0                 # masks out, parents in
        return {"bytes": 4 * (3 * B + sum(used) + 4 * B + 1 + 2 * T + words * T + B * max(used)), "flops": 0}
    hq, hkv, d = HEADS[case["heads"]]
    row = 2 * hkv * (2 * d if case["pages"] == "16" else d + 4)
    if case["kind"] == "accept":
        # a path of three rows that move, each read and written in all layers
        return {"bytes": 2 * case["layers"] * row * sum(min(3, a - 1) for a, _ in lens) + 12 * T + 8 * B * max(a for a, _ in lens), "flops": 0}
    # every token sees at least what is cached, the tree's first token and itself
    return {"bytes": row * sum(a + c for a, c in lens) + 2 * 2 * T * hq * d + 4 * _words(case) * T,
            "flops": 4 * hq * d * sum(a * (c + 1) + a - 1 for a, c in lens)}


# ----------------------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    lens, tables, trees, _ = _layout(case, seed)
    page = case["page"]
    if case["kind"] == "layout":
        width = max(len(t) for t in tables)
        cu, pos, slots = [0], [], []
        for i, (a, c) in enumerate(lens):
            cu.append(cu[-1] + a)
            slots += [tables[i][p // page] * page + p % page for p in range(c, c + a)]
            pos += [c + bin(m).count("1") - 1 for m in _visible([trees[i]])[0]] if trees else range(c, c + a)
        out = {"seq_lens": [a + c for a, c in lens], "cu_q": cu, "last": [x - 1 for x in cu[1:]], "slots": slots,
               "block_tables": [t + [0] * (width - len(t)) for t in tables], "positions": pos}
        if trees:
            out["masks"] = _mask_words(trees, _words(case))
        return {n: torch.tensor(x, dtype=torch.long if n == "last" else I32).cuda() for n, x in out.items()}
    s = prepare(case, seed)
    if case["kind"] == "accept":
        tokens, sampled = _drafts(case, seed, trees)
        wide, at = max(a for a, _ in lens), 0
        tok, paths = [], []
        whole = s["data"].double() if s["scale"] is None else s["data"].view(torch.int8).clone()
        scale = None if s["scale"] is None else s["scale"].double()
        for i, (a, c) in enumerate(lens):
            path = [0]
            while True:
                want = sampled[at + path[-1]]
                step = [j for j in range(a) if trees[i][j] == path[-1] and tokens[at + j] == want]
                if not step:
                    break
                path.append(step[0])
            for n, x in ((0, whole), (1, scale)):
                if x is None:
                    continue
                rows = [x[:, :, tables[i][(c + j) // page], :, (c + j) % page].clone() for j in path]
                for to, r in enumerate(rows):
                    x[:, :, tables[i][(c + to) // page], :, (c + to) % page] = r
            tok.append([sampled[at + j] for j in path] + [-1] * (wide - len(path)))
            paths.append(path + [-1] * (wide - len(path)))
            at += a
        data = whole if s["scale"] is None else whole.view(torch.float8_e4m3fn).double()
        return {"tokens": _ints(tok), "counts": _ints([sum(x >= 0 for x in p) for p in paths]), "path": _ints(paths), "data": data, "scale": scale}
    hq, hkv, d = HEADS[case["heads"]]
    out, at = [], 0
    for i, (a, c) in enumerate(lens):
        ids = torch.tensor(tables[i]).cuda()
        k, v = ((s[n][ids].double() if s[n + "_scale"] is None else s[n][ids].double() * s[n + "_scale"][ids].double()[..., None])
                .transpose(0, 1).reshape(hkv, -1, d)[:, :a + c] for n in ("k", "v"))
        hidden = torch.tensor([[not m >> j & 1 for j in range(a)] for m in _visible([trees[i]])[0]]).cuda()
        q = s["q"][at:at + a].double().view(a, hkv, -1, d)
        heads = []
        for h in range(hkv):
            z = torch.einsum("qgd,kd->gqk", q[:, h], k[h]) / math.sqrt(d)
            z[:, :, c:].masked_fill_(hidden, -math.inf)
            heads.append(torch.einsum("gqk,kd->qgd", torch.softmax(z, -1), v[h]))
        out.append(torch.stack(heads, 1).reshape(a, hq * d))
        at += a
    return torch.cat(out)
