"""Serving from 8-bit cache pages and from pages that a batch shares, as cases whose speed and results can be measured.

Three operators, each a call of ``llmss_b200.ops``: ``rope_kv_write`` into 8-bit pages (rotation of queries and keys, a scale per token and
head, codes), ``attention`` over 8-bit pages, and ``attention`` for groups of sequences that share a prefix, over 16-bit or 8-bit pages.  The
ranges: 1 to 8192 packed tokens, 1 to 64 sequences of unequal lengths, contexts up to 34500 tokens, prefixes up to 8192, the head layouts of
the models that this framework serves, pages of 16 to 64 tokens in scattered order.

``own`` False: plain torch in 32 bits.  ``own`` True: the framework's calls.
"""
import math
import random

import torch

own = False

F32, F64 = torch.float32, torch.float64
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}
PAGE_TYPES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
QMAX = {"int8": 127.0, "fp8": 448.0}
# query heads, key / value heads, head size, rotated columns, style of the rotation
HEADS = {
    "gptj": (16, 16, 256, 64, "pairs"),
    "llama": (32, 32, 128, 128, "halves"),
    "grouped": (32, 8, 128, 128, "halves"),
    "multi_query": (48, 1, 128, 0, "none"),
    "small": (16, 16, 64, 0, "none"),
}
BASE = 10000.0


def listed():
    return [
        # a decode step of a GPT-J-6B layer at the benchmark's batch: the smallest write, where latency counts
        {"name": "write_step", "kind": "write", "heads": "gptj", "seqs": 64, "tokens": 1, "context": 200, "page": 64, "pages": "fp8", "dtype": "bfloat16"},
        # the same for a multi-query model with learned positions, 8-bit integers
        {"name": "write_step_multi_query", "kind": "write", "heads": "multi_query", "seqs": 24, "tokens": 1, "context": 300, "page": 16, "pages": "int8",
         "dtype": "float16"},
        # a prompt round of the engine
        {"name": "write_prompt", "kind": "write", "heads": "llama", "seqs": 8, "tokens": 1024, "context": 0, "page": 64, "pages": "fp8", "dtype": "bfloat16"},
        # one request alone
        {"name": "attend_one", "kind": "attend", "heads": "grouped", "seqs": 1, "tokens": 1, "context": 611, "page": 64, "pages": "int8", "dtype": "bfloat16"},
        # a decode step over a batch of requests at different points of their answers
        {"name": "attend_step", "kind": "attend", "heads": "gptj", "seqs": 64, "tokens": 1, "context": 1040, "page": 64, "pages": "int8", "dtype": "bfloat16"},
        # the same where all query heads read one key head
        {"name": "attend_step_multi_query", "kind": "attend", "heads": "multi_query", "seqs": 32, "tokens": 1, "context": 2000, "page": 16, "pages": "fp8",
         "dtype": "float16"},
        # a few requests with long contexts: the cache is nearly all that is read
        {"name": "attend_long", "kind": "attend", "heads": "grouped", "seqs": 8, "tokens": 1, "context": 24000, "page": 64, "pages": "fp8", "dtype": "bfloat16"},
        # portions of prompts over what is in the cache already
        {"name": "attend_prompt", "kind": "attend", "heads": "grouped", "seqs": 4, "tokens": 1000, "context": 1800, "page": 64, "pages": "int8",
         "dtype": "bfloat16"},
        # a few short requests behind one system prompt
        {"name": "share_few", "kind": "share", "heads": "small", "seqs": 6, "groups": 1, "tokens": 1, "prefix": 520, "context": 40, "page": 16, "pages": "16",
         "dtype": "float16"},
        # a decode step of a full batch behind one long system prompt
        {"name": "share_step", "kind": "share", "heads": "grouped", "seqs": 64, "groups": 1, "tokens": 1, "prefix": 4096, "context": 200, "page": 64,
         "pages": "16", "dtype": "bfloat16"},
        # three prompts with their requests, 8-bit pages
        {"name": "share_step_groups", "kind": "share", "heads": "grouped", "seqs": 48, "groups": 3, "tokens": 1, "prefix": 2500, "context": 300, "page": 64,
         "pages": "int8", "dtype": "bfloat16"},
        # questions of some tens of tokens about one long document
        {"name": "share_questions", "kind": "share", "heads": "llama", "seqs": 16, "groups": 1, "tokens": 40, "prefix": 8000, "context": 0, "page": 64,
         "pages": "16", "dtype": "bfloat16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["write", "attend", "attend", "share", "share"])
    heads = rng.choice(sorted(HEADS))
    hq, hkv, d = HEADS[heads][:3]
    case = {"kind": kind, "heads": heads, "page": rng.choice([16, 32, 64, 64]), "dtype": rng.choice(["bfloat16", "bfloat16", "float16"])}
    case["pages"] = rng.choice(["int8", "fp8"])
    if kind == "write":
        if rng.random() < 0.5:
            case.update(seqs=_log(rng, 1, 64), tokens=1, context=_log(rng, 16, 1000))
            if hkv > 1:
                case["pages"] = "fp8"       # these come back as they lie; turning a large cache of integers into numbers would cost more than the write
        else:
            seqs = _log(rng, 1, 8)
            case.update(seqs=seqs, tokens=_log(rng, 16, 8192 // seqs * 4096 // (hq * d) // 2), context=0, pages="fp8")
        return case
    most = 24000 * 8 * 1024 // (hkv * d)          # cached tokens of all sequences
    if kind == "attend":
        if rng.random() < 0.6:
            seqs = _log(rng, 1, 64)
            case.update(seqs=seqs, tokens=1, context=_log(rng, 16, min(32768, most // seqs // 2)))
        else:
            seqs = _log(rng, 1, 8)
            tokens = _log(rng, 2, min(2500, 2500 * 4096 // (hq * d)) // seqs)
            case.update(seqs=seqs, tokens=tokens, context=_log(rng, 1, 1800))
        return case
    if rng.random() < 0.5:
        case["pages"] = "16"
    seqs = _log(rng, 2, 64)
    tokens = 1 if rng.random() < 0.7 else _log(rng, 2, max(2, 600 // seqs))
    case.update(seqs=seqs, groups=rng.randint(1, min(3, seqs // 2)), tokens=tokens, prefix=_log(rng, 64, min(8000, max(65, most // seqs - 600))),
                context=_log(rng, 1, 400))
    return case


# ----------------------------------------------------------------------------- lengths and pages of a case
def _spread(mean, n):
    """n unequal lengths between half and one and a half times the mean (a function of the case alone, so its work is known)."""
    if mean <= 1:
        return [mean] * n
    return [max(1, round(mean * (0.5 + ((7 * i + 3) % n + 0.5) / n))) for i in range(n)]


def _lengths(case):
    """(new tokens, cached tokens before them, shared tokens at the front, group) of every sequence."""
    n, groups = case["seqs"], case.get("groups", 0)
    new, ctx = _spread(case["tokens"], n), _spread(case["context"], n)
    if not groups:
        return [(a, c, 0, 0) for a, c in zip(new, ctx)]
    group = [i * groups // n for i in range(n)]
    pre = [p // case["page"] * case["page"] for p in _spread(case["prefix"], groups)]       # whole pages are shared
    return [(a, c + pre[g], pre[g], g) for a, c, g in zip(new, ctx, group)]


def _layout(case, seed):
    """Block tables (scattered pages, the first ones shared by a group), lengths and offsets as the engine hands them over."""
    page, lens = case["page"], _lengths(case)
    rng = random.Random(seed)
    need = [-(-(a + c) // page) - p // page for a, c, p, _ in lens]
    shared = {g: p // page for _, _, p, g in lens} if case.get("groups") else {}
    blocks = 1 + sum(need) + sum(shared.values())
    ids = list(range(1, blocks))
    rng.shuffle(ids)
    front, at = {}, 0
    for g, k in sorted(shared.items()):
        front[g] = ids[at:at + k]
        at += k
    tables = []
    for (_, _, _, g), k in zip(lens, need):
        tables.append(front.get(g, []) + ids[at:at + k])
        at += k
    width = max(len(t) for t in tables)

    def ints(v):
        return torch.tensor(v, dtype=torch.int32).cuda()

    cu, pos, slots = [0], [], []
    for (a, c, _, _), t in zip(lens, tables):
        cu.append(cu[-1] + a)
        pos += range(c, c + a)
        slots += [t[p // page] * page + p % page for p in range(c, c + a)]
    s = {"tables": ints([t + [0] * (width - len(t)) for t in tables]), "seq_lens": ints([a + c for a, c, _, _ in lens]), "cu": ints(cu),
         "positions": ints(pos), "slots": ints(slots), "max_q": max(x[0] for x in lens), "max_kv": max(x[0] + x[1] for x in lens), "tokens": cu[-1]}
    if case.get("groups"):
        group = [x[3] for x in lens]
        first = [group.index(g) for g in sorted(shared)] + [len(lens)]
        wide = max(shared.values())
        s.update(first=ints(first), front=ints([front[g] + [0] * (wide - len(front[g])) for g in sorted(shared)]),
                 front_lens=ints([shared[g] * page for g in sorted(shared)]), max_front=wide * page,
                 max_rows=max(cu[b] - cu[a] for a, b in zip(first, first[1:])))
    return s, blocks


def _pages(gen, blocks, hkv, page, d, kind, dtype, channels):
    """Pages as a layer leaves them: keys with some strong channels, values without."""
    x = torch.randn(blocks, hkv, page, d, generator=gen, device="cuda", dtype=F32)
    if channels:
        x *= torch.exp(0.5 * torch.randn(hkv, 1, d, generator=gen, device="cuda"))
    if kind == "16":
        return x.to(dtype), None
    scale = x.abs().amax(-1) / QMAX[kind]
    x /= scale[..., None]
    return (x.round_().to(torch.int8) if kind == "int8" else x.to(torch.float8_e4m3fn)), scale


def prepare(case, seed):
    hq, hkv, d, _, _ = HEADS[case["heads"]]
    dt = DTYPES[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    s, blocks = _layout(case, seed)
    s.update(case=dict(case), blocks=blocks)
    T = s["tokens"]
    if case["kind"] == "write":
        s["qkv"] = torch.randn(T, (hq + 2 * hkv) * d, generator=gen, device="cuda", dtype=F32).to(dt)
        pt = PAGE_TYPES[case["pages"]]
        for n in ("k", "v"):
            s[n] = torch.zeros(blocks, hkv, case["page"], d, device="cuda", dtype=F32).to(pt)
            s[n + "_scale"] = torch.zeros(blocks, hkv, case["page"], device="cuda", dtype=F32)
        return s
    s["q"] = torch.randn(T, hq * d, generator=gen, device="cuda", dtype=F32).to(dt)
    for n in ("k", "v"):
        s[n], s[n + "_scale"] = _pages(gen, blocks, hkv, case["page"], d, case["pages"], dt, n == "k")
    return s


# ----------------------------------------------------------------------------- the plain forms
def _rotate(x, positions, rotary, style, to):
    """x [T, heads, d] with its first ``rotary`` columns turned by position * BASE^(-2 i / rotary); angles in 64 bits."""
    if style == "none":
        return x
    inv = BASE ** (-torch.arange(0, rotary, 2, device=x.device, dtype=F64) / rotary)
    ang = positions.to(F64)[:, None] * inv
    cos, sin = ang.cos().to(to)[:, None], ang.sin().to(to)[:, None]
    y = x.clone()
    if style == "pairs":
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        y[..., 0:rotary:2], y[..., 1:rotary:2] = a * cos - b * sin, b * cos + a * sin
    else:
        a, b = x[..., :rotary // 2], x[..., rotary // 2:rotary]
        y[..., :rotary // 2], y[..., rotary // 2:rotary] = a * cos - b * sin, b * cos + a * sin
    return y


def _write_plain(s):
    hq, hkv, d, rotary, style = HEADS[s["case"]["heads"]]
    kind, page, T = s["case"]["pages"], s["case"]["page"], s["tokens"]
    q, k, v = (x.reshape(T, -1, d).float() for x in s["qkv"].split([hq * d, hkv * d, hkv * d], 1))
    if style != "none":
        s["qkv"][:, :hq * d] = _rotate(q, s["positions"], rotary, style, F32).reshape(T, hq * d).to(s["qkv"].dtype)
        k = _rotate(k, s["positions"], rotary, style, F32)
    at = s["slots"].long()
    block, offset = at // page, at % page
    for n, x in (("k", k), ("v", v)):
        scale = x.abs().amax(-1) / QMAX[kind]
        y = torch.where(scale[..., None] > 0, x / scale[..., None], 0.0)
        codes = y.round().to(torch.int8) if kind == "int8" else y.to(torch.float8_e4m3fn)
        s[n].view(torch.int8)[block, :, offset] = codes.view(torch.int8)
        s[n + "_scale"][block, :, offset] = scale


def _gathered(s, n):
    """Keys or values of every sequence as numbers, [B, heads, tokens of all its table's pages, d]."""
    t = s["tables"].long()
    x = s[n][t].float()
    if s[n + "_scale"] is not None:
        x = x * s[n + "_scale"][t][..., None]
    B, nb, hkv, page, d = x.shape
    return x.transpose(1, 2).reshape(B, hkv, nb * page, d)


def _attend_plain(s):
    hq, hkv, d, _, _ = HEADS[s["case"]["heads"]]
    T, cu, mq = s["tokens"], s["cu"].long(), s["max_q"]
    k, v = _gathered(s, "k"), _gathered(s, "v")
    B, L = k.shape[0], k.shape[2]
    new = cu[1:] - cu[:-1]
    row = torch.arange(mq, device="cuda")
    at = (cu[:-1, None] + row).clamp_(max=T - 1)                                       # [B, mq]; rows behind a sequence's last go nowhere
    pos = (s["seq_lens"].long() - new)[:, None] + row
    q = s["q"].view(T, hkv, hq // hkv, d).float()[at].permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    scores = (q @ k.transpose(-1, -2)).view(B, hkv, hq // hkv, mq, L) * d ** -0.5
    scores = scores.masked_fill_((torch.arange(L, device="cuda") > pos[:, :, None])[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(B, hkv, -1, L) @ v).view(B, hkv, hq // hkv, mq, d).permute(0, 3, 1, 2, 4).reshape(B, mq, hq * d)
    return o[row < new[:, None]].to(s["q"].dtype)                                      # packed again


# ----------------------------------------------------------------------------- the framework's calls
def _batch(s):
    from llmss_b200.engine.batch import BatchInput, SharedPrefix

    batch = BatchInput(tokens=s["positions"], positions=s["positions"], slot_mapping=s["slots"], block_tables=s["tables"], seq_lens=s["seq_lens"],
                       cu_q=s["cu"], last_idx=s["cu"], num_seqs=s["seq_lens"].numel(), max_q=s["max_q"], max_kv=s["max_kv"],
                       is_decode=s["max_q"] == 1, is_fresh_prefill=False)
    if "first" in s:
        batch.prefix = SharedPrefix(block_tables=s["front"], lens=s["front_lens"], first=s["first"], num_groups=s["front_lens"].numel(),
                                    max_len=s["max_front"], max_rows=s["max_rows"])
    return batch


def _own_pages(s):
    from llmss_b200 import ops

    if s["k_scale"] is None:
        return s["k"], s["v"]
    return ops.QuantPages(s["k"], s["k_scale"]), ops.QuantPages(s["v"], s["v_scale"])


def _write_own(s):
    from llmss_b200 import ops

    hq, hkv, d, rotary, style = HEADS[s["case"]["heads"]]
    k, v = _own_pages(s)
    ops.rope_kv_write(s["qkv"], s["positions"], s["slots"], k, v, hq, hkv, d, rotary,
                      {"none": ops.ROPE_NONE, "pairs": ops.ROPE_GPTJ, "halves": ops.ROPE_NEOX}[style], BASE, 0, hq * d, (hq + hkv) * d)


def _attend_own(s):
    from llmss_b200 import ops

    hq, hkv, d, _, _ = HEADS[s["case"]["heads"]]
    k, v = _own_pages(s)
    out = torch.empty_like(s["q"])
    return ops.attention(s["q"], out, _batch(s), k, v, hq, hkv, d, d ** -0.5, 0, 0, 0)


def _written(s):
    """Rotated queries and the cache.  8-bit integers come back as numbers, beside the scales that they are multiples of."""
    hq, _, d, _, _ = HEADS[s["case"]["heads"]]
    k, v = (s[n].to(torch.float16) if s[n].dtype == torch.int8 else s[n] for n in ("k", "v"))
    return {"q": s["qkv"][:, :hq * d], "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def run(state):
    if state["case"]["kind"] == "write":
        if own:
            _write_own(state)
        else:
            _write_plain(state)
        return _written(state)
    return _attend_own(state) if own else _attend_plain(state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    hq, hkv, d, _, style = HEADS[case["heads"]]
    lens = _lengths(case)
    T = sum(x[0] for x in lens)
    if case["kind"] == "write":
        turned = 0 if style == "none" else 2 * 2 * T * hq * d
        return {"bytes": turned + 2 * 2 * T * hkv * d + 2 * T * hkv * (d + 4) + 8 * T, "flops": T * (hq + 2 * hkv) * d * 4}
    row = 2 * hkv * (2 * d if case["pages"] == "16" else d + 4)
    fronts = {g: p for _, _, p, g in lens} if case.get("groups") else {}
    cached = sum(a + c - p for a, c, p, _ in lens) + sum(fronts.values())
    pairs = sum(a * c + a * (a + 1) // 2 for a, c, _, _ in lens)
    return {"bytes": row * cached + 2 * 2 * T * hq * d, "flops": 4 * pairs * hq * d}


# ----------------------------------------------------------------------------- the same from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, d, rotary, style = HEADS[case["heads"]]
    lens, page = _lengths(case), case["page"]
    if case["kind"] == "write":
        x = s["qkv"].double().view(-1, hq + 2 * hkv, d)
        pos = torch.cat([torch.arange(c, c + a, dtype=F64, device="cuda") for a, c, _, _ in lens])
        if style != "none":
            # a turn by an angle is a product with e^(i angle)
            ang = pos[:, None] * torch.exp(torch.arange(rotary // 2, dtype=F64, device="cuda") * (-2 * math.log(BASE) / rotary))
            w = torch.polar(torch.ones_like(ang), ang)[:, None]
            h = x[:, :hq + hkv, :rotary]
            h = h.reshape(*h.shape[:2], -1, 2) if style == "pairs" else h.reshape(*h.shape[:2], 2, -1).transpose(2, 3)
            z = torch.view_as_real(torch.view_as_complex(h.contiguous()) * w)
            x = x.clone()
            x[:, :hq + hkv, :rotary] = (z if style == "pairs" else z.transpose(2, 3)).reshape(*z.shape[:2], rotary)
        got = {"q": x[:, :hq].reshape(-1, hq * d)}
        at = s["slots"].long()
        for n, rows in (("k", x[:, hq:hq + hkv]), ("v", x[:, hq + hkv:])):
            scale = rows.abs().amax(-1) / QMAX[case["pages"]]
            full = torch.zeros(s["blocks"] * page, hkv, dtype=F64, device="cuda")
            full[at] = scale
            got[n + "_scale"] = full.view(s["blocks"], page, hkv).transpose(1, 2)
            got[n] = None                                                              # codes have no value apart from their rounding
        return got
    out = []
    for i, (a, c, _, _) in enumerate(lens):
        ids = s["tables"][i, :-(-(a + c) // page)].long()
        k, v = ((s[n][ids].double() if s[n + "_scale"] is None else s[n][ids].double() * s[n + "_scale"][ids].double()[..., None])
                .transpose(0, 1).reshape(hkv, -1, d)[:, :a + c] for n in ("k", "v"))
        at = int(s["cu"][i])
        q = s["q"][at:at + a].double().view(a, hkv, -1, d)
        seen = torch.arange(a + c, device="cuda") <= torch.arange(c, c + a, device="cuda")[:, None]
        heads = []
        for h in range(hkv):
            z = torch.einsum("qgd,kd->gqk", q[:, h], k[h]) / math.sqrt(d)
            heads.append(torch.einsum("gqk,kd->qgd", torch.softmax(z.masked_fill(~seen, -math.inf), -1), v[h]))
        out.append(torch.stack(heads, 1).reshape(a, hq * d))
    return torch.cat(out)
