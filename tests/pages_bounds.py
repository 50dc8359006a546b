"""Attention over cache pages in 64 bits with the roundings of the 16-bit operands counted one by one: what a result may be off by."""
import torch

from llmss_b200.ops.pages import QuantPages
from pages_oracle import values64

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}          # relative


def sequences(q, k, v, batch, seen, hq, hkv, d, scale):
    """Of every sequence: its first row, scores [hkv, group, rows, keys] (minus infinity where hidden), queries, keys and values, all in 64 bits."""
    keys, values, at = values64(k), values64(v), 0
    for i, (a, L) in enumerate(zip(seen.new, batch.seq_lens.tolist())):
        j, n = seen.front_of.get(i, (0, 0))
        block = torch.tensor([(seen.fronts[j] if p < n else seen.tables[i])[p // seen.page] for p in range(L)], dtype=torch.long, device=keys.device)
        off = torch.arange(L, device=keys.device) % seen.page
        kk, vv = (x[block, :, off].transpose(0, 1) for x in (keys, values))                        # [hkv, L, d]
        rows = q[at:at + a].double().view(a, hkv, hq // hkv, d).permute(1, 2, 0, 3)                # [hkv, group, a, d]
        z = (rows @ kk[:, None].transpose(-1, -2)) * scale
        z = z.masked_fill(torch.arange(L, device=keys.device) > torch.arange(L - a, L, device=keys.device)[:, None], float("-inf"))
        yield at, z, rows, kk, vv
        at += a


def expected(q, k, v, batch, seen, hq, hkv, d, scale):
    """(result, how far an output may be off, results with 16 keys left out that weigh most), each [rows, hq * d] in 64 bits.

    Operands that are rounded to 16 bits on the way are each off by at most half a step, independently of one another, so that what they add to a sum
    is within six times the root of the sum of their squares.  16-bit pages: the probabilities (queries and keys are multiplied as they are).  8-bit
    pages: probabilities, values and keys in f16 (2^-11); a key's moves its score by the root of the sum of (q_i k_i)^2 of 2^-11.  Queries are f16 too:
    exact but for what is 2^-14 of a row's largest and smaller.  Not random: 2^-12 of sum p |v| for the exponential (1.1e-4) and 32-bit sums, 2^-17 of the
    largest sum |q| |k| for scores; below f16's normal numbers 2^-32 per probability and 2^-24 of the largest value.  int8 codes may be multiplied as
    code + 128, up to 2.01 times the largest value, and 128 times the sum taken off: sixteen 32-bit roundings of 2^-24 of that are 2^-19 of the largest
    value."""
    quantised, dtype = isinstance(k, QuantPages), q.dtype
    u = 2.0 ** -11 if quantised else HALF_STEP[dtype]
    rows_of = lambda x: x.permute(2, 0, 1, 3).reshape(x.shape[2], hq * d)
    want, tol, less = [], [], []
    for _, z, rows, kk, vv in sequences(q, k, v, batch, seen, hq, hkv, d, scale):
        a, L = z.shape[2:]
        hidden = z == float("-inf")
        p = torch.nan_to_num(torch.softmax(z, -1)) if L else z                                     # rows without a key: zeros
        vv, kk = vv[:, None], kk[:, None]
        out = p @ vv
        w2 = torch.full_like(p, u * u)
        if quantised:
            w2 = w2 + u * u + (2.0 ** -11 * scale) ** 2 * (rows ** 2 @ (kk ** 2).transpose(-1, -2))
        w2 = p * p * w2
        spread = 6 * torch.sqrt(w2 @ (vv * vv) + w2.sum(-1, keepdim=True) * out * out)
        big = ((rows.abs() @ kk.abs().transpose(-1, -2)) * scale).masked_fill(hidden, 0).amax(-1, keepdim=True) if L else out[..., :1]
        t = spread + (p @ vv.abs()) * (2.0 ** -12 + 2.0 ** -16 * big) + HALF_STEP[dtype] * out.abs()
        if quantised or dtype == torch.float16:
            t = t + 2.0 ** -32 * ((~hidden).double() @ vv.abs())
        if quantised and L:
            t = t + 2.0 ** -19 * vv.abs().amax((-1, -2), keepdim=True)
        if dtype == torch.float16:
            t = t + 2.0 ** -25
        want.append(rows_of(out))
        tol.append(rows_of(t))
        if L > 16:
            n = L // 16 * 16
            top = p[..., :n].unflatten(-1, (-1, 16)).sum(-1).flatten(0, 2).sum(0).argmax()
            gone = z.clone()
            gone[..., 16 * top:16 * top + 16] = float("-inf")
            less.append(rows_of(torch.nan_to_num(torch.softmax(gone, -1)) @ vv))
        else:
            less.append(torch.zeros_like(want[-1]))
    return tuple(torch.cat(x) for x in (want, tol, less))
