"""Plain implementations of the 4-bit cache's operators, for the tests.

Scheduling is a loop over requests that pops and pushes a Python list.
Quantisation and attention are in float64, one request and head at a time,
from the definition; the quotients that decide a code are rounded to binary32
where the format says so (a float64 quotient of two binary32 numbers, rounded
to binary32, is the correctly rounded quotient).
"""
import math

import torch

UNIT = {torch.half: 2.0**-11, torch.bfloat16: 2.0**-8}  # of one rounding


def schedule(new_lens, lens, tables, free, count, rows, page):
    """-> dict of lists; `tables` (list of lists) and `free` are not changed."""
    tables, stack = [list(t) for t in tables], list(free[:count])
    batch, width = len(lens), len(tables[0]) if tables else 0
    out = {"lens": list(lens), "starts": [0], "slots": [-1] * rows, "positions": [0] * rows,
           "fate": [0] * batch}
    for b in range(batch):
        if new_lens[b] < 0:
            stack += tables[b][:-(-lens[b] // page)]
            out["lens"][b] = 0
    pushed = list(stack)
    dry = False
    for b in range(batch):
        new, n = max(new_lens[b], 0), lens[b]
        first = out["starts"][-1]
        out["starts"].append(first + new)
        used, wanted = -(-n // page), -(-(n + new) // page)
        if new == 0:
            continue
        if first + new > rows:
            out["fate"][b] = 3
        elif wanted > width:
            out["fate"][b] = 2
        elif wanted > used and (dry or wanted - used > len(stack)):
            out["fate"][b] = 1
            dry = True
        else:
            for i in range(used, wanted):
                tables[b][i] = stack.pop()
            out["lens"][b] = n + new
        for i in range(new):
            if first + i < rows:
                at = n + i
                out["positions"][first + i] = at
                if out["fate"][b] == 0:
                    out["slots"][first + i] = tables[b][at // page] * page + at % page
    out["free"] = (pushed + list(free[len(pushed):]))[:len(free)]
    out["free_count"] = len(stack)
    out["tables"] = tables
    return out


def quantise(x):
    """(codes, scale, offset) of rows x [..., D], as float64; a row with an
    infinity or a NaN, or whose range overflows, has a NaN scale."""
    y = x.double()
    low = y.amin(-1, keepdim=True)
    scale = ((y.amax(-1, keepdim=True) - low).float().double() / 15).float().to(x.dtype).double()
    scale = torch.where(torch.isfinite(scale) & torch.isfinite(y).all(-1, keepdim=True), scale,
                        torch.full_like(scale, math.nan))
    codes = torch.round(((y - low).float().double() / torch.where(scale > 0, scale, 1.0)).float())
    codes = torch.where(scale > 0, codes.double().clamp(0, 15), 0.0)
    return codes, scale, low


def values(x):
    """What the codes of rows x stand for, float64."""
    codes, scale, low = quantise(x)
    return codes * scale + low


def attention(q, k, v, new, window=0, scale=None):
    """One request: its last `new` tokens' q [new, H, D] over k, v [n, Hkv, D]
    (quantised here).  -> (out, bound), float64: the bound on an element's
    error if weights are rounded once to q's type and all else is 32 bits.

    The weights meet codes that act as if centred on 8: rounding one moves the
    result by a unit of its precision times at most 8 steps of its row's scale.
    Scores are sums of at most a few hundred in 32 bits, so their error times
    the scale, and with it a weight's relative error, is far below 2^-14.
    """
    n, dim, group = k.shape[0], q.shape[2], q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    if n == 0 or new == 0:
        return out, bound
    keys, vals = values(k), values(v)
    steps = quantise(v)[1]
    j = torch.arange(n, device=q.device)
    at = torch.arange(n - new, n, device=q.device)[:, None]
    seen = j <= at
    if window:
        seen &= j > at - window
    for h in range(q.shape[1]):
        s = (q[:, h].double() @ keys[:, h // group].T) * scale
        p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
        out[:, h] = p @ vals[:, h // group]
        size = p @ vals[:, h // group].abs()
        bound[:, h] = (UNIT[q.dtype] * out[:, h].abs() + 8 * UNIT[q.dtype] * (p @ steps[:, h // group])
                       + 2.0**-14 * size + 2.0**-24)
    return out, bound
