"""Oracle of the paged 4-bit key/value cache: the definitions, in plain Python and torch on
the CPU (64-bit sums), one record and one request at a time."""
from __future__ import annotations

import math

import torch

RECORD = 16


def blocks_of(n: int, block: int) -> int:
    return -(-n // block)


def plan(ctx, new, tables, free, n_free, block, n_tokens):
    """The batch's plan from lists; ``tables`` (a list of lists) is updated.  Returns a dict of lists."""
    R, width = len(ctx), len(tables[0]) if tables else 0
    start, slots, positions, seq_lens = [0], [-1] * n_tokens, [0] * n_tokens, []
    wanted = taken = refused = end = 0
    for r in range(R):
        c, n = max(ctx[r], 0), max(new[r], 0)
        first, end = end, end + n
        have, want = blocks_of(c, block), blocks_of(c + n, block)
        fits = ctx[r] >= 0 and new[r] >= 0 and want <= width and end <= n_tokens
        need = want - have if fits else 0
        wanted += need
        granted = fits and (need == 0 or wanted <= n_free)
        if granted:
            for k in range(need):
                tables[r][have + k] = free[n_free - 1 - taken - k]
            taken += need
        else:
            refused += 1
        for j in range(n):
            if first + j < n_tokens:
                positions[first + j] = c + j
                if granted:
                    slots[first + j] = tables[r][(c + j) // block] * block + (c + j) % block
        seq_lens.append(c + n if granted else 0)
        start.append(min(end, n_tokens))
    return dict(query_start=start, positions=positions, slots=slots, seq_lens=seq_lens, n_free=[n_free - taken],
                refused=[refused])


def quantise(x: torch.Tensor, group: int):
    """(codes, scale, minimum) of rows (..., D): int codes, 16-bit scale and minimum (..., D / group).
    The scale is the next smaller number where 15 scale + minimum rounds to infinity.  A row with a
    NaN or an infinity, or whose scale overflows, has NaN parameters and codes 0."""
    g = x.float().unflatten(-1, (-1, group))
    low = g.amin(-1)
    scale = ((g.amax(-1) - low) * torch.tensor(1 / 15, dtype=torch.float32)).to(x.dtype)
    past = torch.isinf((15 * scale.double() + low.double()).float().to(x.dtype)) & torch.isfinite(scale)
    scale = torch.where(past, (scale.view(torch.int16) - 1).view(x.dtype), scale)
    bad = (~torch.isfinite(x)).any(-1, keepdim=True) | (~torch.isfinite(scale)).any(-1, keepdim=True)
    s = scale.float()[..., None]
    code = torch.where(s > 0, torch.round((g - low[..., None]) / s), torch.zeros_like(g))
    code = torch.where(bad[..., None], 0.0, code).clamp(0, 15).int().flatten(-2)
    nan = torch.full_like(scale, math.nan)
    return code, torch.where(bad, nan, scale), torch.where(bad, nan, low.to(x.dtype))


def values(code, scale, low) -> torch.Tensor:
    """What codes stand for, in 64 bits."""
    g = code.double().unflatten(-1, (scale.shape[-1], -1))
    return (g * scale.double()[..., None] + low.double()[..., None]).flatten(-2)


def code_place(kind: str, t: int, d: int, D: int):
    """(byte offset in the record, shift) of the code of token t, dim d."""
    if kind == "k":
        i, c, j, b = d // 32, d % 32 // 8, d % 8 // 2, d % 2
        return t * D // 2 + c * D // 8 + 4 * i + 2 * b + j // 2, 4 * (j % 2)
    i, g, j = d // 32, d % 32 // 4, d % 4
    h, c, b = t // 8, t % 8 // 2, t % 2
    word = ((h * 8 + g) * 4 + c) * (D // 32) + i if D == 128 else ((g * 4 + c) * 2 + h) * (D // 32) + i
    return 8 * D + 4 * word + 2 * b + j // 2, 4 * (j % 2)


def record_bytes(D: int, group: int) -> int:
    return 16 * D + 128 * (D // group)


def write_token(record: torch.Tensor, t: int, kind: str, code, scale, low) -> None:
    """Write token t's codes and parameters of one head into a record (a uint8 vector)."""
    D, NG = code.shape[0], scale.shape[0]
    for d in range(D):
        at, shift = code_place(kind, t, d, D)
        record[at] = (int(record[at]) & ~(15 << shift) & 255) | (int(code[d]) << shift)
    base = 16 * D + (64 * NG if kind == "v" else 0) + t * NG * 4
    record[base:base + 4 * NG] = torch.stack([scale, low], -1).flatten().view(torch.uint8)


def attention(q, k, v, n_new: int, scale=None, window=None):
    """One request: q (n, n_q, D), k and v (L, n_kv, D), all 64-bit; query j sits at position
    L - n + j.  Returns (out (n, n_q, D), spread): spread is sqrt(sum p^2 v^2), the size of the
    output's noise when the summands are rounded independently."""
    n, n_q, D = q.shape
    L, n_kv = k.shape[0], k.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, spread = torch.zeros(n, n_q, D, dtype=torch.float64), torch.zeros(n, n_q, D, dtype=torch.float64)
    for j in range(n):
        pos = L - n_new + j
        lo = max(0, pos - window + 1) if window else 0
        hi = min(L, pos + 1)
        if hi <= lo:
            continue
        kk = k[lo:hi].repeat_interleave(n_q // n_kv, 1)
        vv = v[lo:hi].repeat_interleave(n_q // n_kv, 1)
        p = torch.softmax(torch.einsum("hd,thd->ht", q[j], kk) * scale, -1)
        out[j] = torch.einsum("ht,thd->hd", p, vv)
        spread[j] = torch.einsum("ht,thd->hd", p.square(), vv.square()).sqrt()
    return out, spread
