"""CPU oracle for MXFP4 KV pools and device-built step metadata — TEST INFRASTRUCTURE.

* :func:`quantise`, :func:`values` — OCP MX e2m1 codes with e8m0 scales: the
  scale of a group of 32 is the smallest 2^e with max |x| < 7 * 2^e, e held to
  the row type's range; codes are nearest, ties to even, saturating at 6; a
  group with a NaN has scale byte 255 and codes 0.
* :func:`attend` — softmax attention of one sequence in float64, with a bound
  on what a kernel that rounds P and its output to 16 bits may be off.
* :func:`batch_metadata` — a step's metadata, request by request.

The reference engine has none of these formats; parity is pinned by the
definitions alone, in float64 and Python integers.
"""

from __future__ import annotations

import math

import torch

GROUP = 32
GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
# Exponents of the scales a store may write.
RANGE = {torch.bfloat16: (-125, 125), torch.float16: (-23, 13)}


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., D] 16-bit rows to (codes [..., D/2], scales [..., D/32]), bytes."""
    lo, hi = RANGE[x.dtype]
    g = x.double().unflatten(-1, (-1, GROUP))
    nan = g.isnan().any(-1)
    top = g.abs().nan_to_num(nan=0.0, posinf=math.inf).amax(-1)
    # smallest e with top < 7 * 2^e
    m, e = torch.frexp(torch.where(top.isinf(), torch.full_like(top, 2.0 ** 200), top))
    e = torch.where(top == 0, torch.full_like(e, lo), e - 3 + (m >= 0.875).int()).clamp(lo, hi)
    y = g / torch.exp2(e.double()).unsqueeze(-1)
    a = y.abs().clamp(max=6.0)
    grid = torch.tensor(GRID, dtype=torch.float64)
    d = (a.unsqueeze(-1) - grid).abs()
    best = d.amin(-1, keepdim=True)
    hit = d == best  # two hits on a tie: the even code
    even = torch.arange(8) % 2 == 0
    code = torch.where(hit.sum(-1) > 1, (hit & even).int().argmax(-1), hit.int().argmax(-1))
    code = code + 8 * torch.signbit(g).long()
    code = torch.where(nan.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    scale = torch.where(nan, torch.full_like(e, 255), e + 127)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), scale.to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The float64 rows that (codes, scales) stand for."""
    c = torch.stack((codes % 16, codes // 16), -1).flatten(-2).long()
    v = torch.tensor(GRID + [-x for x in GRID], dtype=torch.float64)[c]
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales == 255, torch.full_like(s, math.nan), s)
    return v * s.repeat_interleave(GROUP, -1)


def rows_at(pool: torch.Tensor, slots: torch.Tensor, block: int, layout: str) -> torch.Tensor:
    """Rows [n, Hkv, w] of a byte pool at slots [n]."""
    return pool[slots // block, slots % block] if layout == "nhd" else pool[slots // block, :, slots % block]


def put_rows(pool, slots, rows, block, layout) -> None:
    for s, r in zip(slots.tolist(), rows):
        if 0 <= s < pool.shape[0] * block:
            if layout == "nhd":
                pool[s // block, s % block] = r
            else:
                pool[s // block, :, s % block] = r


def store(key, value, pool, slots, block, layout) -> None:
    """Quantise rows into pool = (kc, vc, ks, vs) byte tensors, in place."""
    for x, c, s in ((key, pool[0], pool[2]), (value, pool[1], pool[3])):
        codes, scales = quantise(x)
        put_rows(c, slots, codes, block, layout)
        put_rows(s, slots, scales, block, layout)


def attend(q, k, v, seen, scale: float, dtype: torch.dtype, product_bits: float):
    """q [m, Hq, D], k / v [n, Hkv, D] (float64), seen [m, n] bool: the output
    [m, Hq, D] and, elementwise, how far a kernel may be from it that

    * sums Q K^T products with an error of at most 2^-product_bits of the sum
      of their magnitudes (d in a logit after scaling: a weight is off by at
      most exp(2 d) - 1, numerator and denominator),
    * rounds each weight to `dtype` before P V, relative to a reference
      maximum that it may exceed by 2^8 (half a step, u, of each; below f16's
      normal range half its smallest step, of weights that sum to 1 or more;
      below 2^-126 a weight, or an output, may be flushed to zero),
    * sums in float32 and rounds the output once (u |out|).
    """
    u = torch.finfo(dtype).eps / 2
    rep = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    live = seen.any(0)  # what no query sees enters nothing, whatever it holds
    k = torch.where(live[:, None, None], k, torch.zeros_like(k))
    v = torch.where(live[:, None, None], v, torch.zeros_like(v))
    qh, kh, vh = q.double().permute(1, 0, 2), k.permute(1, 0, 2), v.permute(1, 0, 2)
    x = (qh @ kh.transpose(1, 2)) * scale
    d = (qh.abs() @ kh.abs().transpose(1, 2)) * scale * 2.0 ** -product_bits
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(nan=0.0) if not x.isnan().any() else torch.softmax(x, -1)
    p = torch.where(seen.any(-1)[None, :, None], p, torch.zeros_like(p))
    out = p @ vh
    d = d.masked_fill(~seen, 0.0).amax(-1, keepdim=True)
    mass = p @ vh.abs()
    tol = u * out.abs() + (u + torch.expm1(2 * d) + 2.0 ** -16) * mass
    tol = tol + 2.0 ** -126 * (seen.double() @ vh.abs()) + 2.0 ** -126
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 * (seen.double() @ vh.abs()) + 2.0 ** -25
    return out.permute(1, 0, 2), tol.permute(1, 0, 2)


def batch_metadata(lens, done, tables, block, *, max_tokens, rows=None, padded=0, width=None,
                   free=None, count=None, cut=False):
    """Plain integers: dict of lists, and the request tables as they become."""
    tables = [list(t) for t in tables]
    wide = len(tables[0]) if tables else 0
    width = wide if width is None else width
    rows = list(range(len(lens))) if rows is None else rows
    taken = missing = 0
    pos, slots, new, ctx, out = [], [], [], [], []
    for n, c, r in zip(lens, done, rows):
        n = max(0, n)
        c = min(max(0, c), n)
        here = 0 <= r < len(tables)
        cols = min(-(-n // block), wide)
        held = min(-(-c // block), cols) if free is not None and here else cols
        row = list(tables[r][:held]) if here else [-1] * held
        for col in range(held, cols):
            at = count - 1 - taken
            taken += 1
            blk = free[at] if at >= 0 else -1
            missing += at < 0
            row.append(blk)
            tables[r][col] = blk
        for p in range(c, n):
            blk = row[p // block] if p // block < len(row) else -1
            pos.append(p)
            slots.append(blk * block + p % block if blk >= 0 else -1)
        new.append(n - c)
        ctx.append(n)
        out.append((row + [-1] * width)[:width])
    for _ in range(max(0, padded - len(lens))):
        pos.append(0)
        slots.append(-1)
        new.append(1)
        ctx.append(1)
        out.append([0] * width)
    totals = [sum(new), max(new, default=0), max(ctx, default=0), max(0, (count or 0) - taken), missing]
    cu_q, cu_k = [0], [0]
    for m, n in zip(new, ctx):
        kept = min(m, max_tokens - cu_q[-1]) if cut else m
        cu_q.append(cu_q[-1] + kept)
        cu_k.append(cu_k[-1] + n - m + kept)
    fill = max(0, max_tokens - len(pos))
    return {"positions": (pos + [0] * fill)[:max_tokens], "slots": (slots + [-1] * fill)[:max_tokens],
            "cu_q": cu_q, "cu_k": cu_k, "tables": out, "totals": totals, "request_tables": tables}
