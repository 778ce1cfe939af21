"""CPU oracle for the training pass's operators: gradients of varlen attention and of the q/k
prologue, and rotary positions in every form.  TEST INFRASTRUCTURE, NOT PRODUCT CODE.

Only ``tests/`` may import this module.  Written from the definitions in float64, one sequence and
query head at a time.  :func:`varlen_attention_backward` also gives, per element, how far a result
may be that rounds P and dS to the element type before the last products and sums in fp32.
"""

from __future__ import annotations

import math

import torch

F64 = torch.float64
#: Half a step of a type, relative to the value, and half a step below its normal numbers.
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, F64: 0.0}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150, F64: 0.0}
FP32 = 2.0 ** -24


def visible(m: int, n: int, causal: bool) -> torch.Tensor:
    """Which of n keys each of m queries sees; causal: aligned at the sequences' ends."""
    if not causal:
        return torch.ones(m, n, dtype=torch.bool)
    return torch.arange(n)[None, :] <= torch.arange(m)[:, None] + (n - m)


def varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, scale, causal):
    """{"dq", "dk", "dv"} in float64, and the same names with "_off": the largest allowed error.

    The terms of the bounds, with u half a step of the type, d = head_dim and sums of n terms in
    fp32 off by at most n 2^-24 of the sum of magnitudes:
    * S is off by (d + 8) 2^-24 sum |q||k| scale (product, scale, exponent's argument), P by twice
      that, relative (its own and the sum's), and 2^-20 for the exponential, the logarithm and the
      division;
    * dP - delta by (d + 8) 2^-24 (sum |dout||v| + sum |dout||out|);
    * P and dS are rounded: u of each; in f16, where they are scaled by powers of two that keep the
      row's (the sequences') largest |dout|, or 2^-14 of its largest |dP - delta| if that is more, in
      [1, 2) and P's unit at 2^14, also by half a step of the subnormals;
    * the last sums by (rows + 8) 2^-24 of their magnitudes, and u of the result.
    """
    u, tiny = HALF[q.dtype], TINY[q.dtype]
    f16 = q.dtype == torch.float16
    got = {n: torch.zeros(x.shape, dtype=F64) for n, x in (("dq", q), ("dk", k), ("dv", v))}
    off = {n: torch.zeros_like(x) for n, x in got.items()}
    group, d = q.shape[1] // k.shape[1], q.shape[2]
    for s in range(len(cu_q) - 1):
        a, b, c, e = int(cu_q[s]), int(cu_q[s + 1]), int(cu_k[s]), int(cu_k[s + 1])
        if b <= a or e <= c:
            continue
        see = visible(b - a, e - c, causal)
        some = see.any(1, keepdim=True)
        for kv in range(k.shape[1]):
            heads = range(kv * group, (kv + 1) * group)
            kk, vv = k[c:e, kv].to(F64), v[c:e, kv].to(F64)
            tops = {}
            for h in heads:
                do, oo = dout[a:b, h].to(F64), out[a:b, h].to(F64)
                dp = (do @ vv.T - (do * oo).sum(-1, keepdim=True)) * see
                tops[h] = torch.maximum(do.abs().amax(1, keepdim=True),
                                        dp.abs().amax(1, keepdim=True) * 2.0 ** -14)
            top_all = max(float(t.max()) for t in tops.values())
            for h in heads:
                qq, do, oo = (x[a:b, h].to(F64) for x in (q, dout, out))
                x = (qq @ kk.T * scale).masked_fill(~see, -math.inf)
                x = torch.where(some, x, torch.zeros_like(x))
                p = torch.where(some & see, torch.softmax(x, -1), torch.zeros_like(x))
                dp = do @ vv.T - (do * oo).sum(-1, keepdim=True)
                ds = p * dp
                got["dq"][a:b, h] = scale * (ds @ kk)
                got["dk"][c:e, kv] += scale * (ds.T @ qq)
                got["dv"][c:e, kv] += p.T @ do
                rel = (qq.abs() @ kk.abs().T * scale).masked_fill(~see, 0).amax(1, keepdim=True)
                rel = 2 * (d + 8) * FP32 * rel + 2.0 ** -20
                dp_off = (d + 8) * FP32 * (do.abs() @ vv.abs().T + (do * oo).abs().sum(-1, keepdim=True))
                ds_off = (u + rel) * ds.abs() + p * dp_off
                low = TINY[torch.float16] if f16 else 0.0
                dq_each = ds_off + low * tops[h] * see
                sums = (e - c + 8) * FP32
                off["dq"][a:b, h] = scale * ((dq_each + sums * ds.abs()) @ kk.abs())
                sums = (b - a + 8) * group * FP32
                off["dk"][c:e, kv] += scale * ((ds_off + low * top_all * see + sums * ds.abs()).T @ qq.abs())
                pv_off = (u + rel + sums) * p + low * 2.0 ** -14 * see
                off["dv"][c:e, kv] += pv_off.T @ do.abs()
    for n in got:
        off[n] += (u + 2.0 ** -20) * (got[n].abs() + off[n]) + tiny
    return got | {n + "_off": x for n, x in off.items()}


def rotary(x, table, positions, interleaved: bool, inverse: bool):
    """The first table.shape[1] elements of every head of x [T, H, D] rotated, float64: pairs
    (2 i, 2 i + 1) or (i, i + r / 2) as complex numbers times cos + i sin (its conjugate)."""
    part = table.shape[1]
    rows = table[positions.long().clamp(0, table.shape[0] - 1)].to(F64)
    turn = torch.complex(rows[:, :part // 2].contiguous(), rows[:, part // 2:].contiguous())[:, None]
    turn = turn.conj() if inverse else turn
    x = x.to(F64)
    a, b = (x[..., 0:part:2], x[..., 1:part:2]) if interleaved else (x[..., :part // 2], x[..., part // 2:part])
    z = torch.complex(a.contiguous(), b.contiguous()) * turn
    y = x.clone()
    if interleaved:
        y[..., 0:part:2], y[..., 1:part:2] = z.real, z.imag
    else:
        y[..., :part // 2], y[..., part // 2:part] = z.real, z.imag
    return y


def norm_rope(x, weight, eps: float, table, positions):
    """RMS norm, weight and half-split rotation of x [T, H, D] without a rounding, float64."""
    x = x.to(F64)
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    return rotary(n * weight.to(F64), table, positions, False, False)


def norm_rope_backward(dz, x, weight, eps: float, table, positions):
    """(dx, dweight) of :func:`norm_rope` in float64, and the sum over rows of |dweight|'s terms."""
    dy = rotary(dz, table, positions, False, True)
    x, w = x.to(F64), weight.to(F64)
    size = (x.square().mean(-1, keepdim=True) + eps).sqrt()
    n, g = x / size, dy * w
    dx = (g - n * (g * n).mean(-1, keepdim=True)) / size
    return dx, (dy * n).sum((0, 1)), (dy * n).abs().sum((0, 1))
