"""Rotary positions in every form on the GPU, against complex products in float64.

y = a cos - b sin in fp32 (two roundings), rounded once: off by at most 3 2^-24 of |a cos| + |b sin|
and half a step of the result."""

import pytest
import torch

from oracle import attention as oracle
from oracle import gradients as G
from voiceagent_amd import ops
from voiceagent_amd.layers import (AttentionContext, PagedAttention, RotaryScaling,
                                   attention_context, rotary_cos_sin_cache)

pytestmark = pytest.mark.gpu


def _table(part, max_pos=300, seed=0):
    g = torch.Generator().manual_seed(seed)
    angle = torch.rand(max_pos, part // 2, generator=g) * 100
    return torch.cat((angle.cos(), angle.sin()), -1) * 1.07  # (a scaled table's factor)


def _check(got, x, table, pos, interleaved, inverse):
    want = G.rotary(x, table, pos, interleaved, inverse)
    part = table.shape[1]
    mag = x.abs().double().clone()
    a, b = (slice(0, part, 2), slice(1, part, 2)) if interleaved else (slice(0, part // 2), slice(part // 2, part))
    mag[..., a] = mag[..., b] = 1.07 * (x[..., a].abs() + x[..., b].abs()).double()
    off = 3 * 2.0 ** -24 * mag
    off[..., part:] = 0.0
    rounded = G.HALF[x.dtype] * (want.abs() + off) + G.TINY[x.dtype]
    rounded[..., part:] = 0.0  # copied as they are
    assert ((got.double().cpu() - want).abs() <= off + rounded).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("T,hq,hkv,d,part,dtype", [
    (1, 16, 8, 128, 128, torch.bfloat16), (33, 16, 8, 128, 64, torch.float16),
    (40, 3, 1, 80, 80, torch.bfloat16), (257, 5, 2, 96, 24, torch.float32),
    (7, 2, 2, 10, 6, torch.bfloat16), (7, 3, 1, 7, 2, torch.float32), (19, 1, 1, 64, 32, torch.float32),
    (300, 14, 14, 64, 16, torch.bfloat16), (5, 33, 1, 256, 256, torch.float16)])
def test_every_form(dev, interleaved, inverse, T, hq, hkv, d, part, dtype):
    print(f"rotary T={T} {hq}/{hkv} d={d} part={part} {dtype} {interleaved} {inverse}", flush=True)
    g = torch.Generator().manual_seed(T)
    q, k = (torch.randn(T, h, d, generator=g).to(dtype) for h in (hq, hkv))
    table, pos = _table(part), torch.randint(-5, 310, (T,), generator=g)
    got = ops.rotary_embedding(q.to(dev), k.to(dev), table.to(dev), pos.to(dev),
                               interleaved=interleaved, inverse=inverse)
    _check(got[0], q, table, pos, interleaved, inverse)
    _check(got[1], k, table, pos, interleaved, inverse)


def test_halves_agree_with_the_prologues_rotation(dev):
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(50, h, 128, generator=g).to(torch.bfloat16) for h in (4, 2))
    table, pos = oracle.rope_cache(128, 64, 1e4), torch.arange(50)
    got = ops.rotary_embedding(q.to(dev), k.to(dev), table.to(dev)[:, None], pos.to(dev).int())
    want = oracle.apply_rope(q, table, pos), oracle.apply_rope(k, table, pos)
    for a, b in zip(got, want):  # (a fused product may round the other way)
        assert (a.cpu().float() - b.float()).abs().max() <= 2 ** -7 * b.abs().max()
        assert (a.cpu() == b).float().mean() > 0.999


def test_in_place_strided_and_unaligned(dev):
    g = torch.Generator().manual_seed(4)
    table, pos = _table(64), torch.randint(0, 300, (21,), generator=g)
    x = torch.randn(21, 9, 129, generator=g).to(torch.bfloat16)
    on = x.to(dev)
    q, k = on[:, :6, :128], on[:, 6:, 1:]  # rows of odd strides, an odd offset
    none, kk = ops.rotary_embedding(None, k, table.to(dev), pos.to(dev), interleaved=True)
    assert none is None
    _check(kk, x[:, 6:, 1:], table, pos, True, False)
    back = ops.rotary_embedding(q, None, table.to(dev), pos.to(dev), q_out=q)
    assert back[0] is q and back[1] is None
    _check(on[:, :6, :128], x[:, :6, :128], table, pos, False, False)
    assert torch.equal(on[:, 6:].cpu(), x[:, 6:]) and torch.equal(on[..., 128].cpu(), x[..., 128])
    # Into the columns of another buffer.
    to = torch.full((21, 20, 64), 5.0, dtype=torch.bfloat16, device=dev)
    src = x[:, :, :64].contiguous().to(dev)
    ops.rotary_embedding(src[:, :4], src[:, 4:], table.to(dev), pos.to(dev), q_out=to[:, 2:6],
                         k_out=to[:, 10:15])
    _check(to[:, 2:6], x[:, :4, :64], table, pos, False, False)
    _check(to[:, 10:15], x[:, 4:, :64], table, pos, False, False)
    assert (to[:, 6:10] == 5).all() and (to[:, 15:] == 5).all() and (to[:, :2] == 5).all()


def test_no_tokens_and_refusals(dev):
    table, pos = _table(64).to(dev), torch.zeros(8, dtype=torch.int64, device=dev)
    x = torch.zeros(8, 2, 64, dtype=torch.bfloat16, device=dev)
    assert ops.rotary_embedding(x[:0], x[:0], table, pos)[0].shape == (0, 2, 64)
    for bad in [(None, None, table, pos), (x, x[:4], table, pos), (x, x.float(), table, pos),
                (x, x[..., :32], table, pos), (x, x, table.half(), pos), (x, x, table[:, :63], pos),
                (x[..., :32], None, table, pos), (x, x, table, pos[:5]), (x, x, table, pos.float()),
                (x.transpose(1, 2), None, table, pos), (x, x, table.t(), pos)]:
        with pytest.raises(ops.AttentionArgumentError):
            ops.rotary_embedding(*bad)
    with pytest.raises(ops.AttentionArgumentError, match="q_out"):
        ops.rotary_embedding(None, x, table, pos, q_out=x)
    y = torch.zeros_like(x)
    with pytest.raises(ops.AttentionArgumentError, match="overlap the inputs"):
        ops.rotary_embedding(x, y, table, pos, q_out=y)
    with pytest.raises(ops.AttentionArgumentError, match="overlap the inputs"):
        ops.rotary_embedding(x[:4], y[:4], table, pos, q_out=x[1:5])
    with pytest.raises(ops.AttentionArgumentError, match="k_out may not overlap q_out"):
        ops.rotary_embedding(x, x, table, pos, q_out=y, k_out=y)


def test_offsets_past_32_bits(dev):
    # 300 tokens 16 MiB apart, the heads' rows side by side, into the columns behind them.
    n, step = 300, 8 << 20
    buf = torch.empty(n * step, dtype=torch.bfloat16, device=dev)
    view = lambda heads, at: buf.as_strided((n, heads, 64), (step, 64, 1), at * 64)  # noqa: E731
    g = torch.Generator().manual_seed(9)
    x = torch.randn(n, 3, 64, generator=g).to(torch.bfloat16)
    q, k, qo, ko = view(2, 0), view(1, 2), view(2, 3), view(1, 5)
    q.copy_(x[:, :2])
    k.copy_(x[:, 2:])
    table, pos = _table(64), torch.randint(0, 300, (n,), generator=g)
    ops.rotary_embedding(q, k, table.to(dev), pos.to(dev), interleaved=True, q_out=qo, k_out=ko)
    _check(qo, x[:, :2], table, pos, True, False)
    _check(ko, x[:, 2:], table, pos, True, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_autograd_is_the_transposed_rotation(dev, interleaved):
    g = torch.Generator().manual_seed(6)
    table, pos = _table(32).to(dev), torch.randint(0, 300, (30,), generator=g).to(dev)
    q, k = (torch.randn(30, h, 64, generator=g).to(dev).requires_grad_() for h in (3, 1))
    dq, dk = (torch.randn(30, h, 64, generator=g).to(dev) for h in (3, 1))
    out = ops.rotary_embedding(q, k, table, pos, interleaved=interleaved)
    torch.autograd.backward(out, (dq, dk))
    want = ops.rotary_embedding(dq, dk, table, pos, interleaved=interleaved, inverse=True)
    assert torch.equal(q.grad, want[0]) and torch.equal(k.grad, want[1])
    # By differences along a direction (fp32 rows; the rotation is linear).
    way = torch.randn_like(q)
    with torch.no_grad():
        step = ops.rotary_embedding(way, None, table, pos, interleaved=interleaved)[0]
    assert abs((step * dq).sum() - (way * q.grad).sum()) < 1e-2
    # One output used, its gradient expanded.
    q.grad = None
    ops.rotary_embedding(q, k.detach(), table, pos, interleaved=interleaved)[0].sum().backward()
    ones = ops.rotary_embedding(torch.ones_like(q), None, table, pos, interleaved=interleaved,
                                inverse=True)[0]
    assert torch.equal(q.grad, ones)


def test_the_layer_rotates_prompts_and_single_tokens(dev):
    """PagedAttention with a Rotary: a prompt into the cache, then a token, against the rotation
    and the layer without one; without a cache it trains."""
    hq, hkv, d, T = 4, 2, 128, 37
    g = torch.Generator().manual_seed(7)
    table = rotary_cos_sin_cache(d, 64, 1e4, rotary_dim=64,
                                 scaling=RotaryScaling("yarn", 4.0, original_max_position=16)).to(dev)
    assert table.shape == (64, 64)
    q, k, v = (torch.randn(T + 1, h, d, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    pos = torch.arange(T + 1, device=dev)
    slots = torch.arange(T + 1, dtype=torch.int32, device=dev)
    blocks = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev)
    cu = lambda n: torch.tensor([0, n], dtype=torch.int32, device=dev)  # noqa: E731
    outs = []
    for rotated in (False, True):
        layer = PagedAttention(hq, d, d ** -0.5, hkv)
        layer.k_cache, layer.v_cache = torch.zeros(2, 4, 16, hkv, d, dtype=torch.bfloat16, device=dev)
        got = []
        for a, b in ((0, T), (T, T + 1)):
            qq, kk = q[a:b], k[a:b]
            pro = ops.Rotary(table, pos[a:b], True)
            if rotated:
                qq, kk = ops.rotary_embedding(qq, kk, table, pos[a:b], interleaved=True)
                pro = None
            with attention_context(AttentionContext(cu(b - a), cu(b), b - a, b, slots[a:b], blocks)):
                got.append(layer(qq, kk, v[a:b], prologue=pro))
        outs.append(got + [layer.k_cache])
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    layer = PagedAttention(hq, d, d ** -0.5, hkv)
    leaf = q[:T].clone().requires_grad_()
    with attention_context(AttentionContext(cu(T), cu(T), T, T, None, None)):
        out = layer(leaf, k[:T], v[:T], prologue=ops.Rotary(table, pos[:T], True))
    out.backward(torch.ones_like(out))
    assert leaf.grad is not None and torch.isfinite(leaf.grad).all() and leaf.grad.any()
