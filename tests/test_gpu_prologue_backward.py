"""The gradient of the q/k prologue on the GPU, against the definition in float64.

dx is formed in fp32 from x, dz and a row's two sums of head_dim terms, and rounded once: an
element is off by at most half a step of its value and (head_dim + 24) 2^-24 of the magnitudes it
is the difference of.  A weight's gradient is a sum of n = tokens x heads fp32 terms, each of a few
roundings: n + 24 times 2^-24 of the terms' magnitudes, and half a step of the weight's type."""

import pytest
import torch

from oracle import attention as oracle
from oracle import gradients as G
from voiceagent_amd import ops
from voiceagent_amd.layers import AttentionContext, Qwen3AttentionCore, attention_context

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _inputs(T, hq, hkv, d, dtype, wdtype, seed, max_pos=500):
    g = torch.Generator().manual_seed(seed)
    make = lambda h, x=1.0: (torch.randn(T, h, d, generator=g) * x).to(dtype)  # noqa: E731
    w = lambda: (torch.rand(d, generator=g) + 0.5).to(wdtype)  # noqa: E731
    return dict(q=make(hq, 3.0), k=make(hkv, 0.2), dq=make(hq, 2.0 ** -7), dk=make(hkv), qw=w(),
                kw=w(), pos=torch.randint(-3, max_pos + 9, (T,), generator=g),
                table=oracle.rope_cache(d, max_pos, 1e4))


def _pro(c, dev, pos=None):
    return ops.QKPrologue(c["qw"].to(dev), c["kw"].to(dev), EPS, c["table"].to(dev),
                          (c["pos"] if pos is None else pos).to(dev))


def _check_side(dx, dw, dz, x, w, c):
    want, want_w, terms = G.norm_rope_backward(dz, x, w, EPS, c["table"], c["pos"])
    T, heads, d = x.shape
    xx = x.double()
    size = (xx.square().mean(-1, keepdim=True) + EPS).sqrt()
    half = c["table"][c["pos"].clamp(0, c["table"].shape[0] - 1)].double().abs()[:, None]
    cos, sin = (t.repeat(1, 1, 2) for t in half.chunk(2, -1))
    z = dz.double().abs()
    g = (z * cos + z.roll(d // 2, -1) * sin) * w.double().abs()
    n = (xx / size).abs()
    off = (d + 24) * 2.0 ** -24 * (g + n * (g * n).mean(-1, keepdim=True)) / size
    off = off + G.HALF[x.dtype] * (want.abs() + off) + G.TINY[x.dtype]
    assert ((dx.double().cpu() - want).abs() <= off).all()
    if dw is not None:
        off = (T * heads + 24) * 2.0 ** -24 * (g / w.double().abs() * n).sum((0, 1))
        off = off + G.HALF[w.dtype] * (want_w.abs() + off) + G.TINY[w.dtype]
        assert dw.dtype == w.dtype and ((dw.double().cpu() - want_w).abs() <= off).all()


@pytest.mark.parametrize("T,hq,hkv,d,dtype,wdtype", [
    (1, 1, 1, 64, torch.bfloat16, torch.bfloat16), (1, 16, 8, 128, torch.float16, torch.float32),
    (33, 16, 8, 128, torch.bfloat16, torch.bfloat16), (257, 3, 1, 256, torch.bfloat16, torch.float32),
    (65, 5, 2, 64, torch.float32, torch.float32), (40, 14, 14, 64, torch.float16, torch.float16),
    (30, 7, 3, 256, torch.float32, torch.bfloat16), (700, 2, 2, 128, torch.bfloat16, torch.bfloat16),
    (5000, 1, 1, 64, torch.bfloat16, torch.float32)])
def test_gradient_matches_the_definition(dev, T, hq, hkv, d, dtype, wdtype):
    print(f"prologue backward T={T} {hq}/{hkv} d={d} {dtype} {wdtype}", flush=True)
    c = _inputs(T, hq, hkv, d, dtype, wdtype, T)
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(*(c[n].to(dev) for n in ("dq", "dk", "q", "k")),
                                                 _pro(c, dev))
    _check_side(dq, dqw, c["dq"], c["q"], c["qw"], c)
    _check_side(dk, dkw, c["dk"], c["k"], c["kw"], c)


def test_keys_alone_in_place_and_strided(dev):
    c = _inputs(90, 4, 2, 128, torch.bfloat16, torch.bfloat16, 2)
    c["pos"] = c["pos"].int()
    qkv = torch.cat((c["q"], c["k"], c["k"]), 1).to(dev)
    dqkv = torch.cat((c["dq"], c["dk"], c["dk"]), 1).to(dev)
    q, k, _ = qkv.split([4, 2, 2], 1)
    dq, dk, _ = dqkv.split([4, 2, 2], 1)
    none, alone, no_w, w = ops.qk_norm_rope_backward(None, dk, None, k, _pro(c, dev))
    assert none is None and no_w is None
    _check_side(alone, w, c["dk"], c["k"], c["kw"], c)
    both = ops.qk_norm_rope_backward(dq, dk, q, k, _pro(c, dev), dq=dq, dk=dk)
    assert both[0] is dq and torch.equal(dk, alone) and torch.equal(both[3], w)
    _check_side(dq, both[2], c["dq"], c["q"], c["qw"], c)
    assert torch.equal(dqkv[:, 6:].cpu(), c["dk"])


def test_no_tokens(dev):
    c = _inputs(0, 4, 2, 64, torch.bfloat16, torch.bfloat16, 3)
    dq, dk, dqw, dkw = ops.qk_norm_rope_backward(*(c[n].to(dev) for n in ("dq", "dk", "q", "k")),
                                                 _pro(c, dev))
    assert dq.shape == (0, 4, 64) and dk.shape == (0, 2, 64)
    assert not dqw.any() and not dkw.any()


def test_calls_repeat_and_graphs_replay(dev):
    c = _inputs(1500, 6, 2, 128, torch.bfloat16, torch.float32, 4)
    on = [c[n].to(dev) for n in ("dq", "dk", "q", "k")]
    pro = _pro(c, dev)
    first = ops.qk_norm_rope_backward(*on, pro)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.qk_norm_rope_backward(*on, pro)
    for i in range(3):
        on[0].copy_(torch.roll(c["dq"], i, 0))
        want = ops.qk_norm_rope_backward(*on, pro)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, res))
        assert i or all(torch.equal(a, b) for a, b in zip(want, first))


def test_refusals(dev):
    c = _inputs(8, 4, 2, 64, torch.bfloat16, torch.bfloat16, 5)
    dq, dk, q, k = (c[n].to(dev) for n in ("dq", "dk", "q", "k"))
    pro = _pro(c, dev)
    for bad in [(None, dk, q, k), (dq[:4], dk, q, k), (dq, dk[:4], q, k), (dq.float(), dk, q, k),
                (dq, dk, q[:4], k), (dq, dk.transpose(1, 2), q, k)]:
        with pytest.raises(ops.AttentionArgumentError):
            ops.qk_norm_rope_backward(*bad, pro)
    with pytest.raises(ops.AttentionArgumentError, match="match"):
        ops.qk_norm_rope_backward(dq, dk, q, k, pro, dk=q)
    with pytest.raises(ops.AttentionArgumentError, match="dq may not overlap the inputs"):
        ops.qk_norm_rope_backward(dq[:, :2], dk, q[:, :2], k, pro, dq=k)
    with pytest.raises(ops.AttentionArgumentError, match="dq may not overlap the inputs"):
        ops.qk_norm_rope_backward(dq[:, :2], dk, q[:, :2], k, pro, dq=q[:, 1:3])


# ------------------------------------------------------------- the training pass of the core
@pytest.mark.parametrize("fuse", [False, True])
def test_the_core_trains(dev, fuse):
    """Prologue, attention and their gradients together, through the layer's autograd: the results
    of the operators called one by one, bit for bit, and near the definition's."""
    hq, hkv, d, lens = 4, 2, 128, [100, 37, 1, 64]
    T = sum(lens)
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(T, h, d, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv))
    dout = torch.randn(T, hq, d, generator=g).to(torch.bfloat16).to(dev)
    cu = torch.tensor([0, 100, 137, 138, 202], dtype=torch.int32, device=dev)
    pos = torch.cat([torch.arange(n) for n in lens]).to(dev)
    core = Qwen3AttentionCore(hq, d, hkv, max_position=128).to(dev)
    core.varlen_fuse_prologue = fuse
    with torch.no_grad():
        core.q_norm_weight.mul_(torch.rand(d, generator=g).to(dev) + 0.5)
    context = AttentionContext(cu, cu, 100, 100, None, None)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    with attention_context(context):
        out = core(pos, *leaves)
        with torch.no_grad():
            assert torch.equal(out, core(pos, *leaves))
    out.backward(dout)
    with torch.no_grad():
        pro = core.prologue(pos)
        qn, kn = ops.qk_norm_rope(q, k, pro)
        dqn, dkn, dv = ops.varlen_attention_backward(dout, qn, kn, v, out, cu, cu, 100, 100,
                                                     scale=core.scale, causal=True)
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(dqn, dkn, q, k, pro)
    got = (q.grad, k.grad, v.grad, core.q_norm_weight.grad, core.k_norm_weight.grad)
    assert all(torch.equal(a, b) for a, b in zip(got, (dq, dk, dv, dqw, dkw)))
    # Against float64 without any rounding between: each of the chain's 16-bit tensors (n, y, z of
    # both sides, out, dz of both) is off by at most 2^-8 of itself; together under a tenth.
    x = [t.detach().double().cpu().requires_grad_() for t in (q, k, v, core.q_norm_weight, core.k_norm_weight)]
    table = core.cos_sin_cache.cpu()
    qq, kk = (_turned(a, w, core.eps, table, pos.cpu()) for a, w in ((x[0], x[3]), (x[1], x[4])))
    outs = []
    for a, b in zip([0, 100, 137, 138], [100, 137, 138, 202]):
        s = qq[a:b].transpose(0, 1) @ kk[a:b].repeat_interleave(2, 1).permute(1, 2, 0) * core.scale
        s = s.masked_fill(~G.visible(b - a, b - a, True), -1e300)
        outs.append((torch.softmax(s, -1) @ x[2][a:b].repeat_interleave(2, 1).transpose(0, 1)).transpose(0, 1))
    torch.cat(outs).backward(dout.double().cpu())
    for a, t in zip(got, x):
        err = (a.double().cpu() - t.grad).norm() / t.grad.norm()
        assert err < 0.1, err


def _turned(x, w, eps, table, pos):
    """G.norm_rope, differentiable."""
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w
    cos, sin = table[pos.long()].double()[:, None].chunk(2, -1)
    a, b = n.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def test_a_bound_cache_has_no_gradient(dev):
    """Serving is as before: with a cache, weights that ask for a gradient build no graph."""
    hq, hkv, d = 4, 2, 128
    core = Qwen3AttentionCore(hq, d, hkv, max_position=64).to(dev)
    core.k_cache, core.v_cache = torch.zeros(2, 4, 16, hkv, d, dtype=torch.bfloat16, device=dev)
    T = 20
    q, k, v = (torch.randn(T, h, d, device=dev).to(torch.bfloat16) for h in (hq, hkv, hkv))
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
    with attention_context(AttentionContext(cu, cu, T, T, slots, table)):
        out = core(torch.arange(T, device=dev), q, k, v)
    assert not out.requires_grad
