"""The layers' training pass on the GPU: gradients through every choice of launches."""

import pytest
import torch

from voiceagent_amd import ops
from voiceagent_amd.layers import AttentionContext, Qwen3AttentionCore, attention_context

pytestmark = pytest.mark.gpu


def _rows(dev, T, hq, hkv, d, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, h, d, generator=g).to(torch.bfloat16).to(dev) for h in (hq, hkv, hkv, hq)]


def test_a_gradient_of_v_alone(dev):
    """v's gradient is the same whether the layer may leave the query prologue to the launch."""
    hq, hkv, d, T = 4, 2, 128, 90
    q, k, v, dout = _rows(dev, T, hq, hkv, d, 1)
    cu = torch.tensor([0, 50, T], dtype=torch.int32, device=dev)
    core = Qwen3AttentionCore(hq, d, hkv, max_position=64).to(dev).requires_grad_(False)
    pos = torch.cat([torch.arange(50), torch.arange(40)]).to(dev)
    grads = []
    for fuse in (False, True):
        core.varlen_fuse_prologue = fuse
        leaf = v.clone().requires_grad_()
        with attention_context(AttentionContext(cu, cu, 50, 50, None, None)):
            core(pos, q, k, leaf).backward(dout)
        grads.append(leaf.grad)
    assert grads[0].any() and torch.equal(*grads)


@pytest.mark.parametrize("fuse_prologue", [True, False])
@pytest.mark.parametrize("T", [1, 20])
def test_a_bound_cache_builds_no_graph(dev, monkeypatch, fuse_prologue, T):
    """Prompts and single tokens, the prologue inside the launches or ahead of them."""
    hq, hkv, d = 4, 2, 128
    q, k, v, _ = _rows(dev, T, hq, hkv, d, 4)
    core = Qwen3AttentionCore(hq, d, hkv, max_position=64).to(dev)
    core.fuse_prologue = fuse_prologue
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    table = torch.tensor([[0, 1]], dtype=torch.int32, device=dev)
    context = AttentionContext(cu, cu, T, T, slots, table)
    monkeypatch.setattr(ops._QkNormRope, "apply", None)  # (a graph would need it)
    outs = []
    for grad in (True, False):
        core.k_cache, core.v_cache = torch.zeros(2, 4, 16, hkv, d, dtype=torch.bfloat16, device=dev)
        with torch.set_grad_enabled(grad), attention_context(context):
            outs.append(core(torch.arange(T, device=dev), q, k, v))
    assert torch.equal(*outs) and not outs[0].requires_grad


def _prologue(dev, T, d, grad=False):
    g = torch.Generator().manual_seed(9)
    w = torch.ones(d, dtype=torch.bfloat16, device=dev, requires_grad=grad)
    table = torch.rand(T, d, generator=g).to(dev)
    return ops.QKPrologue(w, w, 1e-6, table, torch.arange(T, device=dev))


def test_given_outputs_are_outside_the_graph(dev):
    """In place on rows of a graph: refused in grad mode; otherwise written, and counted."""
    T, d = 12, 64
    q, k, v, _ = _rows(dev, T, 2, 2, d, 2)
    pro, cu = _prologue(dev, T, d, grad=True), torch.tensor([0, T], dtype=torch.int32, device=dev)
    table, pos = pro.cos_sin_cache, pro.positions
    leaf = q.clone().requires_grad_()
    x = leaf * 1
    for call in (lambda: ops.rotary_embedding(x, None, table, pos, q_out=x),
                 lambda: ops.qk_norm_rope(x, k, pro, q_out=x, k_out=k),
                 lambda: ops.varlen_attention(q, k, v, cu, cu, T, T, scale=1.0, causal=True, out=x)):
        with pytest.raises(ops.AttentionArgumentError, match="requires a gradient"):
            call()
    assert x._version == 0 and torch.equal(x, q)
    # Rows outside the graph are written as before, weights that ask for a gradient or not.
    a, b = q.clone(), k.clone()
    got = ops.qk_norm_rope(a, b, pro, q_out=a, k_out=b)
    with torch.no_grad():
        want = ops.qk_norm_rope(q, k, pro)
    assert got[0] is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    assert not a.requires_grad and a._version == b._version == 1


@pytest.mark.parametrize("write", ["rotary", "prologue", "keys", "varlen", "decode", "gradient", "metadata"])
def test_saved_rows_that_are_written_over_are_seen(dev, write):
    """A call that writes where a backward pass has saved rows: the pass raises."""
    T, d = 12, 64
    q, k, v, _ = _rows(dev, T, 2, 2, d, 3)
    pro, cu = _prologue(dev, T, d), torch.tensor([0, T], dtype=torch.int32, device=dev)
    k.requires_grad_()
    if write == "metadata":
        lens = torch.tensor([T], dtype=torch.int32, device=dev)
        req = torch.zeros(1, 4, dtype=torch.int32, device=dev)
        step = lambda out: ops.batch_metadata(lens, lens * 0, req, 16, max_tokens=T, out=out)  # noqa: E731
        made = step(None)
        out = ops.rotary_embedding(None, k, pro.cos_sin_cache, made.positions)[1]
        step(made)
    else:
        out = ops.varlen_attention(q, k, v, cu, cu, T, T, scale=1.0, causal=True)
    with torch.no_grad():
        if write == "rotary":
            ops.rotary_embedding(q, None, pro.cos_sin_cache, pro.positions, q_out=q)
        elif write == "prologue":
            ops.qk_norm_rope(q, v, pro, q_out=q, k_out=v)
        elif write == "keys":
            ops.qk_norm_rope(None, v, pro, k_out=v)
        elif write == "varlen":
            ops.varlen_attention(q, k, v, cu, cu, T, T, scale=1.0, causal=True, out=q)
        elif write == "gradient":
            rows = [torch.ones_like(q) for _ in range(5)]
            ops.varlen_attention_backward(*rows, cu, cu, T, T, scale=1.0, causal=True, dv=v)
        elif write == "decode":
            pool = torch.zeros(2, T, 16, 2, d, dtype=torch.bfloat16, device=dev)
            table = torch.arange(T, dtype=torch.int32, device=dev)[:, None]
            ops.paged_decode(q, *pool, table, torch.ones(T, dtype=torch.int32, device=dev),
                             max_seq_len=1, scale=1.0, out=q)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@pytest.mark.parametrize("d,most", [(128, 40), (64, 40)])
def test_tokens_far_apart(dev, d, most):
    """Rows that the forward takes and the gradient does not as they are: q's tokens 72 MiB apart,
    k's and v's 48."""
    T = 40
    q, k, v, dout = _rows(dev, T, 2, 2, d, 5)
    cu = torch.tensor([0, 25, T], dtype=torch.int32, device=dev)
    buf = torch.empty(T * (36 << 20) + 4096, dtype=torch.bfloat16, device=dev)
    far = [buf.as_strided(t.shape, (step << 20, d, 1), at * 2 * d)
           for at, (t, step) in enumerate(((q, 36), (k, 24), (v, 24)))]
    grads = []
    for rows in ((q, k, v), [f.copy_(t) for f, t in zip(far, (q, k, v))]):
        leaves = [t.detach().requires_grad_() for t in rows]
        out = ops.varlen_attention(*leaves, cu, cu, most, most, scale=0.125, causal=True)
        grads.append(torch.autograd.grad(out, leaves, dout))
    for a, b in zip(*grads):
        assert a.any() and torch.equal(a, b)


def test_gradients_between_one_anothers_heads(dev):
    """dq, dk and dv into one buffer [tokens, heads, 3, elements], as a projection of all three has
    it, and rows rotated there in place."""
    T, h, d = 50, 3, 64
    rows = _rows(dev, T, h, h, d, 6)
    q, k, v, dout = rows
    cu = torch.tensor([0, T], dtype=torch.int32, device=dev)
    out = ops.varlen_attention(q, k, v, cu, cu, T, T, scale=0.125, causal=True)
    want = ops.varlen_attention_backward(dout, q, k, v, out, cu, cu, T, T, scale=0.125, causal=True)
    buf = torch.full((T, h, 3, d), 7.0, dtype=torch.bfloat16, device=dev)
    dq, dk, dv = (buf[:, :, i] for i in range(3))
    ops.varlen_attention_backward(dout, q, k, v, out, cu, cu, T, T, scale=0.125, causal=True, dq=dq,
                                  dk=dk, dv=dv)
    for i in range(3):
        assert torch.equal(buf[:, :, i], want[i])
    pro = _prologue(dev, T, d)
    turned = ops.rotary_embedding(*want[:2], pro.cos_sin_cache, pro.positions)
    ops.rotary_embedding(dq, dk, pro.cos_sin_cache, pro.positions, q_out=dq, k_out=dk)
    for i, t in enumerate((*turned, want[2])):
        assert torch.equal(buf[:, :, i], t)


@pytest.mark.parametrize("dtype,wdtype", [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)])
def test_the_keys_alone_through_autograd(dev, dtype, wdtype):
    """qk_norm_rope(None, k, ...): k's and its weight's gradients, either alone, are those of the
    direct call.  (With both sides the weight's terms are the same and their order another.)"""
    T, d = 33, 128
    q, k, dk = (t.to(dtype) for t in _rows(dev, T, 3, 3, d, 7)[:3])
    pro = _prologue(dev, T, d)
    w = (torch.rand(d, generator=torch.Generator().manual_seed(8)) + 0.5).to(wdtype).to(dev)
    pro = ops.QKPrologue(w, w, 1e-6, pro.cos_sin_cache, pro.positions)
    _, want, _, want_w = ops.qk_norm_rope_backward(None, dk, None, k, pro)
    assert torch.equal(want, ops.qk_norm_rope_backward(dk, dk, q, k, pro)[1])
    for ask_k, ask_w in ((True, True), (True, False), (False, True)):
        kk, ww = k.clone().requires_grad_(ask_k), w.clone().requires_grad_(ask_w)
        none, out = ops.qk_norm_rope(None, kk, ops.QKPrologue(w, ww, 1e-6, pro.cos_sin_cache, pro.positions))
        assert none is None and torch.equal(out, ops.qk_norm_rope(q, k, pro)[1])
        out.backward(dk)
        assert (kk.grad is None) == (not ask_k) and (ww.grad is None) == (not ask_w)
        assert not ask_k or torch.equal(kk.grad, want)
        assert not ask_w or torch.equal(ww.grad, want_w)
