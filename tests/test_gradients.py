"""CPU checks of the training pass: the gradient oracle against torch's autograd and against
differences, and the refusals of bad calls."""

import ctypes

import pytest
import torch

from oracle import gradients as G
from voiceagent_amd import _native as N
from voiceagent_amd import ops

F64 = torch.float64


def _attention(q, k, v, cu_q, cu_k, scale, causal):
    """The forward in float64, differentiable: queries that see no key give zeros."""
    rep = q.shape[1] // k.shape[1]
    outs = []
    for a, b, c, e in zip(cu_q[:-1], cu_q[1:], cu_k[:-1], cu_k[1:]):
        see = G.visible(b - a, e - c, causal)
        kk, vv = (x[c:e].repeat_interleave(rep, 1).transpose(0, 1) for x in (k, v))
        x = (q[a:b].transpose(0, 1) @ kk.transpose(1, 2) * scale).masked_fill(~see, -1e300)
        p = torch.softmax(x, -1) * see if e > c else x
        outs.append((p @ vv).transpose(0, 1))
    return torch.cat(outs)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("hq,hkv", [(4, 2), (3, 3), (6, 2)])
def test_oracle_attention_gradient_is_autograds_and_the_differences(causal, hq, hkv):
    g = torch.Generator().manual_seed(hq)
    lens_q, lens_k = [5, 1, 0, 9, 7], [5, 3, 2, 9, 4]
    cu = lambda x: [sum(x[:i]) for i in range(len(x) + 1)]  # noqa: E731
    cu_q, cu_k = cu(lens_q), cu(lens_k)
    make = lambda n, h: torch.randn(n, h, 16, generator=g, dtype=F64)  # noqa: E731
    q, k, v, w = make(22, hq), make(23, hkv), make(23, hkv), make(22, hq)
    for t in (q, k, v):
        t.requires_grad_()
    out = _attention(q, k, v, cu_q, cu_k, 0.25, causal)
    want = torch.autograd.grad((out * w).sum(), (q, k, v))
    plain = [t.detach() for t in (q, k, v)]
    got = G.varlen_attention_backward(w, *plain, out.detach(), cu_q, cu_k, 0.25, causal)
    for name, x in zip(("dq", "dk", "dv"), want):
        assert (got[name] - x).abs().max() < 1e-12, name
    # Along a random direction, by central differences: the step's third power is left.
    for i, name in enumerate(("dq", "dk", "dv")):
        way = torch.randn(plain[i].shape, generator=g, dtype=F64)
        at = lambda h: (_attention(*[t + h * way if j == i else t for j, t in enumerate(plain)],  # noqa: E731
                                   cu_q, cu_k, 0.25, causal) * w).sum()
        assert abs((at(1e-4) - at(-1e-4)) / 2e-4 - (got[name] * way).sum()) < 1e-5


def test_oracle_prologue_gradient_is_autograds():
    g = torch.Generator().manual_seed(0)
    x, dz = torch.randn(7, 3, 8, generator=g, dtype=F64), torch.randn(7, 3, 8, generator=g, dtype=F64)
    w = torch.randn(8, generator=g, dtype=F64).requires_grad_()
    x.requires_grad_()
    table = torch.randn(20, 8, generator=g)
    pos = torch.randint(0, 20, (7,), generator=g)
    want = torch.autograd.grad((G.norm_rope(x, w, 1e-3, table, pos) * dz).sum(), (x, w))
    dx, dw, _ = G.norm_rope_backward(dz, x.detach(), w.detach(), 1e-3, table, pos)
    assert (dx - want[0]).abs().max() < 1e-12 and (dw - want[1]).abs().max() < 1e-12


@pytest.mark.parametrize("interleaved", [True, False])
def test_oracle_rotary_inverse_is_the_transpose(interleaved):
    g = torch.Generator().manual_seed(1)
    x, y = torch.randn(5, 2, 12, generator=g, dtype=F64), torch.randn(5, 2, 12, generator=g, dtype=F64)
    table, pos = torch.randn(9, 8, generator=g), torch.tensor([0, 8, 3, 3, 1])
    fwd = G.rotary(x, table, pos, interleaved, False)
    back = G.rotary(y, table, pos, interleaved, True)
    assert abs((fwd * y).sum() - (x * back).sum()) < 1e-12
    assert torch.equal(fwd[..., 8:], x[..., 8:])
    one = torch.zeros(1, 1, 12, dtype=F64)
    one[..., 2] = 1.0  # pair (2, 3) or (2, 6), the second or third factor
    turned = G.rotary(one, table, torch.tensor([3]), interleaved, False)
    i, partner = (1, 3) if interleaved else (2, 6)
    assert turned[0, 0, 2] == table[3, i].double() and turned[0, 0, partner] == table[3, 4 + i].double()


# ---------------------------------------------------------------------------------- refusals
def _bwd_args(**over):
    a = N.new_args(N.VarlenBwdArgs)
    for name in ("q", "k", "v", "out", "dout", "dq", "dk", "dv", "cu_seqlens_q", "cu_seqlens_k",
                 "workspace"):
        setattr(a, name, 1 << 20)  # never dereferenced: every call here is refused
    a.num_seqs, a.total_q, a.total_k, a.num_heads, a.num_kv_heads, a.head_dim = 1, 8, 8, 4, 2, 64
    a.scale, a.workspace_bytes = 1.0, 4 * 8 * 4 * 3
    for name, x in over.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("over,says", [
    (dict(num_seqs=-1), "negative"), (dict(dtype=N.VA_F32), "dtype"), (dict(head_dim=96), "head_dim"),
    (dict(num_heads=5), "multiple"), (dict(num_kv_heads=0), "multiple"), (dict(q=None), "query side"),
    (dict(dv=None), "key side"), (dict(cu_seqlens_k=None), "cu_seqlens"), (dict(dq_stride_tok=4), "strides"),
    (dict(dout=(1 << 20) + 8), "aligned"), (dict(scale=0.0), "scale"),
    (dict(total_q=2 ** 31 - 1, total_k=2 ** 31 - 1, num_heads=1024, num_kv_heads=1024), "too many"),
    (dict(workspace=None), "workspace"), (dict(workspace_bytes=63), "workspace"),
])
def test_c_abi_refuses_bad_attention_gradients(over, says):
    assert N.lib().va_varlen_attention_backward(ctypes.byref(_bwd_args(**over)), None) < 0
    assert says in N.last_error()


def test_attention_gradient_without_rows_is_no_call():
    a = _bwd_args(total_q=0, total_k=0)
    assert N.lib().va_varlen_attention_backward(ctypes.byref(a), None) == 0
    a.struct_size -= 8
    assert N.lib().va_varlen_attention_backward(ctypes.byref(a), None) == N.lib().va_varlen_attention_backward(None, None) == -1
    assert N.lib().va_varlen_attention_backward_workspace_bytes(ctypes.byref(a)) == 0
    a = _bwd_args()
    size = N.lib().va_varlen_attention_backward_workspace_bytes
    assert size(ctypes.byref(a)) == 2 * 4 * 8 * 4
    a.dtype = N.VA_F16
    assert size(ctypes.byref(a)) == 3 * 4 * 8 * 4


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ops.AttentionArgumentError, match="GPU"):
        ops.varlen_attention_backward(x, x, x, x, x, cu, cu, 4, 4, scale=1.0, causal=True)


def test_overlap_is_seen():
    x = torch.zeros(4, 6, 8)
    assert not ops._apart(x[:, :2], x[:, 2:])  # views of one buffer's rows: within one another
    assert ops._apart(x[:2], x[2:]) and not ops._apart(x[:3], x[2:])
    assert ops._apart(x[:0], x) and ops._apart(torch.zeros(3), x)
