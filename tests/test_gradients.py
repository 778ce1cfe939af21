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
    (dict(num_seqs=1 << 20, num_heads=32, num_kv_heads=32), "too many"),
    (dict(num_seqs=1 << 20, num_heads=32, num_kv_heads=32, max_seqlen_q=1, max_seqlen_k=1), "too many"),
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
    assert size(ctypes.byref(a)) == 256  # lse and delta of 8 rows of 4 heads, rounded up
    a.dtype = N.VA_F16
    assert size(ctypes.byref(a)) == 512  # and the rows' largest |dout|
    # Few blocks of keys that many queries see: their sums, a share of the queries each.
    a.total_q = a.total_k = 2000
    plain = 3 * 4 * 2000 * 4
    parts, left = divmod(size(ctypes.byref(a)) - (plain + 255) // 256 * 256, (2000 // 64 + 2) * 2 * 2 * 64 * 64 * 4)
    assert left == 0 and 2 <= parts <= 16
    a.total_k = 0
    assert size(ctypes.byref(a)) == (plain + 255) // 256 * 256
    # Short sequences with a kv head to each head take one launch and none.
    a = _bwd_args(num_kv_heads=4, max_seqlen_q=128, max_seqlen_k=5)
    assert size(ctypes.byref(a)) == 0
    for name, x in (("max_seqlen_k", 129), ("max_seqlen_q", 0), ("num_kv_heads", 2)):
        assert size(ctypes.byref(_bwd_args(**{**dict(num_kv_heads=4, max_seqlen_q=128, max_seqlen_k=5), name: x}))) > 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(ops.AttentionArgumentError, match="GPU"):
        ops.varlen_attention_backward(x, x, x, x, x, cu, cu, 4, 4, scale=1.0, causal=True)


def test_overlap_is_seen():
    x = torch.zeros(4, 6, 8)
    assert ops._apart(x[:2], x[2:]) and not ops._apart(x[:3], x[2:])
    assert ops._apart(x[:0], x) and ops._apart(torch.zeros(4, 6, 8), x)
    # Views of one buffer's rows: side by side, or sharing a head, or of other strides.
    assert ops._apart(x[:, :2], x[:, 2:]) and ops._apart(x[:, 3:], x[1:, :3])
    assert not ops._apart(x[:, :3], x[:, 2:]) and not ops._apart(x, x[:, 5:])
    assert not ops._apart(x[:, :2], x.view(8, 3, 8)[:, 2:])
    major = x.view(6, 4, 8).transpose(0, 1)  # heads far apart
    assert ops._apart(major[:2], major[2:]) and not ops._apart(major, major[:, 2:])
    # In place is the same memory, element for element, and only where it is allowed.
    assert ops._in_place(x, x[:]) and not ops._in_place(x[:3], x[1:])
    ops._outputs_apart([("a", x[:, :2], (x[:, :2],))], (x[:, 2:],))
    for given, inputs in (([("a", x[:1].expand(4, 6, 8), ())], ()), ([("a", x, ())], (x,)), ([("a", x[1:], (x[:3],))], (x[:3],)),
                          ([("a", x, ()), ("b", x, ())], ())):
        with pytest.raises(ops.AttentionArgumentError, match="overlap"):
            ops._outputs_apart(given, inputs)


def _rotary_args(**over):
    a = N.new_args(N.RotaryArgs)
    for name in ("q", "k", "q_out", "k_out", "cos_sin_cache", "positions"):
        setattr(a, name, 1 << 20)  # never dereferenced
    a.num_tokens, a.num_heads, a.num_kv_heads, a.head_dim, a.rotary_dim = 4, 2, 2, 64, 32
    a.cos_sin_stride, a.max_position = 32, 10
    for name, x in over.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("over,says", [
    (dict(num_tokens=-1), "num_tokens"), (dict(dtype=9), "dtype"), (dict(num_heads=0, num_kv_heads=0), "heads"),
    (dict(num_heads=-1), "heads"), (dict(rotary_dim=31), "rotary_dim"), (dict(rotary_dim=66), "rotary_dim"),
    (dict(rotary_dim=0), "rotary_dim"), (dict(q=None), "missing"), (dict(k_out=None), "missing"),
    (dict(positions=None), "positions"), (dict(cos_sin_stride=31), "rotary cache"),
    (dict(max_position=0), "rotary cache"), (dict(positions_dtype=2), "positions_dtype"),
    (dict(q=(1 << 20) + 1), "aligned"), (dict(num_tokens=2 ** 31 - 1), "too many"),
])
def test_c_abi_refuses_bad_rotations(over, says):
    assert N.lib().va_rotary(ctypes.byref(_rotary_args(**over)), None) == -1
    assert says in N.last_error()


def test_rotation_of_no_tokens_is_no_call():
    a = _rotary_args(num_tokens=0)
    assert N.lib().va_rotary(ctypes.byref(a), None) == 0
    a.struct_size += 4
    assert N.lib().va_rotary(ctypes.byref(a), None) == -1 and "struct_size" in N.last_error()


def _prologue_args(**over):
    a = N.new_args(N.QkNormRopeBwdArgs)
    for name in ("dq_out", "dk_out", "q", "k", "dq", "dk", "dq_weight", "dk_weight", "workspace"):
        setattr(a, name, 1 << 20)
    a.num_tokens, a.num_heads, a.num_kv_heads, a.head_dim = 4, 2, 2, 64
    pro = a.prologue
    for name in ("q_norm_weight", "k_norm_weight", "cos_sin_cache", "positions"):
        setattr(pro, name, 1 << 20)
    pro.cos_sin_stride, pro.max_position = 64, 10
    a.workspace_bytes = 1 << 30
    for name, x in over.items():
        setattr(pro if hasattr(pro, name) else a, name, x)
    return a


@pytest.mark.parametrize("over,says", [
    (dict(dtype=7), "dtype"), (dict(num_tokens=-1), "num_tokens"), (dict(head_dim=96), "head_dim"),
    (dict(num_heads=0, num_kv_heads=0), "head"), (dict(num_heads=70000), "head"), (dict(q=None), "query side"),
    (dict(dk_weight=None), "key side"), (dict(cos_sin_stride=63), "rotary cache"),
    (dict(q_norm_weight=None), "norm weights"), (dict(weight_dtype=5), "weight_dtype"),
    (dict(positions_dtype=-1), "positions_dtype"), (dict(dk_stride_tok=4), "strides"),
    (dict(dq=(1 << 20) + 4), "aligned"), (dict(workspace=None), "workspace"), (dict(workspace_bytes=8), "workspace"),
    (dict(q_norm_weight=(1 << 20) + 8), "norm weights"), (dict(num_tokens=2 ** 31 - 1, num_heads=50), "too many"),
])
def test_c_abi_refuses_bad_prologue_gradients(over, says):
    assert N.lib().va_qk_norm_rope_backward(ctypes.byref(_prologue_args(**over)), None) < 0
    assert says in N.last_error()


def test_prologue_gradient_workspace():
    size = N.lib().va_qk_norm_rope_backward_workspace_bytes
    assert size(ctypes.byref(_prologue_args(num_tokens=0))) == 0
    assert size(ctypes.byref(_prologue_args(head_dim=96))) == 0
    assert size(ctypes.byref(_prologue_args())) == 2 * 64 * 4  # one workgroup's sums
    most = size(ctypes.byref(_prologue_args(num_tokens=1 << 20)))
    assert most == 1024 * 2 * 64 * 4


def test_cpu_tensors_of_the_prologue_and_the_rotation_are_refused():
    x = torch.zeros(4, 2, 64)
    pos, table, w = torch.zeros(4, dtype=torch.int64), torch.zeros(9, 64), torch.ones(64)
    with pytest.raises(ops.AttentionArgumentError, match="GPU"):
        ops.rotary_embedding(x, x, table, pos)
    with pytest.raises(ops.AttentionArgumentError, match="GPU"):
        ops.qk_norm_rope_backward(x, x, x, x, ops.QKPrologue(w, w, 1e-6, table, pos))


# -------------------------------------------------------------------------------- the tables
def test_rotary_tables():
    import math

    from oracle import attention as oracle
    from voiceagent_amd.layers import RotaryScaling, rotary_cos_sin_cache as table

    # As before without a part or a scaling; in float64 angles with one.
    assert torch.equal(table(64, 100, 1e4), oracle.rope_cache(64, 100, 1e4))
    part = table(128, 100, 1e4, rotary_dim=64)
    assert part.shape == (100, 64) and (part - table(64, 100, 1e4)).abs().max() < 1e-4
    i, p = 5, 77
    angle = p * 1e4 ** (-2 * i / 64)
    assert abs(part[p, i] - math.cos(angle)) < 1e-7 and abs(part[p, 32 + i] - math.sin(angle)) < 1e-7
    # Linear: a position's angles are those of position / factor.
    linear = table(64, 100, 1e4, scaling=RotaryScaling("linear", 4.0))
    assert torch.equal(linear[::4], table(64, 25, 1e4, rotary_dim=64))
    # By the base: the fastest pair as it was, the slowest slower by the factor.
    base = table(64, 100, 1e4, scaling=RotaryScaling("base", 8.0))
    assert torch.equal(base[:, 0], part[:, 0])
    slow = 1e4 ** (-62 / 64) / 8
    assert abs(base[90, 31] - math.cos(90 * slow)) < 1e-7
    # By parts: pairs that turn often as they were, those that hardly turn slower, times a factor.
    yarn = table(64, 100, 1e4, scaling=RotaryScaling("yarn", 8.0, original_max_position=4096))
    factor = 0.1 * math.log(8.0) + 1
    assert abs(yarn[50, 0] - math.cos(50.0) * factor) < 1e-6
    assert abs(yarn[50, 63] - math.sin(50 * 1e4 ** (-62 / 64) / 8) * factor) < 1e-6
    low = math.floor(64 * math.log(4096 / (64 * math.pi)) / (2 * math.log(1e4)))
    high = math.ceil(64 * math.log(4096 / (2 * math.pi)) / (2 * math.log(1e4)))
    j = (low + high) // 2
    ramp = (j - low) / (high - low)
    freq = 1e4 ** (-2 * j / 64) * (1 - ramp + ramp / 8)
    assert abs(yarn[99, j] - math.cos(99 * freq) * factor) < 1e-6
    plain = table(64, 100, 1e4, scaling=RotaryScaling("yarn", 8.0, 4096, attention_factor=1.0))
    assert (plain * factor - yarn).abs().max() < 1e-6
    for bad in (dict(scaling=RotaryScaling("other", 2.0)), dict(scaling=RotaryScaling("linear", 0.5)),
                dict(scaling=RotaryScaling("yarn", 2.0)), dict(rotary_dim=63), dict(rotary_dim=66),
                dict(rotary_dim=2, scaling=RotaryScaling("base", 2.0))):
        with pytest.raises(ValueError):
            table(64, 10, 1e4, **bad)
