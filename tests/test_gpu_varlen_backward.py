"""The gradient of varlen attention on the GPU, against the definition in float64.

Every element is held to the bound that oracle.gradients derives for it (P and dS rounded to the
element type once, sums in fp32, the result rounded)."""

import ctypes

import pytest
import torch

from oracle import gradients as G
from voiceagent_amd import _native as N
from voiceagent_amd import ops
from voiceagent_amd._native import NativeError
from voiceagent_amd.layers import (AttentionContext, PagedAttention, VarlenSelfAttention,
                                   attention_context)

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv")


def _cu(lens, first=0):
    return torch.tensor([first + sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def _inputs(lens_q, lens_k, hq, hkv, d, dtype, seed, *, grad=2.0 ** -6, before=0, behind=0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(lens_q) + before + behind, sum(lens_k) + before + behind
    make = lambda n, h, x=1.0: (torch.randn(n, h, d, generator=g) * x).to(dtype)  # noqa: E731
    q, k, v = make(nq, hq), make(nk, hkv), make(nk, hkv)
    dout, out = make(nq, hq, grad), make(nq, hq, 0.5)  # (out is an input: any values)
    return q, k, v, dout, out, _cu(lens_q, before), _cu(lens_k, before)


def _call(dev, q, k, v, dout, out, cu_q, cu_k, scale, causal, **more):
    on = [t.to(dev) for t in (dout, q, k, v, out, cu_q, cu_k)]
    return ops.varlen_attention_backward(*on, 0, 0, scale=scale, causal=causal, **more)


def _check(got, want):
    for name, x in zip(NAMES, got):
        err = (x.double().cpu() - want[name]).abs()
        worst = (err / want[name + "_off"].clamp_min(1e-300)).max().item()
        assert worst <= 1.0, f"{name}: {worst} of the bound, {err.max().item()}"


LENS = {
    "one": ([1], [1]),
    "few": ([1, 0, 3, 2], [1, 2, 3, 0]),
    "tile": ([31, 32, 33], [31, 32, 33]),
    "block": ([63, 64, 65, 127, 128, 129], [63, 64, 65, 127, 128, 129]),
    "long": ([300, 5, 0, 77], [300, 5, 0, 77]),
    "more keys": ([1, 40, 129, 3], [200, 41, 260, 131]),
    "fewer keys": ([70, 200, 5], [1, 130, 3]),
}


@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d,hq,hkv", [
    (torch.bfloat16, 128, 4, 2), (torch.bfloat16, 64, 3, 3), (torch.float16, 128, 2, 1),
    (torch.float16, 64, 6, 2)])
def test_gradient_matches_the_definition(dev, lens, causal, dtype, d, hq, hkv):
    print(f"varlen backward {lens} causal={causal} {dtype} d={d} {hq}/{hkv}", flush=True)
    lens_q, lens_k = LENS[lens]
    q, k, v, dout, out, cu_q, cu_k = _inputs(lens_q, lens_k, hq, hkv, d, dtype, 3)
    got = _call(dev, q, k, v, dout, out, cu_q, cu_k, d ** -0.5, causal)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, d ** -0.5, causal))


WINDOWS = {
    "encoder": ([104, 104, 33, 13], [104, 104, 33, 13], 104),
    "tiles": ([31, 32, 33, 63, 64, 65], [31, 32, 33, 63, 64, 65], 65),
    "most": ([128, 1, 0, 127, 96, 97], [128, 1, 0, 127, 96, 97], 128),
    "tokens": ([1, 1, 2, 7], [1, 1, 2, 7], 7),
    "sides": ([1, 40, 0, 100, 9, 3], [128, 7, 5, 0, 10, 99], 128),
}


@pytest.mark.parametrize("lens", WINDOWS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_short_sequences_in_one_launch(dev, lens, causal, dtype):
    lens_q, lens_k, most = WINDOWS[lens]
    q, k, v, dout, out, cu_q, cu_k = _inputs(lens_q, lens_k, 3, 3, 64, dtype, 17, before=3, behind=9)
    on = [t.to(dev) for t in (dout, q, k, v, out, cu_q, cu_k)]
    got = ops.varlen_attention_backward(*on, most, most, scale=0.125, causal=causal)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, causal))
    for t in got:
        assert not t[:3].any() and not t[-9:].any()


def test_short_sequences_of_any_values(dev):
    # Small and large gradients, rising maxima, strided rows, NaN outside and in another sequence.
    lens, cu = [104, 50, 104], _cu([104, 50, 104], 7)
    for dtype, size in ((torch.float16, 2.0 ** -20), (torch.float16, 2.0 ** 8), (torch.bfloat16, 2.0 ** -6)):
        q, k, v, dout, out, _, _ = _inputs(lens, lens, 2, 2, 64, dtype, 18, grad=size, before=7, behind=5000)
        q, k = q * 2, k * torch.linspace(0.1, 4, k.shape[0])[:, None, None].to(dtype)
        want = G.varlen_attention_backward(dout, q, k, v, out, cu, cu, 0.125, False)
        for t in (q, k, v, dout, out):
            t[:7] = t[7 + 258:] = float("nan")
        qkv = torch.cat((q, k, v), 1).to(dev).split([2, 2, 2], 1)
        c, o, do = cu.to(dev), out.to(dev), dout.to(dev)
        got = ops.varlen_attention_backward(do, *qkv, o, c, c, 104, 104, scale=0.125, causal=False)
        _check(got, want)
        do[7 + 104] = float("nan")  # the second sequence
        for t, name in zip(ops.varlen_attention_backward(do, *qkv, o, c, c, 104, 104, scale=0.125,
                                                         causal=False), NAMES):
            for at in (slice(7, 111), slice(161, 265)):
                err = (t[at].double().cpu() - want[name][at]).abs()
                assert (err <= want[name + "_off"][at]).all()
            assert not t[265:].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_sequence_longer_than_the_maxima_gets_nan(dev, dtype):
    lens_q, lens_k = [100, 300, 9, 20], [100, 300, 101, 20]
    q, k, v, dout, out, cu_q, cu_k = _inputs(lens_q, lens_k, 2, 2, 64, dtype, 19)
    on = [t.to(dev) for t in (dout, q, k, v, out, cu_q, cu_k)]
    got = ops.varlen_attention_backward(*on, 100, 100, scale=0.125, causal=False)
    want = G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, False)
    for t, name, cu in zip(got, NAMES, (cu_q, cu_k, cu_k)):
        off = (t.double().cpu() - want[name]).abs() <= want[name + "_off"]
        for i, right in enumerate((True, False, False, True)):
            rows = slice(int(cu[i]), int(cu[i + 1]))
            assert off[rows].all() if right else t[rows].isnan().all(), (name, i)


def test_many_sequences(dev):
    # More than a wave's lanes of sequences, some without queries.
    g = torch.Generator().manual_seed(5)
    lens_q = torch.randint(0, 40, (150,), generator=g).tolist()
    lens_k = [n + e for n, e in zip(lens_q, torch.randint(0, 9, (150,), generator=g).tolist())]
    q, k, v, dout, out, cu_q, cu_k = _inputs(lens_q, lens_k, 2, 1, 64, torch.bfloat16, 4)
    for causal in (True, False):
        got = _call(dev, q, k, v, dout, out, cu_q, cu_k, 0.125, causal)
        _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, causal))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.float16, 64)])
def test_enough_blocks_to_fill_the_chip(dev, dtype, d, causal):
    # (The cases above leave most of it idle, where blocks are smaller and their work shared.)
    lens_q = [1, 31, 64, 65, 97, 127, 128, 129, 130, 161, 190, 192, 193, 255, 256, 257, 258]
    lens_k = [n + e for n, e in zip(lens_q, [0, 3, -7, 64, 0, 129] * 3)]
    q, k, v, dout, out, cu_q, cu_k = _inputs(lens_q, lens_k, 16, 16, d, dtype, 16)
    got = _call(dev, q, k, v, dout, out, cu_q, cu_k, d ** -0.5, causal)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, d ** -0.5, causal))


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_and_large_gradients(dev, dtype, size):
    """f16 gradients whose dS would be subnormal (or infinite) as they are."""
    q, k, v, dout, out, cu_q, cu_k = _inputs([600], [600], 2, 1, 64, dtype, 6, grad=size)
    got = _call(dev, q, k, v, dout, out, cu_q, cu_k, 0.125, True)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, True))


def test_large_scores(dev):
    # Maxima that keep rising along the keys: the accumulators are rescaled.
    for dtype in (torch.bfloat16, torch.float16):
        q, k, v, dout, out, cu_q, cu_k = _inputs([260], [260], 2, 2, 64, dtype, 7)
        q, k = q * 2, k * torch.linspace(0.1, 4, 260)[:, None, None].to(dtype)
        got = _call(dev, q, k, v, dout, out, cu_q, cu_k, 0.125, False)
        _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, False))


def test_rows_outside_the_sequences(dev):
    """Rows in front of the first sequence and behind the last hold NaN: they get zeros and reach
    nothing; sequences do not reach one another."""
    q, k, v, dout, out, cu_q, cu_k = _inputs([70, 30], [70, 30], 4, 2, 64, torch.bfloat16, 8,
                                             before=200, behind=333)
    for t in (q, k, v, dout, out):
        t[:200] = t[300:] = float("nan")
    want = G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, 0.125, True)
    got = _call(dev, q, k, v, dout, out, cu_q, cu_k, 0.125, True)
    _check(got, want)
    for t in got:
        assert not t[:200].any() and not t[300:].any()
    # A NaN in the first sequence stays there.
    q[250] = float("nan")
    for t, name in zip(_call(dev, q, k, v, dout, out, cu_q, cu_k, 0.125, True), NAMES):
        err = (t[270:300].double().cpu() - want[name][270:300]).abs()
        assert (err <= want[name + "_off"][270:300]).all()


def test_lengths_past_the_rows_are_held(dev):
    # Cumulative lengths that run past the tensors, or fall: held to the rows there are.
    q, k, v, dout, out, _, _ = _inputs([64], [64], 2, 1, 64, torch.bfloat16, 9)
    cu = torch.tensor([0, 40, 1000, 900], dtype=torch.int32)
    held = torch.tensor([0, 40, 64, 64], dtype=torch.int32)
    got = _call(dev, q, k, v, dout, out, cu, cu, 0.125, True)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, held, held, 0.125, True))


def test_lengths_that_fall_and_rise_stay_in_the_workspace(dev):
    # More blocks than the rows make: results mean nothing, memory behind the workspace stays.
    q, k, v, dout, out, _, _ = (None if t is None else t.to(dev) for t in
                                _inputs([300], [300], 16, 1, 64, torch.bfloat16, 24))
    cu = torch.tensor([0, 300] * 20 + [0], dtype=torch.int32, device=dev)
    grads = [torch.empty_like(t) for t in (q, k, v)]
    a = N.new_args(N.VarlenBwdArgs)
    a.dtype = N.VA_BF16
    for name, t in zip(("q", "k", "v", "out", "dout", "dq", "dk", "dv"), (q, k, v, out, dout, *grads)):
        setattr(a, name, t.data_ptr())
        setattr(a, name + "_stride_tok", t.stride(0))
        setattr(a, name + "_stride_head", t.stride(1))
    a.cu_seqlens_q = a.cu_seqlens_k = cu.data_ptr()
    a.num_seqs, a.total_q, a.total_k = 40, 300, 300
    a.num_heads, a.num_kv_heads, a.head_dim, a.scale = 16, 1, 64, 0.125
    lib = N.lib()
    need = lib.va_varlen_attention_backward_workspace_bytes(ctypes.byref(a))
    assert need > 2 * 16 * 300 * 4 + 256  # the launch has parts
    ws = torch.full((need + (8 << 20),), 85, dtype=torch.uint8, device=dev)
    a.workspace, a.workspace_bytes = ws.data_ptr(), need
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.va_varlen_attention_backward(ctypes.byref(a), stream) == 0
    torch.cuda.synchronize()
    assert (ws[need:] == 85).all()


def test_no_sequences_no_rows(dev):
    q, k, v, dout, out, cu_q, cu_k = _inputs([], [], 2, 1, 64, torch.bfloat16, 1, before=5)
    cu = torch.tensor([5, 5], dtype=torch.int32)
    for t in _call(dev, q, k, v, dout, out, cu, cu, 0.125, True):
        assert not t.any()
    none = [t[:0] for t in (q, k, v, dout, out)]
    for t in _call(dev, *none, cu * 0, cu * 0, 0.125, True):
        assert t.shape[0] == 0
    # Keys without a query in the call, queries without a key.
    dq, dk, dv = _call(dev, q[:0], k, v, dout[:0], out[:0], cu * 0, cu, 0.125, True)
    assert not dk.any() and not dv.any() and dq.numel() == 0
    dq, dk, dv = _call(dev, q, k[:0], v[:0], dout, out, cu, cu * 0, 0.125, True)
    assert not dq.any() and dk.numel() == 0
    on = [t.to(dev) for t in (dout, q, q, q, out, cu * 0, cu)]
    for a, b in ((slice(0), slice(5)), (slice(5), slice(0))):  # the same of short sequences
        call = [on[0][a], on[1][a], on[2][b], on[3][b], on[4][a]]
        for t in ops.varlen_attention_backward(*call, on[5], on[5], 3, 3, scale=0.125, causal=True):
            assert not t.any()


def test_strided_rows_and_gradients_into_one_buffer(dev):
    lens, hq, hkv, d = [90, 37], 4, 2, 128
    q, k, v, dout, out, cu, _ = _inputs(lens, lens, hq, hkv, d, torch.bfloat16, 10)
    want = G.varlen_attention_backward(dout, q, k, v, out, cu, cu, 0.09, True)
    qkv = torch.cat((q, k, v), 1).to(dev)  # [T, Hq + 2 Hkv, D]
    grads = torch.full_like(qkv, 7.0)
    parts = lambda t: t.split([hq, hkv, hkv], 1)  # noqa: E731
    dq, dk, dv = parts(grads)
    back = ops.varlen_attention_backward(
        dout.to(dev), *parts(qkv), out.to(dev), cu.to(dev), cu.to(dev), 90, 90, scale=0.09,
        causal=True, dq=dq, dk=dk, dv=dv)
    assert all(a is b for a, b in zip(back, (dq, dk, dv)))
    _check(parts(grads), want)
    # Head-major tensors: heads far apart, tokens near.
    major = [t.to(dev).transpose(0, 1).contiguous().transpose(0, 1) for t in (dout, q, k, v, out)]
    _check(ops.varlen_attention_backward(*major, cu.to(dev), cu.to(dev), 90, 90, scale=0.09,
                                         causal=True), want)


@pytest.mark.parametrize("d,hkv,most", [(128, 1, 150), (64, 2, 0), (64, 2, 110)])
def test_offsets_past_32_bits(dev, d, hkv, most):
    # Tokens 24 MiB apart in one buffer of 6.6 GB: a tile's last row lies 1.5 GB behind its first.
    lens, step = [110, 150], 12 << 20
    if most == 110:
        lens = [110, 110]
    n = sum(lens)
    buf = torch.empty(n * step + 4096, dtype=torch.bfloat16, device=dev)
    q, k, v, dout, out, cu, _ = _inputs(lens, lens, 2, hkv, d, torch.bfloat16, 21)
    at = 0

    def place(like, fill):
        nonlocal at
        t = buf.as_strided((n, like.shape[1], d), (step, d, 1), at)
        at += like.shape[1] * d
        return t.copy_(like) if fill else t

    on = [place(t, True) for t in (dout, q, k, v, out)]
    dq, dk, dv = (place(t, False) for t in (q, k, v))
    c = cu.to(dev)
    got = ops.varlen_attention_backward(*on, c, c, most, most, scale=0.125, causal=True, dq=dq, dk=dk,
                                        dv=dv)
    _check(got, G.varlen_attention_backward(dout, q, k, v, out, cu, cu, 0.125, True))


def test_calls_repeat_bit_for_bit_on_any_stream(dev):
    lens = [500, 77, 230]
    q, k, v, dout, out, cu, _ = _inputs(lens, lens, 8, 2, 64, torch.float16, 11)
    on = [t.to(dev) for t in (dout, q, k, v, out, cu, cu)]
    first = ops.varlen_attention_backward(*on, 500, 500, scale=0.125, causal=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    results = []
    for i in range(4):
        with torch.cuda.stream(streams[i % 2]):
            results.append(ops.varlen_attention_backward(*on, 500, 500, scale=0.125, causal=True))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_graph_replays(dev):
    lens = [200, 90]
    q, k, v, dout, out, cu, _ = _inputs(lens, lens, 4, 2, 128, torch.bfloat16, 12)
    on = [t.to(dev) for t in (dout, q, k, v, out, cu, cu)]
    call = lambda: ops.varlen_attention_backward(*on, 200, 200, scale=0.09, causal=True)  # noqa: E731
    call()
    graphs = []
    for _ in range(2):  # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = call()
        graphs.append((graph, res))
    for i in range(4):
        on[0].copy_(torch.roll(dout, i, 0))
        want = call()
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(want, res)), i


def test_refusals(dev):
    q, k, v, dout, out, cu, _ = (t.to(dev) for t in _inputs([8], [8], 4, 2, 64, torch.bfloat16, 1))
    call = lambda *a, **kw: ops.varlen_attention_backward(*a, cu, cu, 8, 8, scale=1.0, causal=True, **kw)  # noqa: E731
    for bad in [(dout[:4], q, k, v, out), (dout, q, k, v[:4], out), (dout.half(), q, k, v, out),
                (dout, q[:, :3], k, v, out[:, :3]), (dout, q, k, v, out.transpose(1, 2)),
                (dout.float(), q.float(), k.float(), v.float(), out.float())]:
        with pytest.raises(ops.AttentionArgumentError):
            call(*bad)
    with pytest.raises(ops.AttentionArgumentError, match="overlap"):
        call(dout, q, k, v, out, dq=dout)
    with pytest.raises(ops.AttentionArgumentError, match="match"):
        call(dout, q, k, v, out, dk=q)
    new = torch.zeros_like(k)
    with pytest.raises(ops.AttentionArgumentError, match="dv may not overlap dk"):
        call(dout, q, k, v, out, dk=new, dv=new)
    with pytest.raises(ops.AttentionArgumentError, match="length"):
        ops.varlen_attention_backward(dout, q, k, v, out, cu, cu, -1, 8, scale=1.0, causal=True)
    with pytest.raises(ops.AttentionArgumentError, match="int32"):
        ops.varlen_attention_backward(dout, q, k, v, out, cu.long(), cu, 8, 8, scale=1.0, causal=True)
    wide = torch.zeros(8, 4, 65, dtype=torch.bfloat16, device=dev)[:, :, :64]
    with pytest.raises(NativeError, match="strides"):
        call(wide, q, k, v, out)


# --------------------------------------------------------------------------- through autograd
def test_autograd_of_the_encoder_layer(dev):
    lens, heads, d = [104, 104, 33], 3, 64
    q, k, v, dout, _, cu, _ = _inputs(lens, lens, heads, heads, d, torch.bfloat16, 13, grad=1.0)
    layer = VarlenSelfAttention(heads, d, d ** -0.5)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    out = layer(*leaves, cu.to(dev), 104)
    with torch.no_grad():
        assert torch.equal(out, layer(*leaves, cu.to(dev), 104))
    out.backward(dout.to(dev))
    want = G.varlen_attention_backward(dout, q, k, v, out.detach().cpu(), cu, cu, d ** -0.5, False)
    _check([t.grad for t in leaves], want)
    # A gradient with strides of zero (a plain sum's), and only one that is asked for.
    leaf = k.to(dev).requires_grad_()
    layer(q.to(dev), leaf, v.to(dev), cu.to(dev), 104).sum().backward()
    ones = torch.ones_like(dout)
    want = G.varlen_attention_backward(ones, q, k, v, out.detach().cpu(), cu, cu, d ** -0.5, False)
    err = (leaf.grad.double().cpu() - want["dk"]).abs()
    assert (err <= want["dk_off"]).all()


def test_autograd_of_the_decoder_layer_without_a_cache(dev):
    lens, hq, hkv, d = [130, 70, 9], 4, 2, 128
    q, k, v, dout, _, cu, _ = _inputs(lens, lens, hq, hkv, d, torch.bfloat16, 14, grad=1.0)
    layer = PagedAttention(hq, d, d ** -0.5, hkv)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]
    on = cu.to(dev)
    with attention_context(AttentionContext(on, on, 130, 130, None, None)):
        out = layer(*leaves)
    out.backward(dout.to(dev))
    want = G.varlen_attention_backward(dout, q, k, v, out.detach().cpu(), cu, cu, d ** -0.5, True)
    _check([t.grad for t in leaves], want)


@pytest.mark.parametrize("heads", [(3, 3), (4, 2)])
def test_a_captured_training_step(dev, heads):
    """Forward and gradient in one graph, several replays with eager steps between them."""
    lens, (hq, hkv), d = [104, 60, 1], heads, 64
    q, k, v, dout, _, cu, _ = _inputs(lens, lens, hq, hkv, d, torch.bfloat16, 22, grad=1.0)
    on, do = cu.to(dev), dout.to(dev)
    leaves = [t.to(dev).requires_grad_() for t in (q, k, v)]

    def step(xs):
        out = ops.varlen_attention(*xs, on, on, 104, 104, scale=0.125, causal=True)
        return torch.autograd.grad(out, xs, do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(leaves)
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(torch.roll(q, i, 1))
        graph.replay()
        torch.cuda.synchronize()
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        for a, b in zip(got, want):
            assert torch.equal(a, b), i
