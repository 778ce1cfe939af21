"""The gradient of varlen attention over every choice of launches: a block of keys' queries shared
among workgroups at head_dim 128, and blocks in the order of their work for up to 128 sequences."""

import ctypes

import pytest
import torch

from oracle import gradients as G
from voiceagent_amd import _native as N
from voiceagent_amd import ops

pytestmark = pytest.mark.gpu
NAMES = ("dq", "dk", "dv")


def _inputs(lens_q, lens_k, hq, hkv, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda n, h, x=1.0: (torch.randn(n, h, d, generator=g) * x).to(dtype)  # noqa: E731
    cu = lambda x: torch.tensor([sum(x[:i]) for i in range(len(x) + 1)], dtype=torch.int32)  # noqa: E731
    nq, nk = sum(lens_q), sum(lens_k)
    return (make(nq, hq, 2.0 ** -6), make(nq, hq), make(nk, hkv), make(nk, hkv), make(nq, hq, 0.5),
            cu(lens_q), cu(lens_k))


def _parts(case, causal):
    """Workgroups that share a block's queries, from the workspace that their sums need."""
    dout, q, k, v, out, cu_q, cu_k = case
    a = N.new_args(N.VarlenBwdArgs)
    a.dtype = N.DTYPE_CODES[q.dtype]
    a.num_seqs, a.total_q, a.total_k = cu_q.numel() - 1, q.shape[0], k.shape[0]
    a.num_heads, a.num_kv_heads, a.head_dim, a.causal = q.shape[1], k.shape[1], q.shape[2], causal
    rows = q.shape[0] * q.shape[1] * 4 * (3 if q.dtype == torch.float16 else 2)
    more = N.lib().va_varlen_attention_backward_workspace_bytes(ctypes.byref(a)) - (rows + 255) // 256 * 256
    block = (a.total_k // 64 + a.num_seqs + 1) * a.num_kv_heads * 2 * 64 * a.head_dim * 4
    assert more % block == 0
    return max(more // block, 1)


def _check(dev, case, causal):
    dout, q, k, v, out, cu_q, cu_k = case
    scale = q.shape[2] ** -0.5
    got = ops.varlen_attention_backward(*(t.to(dev) for t in case), 0, 0, scale=scale, causal=causal)
    want = G.varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, scale, causal)
    for name, t in zip(NAMES, got):
        worst = ((t.double().cpu() - want[name]).abs() / want[name + "_off"].clamp_min(1e-300)).max().item()
        assert worst <= 1.0, f"{name}: {worst} of the bound"


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lens_q,lens_k,hq,hkv,d", [
    ([420], [420], 16, 8, 128), ([700, 3], [700, 3], 8, 1, 128), ([190, 0, 330], [450, 70, 331], 8, 2, 128),
    ([513], [129], 8, 1, 128), ([700, 3], [700, 3], 8, 1, 64)])
def test_blocks_whose_queries_are_shared(dev, lens_q, lens_k, hq, hkv, d, dtype, causal):
    """Among them blocks that end inside the sequence, and parts without a step (a sequence of 3
    has 8 of them, for more parts than that)."""
    case = _inputs(lens_q, lens_k, hq, hkv, d, dtype, 41)
    parts = _parts(case, causal)
    print(f"varlen backward parts={parts} {lens_q} {hq}/{hkv} d={d} {dtype} {causal}", flush=True)
    assert parts > 1
    _check(dev, case, causal)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("num_seqs", [63, 64, 65, 100, 127, 128, 129])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(2, 1, 64, torch.bfloat16), (4, 2, 128, torch.float16),
                                            (16, 16, 64, torch.bfloat16)])
def test_the_order_of_many_sequences_blocks(dev, num_seqs, hq, hkv, d, dtype, causal):
    """Lengths from none to several blocks on both sides of a wave's 64 lanes."""
    print(f"varlen backward {num_seqs} sequences {hq}/{hkv} d={d} {dtype} {causal}", flush=True)
    g = torch.Generator().manual_seed(num_seqs)
    of = lambda lo, hi: int(torch.randint(lo, hi, (), generator=g))  # noqa: E731
    top = 60 if hq == 16 else 400
    lens_q = [(0, of(1, 20), of(60, 70), of(1, top))[of(0, 4)] for _ in range(num_seqs)]
    lens_k = [max(n + of(-30, 60), 0) if of(0, 3) == 0 else n for n in lens_q]
    lens_q[0] = lens_k[1] = 0
    lens_q[num_seqs // 3] = lens_k[num_seqs // 3] = lens_q[-2] = lens_k[-2] = 321  # (several blocks)
    _check(dev, _inputs(lens_q, lens_k, hq, hkv, d, dtype, num_seqs), causal)
