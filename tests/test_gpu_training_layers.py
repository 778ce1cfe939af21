"""The layers' training pass on the GPU: gradients through every choice of launches."""

import pytest
import torch

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
