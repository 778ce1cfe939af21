"""Values near f16's limits in the gradient of varlen attention: what is held on the way, dS, may
not become infinite where the gradients themselves are finite."""

import pytest
import torch

from oracle import gradients as G
from voiceagent_amd import ops

pytestmark = pytest.mark.gpu
LARGEST = 65504.0


def _case(lens, hq, hkv, d, causal, which, seed):
    """f16 rows whose values have one channel near the type's limit: every key's, or only the last
    one's of each sequence.  And the output, as the attention gives it."""
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    make = lambda h: torch.randn(T, h, d, generator=g)  # noqa: E731
    q, k, v, dout = make(hq), make(hkv), make(hkv), make(hq) / 64
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    far = (torch.randint(0, 2, (T, hkv), generator=g) * 2 - 1) * 60000.0
    rows = slice(None) if which == "all" else (cu[1:] - 1).long()
    v[rows, :, 5] = far[rows]
    q, k, v, dout = (t.to(torch.float16) for t in (q, k, v, dout))
    out, most = torch.zeros(T, hq, d, dtype=torch.float64), 0.0
    for a, b in zip(cu[:-1].tolist(), cu[1:].tolist()):
        for h in range(hq):
            kk, vv = (x[a:b, h * hkv // hq].double() for x in (k, v))
            s = (q[a:b, h].double() @ kk.T * d ** -0.5).masked_fill(~G.visible(b - a, b - a, causal), -1e300)
            p = torch.softmax(s, -1)
            out[a:b, h] = p @ vv
            do = dout[a:b, h].double()
            dp = do @ vv.T - (do * out[a:b, h].half().double()).sum(-1, keepdim=True)
            unit = 2.0 ** do.abs().amax(1, keepdim=True).log2().floor()
            most = max(most, float((p / p.amax(1, keepdim=True) * dp / unit).abs().max()))
    return q, k, v, dout, out.to(torch.float16), cu, most


@pytest.mark.parametrize("which", ["all", "last"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,hq,hkv,d,most", [
    ([2, 3, 40, 104, 128], 2, 2, 64, 128),  # one launch
    ([2, 3, 40, 129, 300], 4, 2, 128, 0), ([2, 33, 64, 500], 4, 2, 64, 0),  # blocks of 64 queries
    ([300, 65, 257] * 6, 16, 16, 64, 0), ([300, 65, 257] * 6, 16, 16, 128, 0)])  # of 128
def test_values_near_the_types_limit(dev, lens, hq, hkv, d, most, causal, which):
    print(f"varlen backward range {hq}/{hkv} d={d} {causal} {which}", flush=True)
    q, k, v, dout, out, cu, largest = _case(lens, hq, hkv, d, causal, which, 31)
    want = G.varlen_attention_backward(dout, q, k, v, out, cu, cu, d ** -0.5, causal)
    names = ("dq", "dk", "dv")
    assert (which == "last" or largest > 65520) and max(want[n].abs().max() for n in names) < LARGEST / 2
    on = [t.to(dev) for t in (dout, q, k, v, out, cu, cu)]
    got = ops.varlen_attention_backward(*on, most, most, scale=d ** -0.5, causal=causal)
    for t, n in zip(got, names):
        assert torch.isfinite(t).all(), n
        worst = ((t.double().cpu() - want[n]).abs() / want[n + "_off"].clamp_min(1e-300)).max().item()
        assert worst <= 1.0, f"{n}: {worst} of the bound"


def test_a_masked_key_near_the_limit_costs_other_rows_nothing(dev):
    """Rows that do not see the last key have the gradients they have without it, bit for bit."""
    lens, d = [40, 120], 64
    for hq, hkv, most in ((2, 2, 128), (2, 1, 0)):
        q, k, v, dout, out, cu, _ = _case(lens, hq, hkv, d, True, "last", 32)
        on = [t.to(dev) for t in (dout, q, k, v, out, cu, cu)]
        dq = ops.varlen_attention_backward(*on, most, most, scale=0.125, causal=True)[0]
        on[3][(cu[1:] - 1).long().to(dev), :, 5] = 0.0
        plain = ops.varlen_attention_backward(*on, most, most, scale=0.125, causal=True)[0]
        last = (cu[1:] - 1).long()
        rest = [i for i in range(sum(lens)) if i not in last.tolist()]
        assert torch.equal(dq[rest], plain[rest]) and not torch.equal(dq, plain)
