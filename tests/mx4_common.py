"""Random MXFP4 pools and batches shared by the MXFP4 tests."""

import math

import torch

from oracle import mx4 as oracle
from voiceagent_amd import ops


class Pool:
    """An MXFP4 pool on the CPU (bytes) and on the GPU, with `spare` unused blocks."""

    def __init__(self, gen, blocks, block, hkv, d, layout, dtype, dev):
        self.block, self.layout, self.dtype = block, layout, dtype
        dims = (blocks, block, hkv) if layout == "nhd" else (blocks, hkv, block)
        rows = torch.randn(*dims, d, generator=gen) * torch.exp(torch.randn(*dims, 1, generator=gen))
        kc, ks = oracle.quantise(rows.to(dtype))
        vc, vs = oracle.quantise(torch.randn(*dims, d, generator=gen).to(dtype))
        self.cpu = [kc, vc, ks, vs]
        self.gpu = [t.to(dev) for t in self.cpu]

    def args(self):
        k, v, ks, vs = self.gpu
        return (k.view(ops.MXFP4_KV_DTYPE), v.view(ops.MXFP4_KV_DTYPE)), {
            "layout": self.layout, "k_scale": ks.view(ops.MXFP4_SCALE_DTYPE),
            "v_scale": vs.view(ops.MXFP4_SCALE_DTYPE)}

    def rows(self, slots):
        at = lambda t: oracle.rows_at(t, slots, self.block, self.layout)  # noqa: E731
        return (oracle.values(at(self.cpu[0]), at(self.cpu[2])),
                oracle.values(at(self.cpu[1]), at(self.cpu[3])))

    def same(self):
        """Whether the GPU's pool holds exactly the CPU's bytes."""
        return all(torch.equal(g.cpu(), c) for g, c in zip(self.gpu, self.cpu))


def tables_for(gen, lens, block, blocks, dtype=torch.int32, pad=-1, extra=0):
    """Block tables over random distinct blocks; padding behind each context."""
    used = [math.ceil(n / block) for n in lens]
    order = torch.randperm(blocks, generator=gen).tolist()
    width = max(used + [1]) + extra
    rows, at = [], 0
    for u in used:
        rows.append(order[at:at + u] + [pad] * (width - u))
        at += u
    return torch.tensor(rows, dtype=dtype).reshape(len(lens), width)


def slots_of(table, n, block):
    pos = torch.arange(n)
    return table.long()[pos // block] * block + pos % block


def cu(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)


def close(out, ref, tol):
    bad = (out.double().cpu() - ref).abs() > tol
    assert not bad.any(), ((out.double().cpu() - ref).abs() / tol)[bad].max()
