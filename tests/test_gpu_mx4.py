"""MXFP4 KV pools on the GPU: store, load, paged decode and varlen attention
against the float64 oracle (oracle/mx4.py), which also bounds the rounding."""

import math

import pytest
import torch

from oracle import mx4 as oracle
from tests.mx4_common import Pool, close, cu, slots_of, tables_for
from voiceagent_amd import ops
from voiceagent_amd._native import NativeError
from voiceagent_amd.layers.attention import PagedAttention
from voiceagent_amd.layers.context import AttentionContext, attention_context
from voiceagent_amd.layers.qwen3 import Qwen3AttentionCore

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16
# The decode's Q K^T runs on scaled matrix products, which align neighbouring
# products to 13 bits before adding; the varlen kernel's on 16-bit ones.
DECODE_BITS, VARLEN_BITS = 13, 17


# ------------------------------------------------------------- store and load
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hkv, d, block, layout, wide, n", [
    (8, 128, 16, "nhd", False, 37), (8, 128, 16, "hnd", True, 700), (1, 64, 32, "nhd", False, 1),
    (3, 256, 16, "hnd", False, 9), (2, 96, 7, "nhd", True, 50), (5, 32, 1, "hnd", False, 11)])
def test_store_and_load_are_exact(dev, dtype, hkv, d, block, layout, wide, n):
    gen = torch.Generator().manual_seed(n + d)
    blocks = -(-n // block) + 3
    pool = Pool(gen, blocks, block, hkv, d, layout, dtype, dev)
    key = (torch.randn(n, hkv, d, generator=gen) * torch.exp(4 * torch.randn(n, hkv, 1, generator=gen))).to(dtype)
    # Rows strided as a view of a fused projection.
    value = torch.randn(n, hkv + 2, d, generator=gen).to(dtype)[:, 1:-1]
    # The format's corners: ties, limits, subnormals, infinities, NaN.
    special = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.0, -0.25, 7.0, -7.0])
    key[0, 0, :12] = special.to(dtype)
    value[0, 0, :12] = (special * 2.0 ** -13).to(dtype)
    tiny, most = torch.finfo(dtype).tiny, torch.finfo(dtype).max
    if n > 8:
        key[1, 0, :3] = torch.tensor([tiny / 4, tiny, -tiny / 2]).to(dtype)
        key[1, 0, 3:] = 0
        key[2] = 0
        key[3, 0, 5] = math.inf
        value[4, 0, 7] = math.nan
        value[5, 0, :4] = torch.tensor([most, -most, most / 2, 1.0]).to(dtype)
        key[6, 0, 1] = -math.inf
    slots = torch.randperm(blocks * block, generator=gen)[:n].to(torch.int64 if wide else torch.int32)
    if n > 8:
        slots[7], slots[8] = -1, blocks * block  # padding, past the pool
    (kc, vc), kw = pool.args()
    gpu_value = value.to(dev)
    fused = torch.zeros(n, hkv + 2, d, dtype=dtype, device=dev)
    fused[:, 1:-1] = gpu_value
    ops.store_kvcache(key.to(dev), fused[:, 1:-1], kc, vc, slots.to(dev), **kw)
    oracle.store(key, value, pool.cpu, slots, block, layout)
    assert pool.same()
    k, v = ops.load_kvcache(kc, vc, slots.to(dev), dtype, **kw)
    ok = (slots >= 0) & (slots < blocks * block)
    ek, ev = pool.rows(slots.long().clamp(0, blocks * block - 1))
    for got, want in ((k, ek), (v, ev)):
        want[~ok] = 0
        assert torch.equal(got.double().cpu().nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
    assert pool.same()


def test_store_of_nothing(dev):
    gen = torch.Generator().manual_seed(0)
    pool = Pool(gen, 2, 16, 2, 64, "nhd", BF16, dev)
    (kc, vc), kw = pool.args()
    x = torch.zeros(0, 2, 64, dtype=BF16, device=dev)
    slots = torch.zeros(0, dtype=torch.int32, device=dev)
    ops.store_kvcache(x, x, kc, vc, slots, **kw)
    assert ops.load_kvcache(kc, vc, slots, **kw)[0].shape == (0, 2, 64)
    assert pool.same()


# --------------------------------------------------------------------- decode
def run_decode(dev, lens, *, hq=16, hkv=8, d=128, block=16, layout="nhd", dtype=BF16, seed=0,
               cumulative=True, table_dtype=torch.int32, split=0, bound=None, new=False, slots=None,
               mask=None, key_limit=0, table_read_width=0, pad=-1, edit=None, scale=None):
    gen = torch.Generator().manual_seed(seed)
    B = len(lens)
    blocks = sum(-(-n // block) for n in lens) + 5
    pool = Pool(gen, blocks, block, hkv, d, layout, dtype, dev)
    tables = tables_for(gen, lens, block, blocks, table_dtype, pad, extra=1)
    if edit:
        edit(pool, tables)
        pool.gpu = [t.to(dev) for t in pool.cpu]
    q = torch.randn(B, hq + 1, d, generator=gen).to(dtype)[:, :hq]
    more = {}
    if new:
        nk = torch.randn(B, hkv, 2 * d, generator=gen).to(dtype)
        nv = (torch.randn(B, hkv, d, generator=gen) * 3).to(dtype)
        more = {"new_k": nk.to(dev)[..., :d], "new_v": nv.to(dev)}
        if slots is not None:
            more["new_slots"] = slots.to(dev)
    if mask is not None:
        more["valid_mask"] = mask.to(dev)
    (kc, vc), kw = pool.args()
    scale = d ** -0.5 if scale is None else scale
    vec = cu(lens) if cumulative else torch.tensor(lens, dtype=torch.int64)
    out = ops.paged_decode(q.to(dev), kc, vc, tables.to(dev), vec.to(dev), lens_cumulative=cumulative,
                           max_seq_len=max(lens) if bound is None else bound, scale=scale,
                           split_tokens=split, key_limit=key_limit,
                           table_read_width=table_read_width, **more, **kw)
    torch.cuda.synchronize()
    # The oracle: the current row first, then one sequence at a time.
    capacity = blocks * block
    width = tables.shape[1]
    read_width = min(table_read_width, width) if table_read_width else width
    for b, n in enumerate(lens):
        if not new or n < 1:
            continue
        col = (n - 1) // block
        if slots is not None:
            at = int(slots[b])
        else:
            blk = int(tables[b, col]) if col < width else 0
            at = blk * block + (n - 1) % block if 0 <= blk < blocks else -1
        if 0 <= at < capacity:
            oracle.store(nk[b:b + 1, :, :d], nv[b:b + 1], pool.cpu, torch.tensor([at]), block, layout)
    for b, n in enumerate(lens):
        m = min(n, key_limit) if key_limit else n
        if m <= 0:
            assert not out[b].any()
            continue
        pos = torch.arange(m)
        col = pos // block
        blk = torch.where(col < read_width, tables[b].long()[col.clamp(max=width - 1)], 0)
        seen = (blk >= 0) & (blk < blocks)
        if mask is not None:
            seen &= torch.where(pos < mask.shape[1], mask[b][pos.clamp(max=mask.shape[1] - 1)], True)
        k, v = pool.rows(blk.clamp(0, blocks - 1) * block + pos % block)
        if new and m == n and (slots is None or 0 <= int(slots[b]) < capacity) and \
                ((n - 1) // block < read_width or slots is not None or (n - 1) // block >= width):
            kq, ks = oracle.quantise(nk[b, :, :d])
            vq, vs = oracle.quantise(nv[b])
            k[-1], v[-1] = oracle.values(kq, ks), oracle.values(vq, vs)
        ref, tol = oracle.attend(q[b:b + 1], k, v, seen[None], scale, dtype, DECODE_BITS)
        close(out[b:b + 1], ref, tol)
    assert pool.same()
    return out


LENS = [1, 2, 15, 16, 17, 31, 32, 33, 63, 100, 257, 600]


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq, hkv, d", [(16, 8, 128), (8, 8, 128), (8, 2, 64), (16, 2, 128), (4, 2, 256),
                                        (8, 1, 256), (14, 14, 64)])
@pytest.mark.parametrize("layout, block", [("nhd", 16), ("hnd", 16), ("nhd", 48)])
def test_decode(dev, dtype, hq, hkv, d, layout, block):
    run_decode(dev, LENS, hq=hq, hkv=hkv, d=d, dtype=dtype, layout=layout, block=block, seed=hq + d)


@pytest.mark.parametrize("dtype, d", [(BF16, 128), (F16, 64), (BF16, 256)])
@pytest.mark.parametrize("split, bound", [(0, None), (0, 32768), (ops.SPLIT_EXACT, None), (1, None), (700, None)])
def test_decode_splits(dev, dtype, d, split, bound):
    run_decode(dev, [4099, 1, 2050], hq=8, hkv=2, d=d, dtype=dtype, split=split, bound=bound, seed=5)


def test_decode_many_steps_a_wave(dev):
    # One partition: more than 64 steps for every wave (their block ids are read 32 steps at a time).
    run_decode(dev, [17000, 8300], hq=2, hkv=1, split=1 << 20, seed=6)


@pytest.mark.parametrize("new", [False, True])
@pytest.mark.parametrize("cumulative, table_dtype", [(False, torch.int64), (True, torch.int64)])
def test_decode_index_types(dev, new, cumulative, table_dtype):
    run_decode(dev, [5, 40, 300, 0, 16], cumulative=cumulative, table_dtype=table_dtype, new=new, seed=7)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq, hkv, d, layout", [(16, 8, 128, "nhd"), (4, 1, 64, "hnd"), (4, 2, 256, "nhd")])
@pytest.mark.parametrize("split", [0, 256])
def test_decode_current_row(dev, dtype, hq, hkv, d, layout, split):
    run_decode(dev, [1, 16, 17, 32, 33, 255, 900], hq=hq, hkv=hkv, d=d, layout=layout, dtype=dtype,
               new=True, split=split, seed=8)


def test_decode_current_row_slots(dev):
    # Slots other than the position's own, none, and past the pool.
    lens = [40, 33, 17, 1, 64]
    blocks = sum(-(-n // 16) for n in lens) + 5
    for values in ([-1] * 5, [blocks * 16, -1, -1, blocks * 16 + 5, -7]):
        run_decode(dev, lens, new=True, slots=torch.tensor(values, dtype=torch.int64), seed=10)


def test_decode_key_limit_and_read_width(dev):
    lens = [200, 40, 16, 100]
    run_decode(dev, lens, key_limit=50, seed=11)
    run_decode(dev, lens, key_limit=50, new=True, seed=12)
    run_decode(dev, lens, table_read_width=3, seed=13)
    run_decode(dev, lens, table_read_width=3, new=True, seed=14)


@pytest.mark.parametrize("split", [0, 256])
def test_decode_mask(dev, split):
    lens = [300, 40, 17, 1, 600]
    gen = torch.Generator().manual_seed(15)
    mask = torch.rand(5, 333, generator=gen) < 0.5  # narrower than a context: the rest is valid
    mask[1] = False  # a row with nothing left
    mask[0, :290] = False
    run_decode(dev, lens, mask=mask, split=split, seed=16)
    run_decode(dev, lens, mask=mask, new=True, split=split, seed=17, layout="hnd", dtype=F16)
    run_decode(dev, lens, mask=mask[:, 1:], seed=18, hq=4, hkv=1, d=64)


def test_decode_dead_places_hold_anything(dev):
    # NaN groups, huge scales and garbage where a mask, the context's end or a
    # missing block says that nothing is attended.
    lens = [40, 70, 20]
    mask = torch.ones(3, 80, dtype=torch.bool)
    mask[0, 3:9] = False
    mask[1, 64:] = False

    def edit(pool, tables):
        live = torch.zeros(pool.cpu[0].shape[0] * 16, dtype=torch.bool)
        for b, n in enumerate(lens):
            at = slots_of(tables[b], n, 16)
            live[at[mask[b, :n]]] = True
        live[slots_of(tables[2], 20, 16)[16:]] = False
        for t in (2, 3):
            pool.cpu[t].flatten(0, 1)[~live] = 255
        for t in (0, 1):
            pool.cpu[t].flatten(0, 1)[~live] = 0x7f
        tables[2, 1] = 10 ** 6  # a block outside the pool

    out = run_decode(dev, lens, mask=mask, edit=edit, seed=19)
    assert out.isfinite().all()


def test_decode_nan_reaches_its_own_sequence_only(dev):
    gen = torch.Generator().manual_seed(20)
    pool = Pool(gen, 8, 16, 2, 128, "nhd", BF16, dev)
    tables = torch.tensor([[0, 1], [2, 3], [4, 5]], dtype=torch.int32)
    pool.gpu[3][0, 3, 1, 2] = 255  # V, sequence 0, head 1, elements 64 .. 95
    pool.gpu[2][2, 3, 0, 1] = 255  # K, sequence 1, head 0
    (kc, vc), kw = pool.args()
    q = torch.randn(3, 4, 128, generator=gen).to(BF16)
    q[2, 3, 7] = math.inf
    out = ops.paged_decode(q.to(dev), kc, vc, tables.to(dev), torch.tensor([20, 20, 20], device=dev),
                           max_seq_len=20, scale=0.1, **kw).cpu()
    assert out[0, 2:, 64:96].isnan().all() and out[0, 2:, :64].isfinite().all() and out[0, :2].isfinite().all()
    assert out[1, :2].isnan().all() and out[1, 2:].isfinite().all()
    assert out[2, 3].isnan().all() and out[2, :3].isfinite().all()


@pytest.mark.parametrize("d, hq, hkv, dtype", [(128, 16, 8, BF16), (64, 8, 2, F16), (256, 8, 1, BF16)])
@pytest.mark.parametrize("split", [0, 256])
def test_decode_prologue_is_the_standalone_one(dev, d, hq, hkv, dtype, split):
    lens = [1, 17, 300, 700]
    gen = torch.Generator().manual_seed(21)
    blocks = sum(-(-n // 16) for n in lens)
    one, two = (Pool(torch.Generator().manual_seed(3), blocks, 16, hkv, d, "nhd", dtype, dev) for _ in range(2))
    tables = tables_for(gen, lens, 16, blocks).to(dev)
    q, k, v = (torch.randn(4, n, d, generator=gen).to(dtype).to(dev) for n in (hq, hkv, hkv))
    pro = ops.QKPrologue(torch.rand(d, generator=gen).to(dtype).to(dev), torch.rand(d, generator=gen).to(dtype).to(dev),
                         1e-6, torch.randn(800, d, generator=gen).to(dev),
                         torch.tensor([n - 1 for n in lens], device=dev))
    kw = {"max_seq_len": 700, "scale": d ** -0.5, "split_tokens": split}
    vec = torch.tensor(lens, device=dev)
    (kc, vc), more = one.args()
    got = ops.paged_decode(q, kc, vc, tables, vec, new_k=k, new_v=v, prologue=pro, **kw, **more)
    qn, kn = ops.qk_norm_rope(q, k, pro)
    (kc, vc), more = two.args()
    want = ops.paged_decode(qn, kc, vc, tables, vec, new_k=kn, new_v=v, **kw, **more)
    assert torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(one.gpu, two.gpu))


def test_decode_pool_past_4_gib(dev):
    # Codes and scales of one pool past 2^32 bytes: blocks at its far end.
    blocks, hkv, d = 540000, 8, 128
    codes = torch.empty(2, blocks, 16, hkv, d // 2, dtype=torch.uint8, device=dev)
    scales = torch.empty(2, blocks, 16, hkv, d // 32, dtype=torch.uint8, device=dev)
    gen = torch.Generator().manual_seed(22)
    small = Pool(gen, 6, 16, hkv, d, "nhd", BF16, dev)
    at = torch.tensor([blocks - 1, 3, blocks - 7, 530000, 0, blocks - 2], device=dev)
    for i in range(2):
        codes[i, at], scales[i, at] = small.gpu[i], small.gpu[2 + i]
    q = torch.randn(2, 16, d, generator=gen).to(BF16).to(dev)
    near = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=dev)
    (kc, vc), kw = small.args()
    lens = torch.tensor([48, 41], device=dev)
    want = ops.paged_decode(q, kc, vc, near, lens, max_seq_len=48, scale=0.1, **kw)
    far = {"k_scale": scales[0].view(ops.MXFP4_SCALE_DTYPE), "v_scale": scales[1].view(ops.MXFP4_SCALE_DTYPE)}
    big = (codes[0].view(ops.MXFP4_KV_DTYPE), codes[1].view(ops.MXFP4_KV_DTYPE))
    got = ops.paged_decode(q, *big, at[near.long()].int(), lens, max_seq_len=48, scale=0.1, **far)
    assert torch.equal(got, want)
    cq = torch.tensor([0, 16, 25], dtype=torch.int32, device=dev)
    ck = torch.tensor([0, 48, 89], dtype=torch.int32, device=dev)
    qp = torch.randn(25, 16, d, generator=gen).to(BF16).to(dev)
    a = ops.varlen_attention(qp, None, None, cq, ck, 16, 48, scale=0.1, causal=True, k_cache=big[0],
                             v_cache=big[1], block_tables=at[near.long()].int(), **far)
    b = ops.varlen_attention(qp, None, None, cq, ck, 16, 48, scale=0.1, causal=True, k_cache=kc, v_cache=vc,
                             block_tables=near, **kw)
    assert torch.equal(a, b)
    # (stored last: these slots lie in blocks that the calls above read)
    rows = torch.randn(3, hkv, d, generator=gen).to(BF16).to(dev)
    slots = torch.tensor([blocks * 16 - 1, 5, blocks * 16 - 20], dtype=torch.int64, device=dev)
    ops.store_kvcache(rows, rows, *big, slots, **far)
    k, v = ops.load_kvcache(*big, slots, BF16, **far)
    c, s = oracle.quantise(rows.cpu())
    assert torch.equal(k.double().cpu(), oracle.values(c, s)) and torch.equal(k, v)


def test_decode_on_a_side_stream_and_captured(dev):
    gen = torch.Generator().manual_seed(23)
    lens = [3000, 17, 900, 1]
    blocks = sum(-(-n // 16) for n in lens) + 2
    pool = Pool(gen, blocks, 16, 2, 128, "nhd", BF16, dev)
    (kc, vc), kw = pool.args()
    tables = tables_for(gen, lens, 16, blocks).to(dev)
    vec = torch.tensor(lens, device=dev)
    q = torch.randn(4, 8, 128, generator=gen).to(BF16).to(dev)
    nk, nv = (torch.randn(4, 2, 128, generator=gen).to(BF16).to(dev) for _ in range(2))

    def call(out=None):
        return ops.paged_decode(q, kc, vc, tables, vec, max_seq_len=32768, scale=0.1, new_k=nk, new_v=nv,
                                out=out, **kw)

    want = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    outs = [torch.empty_like(q) for _ in range(2)]
    graphs = []
    for out in outs:  # two graphs, which share the capture stream's workspace
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(out)
        graphs.append(g)
    for i in range(3):
        q.copy_(torch.randn(4, 8, 128, generator=gen).to(BF16))
        nk.copy_(torch.randn(4, 2, 128, generator=gen).to(BF16))
        vec.copy_(torch.tensor([3000 - 7 * i, 17, 900 - i, 1 + i]))
        for out in outs:
            out.fill_(7)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = call()
        assert torch.equal(got[0], want) and torch.equal(got[1], want)


# --------------------------------------------------------------------- varlen
def run_varlen(dev, prefixes, qlens, *, hq=16, hkv=8, d=128, block=16, layout="nhd", dtype=BF16, seed=0,
               causal=True, fresh=True, table_dtype=torch.int32, tail=0, edit=None):
    gen = torch.Generator().manual_seed(seed)
    klens = [p + m for p, m in zip(prefixes, qlens)]
    total = sum(qlens) + tail  # rows behind the last sequence
    blocks = sum(-(-n // block) for n in klens) + 3
    pool = Pool(gen, blocks, block, hkv, d, layout, dtype, dev)
    tables = tables_for(gen, klens, block, blocks, table_dtype)
    if edit:
        edit(pool, tables)
        pool.gpu = [t.to(dev) for t in pool.cpu]
    qkv = torch.randn(total, hq + 2 * hkv, d, generator=gen).to(dtype)
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
    slots = torch.full((total,), -1, dtype=table_dtype)
    at = 0
    for b, (p, m) in enumerate(zip(prefixes, qlens)):
        slots[at:at + m] = slots_of(tables[b], p + m, block)[p:].to(table_dtype)
        at += m
    (kc, vc), kw = pool.args()
    gpu = qkv.to(dev)
    out = torch.full((total, hq, d), 5.0, dtype=dtype, device=dev)
    ops.varlen_attention(gpu[:, :hq], gpu[:, hq:hq + hkv] if fresh else None,
                         gpu[:, hq + hkv:] if fresh else None, cu(qlens).to(dev), cu(klens).to(dev),
                         max(qlens), max(klens), scale=d ** -0.5, causal=causal, k_cache=kc, v_cache=vc,
                         block_tables=tables.to(dev), slot_mapping=slots.to(dev) if fresh else None,
                         out=out, **kw)
    torch.cuda.synchronize()
    at = 0
    for b, (p, m, n) in enumerate(zip(prefixes, qlens, klens)):
        if m == 0:
            continue
        pos = torch.arange(n)
        blk = tables[b].long()[pos // block]
        ok = (blk >= 0) & (blk < blocks)
        kk, vv = pool.rows(blk.clamp(0, blocks - 1) * block + pos % block)
        kk[~ok], vv[~ok] = 0, 0  # rows of a block outside the pool read as zeros
        if fresh:
            kk[p:], vv[p:] = k[at:at + m].double(), v[at:at + m].double()
        seen = pos <= torch.arange(p, n)[:, None] if causal else torch.ones(m, n, dtype=torch.bool)
        ref, tol = oracle.attend(q[at:at + m], kk, vv, seen, d ** -0.5, dtype, VARLEN_BITS)
        close(out[at:at + m], ref, tol)
        at += m
    assert (out[at:] == 5.0).all()
    if fresh:
        oracle.store(k, v, pool.cpu, slots, block, layout)
    assert pool.same()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("hq, hkv, d", [(16, 8, 128), (8, 1, 128), (4, 4, 64), (8, 2, 64)])
@pytest.mark.parametrize("layout, block", [("nhd", 16), ("hnd", 48)])
def test_varlen(dev, dtype, hq, hkv, d, layout, block):
    run_varlen(dev, [0, 1, 16, 63, 64, 100, 257, 40], [5, 1, 17, 64, 1, 70, 130, 0], hq=hq, hkv=hkv, d=d,
               dtype=dtype, layout=layout, block=block, seed=d + hq, tail=3)


@pytest.mark.parametrize("d, hq, hkv", [(128, 16, 8), (64, 8, 1), (128, 4, 4)])
@pytest.mark.parametrize("prefixes, qlens", [([5000], [40]), ([3000, 10, 700], [20, 300, 1]),
                                             ([0, 0], [333, 20]), ([2048] * 3, [1, 1, 1])])
def test_varlen_long_prefixes(dev, d, hq, hkv, prefixes, qlens):
    run_varlen(dev, prefixes, qlens, hq=hq, hkv=hkv, d=d, seed=len(prefixes))


@pytest.mark.parametrize("causal", [True, False])
def test_varlen_all_from_the_pool(dev, causal):
    run_varlen(dev, [0, 30, 200], [20, 3, 100], fresh=False, causal=causal, seed=2, table_dtype=torch.int64)


def test_varlen_not_causal(dev):
    run_varlen(dev, [0, 100, 64], [70, 30, 64], causal=False, seed=3)


def test_varlen_blocks_outside_the_pool(dev):
    def edit(pool, tables):
        tables[0, 2] = -1
        tables[1, 0] = 10 ** 6

    run_varlen(dev, [150, 90], [40, 10], edit=edit, seed=4)


@pytest.mark.parametrize("d, hq, hkv", [(128, 8, 2), (64, 4, 1)])
def test_varlen_dead_places_hold_anything(dev, d, hq, hkv):
    # NaN groups in every place that no prefix row holds, the ends of the
    # prefixes' last blocks (inside a tile) among them.
    prefixes = [1, 70, 0, 129]

    def edit(pool, tables):
        live = torch.zeros(pool.cpu[0].shape[0] * 16, dtype=torch.bool)
        for b, n in enumerate(prefixes):
            live[slots_of(tables[b], n, 16)] = True
        for t in (2, 3):
            pool.cpu[t].flatten(0, 1)[~live] = 255
        for t in (0, 1):
            pool.cpu[t].flatten(0, 1)[~live] = 0x7f

    run_varlen(dev, prefixes, [3, 40, 20, 1], hq=hq, hkv=hkv, d=d, edit=edit, seed=5)


# ------------------------------------------------------- heads, views, streams
@pytest.mark.parametrize("hq, hkv, d", [(14, 7, 64), (3, 3, 64), (6, 3, 128), (5, 5, 256)])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_odd_head_counts(dev, hq, hkv, d, layout):
    # At head_dim 64 every second row's scales start inside a word.
    run_decode(dev, [1, 33, 200, 16], hq=hq, hkv=hkv, d=d, layout=layout, new=True, seed=hkv)
    if d <= 128:
        run_varlen(dev, [0, 33, 100], [5, 3, 70], hq=hq, hkv=hkv, d=d, layout=layout, seed=hkv)


@pytest.mark.parametrize("shift", [-100, 100])
def test_scales_of_any_size(dev, shift):
    # Key groups near both ends of the scales' range.
    def edit(pool, tables):
        pool.cpu[2] = (pool.cpu[2].int() + shift).clamp(2, 252).to(torch.uint8)

    run_decode(dev, [40, 300], edit=edit, scale=128 ** -0.5 * 2.0 ** -shift, seed=30)


@pytest.mark.parametrize("d", [64, 128])
def test_pools_inside_larger_tensors(dev, d):
    """Keys and values side by side in one tensor a block, and a pool whose heads
    and slots are transposed: the same results as from a pool of their own."""
    gen = torch.Generator().manual_seed(31)
    blocks, hkv, n = 12, 2, 90
    own = Pool(gen, blocks, 16, hkv, d, "nhd", BF16, dev)
    both = [torch.zeros(blocks, 2, 16, hkv, w, dtype=torch.uint8, device=dev) for w in (d // 2, d // 32)]
    turned = [torch.zeros(2, blocks, hkv, 16, w, dtype=torch.uint8, device=dev).transpose(2, 3)
              for w in (d // 2, d // 32)]
    table = torch.randperm(blocks, generator=gen)[:6].int()[None].to(dev)
    slots = slots_of(table[0].cpu(), n, 16).to(dev)
    rows = [torch.randn(n, hkv, d, generator=gen).to(BF16).to(dev) for _ in range(2)]
    new = [torch.randn(1, hkv, d, generator=gen).to(BF16).to(dev) for _ in range(2)]
    q = torch.randn(40, 8, d, generator=gen).to(BF16).to(dev)

    def run(kc, vc, ks, vs):
        kc, vc = (t.view(ops.MXFP4_KV_DTYPE) for t in (kc, vc))
        kw = {"k_scale": ks.view(ops.MXFP4_SCALE_DTYPE), "v_scale": vs.view(ops.MXFP4_SCALE_DTYPE)}
        ops.store_kvcache(rows[0], rows[1], kc, vc, slots, **kw)
        loaded = ops.load_kvcache(kc, vc, slots, **kw)
        one = ops.paged_decode(q[:1], kc, vc, table, torch.tensor([n + 1], device=dev), max_seq_len=n + 1,
                               scale=0.1, new_k=new[0], new_v=new[1], **kw)
        cq, ck = cu([40]).to(dev), cu([n]).to(dev)
        many = ops.varlen_attention(q, None, None, cq, ck, 40, n, scale=0.1, causal=True, k_cache=kc,
                                    v_cache=vc, block_tables=table, **kw)
        return (*loaded, one, many, *(t[slots // 16, slots % 16] for t in (kc.view(torch.uint8), ks.view(torch.uint8))))

    want = run(own.gpu[0], own.gpu[1], own.gpu[2], own.gpu[3])
    for c, s in ((both[0].unbind(1), both[1].unbind(1)), (turned[0], turned[1])):
        for a, b in zip(run(c[0], c[1], s[0], s[1]), want):
            assert torch.equal(a, b)


def test_wrappers_refuse(dev):
    k, v, ks, vs = ops.mxfp4_kv_pool(4, 16, 2, 128, device=dev)
    kw = {"k_scale": ks, "v_scale": vs}
    x = torch.zeros(3, 2, 128, dtype=BF16, device=dev)
    q = torch.zeros(3, 4, 128, dtype=BF16, device=dev)
    slots = torch.zeros(3, dtype=torch.int32, device=dev)
    table = torch.zeros(3, 2, dtype=torch.int32, device=dev)
    vec = cu([1, 1, 1]).to(dev)

    def store(x=x, k=k, v=v, **more):
        ops.store_kvcache(x, x, k, v, slots, **{**kw, **more})

    def load(k=k, v=v, slots=slots, dtype=BF16, **more):
        ops.load_kvcache(k, v, slots, dtype, **{**kw, **more})

    def decode(q=q, k=k, v=v, **more):
        ops.paged_decode(q, k, v, table, vec, lens_cumulative=True, max_seq_len=20, scale=1.0, **{**kw, **more})

    def varlen(q=q, k=k, v=v, **more):
        ops.varlen_attention(q, None, None, vec, vec, 1, 1, scale=1.0, causal=True, k_cache=k, v_cache=v,
                             block_tables=table, **{**kw, **more})

    wide = torch.zeros(4, 16, 2, 128, dtype=BF16, device=dev)
    odd = [t[:, :, :1] for t in (ks, vs)]
    small = ops.mxfp4_kv_pool(4, 8, 2, 128, device=dev)
    calls = [lambda f=f, m=m: f(**m) for f in (store, load, decode, varlen) for m in (
        {"k_scale": 1.0, "v_scale": 1.0}, {"v_scale": 1.0}, {"k_scale": ks.view(torch.uint8)},
        {"k_scale": odd[0], "v_scale": odd[1]}, {"k": wide, "v": wide}, {"k_scale": ks.cpu(), "v_scale": vs.cpu()},
        {"layout": "dhn"})]
    calls += [lambda: store(x=x.float()), lambda: load(dtype=torch.float32), lambda: decode(q=q.float()),
              lambda: varlen(q=q.float()), lambda: load(slots=slots[None]),
              lambda: decode(no_alloc=True, out=torch.empty_like(q)), lambda: decode(q=q[:, :3]),
              lambda: decode(k=small[0], v=small[1], k_scale=small[2], v_scale=small[3]),
              lambda: varlen(k=small[0], v=small[1], k_scale=small[2], v_scale=small[3]),
              lambda: decode(q=torch.zeros(3, 6, 128, dtype=BF16, device=dev))]
    for i, call in enumerate(calls):
        with pytest.raises((ops.AttentionArgumentError, NativeError, TypeError)):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()


def test_two_streams_at_once(dev):
    gen = torch.Generator().manual_seed(33)
    lens = [5000, 300, 20]
    pool = Pool(gen, 340, 16, 2, 128, "nhd", BF16, dev)
    (kc, vc), kw = pool.args()
    tables = tables_for(gen, lens, 16, 340).to(dev)
    vec = torch.tensor(lens, device=dev)
    qs = [torch.randn(3, 8, 128, generator=gen).to(BF16).to(dev) for _ in range(4)]

    def call(q):
        return ops.paged_decode(q, kc, vc, tables, vec, max_seq_len=5000, scale=0.1, **kw)

    want = [call(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i, q in enumerate(qs * 3):
        with torch.cuda.stream(streams[i % 2]):
            got.append(call(q))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_layer_without_the_fused_store(dev, layout):
    """The layer's unfused path (store, then attention over the pool) against its
    fused one: a decode step is the same; a prompt then attends its rows as stored."""
    gen = torch.Generator().manual_seed(34)
    hq, hkv, d, block = 8, 2, 128, 16
    outs, pools = [], []
    lens = [20, 35]
    pre = torch.randn(55, hq + 2 * hkv, d, generator=gen).to(BF16)
    step = torch.randn(2, hq + 2 * hkv, d, generator=gen).to(BF16)
    tables = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32)
    for fused in (True, False):
        layer = PagedAttention(hq, d, d ** -0.5, hkv)
        pool = ops.mxfp4_kv_pool(6, block, hkv, d, device=dev, layout=layout)
        layer.kv_layout, layer.fuse_store = layout, fused
        layer.k_cache, layer.v_cache, layer.k_scale, layer.v_scale = pool
        for qkv, q, k in ((pre, lens, lens), (step, [1, 1], [21, 36])):
            slots = torch.cat([slots_of(t, n, block)[n - m:] for t, n, m in zip(tables, k, q)])
            gpu = qkv.to(dev)
            with attention_context(AttentionContext(
                    cu_seqlens_q=cu(q).to(dev), cu_seqlens_k=cu(k).to(dev), max_seqlen_q=max(q),
                    max_seqlen_k=max(k), slot_mapping=slots.int().to(dev), block_tables=tables.to(dev))):
                out = layer(gpu[:, :hq], gpu[:, hq:hq + hkv], gpu[:, hq + hkv:])
            outs.append(out)
        pools.append([t.view(torch.uint8).cpu() for t in pool])
    assert all(torch.equal(a, b) for a, b in zip(*pools))
    assert torch.equal(outs[1], outs[3])
    at = 0
    for n in lens:  # the unfused prompt
        q = pre[at:at + n, :hq]
        k, v = (oracle.values(*oracle.quantise(pre[at:at + n, i:i + hkv])) for i in (hq, hq + hkv))
        seen = torch.ones(n, n).tril().bool()
        ref, tol = oracle.attend(q, k, v, seen, d ** -0.5, BF16, VARLEN_BITS)
        close(outs[2][at:at + n], ref, tol)
        at += n


def test_qwen3_core_over_an_mxfp4_pool(dev):
    """The fused decode step is the standalone prologue and the plain layer's step."""
    gen = torch.Generator().manual_seed(35)
    hq, hkv, d, block = 16, 8, 128, 16
    k_lens = [21, 36]
    tables = torch.tensor([[4, 1, 0], [2, 5, 3]], dtype=torch.int32)
    x = torch.randn(2, hq + 2 * hkv, d, generator=gen).to(BF16).to(dev)
    positions = torch.tensor([20, 35], device=dev)
    slots = torch.cat([slots_of(t, n, block)[-1:] for t, n in zip(tables, k_lens)]).int().to(dev)
    context = AttentionContext(cu_seqlens_q=cu([1, 1]).to(dev), cu_seqlens_k=cu(k_lens).to(dev),
                               max_seqlen_q=1, max_seqlen_k=36, slot_mapping=slots,
                               block_tables=tables.to(dev))
    got = []
    for core in (True, False):
        pool = Pool(torch.Generator().manual_seed(36), 6, block, hkv, d, "nhd", BF16, dev)
        (kc, vc), kw = pool.args()
        layer = Qwen3AttentionCore(hq, d, hkv, max_position=64).to(dev)
        layer.k_cache, layer.v_cache, layer.k_scale, layer.v_scale = kc, vc, kw["k_scale"], kw["v_scale"]
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        with attention_context(context):
            if core:
                out = layer(positions, q, k, v)
            else:
                qn, kn = ops.qk_norm_rope(q, k, layer.prologue(positions))
                out = PagedAttention.forward(layer, qn, kn, v)
        got.append((out.reshape(2, -1), pool.gpu))
    assert torch.equal(got[0][0], got[1][0])
    assert all(torch.equal(a, b) for a, b in zip(got[0][1], got[1][1]))


# ------------------------------- decode of long contexts, two heads a workgroup
@pytest.mark.parametrize("dtype, hq, hkv", [(BF16, 4, 2), (F16, 2, 2), (BF16, 16, 2)])
@pytest.mark.parametrize("new", [False, True])
def test_decode_two_long_contexts(dev, dtype, hq, hkv, new):
    run_decode(dev, [16500, 16420], hq=hq, hkv=hkv, dtype=dtype, split=ops.SPLIT_EXACT, new=new, seed=40)


@pytest.mark.parametrize("dtype, hq, hkv, split", [(BF16, 8, 2, 0), (F16, 32, 4, 0), (BF16, 4, 4, 300), (BF16, 16, 8, 0)])
@pytest.mark.parametrize("mask", [False, True])
def test_decode_many_contexts_under_a_bound(dev, dtype, hq, hkv, split, mask):
    # Lengths from none to several partitions; the current rows at their ends.
    lens = [0, 1, 31, 32, 33, 127, 128, 129, 1300, 2500] + [16 * i + 5 for i in range(20)]
    gen = torch.Generator().manual_seed(41)
    m = torch.rand(30, 1400, generator=gen) > 0.3 if mask else None
    if mask:
        m[5] = False
    run_decode(dev, lens, hq=hq, hkv=hkv, dtype=dtype, bound=32768, split=split, new=True, mask=m, seed=42)


def test_decode_pairs_agree_with_single_heads(dev):
    """A pool of 128-byte rows of head pairs against the same rows head-major,
    with the prologue, the current row and two replays of one graph."""
    gen = torch.Generator().manual_seed(43)
    lens = [3000, 17, 900, 1] * 8
    blocks = sum(-(-n // 16) for n in lens)
    pool = Pool(gen, blocks, 16, 2, 128, "nhd", BF16, dev)
    hnd = [t.transpose(1, 2).contiguous() for t in pool.gpu]
    tables = tables_for(gen, lens, 16, blocks).to(dev)
    q, k, v = (torch.randn(32, n, 128, generator=gen).to(BF16).to(dev) for n in (8, 2, 2))
    pro = ops.QKPrologue(torch.rand(128, generator=gen).to(BF16).to(dev),
                         torch.rand(128, generator=gen).to(BF16).to(dev), 1e-6,
                         torch.randn(3000, 128, generator=gen).to(dev),
                         torch.tensor([n - 1 for n in lens], device=dev))
    vec = torch.tensor(lens, device=dev)

    def call(pools, layout, out=None):
        kc, vc = (t.view(ops.MXFP4_KV_DTYPE) for t in pools[:2])
        ks, vs = (t.view(ops.MXFP4_SCALE_DTYPE) for t in pools[2:])
        return ops.paged_decode(q, kc, vc, tables, vec, max_seq_len=32768, scale=0.08, new_k=k, new_v=v,
                                prologue=pro, layout=layout, k_scale=ks, v_scale=vs, out=out)

    one, two = call(hnd, "hnd"), call(pool.gpu, "nhd")
    # (partitions differ, so sums are in another order: half a step of the
    # output each, and P's and the sums' rounding, at values below 4)
    assert (one.float() - two.float()).abs().max() <= 2 * 2.0 ** -8 * 4 + 2 * 2.0 ** -8 * 4
    assert all(torch.equal(a, b.transpose(1, 2)) for a, b in zip(hnd, pool.gpu))
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(pool.gpu, "nhd", out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pool.gpu, "nhd", out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, two)


@pytest.mark.parametrize("hq, hkv, lens", [(16, 8, [2000] * 8), (16, 2, [16500, 30]), (8, 8, [1500] * 31)])
@pytest.mark.parametrize("split", [0, ops.SPLIT_EXACT])
def test_reserved_workspace_holds_every_automatic_split(dev, hq, hkv, lens, split):
    gen = torch.Generator().manual_seed(44)
    blocks = sum(-(-n // 16) for n in lens)
    pool = Pool(gen, blocks, 16, hkv, 128, "nhd", BF16, dev)
    (kc, vc), kw = pool.args()
    tables = tables_for(gen, lens, 16, blocks).to(dev)
    q = torch.randn(len(lens), hq, 128, generator=gen).to(BF16).to(dev)
    vec = torch.tensor(lens, device=dev)
    stream = torch.cuda.Stream()
    ops.reserve_decode_workspace(dev, hq, hkv, 128, stream=stream)
    key = (dev.index or 0, stream.cuda_stream)
    before = ops._WORKSPACES[key]
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        ops.paged_decode(q, kc, vc, tables, vec, max_seq_len=max(lens) if split else 32768, scale=0.1,
                         split_tokens=split, **kw)
    torch.cuda.synchronize()
    assert ops._WORKSPACES[key] is before


def test_fp8_pools_take_scales_of_one_number_as_tensors(dev):
    gen = torch.Generator().manual_seed(45)
    rows = [torch.randn(40, 2, 128, generator=gen).to(BF16).to(dev) for _ in range(2)]
    q = torch.randn(40, 4, 128, generator=gen).to(BF16).to(dev)
    slots = torch.arange(40, dtype=torch.int32, device=dev)
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev)
    lens, cu40 = torch.tensor([40], device=dev), cu([40]).to(dev)
    got = []
    for scale in (0.5, torch.tensor(0.5), torch.tensor([0.5], device=dev)):
        kc, vc = (torch.zeros(4, 16, 2, 128, dtype=torch.uint8, device=dev).view(ops.FP8_KV_DTYPE)
                  for _ in range(2))
        kw = {"k_scale": scale, "v_scale": scale}
        ops.store_kvcache(rows[0], rows[1], kc, vc, slots, **kw)
        one = ops.paged_decode(q[:1], kc, vc, table, lens, max_seq_len=40, scale=0.1, **kw)
        many = ops.varlen_attention(q, None, None, cu40, cu40, 40, 40, scale=0.1, causal=True, k_cache=kc,
                                    v_cache=vc, block_tables=table, **kw)
        got.append((kc.view(torch.uint8), one, many))
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


@pytest.mark.parametrize("d, split", [(64, 256), (128, 0)])
def test_decode_of_more_workgroups_than_a_flat_grid_holds(dev, d, split):
    # 65535 sequences of one token each; at split 256 a bound of 8192 makes 16.8 M workgroups.
    n, hkv = 65535, 8
    k, v, ks, vs = ops.mxfp4_kv_pool(2, 16, hkv, d, device=dev)
    gen = torch.Generator().manual_seed(46)
    rows = [torch.randn(1, hkv, d, generator=gen).to(BF16).to(dev) for _ in range(2)]
    slot = torch.tensor([16], dtype=torch.int32, device=dev)
    ops.store_kvcache(rows[0], rows[1], k, v, slot, k_scale=ks, v_scale=vs)
    _, want = ops.load_kvcache(k, v, slot, k_scale=ks, v_scale=vs)
    q = torch.randn(1, hkv, d, generator=gen).to(BF16).to(dev).expand(n, hkv, d)
    table = torch.ones(1, 512, dtype=torch.int32, device=dev).expand(n, 512)
    out = torch.zeros(n, hkv, d, dtype=BF16, device=dev)
    ops.paged_decode(q, k, v, table, torch.ones(n, dtype=torch.int32, device=dev), max_seq_len=8192, scale=0.1,
                     split_tokens=split, out=out, k_scale=ks, v_scale=vs)
    assert torch.equal(out, want.expand(n, hkv, d))


@pytest.mark.parametrize("d, prefixes, qlens", [(128, [3000, 10, 700], [20, 300, 1]), (64, [2000, 0], [40, 64])])
def test_a_captured_step_replays(dev, d, prefixes, qlens):
    """Store, varlen attention with the fused store and load in one graph: each
    replay, on other rows, is the eager calls' result."""
    gen = torch.Generator().manual_seed(47)
    hq, hkv = 8, 2
    klens = [p + m for p, m in zip(prefixes, qlens)]
    total, blocks = sum(qlens), sum(-(-n // 16) for n in klens)
    pool = Pool(gen, blocks, 16, hkv, d, "nhd", BF16, dev)
    (kc, vc), kw = pool.args()
    tables = tables_for(gen, klens, 16, blocks)
    slots = torch.cat([slots_of(t, n, 16)[p:] for t, n, p in zip(tables, klens, prefixes)]).int().to(dev)
    tables, cq, ck = tables.to(dev), cu(qlens).to(dev), cu(klens).to(dev)
    x = torch.randn(total, hq + 2 * hkv, d, generator=gen).to(BF16).to(dev)
    first = torch.tensor([slots_of(tables[0].cpu(), 5, 16)[i] for i in range(5)], device=dev)

    def step():
        k, v = x[:, hq:hq + hkv], x[:, hq + hkv:]
        ops.store_kvcache(k[:5], v[:5], kc, vc, first, **kw)  # new rows of the first prefix
        out = ops.varlen_attention(x[:, :hq], k, v, cq, ck, max(qlens), max(klens), scale=d ** -0.5,
                                   causal=True, k_cache=kc, v_cache=vc, block_tables=tables,
                                   slot_mapping=slots, **kw)
        return (out, *ops.load_kvcache(kc, vc, slots, **kw))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(3):
        x.copy_(torch.randn(total, hq + 2 * hkv, d, generator=gen).to(BF16))
        graph.replay()
        mine = [t.clone() for t in got]
        state = [t.clone() for t in pool.gpu]
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(mine, want))
        assert all(torch.equal(a, b) for a, b in zip(state, pool.gpu))


def test_varlen_over_a_16_bit_pool_reads_no_scales(dev):
    """k_scale / v_scale belong to FP8 and MXFP4 pools: over a 16-bit pool a tensor
    of any size, on any device, changes nothing and is not waited for."""
    gen = torch.Generator().manual_seed(49)
    kc, vc = (torch.randn(4, 16, 2, 128, generator=gen).to(BF16).to(dev) for _ in range(2))
    q = torch.randn(40, 4, 128, generator=gen).to(BF16).to(dev)
    table = torch.tensor([[0, 2, 1]], dtype=torch.int32, device=dev)
    c40 = cu([40]).to(dev)

    def call(prologue=None, **kw):
        return ops.varlen_attention(q, None, None, c40, c40, 40, 40, scale=0.1, causal=True, k_cache=kc,
                                    v_cache=vc, block_tables=table, prologue=prologue, **kw)

    pro = ops.QKPrologue(*(torch.ones(128, dtype=BF16, device=dev) for _ in range(2)), 1e-6,
                         torch.ones(64, 128, device=dev), torch.arange(40, device=dev))
    want = call(), call(pro)
    for scale in (2.0, None, torch.full((3,), 2.0, device=dev), torch.tensor(2.0, device=dev), torch.ones(2, 2)):
        mode = torch.cuda.get_sync_debug_mode()
        torch.cuda.set_sync_debug_mode("error")
        try:
            got = call(k_scale=scale, v_scale=scale), call(pro, k_scale=scale, v_scale=scale)
        finally:
            torch.cuda.set_sync_debug_mode(mode)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_load_refuses_scales_that_are_no_tensors(dev):
    k, v, ks, vs = ops.mxfp4_kv_pool(4, 16, 2, 128, device=dev)
    slots = torch.zeros(3, dtype=torch.int32, device=dev)
    for k_scale, v_scale in ((1.0, 1.0), (ks, 1.0), (None, vs)):
        with pytest.raises(ops.AttentionArgumentError):
            ops.load_kvcache(k, v, slots, k_scale=k_scale, v_scale=v_scale)


def test_workspaces_of_other_pools_keep_their_size(dev):
    """Two partitions a compute unit are an MXFP4 pool's at head_dim 128 with an even
    number of kv heads; other decodes allocate for one."""
    cus = torch.cuda.get_device_properties(dev).multi_processor_count
    one = (cus * 2 * 2 * 4 + 255) // 256 * 256 + cus * 2 * 128 * 4
    kc, vc = (torch.zeros(128, 16, 2, 128, dtype=BF16, device=dev) for _ in range(2))
    q = torch.zeros(1, 4, 128, dtype=BF16, device=dev)
    table = torch.arange(128, dtype=torch.int32, device=dev)[None]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    key = (dev.index or 0, stream.cuda_stream)
    if key in ops._WORKSPACES:  # another test's, whose graph may hold it
        ops._RETIRED.append(ops._WORKSPACES.pop(key))
    with torch.cuda.stream(stream):
        ops.paged_decode(q, kc, vc, table, torch.tensor([2048], device=dev), max_seq_len=2048, scale=0.1)
    torch.cuda.synchronize()
    assert ops._WORKSPACES[key].numel() == one
    assert ops.decode_workspace_bound(dev, 4, 2, 128, BF16) == one
    assert ops.decode_workspace_bound(dev, 4, 2, 128, ops.MXFP4_KV_DTYPE) > one
    for shape in ((4, 2, 64), (6, 3, 128)):
        both = [ops.decode_workspace_bound(dev, *shape, t) for t in (BF16, ops.MXFP4_KV_DTYPE)]
        assert both[0] == both[1]
    assert ops.decode_workspace_bound(dev, 4, 2, 128) == one


def test_qwen3_core_splits_as_the_plain_layer_does(dev):
    """An eager step that says its exact longest context: the fused step's partitions
    are those of the plain layer's, so the outputs are the same bits."""
    gen = torch.Generator().manual_seed(50)
    hq, hkv, d, block = 16, 8, 128, 16
    k_lens = [9000, 5000, 8100]
    blocks = sum(-(-n // block) for n in k_lens)
    tables = tables_for(gen, k_lens, block, blocks)
    x = torch.randn(3, hq + 2 * hkv, d, generator=gen).to(BF16).to(dev)
    positions = torch.tensor([n - 1 for n in k_lens], device=dev)
    slots = torch.cat([slots_of(t, n, block)[-1:] for t, n in zip(tables, k_lens)]).int().to(dev)
    context = AttentionContext(cu_seqlens_q=cu([1, 1, 1]).to(dev), cu_seqlens_k=cu(k_lens).to(dev), max_seqlen_q=1,
                               max_seqlen_k=9000, slot_mapping=slots, block_tables=tables.to(dev),
                               max_seqlen_k_exact=True)
    got = []
    for core in (True, False):
        pool = Pool(torch.Generator().manual_seed(51), blocks, block, hkv, d, "nhd", BF16, dev)
        (kc, vc), kw = pool.args()
        layer = Qwen3AttentionCore(hq, d, hkv, max_position=9000).to(dev)
        layer.k_cache, layer.v_cache, layer.k_scale, layer.v_scale = kc, vc, kw["k_scale"], kw["v_scale"]
        q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
        with attention_context(context):
            if core:
                out = layer(positions, q, k, v)
            else:
                qn, kn = ops.qk_norm_rope(q, k, layer.prologue(positions))
                out = PagedAttention.forward(layer, qn, kn, v)
        got.append(out.reshape(3, -1))
    assert torch.equal(got[0], got[1])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d, hq, hkv, layout, lens", [(128, 16, 8, "nhd", [40, 300]), (64, 8, 2, "hnd", [40, 300]),
                                                      (256, 4, 2, "nhd", [40, 300]),
                                                      (128, 4, 2, "nhd", [16500, 16420])])
def test_decode_keeps_small_terms_beside_large_ones(dev, dtype, d, hq, hkv, layout, lens):
    """Two channels of the query far larger than the rest, whose products cancel in
    every key: what is left is the other channels' sum.  Q K^T is summed in float32,
    so a logit is off by at most 2^-17 of its products' magnitudes (d additions of a
    step of 2^-24 each, and room), 2^-17 * 2 * 6 * 1024 * scale = 0.01 at d = 64."""
    gen = torch.Generator().manual_seed(48)
    blocks = sum(-(-n // 16) for n in lens)
    pool = Pool(gen, blocks, 16, hkv, d, layout, dtype, dev)
    pool.cpu[0][..., 0] = 7 + 16 * 15  # elements 0 and 1 of every key: 6 and -6
    pool.cpu[2][:] = 127
    pool.gpu = [t.to(dev) for t in pool.cpu]
    tables = tables_for(gen, lens, 16, blocks)
    q = torch.randn(len(lens), hq, d, generator=gen)
    q[..., :2] = 1024.0
    q = q.to(dtype)
    (kc, vc), kw = pool.args()
    scale = d ** -0.5
    out = ops.paged_decode(q.to(dev), kc, vc, tables.to(dev), torch.tensor(lens, device=dev), max_seq_len=max(lens),
                           scale=scale, split_tokens=ops.SPLIT_EXACT, **kw)
    for b, n in enumerate(lens):
        k, v = pool.rows(slots_of(tables[b], n, 16))
        ref, tol = oracle.attend(q[b:b + 1], k, v, torch.ones(1, n, dtype=torch.bool), scale, dtype, VARLEN_BITS)
        close(out[b:b + 1], ref, tol)


@pytest.mark.parametrize("hq, hkv, d", [(16, 8, 128), (8, 2, 64), (4, 2, 256)])
def test_decode_of_the_smallest_f16_values(dev, hq, hkv, d):
    # Keys and values of f16's subnormals, 2^-24 to 2^-15: exact in the products.
    def edit(pool, tables):
        for t in (2, 3):
            pool.cpu[t] = pool.cpu[t].clamp(104, 109)

    run_decode(dev, [40, 300], hq=hq, hkv=hkv, d=d, dtype=F16, edit=edit, scale=2.0 ** 14, new=True, seed=52)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_decode_of_a_query_that_is_not_finite(dev, dtype, bad):
    # One key, whose element beside the bad one is positive, zero or negative.
    k, v, ks, vs = ops.mxfp4_kv_pool(3, 16, 2, 128, device=dev)
    rows = torch.ones(3, 2, 128, dtype=dtype)
    rows[1, :, 5], rows[2, :, 5] = 0.0, -1.0
    slots = torch.tensor([0, 16, 32], dtype=torch.int32, device=dev)
    ops.store_kvcache(rows.to(dev), rows.to(dev), k, v, slots, k_scale=ks, v_scale=vs)
    q = torch.ones(3, 4, 128, dtype=dtype)
    q[:, 1, 5] = bad
    out = ops.paged_decode(q.to(dev), k, v, torch.arange(3, dtype=torch.int32, device=dev)[:, None],
                           torch.ones(3, dtype=torch.int32, device=dev), max_seq_len=1, scale=0.1, k_scale=ks,
                           v_scale=vs).cpu()
    assert out[:, 1].isnan().all()
    for h in (0, 2, 3):
        assert torch.equal(out[:, h], rows[:, h // 2])
