"""MXFP4 pools and device metadata on the CPU: the oracle's own corners and the
refusals of every entry point (bad calls end before any launch)."""

import ctypes
import math

import pytest
import torch

from oracle import mx4 as oracle
from voiceagent_amd import _native as N
from voiceagent_amd import ops
from voiceagent_amd.layers.attention import PagedAttention
from voiceagent_amd.layers.context import AttentionContext, attention_context
from voiceagent_amd.layers.qwen3 import Qwen3AttentionCore


def _row(values, dtype=torch.bfloat16):
    x = torch.zeros(32, dtype=dtype)
    x[: len(values)] = torch.tensor(values, dtype=dtype)
    return x


def test_quantise_ties_and_scale():
    # 6.96875 is the largest bf16 below 7: scale 1, saturates to 6; 7 takes scale 2 -> 3.5 -> 4.
    for top, e, back in ((6.96875, 0, 6.0), (7.0, 1, 8.0), (3.5, 0, 4.0), (4.0, 0, 4.0)):
        c, s = oracle.quantise(_row([top]))
        assert s.item() == 127 + e and oracle.values(c, s)[0].item() == back
    x = _row([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -5.0])
    c, s = oracle.quantise(x)
    assert s.item() == 127
    assert oracle.values(c, s)[:10].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, -0.0, -4.0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantise_limits(dtype):
    lo, hi = oracle.RANGE[dtype]
    for x, s in ((0.0, lo), (torch.finfo(dtype).tiny / 4, lo if dtype == torch.bfloat16 else -18),
                 (torch.finfo(dtype).max, hi), (math.inf, hi)):
        c, e = oracle.quantise(_row([x], dtype))
        assert e.item() == s + 127
        v = oracle.values(c, e)
        assert torch.equal(v.to(dtype).double(), v)  # exact in the rows' type
    c, e = oracle.quantise(_row([1.0, math.nan], dtype))
    assert e.item() == 255 and not c.any() and oracle.values(c, e).isnan().all()


def test_quantise_error_is_at_most_half_a_step():
    gen = torch.Generator().manual_seed(0)
    x = (torch.randn(400, 128, generator=gen) * torch.exp(3 * torch.randn(400, 1, generator=gen))).to(torch.bfloat16)
    c, s = oracle.quantise(x)
    step = torch.exp2(s.double() - 127).repeat_interleave(32, -1)
    assert ((oracle.values(c, s) - x.double()).abs() <= step).all()  # the widest step is 2


# ------------------------------------------------------------------ refusals
def _pool():
    p = N.KvPool(k=1 << 20, v=1 << 20, stride_block=16 * 8 * 64, stride_slot=8 * 64, stride_head=64,
                 block_size=16, num_blocks=8, kv_format=N.VA_KV_MXFP4, k_scale=1.0, v_scale=1.0)
    s = N.Mx4Scales(struct_size=ctypes.sizeof(N.Mx4Scales), k=1 << 21, v=1 << 21,
                    stride_block=16 * 8 * 4, stride_slot=8 * 4, stride_head=4)
    return p, s


def _store_args():
    p, s = _pool()
    a = N.new_args(N.StoreArgs)
    a.dtype, a.key, a.value, a.pool = 0, 1 << 16, 1 << 16, p
    a.key_stride_tok = a.value_stride_tok = 1024
    a.key_stride_head = a.value_stride_head = 128
    a.slot_mapping, a.num_tokens, a.num_kv_heads, a.head_dim = 1 << 16, 4, 8, 128
    return a, s


def _decode_args():
    p, s = _pool()
    a = N.new_args(N.DecodeArgs)
    a.q = a.out = a.block_tables = a.lens = 1 << 16
    a.q_stride_seq = a.out_stride_seq = 2048
    a.q_stride_head = a.out_stride_head = 128
    a.pool, a.num_seqs, a.num_heads, a.num_kv_heads, a.head_dim = p, 2, 16, 8, 128
    a.table_width, a.table_stride_seq, a.max_seq_len, a.scale = 4, 4, 64, 0.1
    return a, s


def _varlen_args():
    p, s = _pool()
    a = N.new_args(N.VarlenArgs)
    a.q = a.k = a.v = a.out = a.cu_seqlens_q = a.cu_seqlens_k = a.block_tables = 1 << 16
    a.q_stride_tok = a.out_stride_tok = 2048
    a.k_stride_tok = a.v_stride_tok = 1024
    a.q_stride_head = a.out_stride_head = a.k_stride_head = a.v_stride_head = 128
    a.pool, a.num_seqs, a.total_q, a.num_heads, a.num_kv_heads, a.head_dim = p, 1, 8, 16, 8, 128
    a.max_seqlen_q, a.max_seqlen_k, a.causal, a.scale, a.table_width = 8, 64, 1, 0.1, 4
    return a, s


CALLS = {"va_store_kvcache_mx4": _store_args, "va_paged_decode_mx4": _decode_args,
         "va_varlen_attention_mx4": _varlen_args}


@pytest.mark.parametrize("fn", sorted(CALLS))
@pytest.mark.parametrize("change, said", [
    (lambda a, s: setattr(s, "struct_size", 8), "struct_size"),
    (lambda a, s: setattr(a, "struct_size", 8), "struct_size"),
    (lambda a, s: setattr(a.pool, "kv_format", N.VA_KV_FP8_E4M3), "kv_format"),
    (lambda a, s: setattr(s, "v", None), "null scale"),
    (lambda a, s: setattr(s, "k", (1 << 21) + 2), "scale pointers"),
    (lambda a, s: setattr(s, "stride_slot", 30), "scale strides"),
    (lambda a, s: setattr(a.pool, "k", (1 << 20) + 8), "aligned"),
    (lambda a, s: setattr(a.pool, "stride_head", 72), "multiples"),
    (lambda a, s: setattr(a, "dtype", N.VA_F32), "dtype"),
])
def test_mx4_entries_refuse(fn, change, said):
    lib = N.lib()
    a, s = CALLS[fn]()
    change(a, s)
    assert getattr(lib, fn)(ctypes.byref(a), ctypes.byref(s), None) < 0
    assert said in N.last_error() and fn in N.last_error().replace("va_varlen_attention:", fn)


@pytest.mark.parametrize("fn, change, said", [
    ("va_paged_decode_mx4", lambda a, s: setattr(a.pool, "block_size", 24), "multiple of 16"),
    ("va_paged_decode_mx4", lambda a, s: setattr(a, "head_dim", 96), "head_dim"),
    ("va_paged_decode_mx4", lambda a, s: setattr(a, "scale", 0.0), "scale"),
    ("va_paged_decode_mx4", lambda a, s: setattr(a.pool, "stride_slot", -512), "non-negative"),
    ("va_varlen_attention_mx4", lambda a, s: setattr(a.pool, "block_size", 24), "multiple of 16"),
    ("va_varlen_attention_mx4", lambda a, s: setattr(a.pool, "k", None), "pool"),
    ("va_varlen_attention_mx4", lambda a, s: setattr(a, "prologue", ctypes.pointer(N.QkPrologue())), "prologue"),
    ("va_store_kvcache_mx4", lambda a, s: setattr(a, "head_dim", 72), "multiple of 32"),
])
def test_mx4_geometry_refusals(fn, change, said):
    lib = N.lib()
    a, s = CALLS[fn]()
    change(a, s)
    assert getattr(lib, fn)(ctypes.byref(a), ctypes.byref(s), None) < 0
    assert said in N.last_error()


def test_other_entries_refuse_mx4_pools():
    lib = N.lib()
    for fn, make in (("va_store_kvcache", _store_args), ("va_paged_decode", _decode_args),
                     ("va_varlen_attention", _varlen_args)):
        a, _ = make()
        assert getattr(lib, fn)(ctypes.byref(a), None) < 0
        assert "kv_format" in N.last_error()


def test_mx4_workspace_needed_only_when_split():
    lib = N.lib()
    a, s = _decode_args()
    assert lib.va_paged_decode_mx4_workspace_bytes(ctypes.byref(a)) == 0
    a.max_seq_len = 16384
    n = lib.va_paged_decode_mx4_workspace_bytes(ctypes.byref(a))
    assert n > 0
    assert lib.va_paged_decode_mx4(ctypes.byref(a), ctypes.byref(s), None) == -3
    assert "workspace" in N.last_error()


def test_batch_metadata_refusals():
    lib = N.lib()

    def args():
        a = N.new_args(N.BatchArgs)
        a.lens = a.num_computed = a.request_tables = a.positions = a.slot_mapping = 1 << 16
        a.cu_seqlens_q = a.cu_seqlens_k = a.block_tables = a.totals = 1 << 16
        a.request_stride = a.request_width = a.table_width = a.table_stride = 8
        a.num_requests, a.num_seqs, a.padded_seqs, a.block_size, a.max_tokens = 4, 4, 4, 16, 64
        return a

    for field, value, said in (
            ("struct_size", 4, "struct_size"), ("padded_seqs", 3, "padded_seqs"),
            ("num_seqs", -1, "padded_seqs"), ("padded_seqs", 70000, "65535"),
            ("block_size", 0, "block_size"), ("max_tokens", -1, "non-negative"),
            ("lens", None, "lengths"), ("positions", None, "positions"), ("totals", None, "output"),
            ("request_stride", 7, "overlap"), ("table_stride", 7, "overlap"),
            ("free_blocks", 1 << 16, "together"), ("index_dtype", 5, "index_dtype")):
        a = args()
        setattr(a, field, value)
        assert lib.va_batch_metadata(ctypes.byref(a), None) == -1, field
        assert said in N.last_error()


def test_wrappers_refuse_cpu_tensors():
    k, v, ks, vs = ops.mxfp4_kv_pool(4, 16, 8, 128, device="cpu")
    assert k.shape == (4, 16, 8, 64) and ks.shape == (4, 16, 8, 4)
    x = torch.zeros(3, 8, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ops.AttentionArgumentError):
        ops.store_kvcache(x, x, k, v, slots, k_scale=ks, v_scale=vs)
    with pytest.raises(ops.AttentionArgumentError):
        ops.load_kvcache(k, v, slots, k_scale=ks, v_scale=vs)
    with pytest.raises(ops.AttentionArgumentError):
        ops.batch_metadata(slots, slots, slots.view(1, 3), 16, max_tokens=3)


def test_batch_metadata_refuses_a_count_inside_its_totals():
    lib = N.lib()
    a = N.new_args(N.BatchArgs)
    a.positions = a.slot_mapping = a.cu_seqlens_q = a.cu_seqlens_k = a.lens = a.num_computed = 1 << 16
    a.totals, a.free_blocks, a.free_capacity = 1 << 17, 1 << 18, 4
    a.num_seqs = a.padded_seqs = 1
    a.block_size = 16
    for entry in range(5):
        a.free_count = (1 << 17) + 4 * entry
        assert lib.va_batch_metadata(ctypes.byref(a), None) == -1
        assert "totals" in N.last_error()


def test_head_dim_64_scale_blocks_start_on_words():
    lib = N.lib()
    for fn, make in CALLS.items():
        a, s = make()
        a.head_dim = 64
        s.stride_head, s.stride_slot, s.stride_block = 2, 6, 16 * 6 + 2
        assert getattr(lib, fn)(ctypes.byref(a), ctypes.byref(s), None) < 0
        assert "block stride" in N.last_error()


def test_load_refusals():
    lib = N.lib()

    def call(change):
        p, s = _pool()
        a = N.new_args(N.LoadArgs)
        a.dtype, a.key, a.value, a.pool = 0, 1 << 16, 1 << 16, p
        a.key_stride_tok = a.value_stride_tok = 1024
        a.key_stride_head = a.value_stride_head = 128
        a.slot_mapping, a.num_tokens, a.num_kv_heads, a.head_dim = 1 << 16, 4, 8, 128
        change(a, s)
        assert lib.va_load_kvcache_mx4(ctypes.byref(a), ctypes.byref(s), None) < 0
        return N.last_error()

    assert "struct_size" in call(lambda a, s: setattr(a, "struct_size", 8))
    assert "empty pool" in call(lambda a, s: setattr(a.pool, "num_blocks", 0))
    assert "kv_format" in call(lambda a, s: setattr(a.pool, "kv_format", N.VA_KV_NATIVE))
    assert "slot_dtype" in call(lambda a, s: setattr(a, "slot_dtype", 9))
    assert "16-byte" in call(lambda a, s: setattr(a, "key", (1 << 16) + 2))
    assert "16-byte" in call(lambda a, s: setattr(a, "value_stride_tok", 1028))
    assert "null" in call(lambda a, s: setattr(a, "slot_mapping", None))
    assert "dtype" in call(lambda a, s: setattr(a, "dtype", N.VA_F32))


@pytest.mark.parametrize("exact", [False, True])
def test_qwen3_core_decodes_as_the_plain_layer_does(monkeypatch, exact):
    """The fused decode step of the prologue's layer gives paged_decode the pool, the
    layout, the scales and the split that the plain layer's gives it."""
    calls = []
    monkeypatch.setattr(ops, "paged_decode", lambda *args, **kw: calls.append((args, kw)) or args[0])
    cu = torch.tensor([0, 5000, 14000], dtype=torch.int32)
    context = AttentionContext(cu_seqlens_q=torch.arange(3, dtype=torch.int32), cu_seqlens_k=cu, max_seqlen_q=1,
                               max_seqlen_k=9000, slot_mapping=torch.zeros(2, dtype=torch.int32),
                               block_tables=torch.zeros(2, 600, dtype=torch.int32), max_seqlen_k_exact=exact)
    layer = Qwen3AttentionCore(4, 128, 2, max_position=8)
    layer.k_cache, layer.v_cache, layer.k_scale, layer.v_scale = ops.mxfp4_kv_pool(2, 16, 2, 128, device="cpu",
                                                                                   layout=ops.LAYOUT_HND)
    layer.kv_layout = ops.LAYOUT_HND
    q, k, v = (torch.zeros(2, n, 128, dtype=torch.bfloat16) for n in (4, 2, 2))
    positions = torch.tensor([4999, 8999])
    with attention_context(context):
        layer(positions, q, k, v)
        PagedAttention.forward(layer, q, k, v, layer.prologue(positions))
    (a, kw), (b, plain) = calls
    assert all(x is y for x, y in zip(a, b)) and kw.keys() == plain.keys()
    pro, other = kw.pop("prologue"), plain.pop("prologue")
    assert pro.positions is other.positions and pro.eps == other.eps
    assert all(kw[n] is plain[n] or kw[n] == plain[n] for n in kw)
    assert kw["split_tokens"] == (ops.SPLIT_EXACT if exact else 0)
