"""Tensor-level entry points over the C ABI.

Each function validates shapes, dtypes, devices and strides on the host
(shape metadata only: no device synchronisation), fills the argument struct
and launches on torch's current stream.  The HIP library is the only compute
path: CPU tensors or a missing library raise.
"""

from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass

import torch

from voiceagent_amd import _native as N

# split_tokens for a max_seq_len that is the batch's exact longest context
# (an eager step's): the automatic split with fixed partitions at any length
# (va_paged_decode, VA_SPLIT_EXACT).
SPLIT_EXACT = N.VA_SPLIT_EXACT
LAYOUT_NHD = "nhd"  # [num_blocks, block_size, Hkv, D]  (engine, model_runner.py:116-131)
LAYOUT_HND = "hnd"  # [pages, Hkv, page_size, D]        (TTS, qwen_tts_outer_paged_cache.py:116-119)
# An FP8 KV pool holds OCP e4m3 codes (torch.float8_e4m3fn); an element's
# value is code * k_scale (keys) or code * v_scale (values).
FP8_KV_DTYPE = torch.float8_e4m3fn
# An MXFP4 KV pool holds 4-bit e2m1 codes, two to a byte (the even element in
# the low half): a float4_e2m1fn_x2 pool whose last dimension is head_dim / 2.
# k_scale / v_scale are then float8_e8m0fnu tensors of the pool's shape with a
# last dimension of head_dim / 32: one power of two per 32 elements of a row.
MXFP4_KV_DTYPE = torch.float4_e2m1fn_x2
MXFP4_SCALE_DTYPE = torch.float8_e8m0fnu
MXFP4_GROUP = 32


class AttentionArgumentError(ValueError):
    """Host-side contract violation detected before launch."""


def _require(cond: bool, msg: str) -> None:
    if not cond:
        raise AttentionArgumentError(msg)


def _check_gpu(*tensors: torch.Tensor | None) -> torch.device:
    device = None
    for t in tensors:
        if t is None:
            continue
        _require(t.is_cuda, "attention kernels need GPU tensors (there is no CPU path)")
        if device is None:
            device = t.device
        _require(t.device == device, "all tensors must be on the same device")
    return device


def _dtype_code(t: torch.Tensor) -> int:
    _require(t.dtype in N.DTYPE_CODES, f"unsupported dtype {t.dtype}")
    return N.DTYPE_CODES[t.dtype]


def _index_code(t: torch.Tensor, what: str) -> int:
    _require(t.dtype in N.INDEX_CODES, f"{what} must be int32 or int64, got {t.dtype}")
    return N.INDEX_CODES[t.dtype]


def _rows(t: torch.Tensor, what: str) -> None:
    _require(t.stride(-1) == 1, f"{what}: the last dimension must be contiguous")


def _plain_output(t: torch.Tensor | None, what: str) -> None:
    """Refuses a given output that would claim a gradient that the call does not have: written
    through its pointer it keeps its place in autograd's graph."""
    _require(t is None or not t.requires_grad or not torch.is_grad_enabled(),
             f"{what} requires a gradient, and a call with outputs has none "
             "(call without outputs, or in torch.no_grad())")


def _written(*outs: torch.Tensor | None) -> None:
    """Counts given outputs as changed, as torch's own in-place calls do, so that a backward pass
    that saved their rows before raises instead of reading others."""
    torch.autograd.graph.increment_version([t for t in outs if t is not None])


def _pool_matches(pool: torch.Tensor, dtype: torch.dtype) -> bool:
    """A pool of `dtype` itself, or an FP8 pool for 16-bit data."""
    return pool.dtype == dtype or (pool.dtype == FP8_KV_DTYPE and
                                   dtype in (torch.bfloat16, torch.float16))


def kv_pool(k_cache: torch.Tensor, v_cache: torch.Tensor, layout: str = LAYOUT_NHD,
            k_scale: float = 1.0, v_scale: float = 1.0) -> N.KvPool:
    """Describe a paged K/V pool pair (4-D, NHD or HND) for the C ABI; an
    FP8 (float8_e4m3fn) pool carries its k_scale / v_scale."""
    _require(k_cache.dim() == 4, "KV pool must be 4-D")
    _require(
        v_cache.shape == k_cache.shape and v_cache.stride() == k_cache.stride(),
        "key and value pools must have identical shapes and strides",
    )
    _require(v_cache.dtype == k_cache.dtype, "key and value pools must share a dtype")
    _rows(k_cache, "KV pool")
    pool = N.KvPool()
    pool.k = k_cache.data_ptr()
    pool.v = v_cache.data_ptr()
    if layout == LAYOUT_NHD:
        nb, bs, _, _ = k_cache.shape
        pool.stride_block, pool.stride_slot, pool.stride_head = (
            k_cache.stride(0),
            k_cache.stride(1),
            k_cache.stride(2),
        )
    elif layout == LAYOUT_HND:
        nb, _, bs, _ = k_cache.shape
        pool.stride_block, pool.stride_slot, pool.stride_head = (
            k_cache.stride(0),
            k_cache.stride(2),
            k_cache.stride(1),
        )
    else:
        raise AttentionArgumentError(f"unknown pool layout {layout!r}")
    pool.block_size = int(bs)
    pool.num_blocks = int(nb)
    if k_cache.dtype == FP8_KV_DTYPE:
        _require(k_scale > 0 and v_scale > 0, "FP8 pool scales must be positive")
        pool.kv_format = N.VA_KV_FP8_E4M3
        pool.k_scale = float(k_scale)
        pool.v_scale = float(v_scale)
    else:
        pool.kv_format = N.VA_KV_NATIVE
        pool.k_scale = pool.v_scale = 1.0
    return pool


def mxfp4_kv_pool(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int, *,
                  device: torch.device | str, layout: str = LAYOUT_NHD
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """An MXFP4 pool of zeros: (k_cache, v_cache, k_scale, v_scale)."""
    _require(head_dim % MXFP4_GROUP == 0, "head_dim must be a multiple of 32")
    _require(layout in (LAYOUT_NHD, LAYOUT_HND), f"unknown pool layout {layout!r}")
    dims = ((num_blocks, block_size, num_kv_heads) if layout == LAYOUT_NHD
            else (num_blocks, num_kv_heads, block_size))

    def zeros(width: int, dtype: torch.dtype) -> torch.Tensor:
        return torch.zeros(2, *dims, width, dtype=torch.uint8, device=device).view(dtype)

    codes = zeros(head_dim // 2, MXFP4_KV_DTYPE)
    scales = zeros(head_dim // MXFP4_GROUP, MXFP4_SCALE_DTYPE)
    return codes[0], codes[1], scales[0], scales[1]


def _mx4_structs(k_cache: torch.Tensor, v_cache: torch.Tensor, layout: str, k_scale, v_scale,
                 dtype: torch.dtype) -> tuple[N.KvPool, N.Mx4Scales]:
    """The pool and scale descriptions of an MXFP4 pool that `dtype` rows go
    to or come from."""
    _require(k_cache.dtype == MXFP4_KV_DTYPE and v_cache.dtype == MXFP4_KV_DTYPE,
             f"tensor scales need an MXFP4 (float4_e2m1fn_x2) pool, got {k_cache.dtype}")
    _require(dtype in (torch.bfloat16, torch.float16), "an MXFP4 pool needs 16-bit rows")
    _require(isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)
             and k_scale.dtype == v_scale.dtype == MXFP4_SCALE_DTYPE,
             "an MXFP4 pool needs k_scale and v_scale tensors of float8_e8m0fnu")
    _check_gpu(k_cache, v_cache, k_scale, v_scale)
    _require(k_cache.dim() == 4, "KV pool must be 4-D")
    _require(v_cache.shape == k_cache.shape and v_cache.stride() == k_cache.stride(),
             "key and value pools must have identical shapes and strides")
    _require(k_scale.shape == k_cache.shape[:3] + (k_cache.shape[3] * 2 // MXFP4_GROUP,)
             and k_cache.shape[3] * 2 % MXFP4_GROUP == 0,
             "k_scale must have the pool's shape with a last dimension of head_dim / 32")
    _require(v_scale.shape == k_scale.shape and v_scale.stride() == k_scale.stride(),
             "k_scale and v_scale must have identical shapes and strides")
    _rows(k_cache, "KV pool")
    _require(k_scale.stride(3) == 1 or k_scale.shape[3] == 1,
             "k_scale: the last dimension must be contiguous")
    _require(layout in (LAYOUT_NHD, LAYOUT_HND), f"unknown pool layout {layout!r}")
    slot, head = (1, 2) if layout == LAYOUT_NHD else (2, 1)
    pool = N.KvPool(k=k_cache.data_ptr(), v=v_cache.data_ptr(), stride_block=k_cache.stride(0),
                    stride_slot=k_cache.stride(slot), stride_head=k_cache.stride(head),
                    block_size=k_cache.shape[slot], num_blocks=k_cache.shape[0],
                    kv_format=N.VA_KV_MXFP4, k_scale=1.0, v_scale=1.0)
    scales = N.Mx4Scales(struct_size=ctypes.sizeof(N.Mx4Scales), k=k_scale.data_ptr(),
                         v=v_scale.data_ptr(), stride_block=k_scale.stride(0),
                         stride_slot=k_scale.stride(slot), stride_head=k_scale.stride(head))
    return pool, scales


def _number(scale: float | torch.Tensor) -> float:
    """An FP8 pool's scale (other pools ignore theirs)."""
    _require(not isinstance(scale, torch.Tensor) or scale.numel() == 1,
             "tensor scales need an MXFP4 (float4_e2m1fn_x2) pool, or hold one number")
    return float(scale)


def _mx4_call(name: str, args, scales: N.Mx4Scales, device: torch.device) -> None:
    """Launch an MXFP4 entry point on the current stream of `device`."""
    index = _device_index(device)
    with _current(index):
        N.check(name, getattr(N.lib(), name)(ctypes.byref(args), ctypes.byref(scales),
                                             _raw_stream(index)))


def pool_heads(k_cache: torch.Tensor, layout: str) -> tuple[int, int]:
    """(num_kv_heads, head_dim) of a pool."""
    d = int(k_cache.shape[3]) * (2 if k_cache.dtype == MXFP4_KV_DTYPE else 1)
    if layout == LAYOUT_NHD:
        return int(k_cache.shape[2]), d
    return int(k_cache.shape[1]), d


# --------------------------------------------------------------------- store
def store_kvcache(
    key: torch.Tensor,
    value: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    layout: str = LAYOUT_NHD,
    k_scale: float | torch.Tensor = 1.0,
    v_scale: float | torch.Tensor = 1.0,
) -> None:
    """Write key[i] / value[i] ([N, Hkv, D]) to pool slot slot_mapping[i]; -1 skips.
    An FP8 pool receives e4m3 codes of key / k_scale and value / v_scale.  An
    MXFP4 pool receives e2m1 codes, and k_scale / v_scale (its scale tensors)
    the groups' scales: the smallest power of two 2^e with max |x| < 7 * 2^e."""
    if k_cache.dtype is MXFP4_KV_DTYPE:
        return _store_mx4(key, value, k_cache, v_cache, slot_mapping, layout, k_scale, v_scale)
    fast = _FAST if _FAST_LOADED else _fast_calls()
    if fast is not None and layout in (LAYOUT_NHD, LAYOUT_HND):
        index = key.get_device()
        if index >= 0 and index == torch.cuda.current_device():
            rc = fast.store_kvcache(key, value, k_cache, v_cache, slot_mapping,
                                    layout == LAYOUT_HND,
                                    k_scale if k_scale.__class__ is float else _number(k_scale),
                                    v_scale if v_scale.__class__ is float else _number(v_scale),
                                    index, _raw_stream(index))
            if rc == 0:
                return
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_store_kvcache", rc)
    device = _check_gpu(key, value, k_cache, v_cache, slot_mapping)
    _require(key.dim() == 3 and value.shape == key.shape, "key/value must be [N, Hkv, D]")
    _rows(key, "key")
    _rows(value, "value")
    hkv, d = pool_heads(k_cache, layout)
    _require(key.shape[1] == hkv and key.shape[2] == d, "key/value heads must match the pool")
    _require(key.dtype == value.dtype and _pool_matches(k_cache, key.dtype),
             "key/value/pool dtypes must match (or the pool be FP8 for 16-bit rows)")
    _require(slot_mapping.dim() == 1 and slot_mapping.numel() == key.shape[0],
             "slot_mapping must have one entry per token")
    _require(slot_mapping.is_contiguous(), "slot_mapping must be contiguous")
    args = N.new_args(N.StoreArgs)
    args.dtype = _dtype_code(key)
    args.key = key.data_ptr()
    args.value = value.data_ptr()
    args.key_stride_tok, args.key_stride_head = key.stride(0), key.stride(1)
    args.value_stride_tok, args.value_stride_head = value.stride(0), value.stride(1)
    args.pool = kv_pool(k_cache, v_cache, layout, _number(k_scale), _number(v_scale))
    args.slot_mapping = slot_mapping.data_ptr()
    args.slot_dtype = _index_code(slot_mapping, "slot_mapping")
    args.num_tokens = int(key.shape[0])
    args.num_kv_heads = hkv
    args.head_dim = d
    N.call("va_store_kvcache", args, device)


def _rows_args(args, key, value, pool, slot_mapping, hkv, d):
    """Fill the fields that the store's and the load's arguments share."""
    _require(key.dim() == 3 and value.shape == key.shape, "key/value must be [N, Hkv, D]")
    _rows(key, "key")
    _rows(value, "value")
    _require(key.shape[1] == hkv and key.shape[2] == d, "key/value heads must match the pool")
    _require(key.dtype == value.dtype, "key and value must share a dtype")
    _require(slot_mapping.dim() == 1 and slot_mapping.numel() == key.shape[0],
             "slot_mapping must have one entry per token")
    _require(slot_mapping.is_contiguous(), "slot_mapping must be contiguous")
    args.dtype = _dtype_code(key)
    args.key = key.data_ptr()
    args.value = value.data_ptr()
    args.key_stride_tok, args.key_stride_head = key.stride(0), key.stride(1)
    args.value_stride_tok, args.value_stride_head = value.stride(0), value.stride(1)
    args.pool = pool
    args.slot_mapping = slot_mapping.data_ptr()
    args.slot_dtype = _index_code(slot_mapping, "slot_mapping")
    args.num_tokens = int(key.shape[0])
    args.num_kv_heads = hkv
    args.head_dim = d
    return args


def _fast_on(t: torch.Tensor, layout: str):
    """(fast-path module, device index) for a call on t's device when that is
    the current one, else (None, -1)."""
    fast = _FAST if _FAST_LOADED else _fast_calls()
    if fast is not None and layout in (LAYOUT_NHD, LAYOUT_HND):
        index = t.get_device()
        if index >= 0 and index == torch.cuda.current_device():
            return fast, index
    return None, -1


def _store_mx4(key, value, k_cache, v_cache, slot_mapping, layout, k_scale, v_scale) -> None:
    fast, index = _fast_on(key, layout)
    if fast is not None and isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor):
        rc = fast.store_kvcache_mx4(key, value, k_cache, v_cache, slot_mapping,
                                    layout == LAYOUT_HND, k_scale, v_scale, index,
                                    _raw_stream(index))
        if rc == 0:
            return
        if _FAST_NOT_TAKEN < rc < 0:
            N.check("va_store_kvcache_mx4", rc)
    device = _check_gpu(key, value, k_cache, v_cache, slot_mapping)
    pool, scales = _mx4_structs(k_cache, v_cache, layout, k_scale, v_scale, key.dtype)
    _check_gpu(key, k_scale)
    hkv, d = pool_heads(k_cache, layout)
    args = _rows_args(N.new_args(N.StoreArgs), key, value, pool, slot_mapping, hkv, d)
    _mx4_call("va_store_kvcache_mx4", args, scales, device)


def load_kvcache(
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    dtype: torch.dtype = torch.bfloat16,
    *,
    layout: str = LAYOUT_NHD,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
) -> tuple[torch.Tensor, torch.Tensor]:
    """The K and V rows [N, Hkv, D] that an MXFP4 pool holds at slot_mapping,
    as values of `dtype` (exact in the type they were stored from); slots
    outside the pool read as zeros.  A 16-bit or FP8 pool's rows are read by
    indexing it."""
    fast, index = _fast_on(k_cache, layout)
    if (fast is not None and dtype in (torch.bfloat16, torch.float16) and
            isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)):
        rc, key, value = fast.load_kvcache_mx4(k_cache, v_cache, slot_mapping,
                                               dtype == torch.float16, layout == LAYOUT_HND,
                                               k_scale, v_scale, index, _raw_stream(index))
        if rc == 0:
            return key, value
        if _FAST_NOT_TAKEN < rc < 0:
            N.check("va_load_kvcache_mx4", rc)
    device = _check_gpu(k_cache, v_cache, slot_mapping)
    pool, scales = _mx4_structs(k_cache, v_cache, layout, k_scale, v_scale, dtype)
    _check_gpu(k_cache, k_scale)
    hkv, d = pool_heads(k_cache, layout)
    _require(slot_mapping.dim() == 1, "slot_mapping must be a vector")
    shape = (int(slot_mapping.numel()), hkv, d)
    key = torch.empty(shape, dtype=dtype, device=device)
    value = torch.empty(shape, dtype=dtype, device=device)
    args = _rows_args(N.new_args(N.LoadArgs), key, value, pool, slot_mapping, hkv, d)
    _mx4_call("va_load_kvcache_mx4", args, scales, device)
    return key, value


# ---------------------------------------------------------- q/k prologue
@dataclass(frozen=True)
class QKPrologue:
    """Qwen3's per-head q/k prologue (qwen_asr_vllm/models/qwen3.py:42-48):
    RMSNorm with ``q_norm_weight`` / ``k_norm_weight`` and ``eps``
    (layers/layernorm.py:19-25), then the half-split rotary embedding read from
    the fp32 ``cos_sin_cache`` ([max_position, D] or the reference's
    [max_position, 1, D] buffer) at ``positions`` (layers/rotary_embedding.py:9-32)."""

    q_norm_weight: torch.Tensor
    k_norm_weight: torch.Tensor
    eps: float
    cos_sin_cache: torch.Tensor
    positions: torch.Tensor


def _prologue_struct(pro: QKPrologue, head_dim: int, n_positions: int) -> N.QkPrologue:
    for name, w in (("q_norm_weight", pro.q_norm_weight), ("k_norm_weight", pro.k_norm_weight)):
        _require(w.dim() == 1 and w.numel() == head_dim and w.is_contiguous(),
                 f"{name} must be a contiguous [head_dim] vector")
    _require(pro.q_norm_weight.dtype == pro.k_norm_weight.dtype,
             "q_norm_weight and k_norm_weight must share a dtype")
    cs = pro.cos_sin_cache
    if cs.dim() == 3:
        _require(cs.shape[1] == 1, "cos_sin_cache must be [max_position, (1,) head_dim]")
        cs = cs[:, 0]
    _require(cs.dim() == 2 and cs.shape[1] == head_dim and cs.dtype == torch.float32
             and cs.stride(-1) == 1,
             "cos_sin_cache must be an fp32 [max_position, head_dim] table (cos | sin)")
    pos = pro.positions
    _require(pos.dim() == 1 and pos.numel() >= n_positions and pos.is_contiguous(),
             f"positions must be a contiguous vector of at least {n_positions} entries")
    st = N.QkPrologue()
    st.q_norm_weight = pro.q_norm_weight.data_ptr()
    st.k_norm_weight = pro.k_norm_weight.data_ptr()
    st.weight_dtype = _dtype_code(pro.q_norm_weight)
    st.eps = float(pro.eps)
    st.cos_sin_cache = cs.data_ptr()
    st.cos_sin_stride = cs.stride(0)
    st.max_position = int(cs.shape[0])
    st.positions_dtype = _index_code(pos, "positions")
    st.positions = pos.data_ptr()
    return st


def qk_norm_rope(
    q: torch.Tensor | None,
    k: torch.Tensor,
    prologue: QKPrologue,
    *,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor]:
    """Apply the Qwen3 q/k prologue to q [T, Hq, D] and k [T, Hkv, D] (one
    position per token).  Outputs are allocated contiguous when not given and
    may be q / k themselves (in place).  ``q`` None: the keys alone (a
    prefill whose varlen launch applies the query prologue itself); the
    first result is then None.  Without outputs the call is differentiable in q,
    k and the norm weights (:func:`qk_norm_rope_backward`); with outputs it has
    no gradient, and in grad mode they may not require one."""
    if q_out is not None or k_out is not None:
        _plain_output(q_out, "q_out")
        _plain_output(k_out, "k_out")
    elif torch.is_grad_enabled():
        qw, kw = prologue.q_norm_weight, prologue.k_norm_weight
        if q is None:
            if k.requires_grad or kw.requires_grad:
                return None, _KNormRope.apply(k, kw, prologue)
        elif q.requires_grad or k.requires_grad or qw.requires_grad or kw.requires_grad:
            return _QkNormRope.apply(q, k, qw, kw, prologue)
    if q is None:
        return None, _k_norm_rope(k, prologue, k_out)
    fast = _FAST if _FAST_LOADED else _fast_calls()
    if fast is not None:
        index = q.get_device()
        if index >= 0 and index == torch.cuda.current_device():
            if q_out is None:
                q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            if k_out is None:
                k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            rc = fast.qk_norm_rope(q, k, q_out, k_out, prologue.q_norm_weight,
                                   prologue.k_norm_weight, float(prologue.eps),
                                   prologue.cos_sin_cache, prologue.positions, index,
                                   _raw_stream(index))
            if rc == 0:
                return q_out, k_out
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_qk_norm_rope", rc)
    device = _check_gpu(q, k, q_out, k_out, prologue.q_norm_weight, prologue.k_norm_weight,
                        prologue.cos_sin_cache, prologue.positions)
    _require(q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0] and
             q.shape[2] == k.shape[2], "q must be [T, Hq, D] and k [T, Hkv, D]")
    _require(q.dtype == k.dtype, "q and k must share a dtype")
    _rows(q, "q")
    _rows(k, "k")
    T, hq, d = (int(x) for x in q.shape)
    hkv = int(k.shape[1])
    if q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=device)
    _require(q_out.shape == q.shape and q_out.dtype == q.dtype, "q_out must match q")
    _require(k_out.shape == k.shape and k_out.dtype == k.dtype, "k_out must match k")
    _rows(q_out, "q_out")
    _rows(k_out, "k_out")
    args = N.new_args(N.QkNormRopeArgs)
    args.dtype = _dtype_code(q)
    args.q, args.q_stride_tok, args.q_stride_head = q.data_ptr(), q.stride(0), q.stride(1)
    args.k, args.k_stride_tok, args.k_stride_head = k.data_ptr(), k.stride(0), k.stride(1)
    args.q_out = q_out.data_ptr()
    args.q_out_stride_tok, args.q_out_stride_head = q_out.stride(0), q_out.stride(1)
    args.k_out = k_out.data_ptr()
    args.k_out_stride_tok, args.k_out_stride_head = k_out.stride(0), k_out.stride(1)
    args.num_tokens, args.num_heads, args.num_kv_heads, args.head_dim = T, hq, hkv, d
    args.prologue = _prologue_struct(prologue, d, T)
    N.call("va_qk_norm_rope", args, device)
    _written(q_out, k_out)
    return q_out, k_out


def _k_norm_rope(k: torch.Tensor, prologue: QKPrologue,
                 k_out: torch.Tensor | None) -> torch.Tensor:
    """The key side of qk_norm_rope alone (num_heads = 0 in the C ABI)."""
    device = _check_gpu(k, k_out, prologue.k_norm_weight, prologue.cos_sin_cache,
                        prologue.positions)
    _require(k.dim() == 3, "k must be [T, Hkv, D]")
    _rows(k, "k")
    T, hkv, d = (int(x) for x in k.shape)
    if k_out is None:
        k_out = torch.empty(k.shape, dtype=k.dtype, device=device)
    _require(k_out.shape == k.shape and k_out.dtype == k.dtype, "k_out must match k")
    _rows(k_out, "k_out")
    args = N.new_args(N.QkNormRopeArgs)
    args.dtype = _dtype_code(k)
    args.k, args.k_stride_tok, args.k_stride_head = k.data_ptr(), k.stride(0), k.stride(1)
    args.k_out = k_out.data_ptr()
    args.k_out_stride_tok, args.k_out_stride_head = k_out.stride(0), k_out.stride(1)
    args.num_tokens, args.num_heads, args.num_kv_heads, args.head_dim = T, 0, hkv, d
    args.prologue = _prologue_struct(prologue, d, T)
    N.call("va_qk_norm_rope", args, device)
    _written(k_out)
    return k_out


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [rows, heads, elements] tensors are seen to share no memory: one ends before
    the other begins, or their rows (or heads) lie side by side in one buffer's."""
    if a.numel() == 0 or b.numel() == 0:
        return True
    size = a.element_size()

    def reach(t, step=0):  # bytes from the first element to behind the last, but for whole steps
        return t.element_size() + sum(
            (n - 1) * st * t.element_size() for n, st in zip(t.shape, t.stride())
            if not step or st * t.element_size() % step)

    pa, pb = a.data_ptr(), b.data_ptr()
    if pa + reach(a) <= pb or pb + reach(b) <= pa:
        return True
    for dim in (0, 1):
        step = a.stride(dim) * size
        if step > 0 and b.stride(dim) * b.element_size() == step:
            wa, wb, at = reach(a, step), reach(b, step), (pb - pa) % step
            if wa <= at and at + wb <= step:
                return True
    return False


def _rows_apart(t: torch.Tensor) -> bool:
    """Whether no two elements of a tensor are seen to share memory: from the smallest stride on,
    a dimension steps past all that the ones before it reach."""
    reach = 1
    for st, n in sorted((st, n) for n, st in zip(t.shape, t.stride()) if n > 1):
        if st < reach:
            return False
        reach += (n - 1) * st
    return True


def _in_place(new: torch.Tensor, old: torch.Tensor) -> bool:
    """Whether two tensors of one shape are the same memory, element for element."""
    return new.data_ptr() == old.data_ptr() and new.stride() == old.stride()


def _outputs_apart(given, inputs) -> None:
    """Refuses outputs that share memory with one another or with an input, but for what may be
    written in place.  given: (name, tensor, the inputs it may replace)."""
    for i, (name, t, own) in enumerate(given):
        _plain_output(t, name)
        _require(_rows_apart(t), f"{name}'s rows may not overlap")
        for x in inputs:
            _require(_apart(t, x) or (any(x is o for o in own) and _in_place(t, x)),
                     f"{name} may not overlap the inputs")
        for other, u, _ in given[:i]:
            _require(_apart(t, u), f"{name} may not overlap {other}")


def qk_norm_rope_backward(
    dq_out: torch.Tensor | None,
    dk_out: torch.Tensor,
    q: torch.Tensor | None,
    k: torch.Tensor,
    prologue: QKPrologue,
    *,
    dq: torch.Tensor | None = None,
    dk: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """(dq, dk, dq_norm_weight, dk_norm_weight) of :func:`qk_norm_rope`, from the
    gradients of its outputs and its inputs q [T, Hq, D], k [T, Hkv, D]; the
    weights' sum over all tokens and heads.  fp32, rounded once: the forward's
    roundings to the element type count as the identity.  ``dq`` / ``dk`` may be
    dq_out / dk_out or q / k themselves, and share no memory otherwise.  ``dq_out`` and ``q`` None: the keys
    alone (dq and dq_norm_weight are then None).  Two launches, no atomics."""
    if q is not None and dq_out is not None and dq is None and dk is None:
        fast, index = _fast_on(k, LAYOUT_NHD)
        if fast is not None:
            rc, made = fast.qk_norm_rope_backward(
                dq_out, dk_out, q, k, prologue.q_norm_weight, prologue.k_norm_weight,
                float(prologue.eps), prologue.cos_sin_cache, prologue.positions, index,
                _raw_stream(index))
            if rc == 0:
                return tuple(made)
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_qk_norm_rope_backward", rc)
    _require((q is None) == (dq_out is None), "q and dq_out must be given together")
    _require(q is not None or dq is None, "dq without q")
    device = _check_gpu(dq_out, dk_out, q, k, dq, dk, prologue.q_norm_weight,
                        prologue.k_norm_weight, prologue.cos_sin_cache, prologue.positions)
    sides = [("k", dk_out, k, dk)] if q is None else [("q", dq_out, q, dq), ("k", dk_out, k, dk)]
    _require(k.dim() == 3, "k must be [T, Hkv, D]")
    T, hkv, d = (int(x) for x in k.shape)
    args = N.new_args(N.QkNormRopeBwdArgs)
    args.dtype = _dtype_code(k)
    args.num_tokens, args.num_kv_heads, args.head_dim = T, hkv, d
    results = {"q": None, "k": None, "qw": None, "kw": None}
    given = []
    for name, dz, x, dx in sides:
        _require(x.dim() == 3 and x.shape[0] == T and x.shape[2] == d and x.dtype == k.dtype,
                 "q must be [T, Hq, D] and k [T, Hkv, D] of one dtype")
        _require(dz.shape == x.shape and dz.dtype == x.dtype, f"d{name}_out must match {name}")
        if dx is None:
            dx = torch.empty(x.shape, dtype=x.dtype, device=device)
        else:
            _require(dx.shape == x.shape and dx.dtype == x.dtype, f"d{name} must match {name}")
            given.append((f"d{name}", dx, (dz, x)))
        for field, t in ((f"d{name}_out", dz), (name, x), (f"d{name}", dx)):
            _rows(t, field)
            tok, head = _row_strides(t)
            setattr(args, field, t.data_ptr())
            setattr(args, field + "_stride_tok", tok)
            setattr(args, field + "_stride_head", head)
        weight = prologue.q_norm_weight if name == "q" else prologue.k_norm_weight
        results[name], results[name + "w"] = dx, torch.empty(d, dtype=weight.dtype, device=device)
        setattr(args, f"d{name}_weight", results[name + "w"].data_ptr())
    _outputs_apart(given, [t for _, dz, x, _ in sides for t in (dz, x)])
    args.num_heads = 0 if q is None else int(q.shape[1])
    args.prologue = _prologue_struct(prologue, d, T)
    lib = N.lib()
    index = _device_index(device)
    with _current(index):
        nbytes = lib.va_qk_norm_rope_backward_workspace_bytes(ctypes.byref(args))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)  # this call's alone
        args.workspace = ws.data_ptr()
        args.workspace_bytes = nbytes
        N.check("va_qk_norm_rope_backward",
                lib.va_qk_norm_rope_backward(ctypes.byref(args), _raw_stream(index)))
    _written(*(t for _, t, _ in given))
    return results["q"], results["k"], results["qw"], results["kw"]


class _QkNormRope(torch.autograd.Function):
    """qk_norm_rope with its gradient."""

    @staticmethod
    def forward(ctx, q, k, q_norm_weight, k_norm_weight, prologue):
        ctx.save_for_backward(q, k, q_norm_weight, k_norm_weight, prologue.cos_sin_cache,
                              prologue.positions)
        ctx.eps = prologue.eps
        return qk_norm_rope(q, k, prologue)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq_out, dk_out):
        q, k, qw, kw, cos_sin, positions = ctx.saved_tensors
        grads = qk_norm_rope_backward(_whole_rows(dq_out), _whole_rows(dk_out), q, k,
                                      QKPrologue(qw, kw, ctx.eps, cos_sin, positions))
        return (*(g if need else None for g, need in zip(grads, ctx.needs_input_grad)), None)


class _KNormRope(torch.autograd.Function):
    """The key side of qk_norm_rope alone, with its gradient."""

    @staticmethod
    def forward(ctx, k, k_norm_weight, prologue):
        ctx.save_for_backward(k, prologue.q_norm_weight, k_norm_weight, prologue.cos_sin_cache,
                              prologue.positions)
        ctx.eps = prologue.eps
        return _k_norm_rope(k, prologue, None)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dk_out):
        k, qw, kw, cos_sin, positions = ctx.saved_tensors
        _, dk, _, dkw = qk_norm_rope_backward(None, _whole_rows(dk_out), None, k,
                                              QKPrologue(qw, kw, ctx.eps, cos_sin, positions))
        return (*(g if need else None for g, need in zip((dk, dkw), ctx.needs_input_grad)), None)


# -------------------------------------------------------------------- rotary
@dataclass(frozen=True)
class Rotary:
    """Rotary positions without a norm, for attention layers' ``prologue``: see
    :func:`rotary_embedding`."""

    cos_sin_cache: torch.Tensor
    positions: torch.Tensor
    interleaved: bool = False


def rotary_embedding(
    q: torch.Tensor | None,
    k: torch.Tensor | None,
    cos_sin_cache: torch.Tensor,
    positions: torch.Tensor,
    *,
    interleaved: bool = False,
    inverse: bool = False,
    q_out: torch.Tensor | None = None,
    k_out: torch.Tensor | None = None,
) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Rotate the first r elements of every head of q [T, Hq, D] and k [T, Hkv, D]
    (either may be None) at the tokens' positions.  ``cos_sin_cache`` is an fp32
    [max_position, (1,) r] table, cosines | sines, r even and at most D
    (:func:`voiceagent_amd.layers.rotary_cos_sin_cache` makes one, scaled or
    not); pairs are elements (i, i + r/2), or (2 i, 2 i + 1) when
    ``interleaved``.  Elements from r on are copied.  ``inverse``: the
    transposed rotation, the gradient of the other.  fp32, rounded once (16-bit
    or fp32 rows, any head_dim and strides; rows of 16-byte multiples go 16
    bytes at a time).  Positions are held to the table.  Outputs may be q / k
    themselves, and share no memory otherwise; without outputs the call is
    differentiable in q and k (the table is a constant), with outputs it has no
    gradient, and in grad mode they may not require one."""
    if q_out is not None or k_out is not None:
        _plain_output(q_out, "q_out")
        _plain_output(k_out, "k_out")
    elif (torch.is_grad_enabled() and
            ((q is not None and q.requires_grad) or (k is not None and k.requires_grad))):
        return _Rotary.apply(q, k, cos_sin_cache, positions, interleaved, inverse)
    if q is not None and k is not None and q_out is None and k_out is None:
        fast, index = _fast_on(q, LAYOUT_NHD)
        if fast is not None:
            rc, made = fast.rotary(q, k, cos_sin_cache, positions, bool(interleaved),
                                   bool(inverse), index, _raw_stream(index))
            if rc == 0:
                return made[0], made[1]
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_rotary", rc)
    device = _check_gpu(q, k, cos_sin_cache, positions, q_out, k_out)
    _require(q is not None or k is not None, "q or k must be given")
    like = k if q is None else q
    _require(like.dim() == 3, "q and k must be [T, heads, D]")
    T, _, d = (int(x) for x in like.shape)
    for n in (*like.shape, *(() if k is None else k.shape), *cos_sin_cache.shape[:1]):
        _length(n, "every size")  # (the argument block's are 32-bit)
    args = N.new_args(N.RotaryArgs)
    args.dtype = _dtype_code(like)
    args.num_tokens, args.head_dim = T, d
    outs, given = [], []
    for name, x, y in (("q", q, q_out), ("k", k, k_out)):
        if x is None:
            _require(y is None, f"{name}_out without {name}")
            outs.append(None)
            continue
        _require(x.dim() == 3 and x.shape[0] == T and x.shape[2] == d and x.dtype == like.dtype,
                 "q must be [T, Hq, D] and k [T, Hkv, D] of one dtype")
        if y is None:
            y = torch.empty(x.shape, dtype=x.dtype, device=device)
        else:
            _require(y.shape == x.shape and y.dtype == x.dtype, f"{name}_out must match {name}")
            given.append((f"{name}_out", y, (x,)))
        for field, t in ((name, x), (name + "_out", y)):
            _require(t.stride(2) == 1 or d == 1, f"{field}: the last dimension must be contiguous")
            tok, head = _row_strides(t)
            setattr(args, field, t.data_ptr())
            setattr(args, field + "_stride_tok", tok)
            setattr(args, field + "_stride_head", head)
        outs.append(y)
    _outputs_apart(given, [x for x in (q, k) if x is not None])
    args.num_heads = 0 if q is None else int(q.shape[1])
    args.num_kv_heads = 0 if k is None else int(k.shape[1])
    cs = cos_sin_cache
    if cs.dim() == 3:
        _require(cs.shape[1] == 1, "cos_sin_cache must be [max_position, (1,) rotary_dim]")
        cs = cs[:, 0]
    _require(cs.dim() == 2 and cs.dtype == torch.float32 and cs.stride(-1) == 1 and
             0 < cs.shape[1] <= d and cs.shape[1] % 2 == 0,
             "cos_sin_cache must be an fp32 [max_position, rotary_dim] table (cos | sin), "
             "rotary_dim even and at most head_dim")
    _require(positions.dim() == 1 and positions.numel() >= T and positions.is_contiguous(),
             f"positions must be a contiguous vector of at least {T} entries")
    args.rotary_dim, args.interleaved, args.inverse = cs.shape[1], bool(interleaved), bool(inverse)
    args.cos_sin_cache, args.cos_sin_stride = cs.data_ptr(), cs.stride(0)
    args.max_position = int(cs.shape[0])
    args.positions_dtype = _index_code(positions, "positions")
    args.positions = positions.data_ptr()
    N.call("va_rotary", args, device)
    _written(*(t for _, t, _ in given))
    return outs[0], outs[1]


class _Rotary(torch.autograd.Function):
    """rotary_embedding with its gradient, the transposed rotation."""

    @staticmethod
    def forward(ctx, q, k, cos_sin_cache, positions, interleaved, inverse):
        ctx.save_for_backward(cos_sin_cache, positions)
        ctx.form = (interleaved, inverse)
        ctx.set_materialize_grads(False)
        return rotary_embedding(q, k, cos_sin_cache, positions, interleaved=interleaved,
                                inverse=inverse)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk):
        cos_sin, positions = ctx.saved_tensors
        interleaved, inverse = ctx.form
        dq, dk = (g if g is not None and need else None
                  for g, need in zip((dq, dk), ctx.needs_input_grad))
        if dq is not None or dk is not None:
            dq, dk = (g if g is None or g.stride(2) == 1 else g.contiguous() for g in (dq, dk))
            dq, dk = rotary_embedding(dq, dk, cos_sin, positions, interleaved=interleaved,
                                      inverse=not inverse)
        return dq, dk, None, None, None, None


# -------------------------------------------------------------------- decode
_WORKSPACES: dict[tuple[int, int], torch.Tensor] = {}
# Workspaces replaced by a larger one.  They are never freed: a HIP graph
# captured while one was current keeps its address, and memory returned to
# torch's allocator (a graph's private pool included) could be handed to
# another tensor that the graph's replays would then overwrite.
_RETIRED: list[torch.Tensor] = []
_CUS: dict[int, int] = {}  # compute units per device index


def _device_index(device: torch.device) -> int:
    return device.index if device.index is not None else torch.cuda.current_device()


def _raw_stream(index: int) -> int:
    """Handle of torch's current stream on device `index`."""
    return torch._C._cuda_getCurrentRawStream(index)


class _current:
    """Make device `index` current for the block (the library plans launches
    for, and launches on, the current device); a no-op when it already is."""

    __slots__ = ("index", "prev")

    def __init__(self, index: int):
        self.index = index
        self.prev = -1

    def __enter__(self):
        cur = torch._C._cuda_getDevice()
        if cur != self.index:
            self.prev = cur
            torch._C._cuda_setDevice(self.index)
        return self

    def __exit__(self, *exc):
        if self.prev >= 0:
            torch._C._cuda_setDevice(self.prev)
        return False


_DECODE_ARGS_SIZE = ctypes.sizeof(N.DecodeArgs)
_VARLEN_ARGS_SIZE = ctypes.sizeof(N.VarlenArgs)
_VARLEN_BWD_ARGS_SIZE = ctypes.sizeof(N.VarlenBwdArgs)

# Host fast path (csrc/host/fast_calls.cpp, the ``_fast_calls`` module next
# to the library): the same checks and the same C-ABI call in C++, for the
# common paged_decode / varlen_attention / store_kvcache / qk_norm_rope /
# load_kvcache / batch_metadata / rotary_embedding calls and the gradients.  It launches nothing for a
# call it does not take, and the Python path below then runs (and raises the
# error for a bad argument), so results and errors are the same either way.
_FAST_NOT_TAKEN = -1000
_FAST = None
_FAST_LOADED = False


def _fast_calls():
    """The fast-path module with the library's entry points handed to it, or
    None when it is not built or does not load."""
    global _FAST, _FAST_LOADED
    if not _FAST_LOADED:
        _FAST_LOADED = True
        from voiceagent_amd.build import FAST_MODULE, FAST_PATH

        if FAST_PATH.exists():
            import importlib.util

            try:
                spec = importlib.util.spec_from_file_location(FAST_MODULE, FAST_PATH)
                mod = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(mod)
            except ImportError:
                return None
            lib = N.lib()

            def addr(fn):
                return ctypes.cast(fn, ctypes.c_void_p).value

            mod.set_entries(addr(lib.va_paged_decode), addr(lib.va_paged_decode_workspace_bytes),
                            addr(lib.va_varlen_attention),
                            addr(lib.va_varlen_split_workspace_bytes), addr(lib.va_store_kvcache),
                            addr(lib.va_qk_norm_rope))
            mod.set_mx4_entries(addr(lib.va_store_kvcache_mx4), addr(lib.va_load_kvcache_mx4),
                                addr(lib.va_paged_decode_mx4),
                                addr(lib.va_paged_decode_mx4_workspace_bytes),
                                addr(lib.va_varlen_attention_mx4), addr(lib.va_batch_metadata))
            mod.set_train_entries(addr(lib.va_varlen_attention_backward),
                                  addr(lib.va_varlen_attention_backward_workspace_bytes),
                                  addr(lib.va_qk_norm_rope_backward),
                                  addr(lib.va_qk_norm_rope_backward_workspace_bytes),
                                  addr(lib.va_rotary))
            _FAST = mod
    return _FAST
_POOLS: dict[tuple, N.KvPool] = {}  # pool descriptions by tensor identity and geometry


def _pool_struct(k_cache, v_cache, layout, k_scale, v_scale) -> N.KvPool:
    """kv_pool(...), cached: engine pools live for the whole run, and the
    description depends only on the key's fields."""
    key = (k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape, k_cache.stride(),
           v_cache.shape, v_cache.stride(), k_cache.dtype, v_cache.dtype, layout,
           _number(k_scale), _number(v_scale))
    pool = _POOLS.get(key)
    if pool is None:
        pool = kv_pool(k_cache, v_cache, layout, key[-2], key[-1])
        if len(_POOLS) >= 1024:
            _POOLS.clear()
        _POOLS[key] = pool
    return pool


def decode_workspace_bound(device: torch.device, num_heads: int, num_kv_heads: int,
                           head_dim: int, kv_dtype: torch.dtype | None = None) -> int:
    """Bytes that covers every automatic split (split_tokens = 0) of a decode
    with these heads on `device`, whatever the batch and lengths: the split
    gives at most one partition per compute unit over all (sequence, kv head)
    pairs, each holding (m, l) and head_dim floats per query head of the
    group, with the (m, l) block rounded to 256 bytes.  Over an MXFP4 pool at
    head_dim 128 a workgroup may serve two kv heads, and there may be two
    partitions per compute unit.  ``kv_dtype``: the pool's (None: not MXFP4)."""
    index = _device_index(device)
    cus = _CUS.get(index)
    if cus is None:
        cus = _CUS[index] = torch.cuda.get_device_properties(index).multi_processor_count
    group = max(1, num_heads // max(1, num_kv_heads))
    if kv_dtype is MXFP4_KV_DTYPE and head_dim == 128 and num_kv_heads % 2 == 0:
        cus *= 2
    return (cus * group * 2 * 4 + 255) // 256 * 256 + cus * group * head_dim * 4


def decode_workspace(device: torch.device, nbytes: int, floor: int = 0,
                     stream: torch.cuda.Stream | None = None, kind: str = "decode"
                     ) -> torch.Tensor | None:
    """Partial-result workspace of the decode launches on `stream` (torch's
    current stream of `device` by default): no initialisation needed.  One
    per stream: launches on one stream are ordered, while decodes on two
    streams (an ASR engine and a TTS talker, say) may run at once and must not
    share their partials.  The first allocation takes at least `floor` bytes;
    a later, larger need allocates anew (doubling) and retires, without
    freeing, the old buffer."""
    if nbytes == 0:
        return None
    if stream is None:
        stream = torch.cuda.current_stream(device)
    key = (_device_index(device), stream.cuda_stream)
    if kind != "decode":
        key = key + (kind,)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < nbytes:
        size = max(nbytes, floor if ws is None else 2 * ws.numel())
        if ws is not None:
            _RETIRED.append(ws)
        ws = torch.empty(size, dtype=torch.uint8, device=device)
        _WORKSPACES[key] = ws
    return ws


# Stream of the last no_alloc decode per device (their scratch buffer is
# shared by every stream of a GPU).
_NOALLOC_STREAM: dict[int, torch.cuda.Stream] = {}


def _order_noalloc(index: int) -> None:
    """Order a no_alloc decode after the previous one on its GPU when they
    run on different streams: the current stream waits (on the GPU) for the
    other.  Skipped under graph capture, where a wait on work outside the
    capture is not allowed."""
    cur = torch.cuda.current_stream(index)
    prev = _NOALLOC_STREAM.get(index)
    if (prev is not None and prev.cuda_stream != cur.cuda_stream
            and not torch.cuda.is_current_stream_capturing()):
        cur.wait_stream(prev)
    _NOALLOC_STREAM[index] = cur


def reserve_decode_workspace(device: torch.device, num_heads: int, num_kv_heads: int,
                             head_dim: int, stream: torch.cuda.Stream | None = None,
                             kv_dtype: torch.dtype | None = None) -> None:
    """Allocate the decode workspace of `stream` (torch's current stream by
    default) up front, at the size every automatic split needs over a pool of
    ``kv_dtype`` (None: over any), e.g. before HIP graph capture.
    ``torch.cuda.graph`` captures on a stream of its own unless it is given
    one: pass that stream here to reserve for it."""
    device = torch.device(device)
    bound = decode_workspace_bound(device, num_heads, num_kv_heads, head_dim,
                                   MXFP4_KV_DTYPE if kv_dtype is None else kv_dtype)
    decode_workspace(device, bound, floor=bound, stream=stream)


def paged_decode(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_tables: torch.Tensor,
    lens: torch.Tensor,
    *,
    max_seq_len: int,
    scale: float,
    lens_cumulative: bool = False,
    layout: str = LAYOUT_NHD,
    valid_mask: torch.Tensor | None = None,
    new_k: torch.Tensor | None = None,
    new_v: torch.Tensor | None = None,
    new_slots: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    split_tokens: int = 0,
    prologue: QKPrologue | None = None,
    key_limit: int = 0,
    table_read_width: int = 0,
    no_alloc: bool = False,
    k_scale: float | torch.Tensor = 1.0,
    v_scale: float | torch.Tensor = 1.0,
) -> torch.Tensor:
    """One-token paged GQA attention.

    q: [B, Hq, D]; out: [B, Hq, D] (allocated if None; it has no gradient, and
    in grad mode may not require one); lens: per-sequence
    context lengths [B], or cu_seqlens_k [B + 1] with ``lens_cumulative``.
    ``new_k``/``new_v`` ([B, Hkv, D]) are written at position len-1 (or at
    ``new_slots[b]``) and used for that position in the same launch.  With a
    ``prologue``, q and new_k are raw projections, normalised and rotated at
    ``prologue.positions[b]`` inside the launch.  ``key_limit`` (> 0) leaves
    tokens at or past it unattended and ``table_read_width`` (> 0) makes the
    attention read block 0 for table columns at or past it (the TTS kernel's
    kernel_seq_len / kernel_page_count bounds); the current row is written at
    len - 1 either way.  ``no_alloc`` launches va_paged_decode_noalloc, which
    keeps the split partials in the library's own scratch buffer instead of a
    workspace; ``out`` must then be given, so that nothing is allocated.  That
    buffer is one per GPU, shared by every stream: no_alloc calls on two
    streams would race on it, so a no_alloc call issued on another stream than
    the previous one on its GPU first makes its stream wait for that stream
    (on the GPU, outside graph capture; under capture the caller must order
    them).
    An FP8 (float8_e4m3fn) pool is read as code * k_scale / v_scale, and the
    current row is stored into it quantised; so is an MXFP4 pool, with its
    scale tensors as k_scale / v_scale (16-bit q, head_dim 64 / 128 / 256,
    groups of 1 / 2 / 4 / 8, blocks of a multiple of 16 tokens, not with
    ``no_alloc``).  ``split_tokens``: 0 splits
    contexts automatically; ``SPLIT_EXACT`` does too, for a ``max_seq_len``
    that is the batch's exact longest context (partitions fixed from it); a
    positive value fixes the partition size.
    """
    if out is not None:
        _plain_output(out, "out")
    mx4 = k_cache.dtype is MXFP4_KV_DTYPE
    fast = _FAST if _FAST_LOADED else _fast_calls()
    if (fast is not None and not no_alloc and layout in (LAYOUT_NHD, LAYOUT_HND) and
            (not mx4 or (isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)))):
        index = q.get_device()
        if index >= 0 and index == torch.cuda.current_device():
            if out is None:
                out = torch.empty_like(q)
            stream = _raw_stream(index)
            pro = prologue
            rc = (fast.paged_decode_mx4 if mx4 else fast.paged_decode)(
                q, k_cache, v_cache, block_tables, lens, out, new_k, new_v, new_slots,
                valid_mask, None if pro is None else pro.q_norm_weight,
                None if pro is None else pro.k_norm_weight,
                0.0 if pro is None else float(pro.eps),
                None if pro is None else pro.cos_sin_cache,
                None if pro is None else pro.positions, _WORKSPACES.get((index, stream)),
                lens_cumulative, layout == LAYOUT_HND,
                int(max_seq_len), float(scale), int(split_tokens), int(key_limit),
                int(table_read_width),
                k_scale if mx4 or k_scale.__class__ is float else _number(k_scale),
                v_scale if mx4 or v_scale.__class__ is float else _number(v_scale), index, stream)
            if rc == 0:
                return out
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_paged_decode_mx4" if mx4 else "va_paged_decode", rc)
            # Not taken, or a workspace is needed first: the path below.
    device = _check_gpu(q, k_cache, v_cache, block_tables, lens, valid_mask, new_k, new_v,
                        new_slots, out)
    if prologue is not None:
        _check_gpu(q, prologue.q_norm_weight, prologue.k_norm_weight, prologue.cos_sin_cache,
                   prologue.positions)
    _require(not no_alloc or out is not None, "no_alloc needs the output tensor (out=...)")
    _require(not no_alloc or not mx4, "no_alloc takes no MXFP4 pool")
    _require(q.dim() == 3, "q must be [num_seqs, num_heads, head_dim]")
    qs = q.stride()
    _require(qs[2] == 1, "q: the last dimension must be contiguous")
    B, hq, d = q.shape
    hkv, pd = pool_heads(k_cache, layout)
    _require(pd == d, f"head_dim mismatch: q {d}, pool {pd}")
    _require(hq % hkv == 0, "num_heads must be a multiple of num_kv_heads")
    if mx4:
        pool, scales = _mx4_structs(k_cache, v_cache, layout, k_scale, v_scale, q.dtype)
        _check_gpu(q, k_scale)
    else:
        _require(_pool_matches(k_cache, q.dtype),
                 "q and the KV pool must share a dtype (or the pool be FP8 for 16-bit q)")
        pool = _pool_struct(k_cache, v_cache, layout, k_scale, v_scale)
    bts = block_tables.stride()
    _require(block_tables.dim() == 2 and block_tables.shape[0] >= B,
             "block_tables must be [num_seqs, width]")
    _require(bts[1] == 1, "block_tables rows must be contiguous")
    expect = B + 1 if lens_cumulative else B
    _require(lens.dim() == 1 and lens.numel() >= expect and lens.is_contiguous(),
             f"lens must be a contiguous vector of at least {expect} entries")
    if out is None:
        out = torch.empty_like(q)
    os_ = out.stride()
    _require(out.shape == q.shape and out.dtype == q.dtype, "out must match q")
    _require(os_[2] == 1, "out: the last dimension must be contiguous")
    _require(key_limit >= 0 and table_read_width >= 0,
             "key_limit and table_read_width must be non-negative")
    fields = dict(
        struct_size=_DECODE_ARGS_SIZE, dtype=_dtype_code(q), q=q.data_ptr(),
        q_stride_seq=qs[0], q_stride_head=qs[1], out=out.data_ptr(), out_stride_seq=os_[0],
        out_stride_head=os_[1], pool=pool,
        block_tables=block_tables.data_ptr(),
        table_dtype=_index_code(block_tables, "block_tables"), table_stride_seq=bts[0],
        table_width=block_tables.shape[1], lens=lens.data_ptr(),
        lens_dtype=_index_code(lens, "lens"),
        lens_kind=N.VA_LENS_CUMULATIVE if lens_cumulative else N.VA_LENS_PER_SEQ,
        num_seqs=B, num_heads=hq, num_kv_heads=hkv, head_dim=d, max_seq_len=int(max_seq_len),
        split_tokens=int(split_tokens), scale=float(scale), key_limit=int(key_limit),
        table_read_width=int(table_read_width))
    if valid_mask is not None:
        _require(valid_mask.dim() == 2 and valid_mask.shape[0] >= B and
                 valid_mask.dtype == torch.bool and valid_mask.stride(-1) == 1,
                 "key_valid_mask must be a [num_seqs, max_seq] bool tensor")
        fields.update(valid_mask=valid_mask.data_ptr(), valid_stride_seq=valid_mask.stride(0),
                      valid_len=valid_mask.shape[1])
    _require((new_k is None) == (new_v is None), "new_k and new_v must be given together")
    if new_k is not None:
        nks, nvs = new_k.stride(), new_v.stride()
        _require(new_k.shape == (B, hkv, d) and new_v.shape == new_k.shape,
                 "new_k/new_v must be [num_seqs, num_kv_heads, head_dim]")
        _require(new_k.dtype == new_v.dtype == q.dtype, "new_k/new_v must match q's dtype")
        _require(nks[2] == 1 and nvs[2] == 1, "new_k/new_v: the last dimension must be contiguous")
        fields.update(new_k=new_k.data_ptr(), new_k_stride_seq=nks[0], new_k_stride_head=nks[1],
                      new_v=new_v.data_ptr(), new_v_stride_seq=nvs[0], new_v_stride_head=nvs[1])
    if new_slots is not None:
        _require(new_k is not None, "new_slots requires new_k/new_v")
        _require(new_slots.dim() == 1 and new_slots.numel() >= B and new_slots.is_contiguous(),
                 "new_slots must be a contiguous [num_seqs] vector")
        fields.update(new_slots=new_slots.data_ptr(),
                      new_slots_dtype=_index_code(new_slots, "new_slots"))
    pro_struct = None
    if prologue is not None:
        pro_struct = _prologue_struct(prologue, d, B)  # kept alive through the call
        fields["prologue"] = ctypes.pointer(pro_struct)
    args = N.DecodeArgs(**fields)
    lib = N.lib()
    index = _device_index(device)
    with _current(index):  # the split plan depends on the device's CU count
        if no_alloc:
            _order_noalloc(index)
            N.check("va_paged_decode_noalloc",
                    lib.va_paged_decode_noalloc(ctypes.byref(args), _raw_stream(index)))
            return out
        nbytes = (lib.va_paged_decode_mx4_workspace_bytes if mx4
                  else lib.va_paged_decode_workspace_bytes)(ctypes.byref(args))
        if nbytes:
            ws = decode_workspace(device, nbytes, floor=decode_workspace_bound(
                device, hq, hkv, d, k_cache.dtype))
            args.workspace = ws.data_ptr()
            args.workspace_bytes = ws.numel()
        if mx4:
            N.check("va_paged_decode_mx4",
                    lib.va_paged_decode_mx4(ctypes.byref(args), ctypes.byref(scales),
                                            _raw_stream(index)))
        else:
            N.check("va_paged_decode", lib.va_paged_decode(ctypes.byref(args), _raw_stream(index)))
    _written(out)
    return out


# -------------------------------------------------------------------- varlen
def varlen_attention(
    q: torch.Tensor,
    k: torch.Tensor | None,
    v: torch.Tensor | None,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    *,
    scale: float,
    causal: bool,
    k_cache: torch.Tensor | None = None,
    v_cache: torch.Tensor | None = None,
    block_tables: torch.Tensor | None = None,
    slot_mapping: torch.Tensor | None = None,
    layout: str = LAYOUT_NHD,
    out: torch.Tensor | None = None,
    k_scale: float | torch.Tensor = 1.0,
    v_scale: float | torch.Tensor = 1.0,
    prologue: QKPrologue | None = None,
) -> torch.Tensor:
    """Packed variable-length attention (flash_attn_varlen_func semantics).

    Causal attention is bottom-right aligned: query i of a sequence with
    (q_len, k_len) sees keys j <= k_len - q_len + i.  With a pool, keys
    j < k_len - q_len are read through ``block_tables``; the others from
    ``k``/``v`` rows aligned with the queries (all from the pool if ``k`` is
    None).  ``slot_mapping`` fuses store_kvcache of k/v into the same launch.
    ``max_seqlen_q`` must be at least every q_len, as for flash-attn: it sizes
    the launch, and query rows past it are not computed.  Key ranges come from
    ``cu_seqlens_k``; ``max_seqlen_k`` only bounds the context lengths for the
    launch's choice of items (the block table may be wider).  An FP8 pool
    (float8_e4m3fn codes, values code * k_scale / v_scale) is converted tile
    by tile inside the kernel (no workspace); its new rows are stored
    quantised after the attention.  An MXFP4 pool (:func:`mxfp4_kv_pool`, blocks
    of a multiple of 16 tokens), with its scale tensors as k_scale / v_scale, is
    converted inside the kernel too, which also stores the new rows; the new
    rows themselves are attended as given.  With a ``prologue`` (causal,
    head_dim 128, a 16-bit pool or none), q holds the raw query projections and
    the launch normalises and rotates them at ``prologue.positions`` (one per
    query token); k and the pool must hold processed keys.

    Without a pool, a prologue or ``out`` the call is differentiable in q, k
    and v (:func:`varlen_attention_backward`); the others return tensors without
    a gradient (in grad mode ``out`` may not require one).
    """
    if out is not None:
        _plain_output(out, "out")
    if (k_cache is None and out is None and prologue is None and k is not None and v is not None
            and (q.requires_grad or k.requires_grad or v.requires_grad)
            and torch.is_grad_enabled()):
        return _VarlenAttention.apply(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q,
                                      max_seqlen_k, scale, causal)
    pool_dtype = None if k_cache is None else k_cache.dtype
    mx4 = pool_dtype is MXFP4_KV_DTYPE
    if (not mx4 and pool_dtype is not FP8_KV_DTYPE and
            not (k_scale.__class__ is float and v_scale.__class__ is float)):
        # A 16-bit pool, or none, has no scales: whatever is given is not read,
        # but an MXFP4 pool's belong to codes.
        _require(MXFP4_SCALE_DTYPE not in (getattr(k_scale, "dtype", None),
                                           getattr(v_scale, "dtype", None)),
                 f"float8_e8m0fnu scales need an MXFP4 pool, got {pool_dtype}")
        k_scale = v_scale = 1.0
    fast = _FAST if _FAST_LOADED else _fast_calls()
    if (fast is not None and prologue is None and layout in (LAYOUT_NHD, LAYOUT_HND) and
            pool_dtype is not FP8_KV_DTYPE and
            (not mx4 or (isinstance(k_scale, torch.Tensor) and isinstance(v_scale, torch.Tensor)))):
        index = q.get_device()
        if index >= 0 and index == torch.cuda.current_device():
            if out is None:
                out = torch.empty_like(q)
            more = (k_scale, v_scale, index) if mx4 else (index,)
            rc = (fast.varlen_attention_mx4 if mx4 else fast.varlen_attention)(
                q, k, v, cu_seqlens_q, cu_seqlens_k, int(max_seqlen_q), int(max_seqlen_k),
                float(scale), bool(causal), k_cache, v_cache, block_tables, slot_mapping, out,
                layout == LAYOUT_HND, *more, _raw_stream(index))
            if rc == 0:
                return out
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_varlen_attention_mx4" if mx4 else "va_varlen_attention", rc)
    device = _check_gpu(q, k, v, cu_seqlens_q, cu_seqlens_k, k_cache, v_cache, block_tables,
                        slot_mapping, out)
    _require(q.dim() == 3, "q must be [total_q, num_heads, head_dim]")
    qs = q.stride()
    _require(qs[2] == 1, "q: the last dimension must be contiguous")
    total_q, hq, d = q.shape
    _require(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32,
             "cu_seqlens must be int32")
    _require(cu_seqlens_q.dim() == 1 and cu_seqlens_q.numel() >= 2 and
             cu_seqlens_k.numel() == cu_seqlens_q.numel(), "cu_seqlens must be [num_seqs + 1]")
    _require(cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous(),
             "cu_seqlens must be contiguous")
    num_seqs = cu_seqlens_q.numel() - 1
    fields = {}
    scales = None  # an MXFP4 pool's
    if k_cache is not None:
        _require(v_cache is not None and block_tables is not None,
                 "a KV pool needs v_cache and block_tables")
        hkv, pd = pool_heads(k_cache, layout)
        _require(pd == d, "pool head_dim must match q")
        if mx4:
            pool, scales = _mx4_structs(k_cache, v_cache, layout, k_scale, v_scale, q.dtype)
            _check_gpu(q, k_scale)
        else:
            _require(_pool_matches(k_cache, q.dtype),
                     "pool dtype must match q (or the pool be FP8 for 16-bit q)")
            pool = _pool_struct(k_cache, v_cache, layout, k_scale, v_scale)
        bts = block_tables.stride()
        _require(block_tables.dim() == 2 and block_tables.shape[0] >= num_seqs and bts[1] == 1,
                 "block_tables must be [num_seqs, width]")
        fields.update(pool=pool,
                      block_tables=block_tables.data_ptr(),
                      table_dtype=_index_code(block_tables, "block_tables"),
                      table_stride_seq=bts[0], table_width=block_tables.shape[1])
    else:
        _require(k is not None and v is not None, "k and v are required without a KV pool")
        hkv = k.shape[1]
    if k is not None:
        _require(v is not None and k.dim() == 3 and v.shape == k.shape,
                 "k/v must be [tokens, num_kv_heads, head_dim]")
        _require(k.shape[1] == hkv and k.shape[2] == d, "k/v heads must match")
        _require(k.dtype == v.dtype == q.dtype, "q/k/v dtypes must match")
        ks, vs = k.stride(), v.stride()
        _require(ks[2] == 1 and vs[2] == 1, "k/v: the last dimension must be contiguous")
        fields.update(k=k.data_ptr(), k_stride_tok=ks[0], k_stride_head=ks[1], v=v.data_ptr(),
                      v_stride_tok=vs[0], v_stride_head=vs[1])
    _require(hq % hkv == 0, "num_heads must be a multiple of num_kv_heads")
    if slot_mapping is not None:
        _require(k_cache is not None and k is not None, "slot_mapping needs a pool and k/v")
        _require(slot_mapping.dim() == 1 and slot_mapping.numel() == total_q and
                 slot_mapping.is_contiguous(), "slot_mapping must have one entry per query")
        fields.update(slot_mapping=slot_mapping.data_ptr(),
                      slot_dtype=_index_code(slot_mapping, "slot_mapping"))
    pro_struct = None
    if prologue is not None:
        _check_gpu(q, prologue.q_norm_weight, prologue.cos_sin_cache, prologue.positions)
        pro_struct = _prologue_struct(prologue, d, total_q)  # kept alive through the call
        fields["prologue"] = ctypes.pointer(pro_struct)
    if out is None:
        out = torch.empty_like(q)
    os_ = out.stride()
    _require(out.shape == q.shape and out.dtype == q.dtype, "out must match q")
    _require(os_[2] == 1, "out: the last dimension must be contiguous")
    args = N.VarlenArgs(
        struct_size=_VARLEN_ARGS_SIZE, dtype=_dtype_code(q), q=q.data_ptr(), q_stride_tok=qs[0],
        q_stride_head=qs[1], out=out.data_ptr(), out_stride_tok=os_[0], out_stride_head=os_[1],
        cu_seqlens_q=cu_seqlens_q.data_ptr(), cu_seqlens_k=cu_seqlens_k.data_ptr(),
        num_seqs=num_seqs, total_q=total_q, num_heads=hq, num_kv_heads=hkv, head_dim=d,
        max_seqlen_q=int(max_seqlen_q), max_seqlen_k=int(max_seqlen_k),
        causal=1 if causal else 0, scale=float(scale), **fields)
    lib = N.lib()
    index = _device_index(device)
    with _current(index):
        nbytes = lib.va_varlen_split_workspace_bytes(ctypes.byref(args))
        if nbytes:
            # A tensor of this call alone: torch's allocator hands its memory
            # out again in the order of this stream (or of the captured graph).
            # Without it the launch runs unsplit, as it also does when memory
            # is short.
            try:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
                args.workspace = ws.data_ptr()
                args.workspace_bytes = nbytes
            except torch.OutOfMemoryError:
                pass
        if scales is not None:
            N.check("va_varlen_attention_mx4",
                    lib.va_varlen_attention_mx4(ctypes.byref(args), ctypes.byref(scales),
                                                _raw_stream(index)))
        else:
            N.check("va_varlen_attention",
                    lib.va_varlen_attention(ctypes.byref(args), _raw_stream(index)))
    _written(out)
    return out


# ---------------------------------------------------------- varlen, backward
def _whole_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it whose rows the kernels can read: 16-byte aligned, the
    last dimension contiguous (autograd hands on expanded and offset gradients)."""
    step = 16 // t.element_size()
    if (t.stride(-1) != 1 or t.data_ptr() % 16 or
            any(st % step for st, n in zip(t.stride()[:-1], t.shape) if n > 1)):
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _near_rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy of it where its tokens are farther apart than the attention's gradient takes
    (32 MiB: lane offsets in a tile are 32-bit) and the attention itself does."""
    if t.shape[0] > 1 and t.stride(0) * t.element_size() >= 1 << 25:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _row_strides(t: torch.Tensor) -> tuple[int, int]:
    """Strides of tokens and heads; a dimension of one has none to speak of
    (torch leaves any number there)."""
    n, h, _ = t.shape
    return (t.stride(0) if n > 1 else 0), (t.stride(1) if h > 1 else 0)


def _length(n: int, name: str) -> int:
    n = int(n)
    _require(0 <= n < 2 ** 31, f"{name} must be a length, from 0 to under 2^31")
    return n


def varlen_attention_backward(
    dout: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    out: torch.Tensor,
    cu_seqlens_q: torch.Tensor,
    cu_seqlens_k: torch.Tensor,
    max_seqlen_q: int,
    max_seqlen_k: int,
    *,
    scale: float,
    causal: bool,
    dq: torch.Tensor | None = None,
    dk: torch.Tensor | None = None,
    dv: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dq, dk, dv) of :func:`varlen_attention` without a pool, from the output's
    gradient ``dout`` and the output itself ([total_q, Hq, D]).

    q, k, v, cu_seqlens, scale and causal are those of the forward call (16-bit
    rows, head_dim 64 or 128, tokens under 32 MiB apart; any group size); k and
    v of ``cu_seqlens_k``'s rows, [total_k, Hkv, D].  The probabilities are recomputed.  The maxima
    must be at least every length, as in the forward call, or 0 if they are not
    known: sequences of at most 128 rows at head_dim 64, with as many kv heads as
    heads, take one launch, in which a longer sequence than the maxima say gets
    NaN; others take two or three and go by the cumulative lengths.  Rows outside every
    sequence, queries that see no key and keys that no query sees get zeros.
    ``dq``, ``dk``, ``dv``: tensors to write into (views of one buffer, say); they
    may not overlap the inputs.  All launches are on the current stream, without
    atomics: the results repeat bit for bit."""
    if dq is None and dk is None and dv is None:
        fast, index = _fast_on(q, LAYOUT_NHD)
        if fast is not None:
            rc, made = fast.varlen_attention_backward(dout, q, k, v, out, cu_seqlens_q,
                                                      cu_seqlens_k, int(max_seqlen_q),
                                                      int(max_seqlen_k), float(scale),
                                                      bool(causal), index, _raw_stream(index))
            if rc == 0:
                return tuple(made)
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_varlen_attention_backward", rc)
    device = _check_gpu(dout, q, k, v, out, cu_seqlens_q, cu_seqlens_k, dq, dk, dv)
    _require(q.dim() == 3, "q must be [total_q, num_heads, head_dim]")
    _require(out.shape == q.shape and dout.shape == q.shape, "out and dout must match q")
    _require(k.dim() == 3 and v.shape == k.shape and k.shape[2] == q.shape[2],
             "k/v must be [total_k, num_kv_heads, head_dim]")
    _require(q.dtype == k.dtype == v.dtype == out.dtype == dout.dtype,
             "dout/q/k/v/out dtypes must match")
    _require(q.dtype in (torch.bfloat16, torch.float16), "varlen attention needs 16-bit rows")
    total_q, hq, d = q.shape
    total_k, hkv, _ = k.shape
    _require(hkv > 0 and hq % hkv == 0 and hq > 0, "num_heads must be a multiple of num_kv_heads")
    _require(cu_seqlens_q.dtype == torch.int32 and cu_seqlens_k.dtype == torch.int32,
             "cu_seqlens must be int32")
    _require(cu_seqlens_q.dim() == 1 and cu_seqlens_q.numel() >= 2 and
             cu_seqlens_k.shape == cu_seqlens_q.shape, "cu_seqlens must be [num_seqs + 1]")
    _require(cu_seqlens_q.is_contiguous() and cu_seqlens_k.is_contiguous(),
             "cu_seqlens must be contiguous")
    for n in (*q.shape, *k.shape, cu_seqlens_q.numel()):
        _length(n, "every size")
    given = []
    for name, t, like in (("dq", dq, q), ("dk", dk, k), ("dv", dv, v)):
        if t is not None:
            _require(t.shape == like.shape and t.dtype == like.dtype, f"{name} must match {name[1]}")
            given.append((name, t, ()))
    _outputs_apart(given, (dout, q, k, v, out))
    dq = torch.empty(q.shape, dtype=q.dtype, device=device) if dq is None else dq
    dk = torch.empty(k.shape, dtype=k.dtype, device=device) if dk is None else dk
    dv = torch.empty(k.shape, dtype=k.dtype, device=device) if dv is None else dv
    args = N.VarlenBwdArgs(
        struct_size=_VARLEN_BWD_ARGS_SIZE, dtype=_dtype_code(q),
        cu_seqlens_q=cu_seqlens_q.data_ptr(), cu_seqlens_k=cu_seqlens_k.data_ptr(),
        num_seqs=cu_seqlens_q.numel() - 1, total_q=total_q, total_k=total_k, num_heads=hq,
        num_kv_heads=hkv, head_dim=d, max_seqlen_q=_length(max_seqlen_q, "max_seqlen_q"),
        max_seqlen_k=_length(max_seqlen_k, "max_seqlen_k"), causal=1 if causal else 0,
        scale=float(scale))
    for name, t in (("q", q), ("k", k), ("v", v), ("out", out), ("dout", dout), ("dq", dq),
                    ("dk", dk), ("dv", dv)):
        _require(t.stride(2) == 1, f"{name}: the last dimension must be contiguous")
        tok, head = _row_strides(t)
        setattr(args, name, t.data_ptr())
        setattr(args, name + "_stride_tok", tok)
        setattr(args, name + "_stride_head", head)
    lib = N.lib()
    index = _device_index(device)
    with _current(index):
        # Two or three floats a query row, for this call alone: torch's allocator
        # hands them out again in the order of this stream (or captured graph).
        nbytes = lib.va_varlen_attention_backward_workspace_bytes(ctypes.byref(args))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        args.workspace = ws.data_ptr()
        args.workspace_bytes = nbytes
        N.check("va_varlen_attention_backward",
                lib.va_varlen_attention_backward(ctypes.byref(args), _raw_stream(index)))
    _written(*(t for _, t, _ in given))
    return dq, dk, dv


class _VarlenAttention(torch.autograd.Function):
    """varlen_attention without a pool, with its gradient."""

    @staticmethod
    def forward(ctx, q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k, scale, causal):
        out = varlen_attention(q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
                               scale=scale, causal=causal)
        ctx.save_for_backward(q, k, v, out, cu_seqlens_q, cu_seqlens_k)
        ctx.call = (max_seqlen_q, max_seqlen_k, scale, causal)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, out, cu_q, cu_k = ctx.saved_tensors
        max_q, max_k, scale, causal = ctx.call
        dout, q, k, v = (_near_rows(t) for t in (_whole_rows(dout), q, k, v))
        grads = varlen_attention_backward(dout, q, k, v, out, cu_q, cu_k, max_q, max_k, scale=scale,
                                          causal=causal)
        wanted = (g if need else None for g, need in zip(grads, ctx.needs_input_grad))
        return (*wanted, None, None, None, None, None, None)


# ------------------------------------------------------------- step metadata
@dataclass(frozen=True)
class BatchMetadata:
    """A step's attention metadata on the GPU (see :func:`batch_metadata`)."""

    positions: torch.Tensor  # [max_tokens] int64
    slot_mapping: torch.Tensor  # [max_tokens] int32
    cu_seqlens_q: torch.Tensor  # [rows + 1] int32
    cu_seqlens_k: torch.Tensor  # [rows + 1] int32
    block_tables: torch.Tensor  # [rows, table_width] int32
    totals: torch.Tensor
    """[5] int32: tokens, longest query, longest context, free blocks left, blocks missing."""

    @property
    def free_count(self) -> torch.Tensor:
        """[1] int32: the free list's count after the step."""
        return self.totals[3:4]


def batch_metadata(
    lens: torch.Tensor,
    num_computed: torch.Tensor,
    request_tables: torch.Tensor,
    block_size: int,
    *,
    max_tokens: int,
    rows: torch.Tensor | None = None,
    padded_batch: int = 0,
    table_width: int | None = None,
    free_blocks: torch.Tensor | None = None,
    free_count: torch.Tensor | None = None,
    out: BatchMetadata | None = None,
    cut: bool = False,
) -> BatchMetadata:
    """Positions, slots, cumulative lengths and block tables of a step, built
    on the GPU from the requests' lengths (engine/model_runner.py:183-233,
    engine/graph_runner.py:150-191 build them on the host).

    Request i has ``num_computed[i]`` tokens behind it and ``lens[i]`` after the
    step (int32 or int64 [B]); its block table is row ``rows[i]`` (int32; row i
    without it) of ``request_tables`` ([requests, width] int32).  Its new tokens'
    positions and slots follow those of the requests before it; entries up to
    ``max_tokens`` behind the last token are 0 and -1, and tokens past it are
    not written.  The cumulative lengths count those tokens too, and attention
    over ``max_tokens`` rows may be given them only where ``totals[0]``, the
    step's tokens, is no more; with ``cut`` they stop at ``max_tokens`` (the
    keys of a request that is cut end with its queries), and may be given to
    attention whatever the lengths say.  ``block_tables`` row i holds the request's blocks, then -1
    (``table_width`` columns, request_tables' width by default).  Rows B ..
    ``padded_batch`` - 1 are a captured decode graph's padding: one token at
    position 0 with slot -1, table row 0, key length 1.  A row or column outside
    request_tables, or a negative block id, gives slot -1.

    With ``free_blocks`` ([n] int32) and ``free_count`` ([1] int32), requests
    hold the blocks of their computed tokens, and the blocks of their new
    columns are taken from the list's end, in request order: the k-th taken is
    ``free_blocks[free_count - 1 - k]``.  They are written into request_tables
    (``rows`` must be distinct; a request whose row is outside it takes none);
    columns that the list does not reach get -1 there, and so do their slots.
    ``free_count`` itself is not changed: the
    count left is ``totals[3]`` (``result.free_count``), the blocks that were
    missing ``totals[4]`` (an ``out`` that free_count lies in is refused: copy
    the count left into it after the launch).  A step that lacked blocks, or had
    more tokens than ``max_tokens``, is to be made again from the list and the
    ``num_computed`` it began with: columns below ``num_computed`` are held
    whatever the table says, so those that got -1 would stay without a block.

    ``out``: tensors of an earlier result of the same sizes to write into (a
    captured graph's static buffers); they may not overlap the inputs."""
    if out is None and (table_width is None or table_width >= 0):
        fast, index = _fast_on(lens, LAYOUT_NHD)
        if fast is not None:
            rc, made = fast.batch_metadata(lens, num_computed, request_tables, int(block_size),
                                           int(max_tokens), rows, int(padded_batch),
                                           -1 if table_width is None else int(table_width),
                                           free_blocks, free_count, bool(cut), index,
                                           _raw_stream(index))
            if rc == 0:
                return BatchMetadata(*made)
            if _FAST_NOT_TAKEN < rc < 0:
                N.check("va_batch_metadata", rc)
    device = _check_gpu(lens, num_computed, request_tables, rows, free_blocks, free_count)
    _require(lens.dim() == 1 and num_computed.shape == lens.shape and lens.is_contiguous()
             and num_computed.is_contiguous(), "lens and num_computed must be [B] vectors")
    _require(lens.dtype == num_computed.dtype, "lens and num_computed must share a dtype")
    _require(request_tables.dim() == 2 and request_tables.dtype == torch.int32
             and request_tables.stride(1) == 1, "request_tables must be int32 [requests, width]")
    _require(block_size > 0, "block_size must be positive")
    B = int(lens.numel())
    if rows is not None:
        _require(rows.dtype == torch.int32 and rows.dim() == 1 and rows.numel() >= B
                 and rows.is_contiguous(), "rows must be a contiguous int32 [B] vector")
    _require((free_blocks is None) == (free_count is None),
             "free_blocks and free_count must be given together")
    if free_blocks is not None:
        _require(free_blocks.dtype == torch.int32 and free_blocks.dim() == 1
                 and free_blocks.is_contiguous(), "free_blocks must be a contiguous int32 vector")
        _require(free_count.dtype == torch.int32 and free_count.numel() == 1,
                 "free_count must be one int32")
    size = max(B, int(padded_batch))
    width = int(request_tables.shape[1]) if table_width is None else int(table_width)
    _require(max_tokens >= 0 and width >= 0, "max_tokens and table_width must be non-negative")
    if out is None:
        i32 = {"dtype": torch.int32, "device": device}
        out = BatchMetadata(torch.empty(max_tokens, dtype=torch.int64, device=device),
                            torch.empty(max_tokens, **i32), torch.empty(size + 1, **i32),
                            torch.empty(size + 1, **i32), torch.empty(size, width, **i32),
                            torch.empty(5, **i32))
    else:
        _check_gpu(lens, out.positions, out.slot_mapping, out.cu_seqlens_q, out.cu_seqlens_k,
                   out.block_tables, out.totals)
        for t, n, dtype in ((out.positions, max_tokens, torch.int64),
                            (out.slot_mapping, max_tokens, torch.int32),
                            (out.cu_seqlens_q, size + 1, torch.int32),
                            (out.cu_seqlens_k, size + 1, torch.int32),
                            (out.totals, 5, torch.int32)):
            _require(t.dim() == 1 and t.numel() == n and t.dtype == dtype and t.is_contiguous(),
                     "out: tensors must have the sizes and types of this call's result")
        _require(out.block_tables.shape == (size, width) and out.block_tables.dtype == torch.int32
                 and out.block_tables.stride(1) == 1,
                 "out: block_tables must be int32 [rows, table_width]")
    args = N.BatchArgs(
        struct_size=ctypes.sizeof(N.BatchArgs), index_dtype=_index_code(lens, "lens"),
        lens=lens.data_ptr(), num_computed=num_computed.data_ptr(),
        request_tables=request_tables.data_ptr(), request_stride=request_tables.stride(0),
        num_requests=request_tables.shape[0], request_width=request_tables.shape[1],
        rows=N.ptr(rows), num_seqs=B, padded_seqs=size, block_size=int(block_size),
        max_tokens=int(max_tokens), positions=out.positions.data_ptr(),
        slot_mapping=out.slot_mapping.data_ptr(), cu_seqlens_q=out.cu_seqlens_q.data_ptr(),
        cu_seqlens_k=out.cu_seqlens_k.data_ptr(), block_tables=out.block_tables.data_ptr(),
        table_stride=out.block_tables.stride(0), table_width=width,
        totals=out.totals.data_ptr(), free_blocks=N.ptr(free_blocks), free_count=N.ptr(free_count),
        free_capacity=0 if free_blocks is None else free_blocks.numel(), cut=bool(cut))
    index = _device_index(device)
    with _current(index):
        N.check("va_batch_metadata",
                N.lib().va_batch_metadata(ctypes.byref(args), _raw_stream(index)))
    _written(out.positions, out.slot_mapping, out.cu_seqlens_q, out.cu_seqlens_k, out.block_tables,
             out.totals)
    return out


def default_scale(head_dim: int) -> float:
    return 1.0 / math.sqrt(head_dim)
