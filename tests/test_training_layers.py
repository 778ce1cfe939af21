"""CPU checks of the layers' host logic in a training pass: which calls a layer makes, and in
which grad mode, with the operators stood in for."""

import pytest
import torch

from voiceagent_amd import ops
from voiceagent_amd.layers import (AttentionContext, PagedAttention, Qwen3AttentionCore,
                                   attention_context)

HQ, HKV, D, T = 4, 2, 128, 6


@pytest.fixture
def calls(monkeypatch):
    """The operators a layer calls: (name, whether grad mode was on, whether a prologue went along)."""
    made = []

    def stand_in(name, result):
        def call(*args, prologue=None, **kw):
            made.append((name, torch.is_grad_enabled(), prologue is not None))
            return result(*args)
        monkeypatch.setattr(ops, name, call)

    stand_in("qk_norm_rope", lambda q, k, pro: (q, k))
    stand_in("rotary_embedding", lambda q, k, *rest: (q, k))
    stand_in("varlen_attention", lambda q, k, v, *rest: q)
    stand_in("paged_decode", lambda q, *rest: q)
    stand_in("store_kvcache", lambda *rest: None)
    return made


def _rows(*asks):
    rows = [torch.zeros(T, h, D, dtype=torch.bfloat16) for h in (HQ, HKV, HKV)]
    for t, ask in zip(rows, asks):
        t.requires_grad_(ask)
    return rows


def _context(slots=None):
    cu = torch.tensor([0, T], dtype=torch.int32)
    return attention_context(AttentionContext(cu, cu, T, T, slots, None))


@pytest.mark.parametrize("asks", ["none", "q", "k", "v", "q weight", "k weight"])
def test_a_launch_with_the_prologue_takes_nothing_that_asks_for_a_gradient(calls, asks):
    """A launch that applies the query prologue has no gradient: whatever asks for one goes through
    the prologue's own call, v alone too."""
    core = Qwen3AttentionCore(HQ, D, HKV, max_position=16)
    core.varlen_fuse_prologue = True
    core.q_norm_weight.requires_grad_(asks == "q weight")
    core.k_norm_weight.requires_grad_(asks == "k weight")
    with _context():
        core(torch.arange(T), *_rows(*(asks == name for name in "qkv")))
    fused = asks == "none"
    assert calls == [("qk_norm_rope", True, False), ("varlen_attention", True, fused)]
    calls.clear()
    with torch.no_grad(), _context():
        core(torch.arange(T), *_rows(*(asks == name for name in "qkv")))
    assert calls == [("qk_norm_rope", False, False), ("varlen_attention", False, True)]


@pytest.mark.parametrize("fuse_prologue,fuse_store", [(True, True), (True, False), (False, True), (False, False)])
@pytest.mark.parametrize("asks", ["weights", "rows"])
def test_over_a_cache_the_prologue_runs_without_a_graph(calls, fuse_prologue, fuse_store, asks):
    """Serving without torch.no_grad(): the prologue saves nothing for a backward pass that cannot
    be, however the layer's launches are chosen."""
    core = Qwen3AttentionCore(HQ, D, HKV, max_position=16)  # (its weights ask for a gradient)
    core.requires_grad_(asks == "weights")
    core.fuse_prologue, core.fuse_store = fuse_prologue, fuse_store
    core.k_cache = core.v_cache = torch.zeros(4, 16, HKV, D, dtype=torch.bfloat16)
    with _context(torch.arange(T)):
        core(torch.arange(T), *_rows(*[asks == "rows"] * 3))
    assert [on for name, on, _ in calls if name == "qk_norm_rope"] == [False]
    core.k_cache = torch.tensor([])
    calls.clear()
    with _context():
        core(torch.arange(T), *_rows(*[asks == "rows"] * 3))
    assert [on for name, on, _ in calls if name == "qk_norm_rope"] == [True]


# ------------------------------------------------------------------ given outputs in grad mode
def test_outputs_that_require_a_gradient_are_refused():
    """Written through its pointer, such an output would keep its old place in the graph: the
    gradient of what is written flowed on as if nothing had been done to it."""
    leaf = torch.zeros(4, 2, 64, requires_grad=True)
    x, table, pos, w = leaf * 1, torch.zeros(9, 64), torch.zeros(4, dtype=torch.int64), torch.ones(64)
    y, cu = torch.zeros(4, 2, 64), torch.tensor([0, 4], dtype=torch.int32)
    pro = ops.QKPrologue(w, w, 1e-6, table, pos)
    bad = [lambda: ops.rotary_embedding(x, y, table, pos, q_out=x),
           lambda: ops.rotary_embedding(y, x, table, pos, q_out=y, k_out=x),
           lambda: ops.rotary_embedding(leaf, None, table, pos, q_out=leaf),
           lambda: ops.rotary_embedding(y, None, table, pos, q_out=x),
           lambda: ops.qk_norm_rope(x, y, pro, q_out=x, k_out=y),
           lambda: ops.qk_norm_rope(y, x, pro, k_out=x),
           lambda: ops.qk_norm_rope(None, x, pro, k_out=x),
           lambda: ops.varlen_attention(y, y, y, cu, cu, 4, 4, scale=1.0, causal=True, out=x),
           lambda: ops.paged_decode(y, y[None], y[None], cu[None], cu, max_seq_len=1, scale=1.0, out=x),
           lambda: ops._outputs_apart([("dq", x, ())], ())]
    for call in bad:
        with pytest.raises(ops.AttentionArgumentError, match="requires a gradient"):
            call()
    # Without a graph nothing is falsified: the next check is what refuses the CPU's tensors.
    with torch.no_grad():
        for call in bad[:-1]:
            with pytest.raises(ops.AttentionArgumentError, match="GPU"):
                call()
        bad[-1]()


def test_written_outputs_count_as_changed():
    x = torch.zeros(3, requires_grad=True)
    y = x * 1
    z = y.square()  # saves y
    with torch.no_grad():
        ops._written(y, None)
    assert y._version == 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with torch.inference_mode():
        ops._written(torch.zeros(2))  # (has no count)


# ------------------------------------------------------------------------------ given outputs
def test_outputs_whose_rows_overlap_are_refused():
    x = torch.zeros(4096)
    for sizes, strides in (((8, 4, 64), (32, 8, 1)), ((8, 4, 64), (256, 32, 1)),  # heads
                           ((8, 4, 64), (128, 64, 1)), ((8, 4, 64), (64, 512 - 64, 1)),  # tokens
                           ((8, 4, 64), (256, 0, 1)), ((8, 4, 64), (0, 64, 1)), ((2, 1, 64), (63, 1, 1))):
        t = x.as_strided(sizes, strides)
        assert len({i for i in torch.arange(4096).as_strided(sizes, strides).flatten().tolist()}) < t.numel()
        with pytest.raises(ops.AttentionArgumentError, match="dq's rows may not overlap"):
            ops._outputs_apart([("dq", t, ())], ())
    # Rows side by side, far apart, heads ahead of tokens, one of either, none.
    for sizes, strides in (((8, 4, 64), (256, 64, 1)), ((8, 4, 64), (500, 100, 1)), ((8, 4, 64), (64, 512, 1)),
                           ((8, 1, 64), (64, 0, 1)), ((1, 4, 64), (1, 64, 1)), ((1, 1, 64), (0, 0, 1)),
                           ((0, 4, 64), (0, 64, 1))):
        t = x.as_strided(sizes, strides)
        assert len({i for i in torch.arange(4096).as_strided(sizes, strides).flatten().tolist()}) == t.numel()
        ops._outputs_apart([("dq", t, ())], ())


# ------------------------------------------------------------- rows that only the forward takes
def test_rows_far_apart_reach_the_gradient_as_copies(monkeypatch):
    """The attention takes q at any distance between tokens and k and v up to 64 MiB, its gradient
    under 32: autograd copies rows that are farther apart."""
    step = 1 << 24  # elements of 2 bytes: 32 MiB
    buf = torch.zeros(step + 4096, dtype=torch.bfloat16)
    seen = {}

    def backward(dout, q, k, v, out, *rest, **kw):
        seen.update(dout=dout, q=q, k=k, v=v)
        return q, k, v

    monkeypatch.setattr(ops, "varlen_attention", lambda q, *rest, **kw: torch.zeros(q.shape, dtype=q.dtype))
    monkeypatch.setattr(ops, "varlen_attention_backward", backward)
    cu = torch.tensor([0, 2], dtype=torch.int32)
    for st, copied in ((step, True), (step - 8, False)):
        far = {n: buf.as_strided((2, 2, 64), (st, 64, 1), i * 128) for i, n in enumerate(("q", "k", "v", "dout"))}
        rows = [far[n].detach().requires_grad_() for n in "qkv"]
        out = ops._VarlenAttention.apply(*rows, cu, cu, 2, 2, 1.0, True)
        out.backward(far["dout"])
        for n, t in seen.items():
            assert (t.data_ptr() != far[n].data_ptr()) == copied, n
            assert t.stride(0) * 2 < 1 << 25 and torch.equal(t, far[n])
    one = buf.as_strided((1, 2, 64), (step, 64, 1))  # a single row has no distance
    assert ops._near_rows(one) is one


def test_heads_between_one_anothers_are_apart():
    """q, k and v of a buffer [tokens, heads, 3, elements] share nothing; whatever is called apart
    is so, element by element."""
    T, H, D3 = 5, 3, 8
    for dims in ((T, H, 3, D3), (H, T, 3, D3)):
        buf = torch.zeros(dims)
        parts = [buf[:, :, i] for i in range(3)]
        if dims[0] == H:
            parts = [t.transpose(0, 1) for t in parts]
        ops._outputs_apart([("dq", parts[0], ()), ("dk", parts[1], ()), ("dv", parts[2], ())], ())
        assert not ops._apart(parts[0], parts[0]) and not ops._apart(parts[1], buf.view(T, H, 24) if dims[0] == T
                                                                     else buf.view(H, T, 24).transpose(0, 1))
    g = torch.Generator().manual_seed(0)
    memory, at = torch.zeros(4000), torch.arange(4000)
    pick = lambda *xs: xs[int(torch.randint(len(xs), (), generator=g))]  # noqa: E731
    seen = [0, 0]
    for _ in range(3000):
        views, where = [], []
        for _ in range(2):
            sizes = (pick(1, 2, 5), pick(1, 3, 4), 8)
            strides = (pick(8, 16, 24, 32, 64, 72, 96, 120, 7), pick(8, 16, 24, 40, 64, 7), 1)
            offset = pick(0, 8, 16, 24, 32, 48, 96, 500, 3)
            views.append(memory.as_strided(sizes, strides, offset))
            where.append(set(at.as_strided(sizes, strides, offset).flatten().tolist()))
        share = bool(where[0] & where[1])
        seen[share] += 1
        assert not (share and ops._apart(*views)), (views[0].shape, views[0].stride(), views[1].shape, views[1].stride())
    assert min(seen) > 500


def test_an_output_without_its_input_is_refused():
    x, w = torch.zeros(4, 2, 64), torch.ones(64)
    pro = ops.QKPrologue(w, w, 1e-6, torch.zeros(9, 64), torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ops.AttentionArgumentError, match="dq without q"):
        ops.qk_norm_rope_backward(None, x, None, x, pro, dq=torch.zeros(4, 2, 64))


def test_sizes_past_the_argument_blocks_32_bits_are_refused(monkeypatch):
    """2^32 + 4 tokens would be 4 of them there."""
    monkeypatch.setattr(ops, "_check_gpu", lambda *tensors: torch.device("cpu"))  # (host checks alone)
    table, pos, cu = torch.zeros(9, 2), torch.zeros(4, dtype=torch.int64), torch.tensor([0, 4], dtype=torch.int32)
    x, many = torch.zeros(4, 1, 2), torch.zeros(1, 1, 2).expand(2 ** 32 + 4, 1, 2)
    for call in (lambda: ops.rotary_embedding(many, None, table, pos, q_out=many),
                 lambda: ops.rotary_embedding(x, torch.zeros(1, 1, 1).expand(4, 2 ** 32 + 1, 2), table, pos, q_out=x),
                 lambda: ops.rotary_embedding(x, None, torch.zeros(1, 2).expand(2 ** 32 + 1, 2), pos, q_out=x),
                 lambda: ops.varlen_attention_backward(
                     *[t.bfloat16() for t in (x, x)], *[torch.zeros(1, 1, 2, dtype=torch.bfloat16).expand(2 ** 32 + 4, 1, 2)] * 2,
                     x.bfloat16(), cu, cu, 4, 4, scale=1.0, causal=True, dq=x.bfloat16())):
        with pytest.raises(ops.AttentionArgumentError, match=r"under 2\^31"):
            call()
