"""Operators of a 4-bit KV cache, each in a plain form and through its public entry point.

The cache holds K and V rows as OCP MXFP4: 4-bit e2m1 codes, two to a byte (the even element in
the low half), with one power-of-two scale (e8m0, a biased exponent) for each 32 elements of a
row.  A case is one of four kinds of call:

store    new K/V rows are quantised into the pool at their slots, and read back from it.
decode   one query token per sequence over the pool; ``fused``: the current K/V rows are stored
         in the same call and attended as stored.
prefill  prompts (and decoding sequences beside them) over a cached prefix in the pool, the new
         rows in 16 bits, stored in the same call.
batch    a step's positions, slots, cumulative lengths and block tables, built on the GPU from
         the requests' lengths; ``alloc``: the new tokens' blocks are taken from a free list.

Geometry is the decoder's (16 query heads, 8 KV heads, head_dim 128, blocks of 16 tokens) where a
case does not say otherwise.  Lengths follow from the case alone; the seed makes the values, the
block order and the slots.
"""

from __future__ import annotations

import math
import random

import torch

own = False

GROUP = 32
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
#: Range of the scales' biased exponents: the largest and smallest code value times the scale stay
#: representable in the rows' type.
SCALE_RANGE = {torch.bfloat16: (2, 252), torch.float16: (104, 140)}
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # The rows of one decode step of 32 sequences, stored on their own.
        store("store-32", 32),
        # The rows of a burst of prompts (32 of 50-450 tokens).
        store("store-8561", 8561),
        # One user speaking: a step of a single 30 s utterance.
        decode("decode-1", 1, 430, 430),
        # The serving batch: 32 utterances of a few seconds to half a minute, the current rows
        # stored in the same call.
        decode("decode-32", 32, 60, 600, fused=True),
        # A full server.
        decode("decode-256", 256, 60, 600),
        # Long-form audio: contexts of thousands of tokens.
        decode("decode-8-long", 8, 4096, 16384),
        # The talker over its head-major pool, with leading padding masked, 64-bit tables.
        decode("talker-4", 4, 1100, 1500, fused=True, mask=True, layout="hnd", wide=True, dtype="f16"),
        # Streams that add a few seconds of audio to a cached context.
        prefill("prefill-4-prefix", prompts=4, lo=200, hi=300, plo=2048, phi=8192),
        # A short chunk at the end of a long recording.
        prefill("prefill-1-chunk", prompts=1, lo=61, hi=61, plo=16384, phi=16384),
        # A continuous-batching step: 28 decoding sequences and 4 prompts over cached prefixes.
        prefill("mixed-32", prompts=4, lo=50, hi=450, plo=64, phi=512, decodes=28, dlo=60, dhi=600),
        # A decode step of 32 sequences in a bucket of 64 rows.
        batch("batch-32", 32, lo=60, hi=600, new=1, padded=64, width=64),
        # A burst of 256 prompts, blocks taken from the free list.
        batch("batch-256", 256, lo=50, hi=450, new=0, width=2048, alloc=True),
    ]


def store(name, rows, *, hkv=8, d=128, block=16, layout="nhd", dtype="bf16", wide=False, mix=0):
    return {"name": name, "kind": "store", "rows": rows, "hkv": hkv, "d": d, "block": block,
            "layout": layout, "dtype": dtype, "wide": wide, "mix": mix}


def decode(name, batch, lo, hi, *, hq=16, hkv=8, d=128, block=16, layout="nhd", dtype="bf16",
           fused=False, mask=False, wide=False, exact=True, mix=0):
    return {"name": name, "kind": "decode", "batch": batch, "lo": lo, "hi": hi, "hq": hq, "hkv": hkv,
            "d": d, "block": block, "layout": layout, "dtype": dtype, "fused": fused, "mask": mask,
            "wide": wide, "exact": exact, "mix": mix}


def prefill(name, *, prompts, lo, hi, plo, phi, decodes=0, dlo=0, dhi=0, hq=16, hkv=8, d=128,
            block=16, layout="nhd", dtype="bf16", mix=0):
    return {"name": name, "kind": "prefill", "prompts": prompts, "lo": lo, "hi": hi, "plo": plo,
            "phi": phi, "decodes": decodes, "dlo": dlo, "dhi": dhi, "hq": hq, "hkv": hkv, "d": d,
            "block": block, "layout": layout, "dtype": dtype, "mix": mix}


def batch(name, requests, *, lo, hi, new, width, padded=0, block=16, alloc=False, wide=False, mix=0):
    """``new``: tokens that each request adds (0: all of its tokens are new)."""
    return {"name": name, "kind": "batch", "requests": requests, "lo": lo, "hi": hi, "new": new,
            "width": width, "padded": padded, "block": block, "alloc": alloc, "wide": wide, "mix": mix}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 8), (16, 8), (32, 8), (16, 16), (8, 1), (16, 4)]


def draw(rng):
    """One more case of the listed ranges: no decode reads more than decode-8-long, no prefill
    multiplies more than prefill-4-prefix, no store or batch writes more than the listed ones."""
    kind = rng.choice(["store", "decode", "decode", "prefill", "prefill", "batch"])
    mix = rng.randrange(1, 1 << 20)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    layout = rng.choice(["nhd", "nhd", "hnd"])
    block = rng.choice([16, 16, 32, 64, 256])
    hq, hkv = rng.choice(HEADS)
    if kind == "store":
        d = rng.choice([64, 128, 128, 256])
        case = store("", _log(rng, 1, 8561 * 8 * 128 // (hkv * d)), hkv=hkv, d=d, block=block,
                     layout=layout, dtype=dtype, wide=rng.random() < 0.3, mix=mix)
    elif kind == "decode":
        d = rng.choice([64, 128, 128, 128, 256])
        most = 80000 * 8 * 128 // (hkv * d)  # tokens in all
        size = _log(rng, 1, 300)
        hi = _log(rng, 4, max(8, min(16384, most // size)))
        case = decode("", size, max(1, int(hi * rng.uniform(0.05, 1.0))), hi, hq=hq, hkv=hkv, d=d,
                      block=block, layout=layout, dtype=dtype, fused=rng.random() < 0.5,
                      mask=rng.random() < 0.3, wide=rng.random() < 0.3, exact=rng.random() < 0.7, mix=mix)
    elif kind == "prefill":
        d = rng.choice([64, 128, 128])
        prompts = _log(rng, 1, 12)
        hi = _log(rng, 2, 700 // prompts ** 0.75 + 2)
        phi = _log(rng, 32, 8192 / prompts ** 0.5)
        decodes = rng.choice([0, _log(rng, 1, 32)])
        dhi = _log(rng, 16, 2000 / max(1, decodes) ** 0.4 + 16)
        case = prefill("", prompts=prompts, lo=max(1, int(hi * rng.uniform(0.2, 1.0))), hi=hi,
                       plo=int(phi * rng.uniform(0.0, 1.0)), phi=phi, decodes=decodes,
                       dlo=max(1, dhi // 8), dhi=dhi, hq=hq, hkv=hkv, d=d, block=block, layout=layout,
                       dtype=dtype, mix=mix)
    else:
        requests = _log(rng, 1, 256)
        hi = _log(rng, 16, max(32, min(16384, 100000 // requests)))
        new = rng.choice([1, 0, _log(rng, 1, hi)])
        case = batch("", requests, lo=max(1, int(hi * rng.uniform(0.05, 1.0))), hi=hi, new=new,
                     width=-(-hi // block) + rng.choice([0, 0, 7, 100]),
                     padded=rng.choice([0, requests + rng.randrange(0, 9)]), block=block,
                     alloc=rng.random() < 0.5, wide=rng.random() < 0.3, mix=mix)
    del case["name"]
    return case


def lengths(case):
    """(computed, context) lengths of the case's sequences, the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "decode":
        lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
        return [n - 1 for n in lens], lens
    if case["kind"] == "prefill":
        pre = [rng.randint(case["plo"], case["phi"]) for _ in range(case["prompts"])]
        lens = [p + rng.randint(case["lo"], case["hi"]) for p in pre]
        more = [rng.randint(case["dlo"], case["dhi"]) for _ in range(case["decodes"])]
        return pre + [n - 1 for n in more], lens + more
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["requests"])]
    return [max(0, n - case["new"]) if case["new"] else 0 for n in lens], lens


def work(case):
    """Bytes and operations of one pass: each cached row that a query sees read once, q, new rows
    and outputs once."""
    row = lambda: case["hkv"] * case["d"] * (0.5 + 1 / GROUP) * 2  # noqa: E731  K and V of a token
    if case["kind"] == "store":
        n = case["rows"]
        # The 16-bit rows in, the codes out; read back: the codes in, the 16-bit rows out.
        return {"bytes": n * 2 * (case["hkv"] * case["d"] * 4 + row()), "flops": n * case["hkv"] * case["d"] * 2 * 2}
    if case["kind"] == "batch":
        done, lens = lengths(case)
        tokens = sum(lens) - sum(done) + max(0, case["padded"] - len(lens))
        rows = max(case["padded"], len(lens))
        return {"bytes": tokens * 12 + rows * (case["width"] * 4 + 12 + 8) + sum(-(-n // case["block"]) for n in lens) * 4, "flops": tokens}
    done, lens = lengths(case)
    new = [n - p for p, n in zip(done, lens)]
    width = case["hq"] * case["d"]
    flops = 4 * width * sum(m * p + m * (m + 1) // 2 for p, m in zip(done, new))
    tokens = sum(new)
    if case["kind"] == "decode":
        bytes_ = sum(lens) * row() + tokens * width * 2 * 2
        if case["fused"]:  # new rows in, codes out, and read back
            bytes_ += tokens * (case["hkv"] * case["d"] * 8 + 2 * row())
        return {"bytes": bytes_, "flops": flops}
    return {"bytes": sum(done) * row() + tokens * (width * 4 + case["hkv"] * case["d"] * 8 + 2 * row()), "flops": flops}


# ------------------------------------------------------------------------------- the plain forms
def quantise(x):
    """x [..., D] (16-bit) to (codes [..., D/2], scales [..., D/32]), bytes.  The scale is the
    smallest power of two 2^e with max |x| < 7 * 2^e: the largest element is then off by at most
    one 2^e, half the widest step of the grid; the codes are rounded to nearest, ties to even."""
    lo, hi = SCALE_RANGE[x.dtype]
    g = x.float().unflatten(-1, (-1, GROUP))
    amax = g.abs().amax(-1)
    e = (((amax.view(torch.int32) + 0x200000) >> 23) - 2).clamp(lo, hi)
    inv = ((254 - e) << 23).view(torch.float32)  # 2^-(e - 127)
    y = g.abs() * inv.unsqueeze(-1)
    c = ((y > 0.25).int() + (y >= 0.75).int() + (y > 1.25).int() + (y >= 1.75).int() + (y > 2.5).int()
         + (y >= 3.5).int() + (y > 5.0).int())
    c = (c + torch.signbit(g).int() * 8).flatten(-2)
    return (c[..., 0::2] + c[..., 1::2] * 16).to(torch.uint8), e.to(torch.uint8)


def values(codes, scales):
    """The rows that (codes, scales) stand for, in 32 bits."""
    grid = torch.tensor(GRID + tuple(-v for v in GRID), dtype=torch.float32, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    s = (scales.int() << 23).view(torch.float32)
    return (grid[c].unflatten(-1, (-1, GROUP)) * s.unsqueeze(-1)).flatten(-2)


def rows_at(pool, slots, block, layout):
    """Rows [..., Hkv, n] of a byte pool at slots [...]."""
    blk, off = slots // block, slots % block
    return pool[blk, off] if layout == "nhd" else pool[blk, :, off]


def put_rows(pool, slots, rows, block, layout):
    blk, off = slots // block, slots % block
    if layout == "nhd":
        pool[blk, off] = rows
    else:
        pool[blk, :, off] = rows


def plain_store(s):
    """The new rows into the pools; what the pools then hold for them, in the rows' type."""
    got = []
    for x, codes, scales in ((s["new_k"], s["kc"], s["ks"]), (s["new_v"], s["vc"], s["vs"])):
        c, e = quantise(x)
        put_rows(codes, s["slots"].long(), c, s["block"], s["layout"])
        put_rows(scales, s["slots"].long(), e, s["block"], s["layout"])
        got.append(values(c, e).to(x.dtype))
    return got


def plain_cached(s, pos):
    """K and V [B, L, Hkv, D] of the positions pos [B, L] through the block tables."""
    slots = s["tables"].long().clamp(min=0).gather(1, pos // s["block"]) * s["block"] + pos % s["block"]
    at = lambda pool: rows_at(pool, slots, s["block"], s["layout"])  # noqa: E731
    return values(at(s["kc"]), at(s["ks"])), values(at(s["vc"]), at(s["vs"]))


def plain_softmax(x, live):
    x = torch.where(live, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, torch.zeros_like(p))


def plain_decode(s):
    got = plain_store(s) if s["fused"] else []
    q = s["q"].float()
    size, hq, d = q.shape
    lens = s["lens"].long().unsqueeze(1)
    pos = torch.arange(s["longest"], device=q.device).unsqueeze(0).minimum(lens - 1)
    k, v = plain_cached(s, pos)
    live = torch.arange(s["longest"], device=q.device).unsqueeze(0) < lens
    if s["valid"] is not None:
        live = live & s["valid"]
    hkv = k.shape[2]
    x = torch.matmul(q.view(size, hkv, hq // hkv, d) * s["scale"], k.permute(0, 2, 3, 1).contiguous())
    p = plain_softmax(x, live[:, None, None, :])
    out = torch.matmul(p, v.transpose(1, 2).contiguous()).view(size, hq, d)
    return {"out": out.to(s["q"].dtype), "stored": got}


def plain_prefill(s):
    got = plain_store(s)
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    qlen, klen = cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1]
    prefix = klen - qlen
    size, most_q, most_k = qlen.numel(), s["most_q"], s["longest"]
    qi = torch.arange(most_q, device=DEV)
    kj = torch.arange(most_k, device=DEV).unsqueeze(0).minimum(klen.unsqueeze(1) - 1)
    q = s["q"].float()[(cu_q[:-1, None] + qi.minimum(qlen[:, None] - 1))]  # [S, q, Hq, D]
    kp, vp = plain_cached(s, kj.minimum((prefix - 1).clamp(min=0).unsqueeze(1)))
    fresh = cu_q[:-1, None] + (kj - prefix[:, None]).clamp(min=0)
    old = (kj < prefix[:, None])[..., None, None]
    k = torch.where(old, kp, s["new_k"].float()[fresh])
    v = torch.where(old, vp, s["new_v"].float()[fresh])
    hq, d, hkv = q.shape[2], q.shape[3], k.shape[2]
    q = q.view(size, most_q, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(size, hkv, -1, d)
    x = torch.matmul(q * s["scale"], k.permute(0, 2, 3, 1).contiguous()).view(size, hkv, -1, most_q, most_k)
    live = torch.arange(most_k, device=DEV) <= (prefix[:, None] + qi)[..., None]
    p = plain_softmax(x, live[:, None, None]).flatten(2, 3)
    out = torch.matmul(p, v.transpose(1, 2).contiguous()).view(size, hkv, -1, most_q, d)
    out = out.permute(0, 3, 1, 2, 4).reshape(size, most_q, hq, d)[qi < qlen[:, None]]
    return {"out": out.to(s["q"].dtype), "stored": got}


def plain_batch(s):
    bs, width = s["block"], s["width"]
    done, lens, rows = s["done"].long(), s["lens"].long(), s["rows"].long()
    size, padded = lens.numel(), max(s["padded"], lens.numel())
    one = torch.ones(padded - size, dtype=torch.int64, device=DEV)
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    cu_q = torch.cat((zero, torch.cat((lens - done, one)).cumsum(0)))
    cu_k = torch.cat((zero, torch.cat((lens, one)).cumsum(0)))
    held, cols = (done + bs - 1) // bs, (lens + bs - 1) // bs
    need = cols - held if s["free"] is not None else torch.zeros_like(held)
    first = need.cumsum(0) - need
    col = torch.arange(width, device=DEV)
    table = s["table"][rows].long()
    left = missing = torch.zeros((), dtype=torch.int64, device=DEV)
    if s["free"] is not None:
        count = s["count"].long()[0]
        at = first[:, None] + col - held[:, None]
        taken = torch.where(at < count, s["free"].long()[(count - 1 - at).clamp(0, s["free"].numel() - 1)], -1)
        fresh = (col >= held[:, None]) & (col < cols[:, None])
        table = torch.where(fresh, taken, table)
        s["table"][rows] = table.int()
        left, missing = (count - need.sum()).clamp(min=0), (need.sum() - count).clamp(min=0)
    table = torch.where(col < cols[:, None], table, -1)
    t = torch.arange(s["tokens"], device=DEV)
    seq = torch.searchsorted(cu_q[1:], t, right=True)
    real = seq < size
    seq = seq.clamp(max=size - 1)
    pos = torch.where(real, done[seq] + t - cu_q[seq], 0)
    blk = table[seq, (pos // bs).clamp(max=width - 1)]
    slot = torch.where(real & (blk >= 0), blk * bs + pos % bs, -1)
    tables = torch.cat((table, torch.zeros(padded - size, width, dtype=torch.int64, device=DEV)))
    totals = torch.stack((cu_q[-1], (cu_q[1:] - cu_q[:-1]).amax(), (cu_k[1:] - cu_k[:-1]).amax(), left, missing))
    return {"positions": pos, "slots": slot.int(), "cu_q": cu_q.int(), "cu_k": cu_k.int(),
            "tables": tables.int(), "totals": totals.int(), "request_tables": s["table"]}


# ------------------------------------------------------------------------------------ the inputs
def _rows(gen, n, heads, d, dtype):
    """K or V rows: normal values, a few channels several times larger, as keys have them."""
    x = torch.randn(n, heads, d, generator=gen, device=DEV)
    gain = torch.ones(heads, d, device=DEV)
    gain[:, 5::37] = 4.0
    return (x * gain).to(dtype)


def _pool(gen, blocks, case, dtype):
    """A byte pool pair (codes, scales) of quantised rows, in the case's layout."""
    hkv, d, block = case["hkv"], case["d"], case["block"]
    shape = (blocks, block, hkv) if case["layout"] == "nhd" else (blocks, hkv, block)
    codes = torch.empty(shape + (d // 2,), dtype=torch.uint8, device=DEV)
    scales = torch.empty(shape + (d // GROUP,), dtype=torch.uint8, device=DEV)
    step = max(1, (1 << 24) // (block * hkv * d))
    for i in range(0, blocks, step):
        n = min(step, blocks - i)
        c, e = quantise(_rows(gen, n * block, hkv, d, dtype).view(n, block, hkv, d))
        if case["layout"] == "hnd":
            c, e = c.transpose(1, 2), e.transpose(1, 2)
        codes[i:i + n], scales[i:i + n] = c, e
    return codes, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    if case["kind"] == "batch":
        return _prepare_batch(case, gen)
    dtype = DTYPES[case["dtype"]]
    hkv, d, block = case["hkv"], case["d"], case["block"]
    index = torch.int64 if case.get("wide") else torch.int32
    s = {"kind": case["kind"], "block": block, "layout": case["layout"], "dtype": dtype}
    if case["kind"] == "store":
        n = case["rows"]
        blocks = -(-n // block) + 3
        s["slots"] = torch.randperm(blocks * block, generator=gen, device=DEV)[:n].to(index)
        s["new_k"], s["new_v"] = _rows(gen, n, hkv, d, dtype), _rows(gen, n, hkv, d, dtype)
    else:
        done, lens = lengths(case)
        used = [-(-n // block) for n in lens]
        blocks = sum(used) + 3
        order = torch.randperm(blocks, generator=gen, device=DEV).int()
        size, longest = len(lens), max(lens)
        first = torch.tensor([sum(used[:i]) for i in range(size)], device=DEV)
        col = torch.arange(max(used), device=DEV)
        mine = col < torch.tensor(used, device=DEV)[:, None]
        s["tables"] = torch.where(mine, order[(first[:, None] + col).clamp(max=blocks - 1)], -1).to(index)
        new = [n - p for p, n in zip(done, lens)]
        tokens = sum(new)
        seq = torch.repeat_interleave(torch.arange(size), torch.tensor(new)).to(DEV)
        pos = torch.cat([torch.arange(p, n) for p, n in zip(done, lens)]).to(DEV)
        s["slots"] = (s["tables"][seq, pos // block] * block + pos % block).to(index)
        s["q"] = torch.randn(tokens, case["hq"], d, generator=gen, device=DEV).to(dtype)
        s["new_k"], s["new_v"] = _rows(gen, tokens, hkv, d, dtype), _rows(gen, tokens, hkv, d, dtype)
        cu = lambda v: torch.tensor([sum(v[:i]) for i in range(size + 1)], dtype=torch.int32, device=DEV)  # noqa: E731
        s.update(longest=longest, scale=d ** -0.5, cu_q=cu(new), cu_k=cu(lens), most_q=max(new))
        if case["kind"] == "decode":
            s.update(lens=torch.tensor(lens, device=DEV).to(index), fused=case["fused"], wide=case["wide"],
                     exact=case["exact"], valid=None)
            if case["mask"]:  # leading padding, up to a quarter of a context
                pad = (torch.rand(size, generator=gen, device=DEV) * 0.25 * s["lens"]).long()
                s["valid"] = torch.arange(longest, device=DEV) >= pad[:, None]
    s["kc"], s["ks"] = _pool(gen, blocks, case, dtype)
    s["vc"], s["vs"] = _pool(gen, blocks, case, dtype)
    return s


def _prepare_batch(case, gen):
    done, lens = lengths(case)
    block, width, size = case["block"], case["width"], len(lens)
    index = torch.int64 if case["wide"] else torch.int32
    requests = size + 5  # rows of the server's request table, some of them idle
    cols = [-(-n // block) for n in lens]
    blocks = requests * 2 + sum(cols) + 11
    order = torch.randperm(blocks, generator=gen, device=DEV).int()
    rows = torch.randperm(requests, generator=gen, device=DEV)[:size].int()
    held = [-(-n // block) for n in done] if case["alloc"] else cols
    first = torch.tensor([sum(held[:i]) for i in range(size)], device=DEV)
    col = torch.arange(width, device=DEV)
    mine = col < torch.tensor(held, device=DEV)[:, None]
    table = torch.full((requests, width), -1, dtype=torch.int32, device=DEV)
    table[rows.long()] = torch.where(mine, order[(first[:, None] + col).clamp(max=blocks - 1)], -1)
    tokens = sum(lens) - sum(done) + max(0, case["padded"] - size)
    s = {"kind": "batch", "block": block, "width": width, "padded": case["padded"], "table": table,
         "rows": rows, "done": torch.tensor(done, device=DEV).to(index), "tokens": tokens + 3,
         "lens": torch.tensor(lens, device=DEV).to(index), "free": None, "count": None}
    if case["alloc"]:
        s["free"] = order[sum(held):].contiguous()
        s["count"] = torch.tensor([s["free"].numel()], dtype=torch.int32, device=DEV)
    return s


# --------------------------------------------------------------------------------------- a pass
def run(s):
    if own:
        return own_run(s)
    if s["kind"] == "store":
        return {"stored": plain_store(s)}
    if s["kind"] == "decode":
        return plain_decode(s)
    if s["kind"] == "prefill":
        return plain_prefill(s)
    return plain_batch(s)


def own_run(s):
    from voiceagent_amd import ops

    if s["kind"] == "batch":
        m = ops.batch_metadata(s["lens"], s["done"], s["table"], s["block"], max_tokens=s["tokens"],
                               rows=s["rows"], padded_batch=s["padded"], free_blocks=s["free"],
                               free_count=s["count"])
        return {"positions": m.positions, "slots": m.slot_mapping, "cu_q": m.cu_seqlens_q,
                "cu_k": m.cu_seqlens_k, "tables": m.block_tables, "totals": m.totals,
                "request_tables": s["table"]}
    kc, vc = s["kc"].view(ops.MXFP4_KV_DTYPE), s["vc"].view(ops.MXFP4_KV_DTYPE)
    cache = {"layout": s["layout"], "k_scale": s["ks"].view(ops.MXFP4_SCALE_DTYPE),
             "v_scale": s["vs"].view(ops.MXFP4_SCALE_DTYPE)}
    if s["kind"] == "store":
        ops.store_kvcache(s["new_k"], s["new_v"], kc, vc, s["slots"], **cache)
        return {"stored": list(ops.load_kvcache(kc, vc, s["slots"], s["dtype"], **cache))}
    if s["kind"] == "decode":
        more = {"new_k": s["new_k"], "new_v": s["new_v"], "new_slots": s["slots"]} if s["fused"] else {}
        out = ops.paged_decode(s["q"], kc, vc, s["tables"], s["lens"] if s["wide"] else s["cu_k"],
                               lens_cumulative=not s["wide"], scale=s["scale"], valid_mask=s["valid"],
                               max_seq_len=s["longest"] if s["exact"] else max(32768, s["longest"]),
                               split_tokens=ops.SPLIT_EXACT if s["exact"] else 0, **more, **cache)
        got = list(ops.load_kvcache(kc, vc, s["slots"], s["dtype"], **cache)) if s["fused"] else []
        return {"out": out, "stored": got}
    out = ops.varlen_attention(s["q"], s["new_k"], s["new_v"], s["cu_q"], s["cu_k"], s["most_q"],
                               s["longest"], scale=s["scale"], causal=True, k_cache=kc, v_cache=vc,
                               block_tables=s["tables"], slot_mapping=s["slots"], **cache)
    return {"out": out, "stored": list(ops.load_kvcache(kc, vc, s["slots"], s["dtype"], **cache))}


# ----------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    """What the definitions give in 64 bits, one sequence at a time."""
    if case["kind"] == "batch":
        return None
    s = prepare(case, seed)
    edges = torch.tensor([(a + b) / 2 for a, b in zip(GRID, GRID[1:])], dtype=torch.float64, device=DEV)
    grid = torch.tensor(GRID, dtype=torch.float64, device=DEV)

    def as_stored(x):
        """x rounded to the cache's values."""
        lo, hi = SCALE_RANGE[x.dtype]
        g = x.double().unflatten(-1, (-1, GROUP))
        m, e = torch.frexp(g.abs().amax(-1, keepdim=True))  # max = m 2^e, m in [1/2, 1)
        e = torch.where(m == 0, lo - 127, (e - 3 + (m >= 0.875).int()).clamp(lo - 127, hi - 127))
        step = torch.ldexp(torch.ones_like(m), e)
        y = g / step
        i = torch.bucketize(y.abs(), edges)  # a value on an edge falls to the lower code
        tie = (y.abs() == edges[i.clamp(max=6)]) & (i < 7) & (i % 2 == 1)
        return (torch.sign(y) * grid[i + tie.long()] * step).flatten(-2)

    def cached(codes, scales, slots):
        c, e = (rows_at(p, slots, s["block"], s["layout"]) for p in (codes, scales))
        n = torch.stack((c % 16, c // 16), -1).flatten(-2).long()
        v = torch.where(n >= 8, -grid[n % 8], grid[n % 8])
        return v * torch.exp2(e.double() - 127).repeat_interleave(GROUP, -1)

    stored = [as_stored(s["new_k"]), as_stored(s["new_v"])]
    if case["kind"] == "store":
        return {"stored": stored}
    done, lens = lengths(case)
    outs, at = [], 0
    for b, (p, n) in enumerate(zip(done, lens)):
        m = n - p
        pos = torch.arange(n, device=DEV)
        slots = s["tables"][b].long()[pos // s["block"]] * s["block"] + pos % s["block"]
        k, v = cached(s["kc"], s["ks"], slots), cached(s["vc"], s["vs"], slots)
        if case["kind"] == "prefill":
            k[p:], v[p:] = s["new_k"][at:at + m].double(), s["new_v"][at:at + m].double()
        elif case["fused"]:
            k[p:], v[p:] = stored[0][at:at + m], stored[1][at:at + m]
        rep = case["hq"] // case["hkv"]
        k, v = (t.repeat_interleave(rep, 1).permute(1, 0, 2) for t in (k, v))  # [Hq, n, D]
        x = s["q"][at:at + m].double().permute(1, 0, 2) @ k.transpose(1, 2).contiguous() * s["scale"]
        seen = pos <= torch.arange(p, n, device=DEV)[:, None]
        if s.get("valid") is not None:
            seen = seen & s["valid"][b, :n]
        x = x.masked_fill(~seen, -math.inf)
        w = torch.nan_to_num(torch.softmax(x, -1), nan=0.0)
        outs.append((w @ v.contiguous()).permute(1, 0, 2))
        at += m
    fused = case["kind"] == "prefill" or case["fused"]
    return {"out": torch.cat(outs), "stored": stored if fused else []}
