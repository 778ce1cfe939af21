"""Operators of the attention core's training pass, each in a plain form and through its public entry point.

A case is one of three kinds of call:

attention  the gradient of variable-length attention over packed sequences: dq, dk and dv from the output's gradient,
           with the probabilities recomputed from q and k.  Causal, aligned at the sequences' ends (``extra``: keys
           that a sequence has more than queries), or not causal (the audio encoder's windows).
prologue   the gradient of the q/k prologue (RMS norm of every head row, its weight, the half-split rotation): dq, dk
           and the two weights' gradients, which sum over all tokens and heads.
rotary     rotary positions in their other forms: pairs interleaved or halves, the first ``part`` elements of a head,
           a table scaled for long contexts; ``inverse``: the rotation's gradient.

Geometry is the decoder's (16 query heads, 8 KV heads, head_dim 128) or the audio encoder's (14 heads of 64, windows of
104 tokens) where a case does not say otherwise.  Lengths follow from the case alone; the seed makes the values.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEV = "cuda"
EPS = 1e-6
WINDOW = 104


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # The encoder over a single 30 s clip: four windows.
        attention("attention-clip", 4, 78, 104, hq=14, hkv=14, d=64, causal=False),
        # The encoder over a burst of 32 clips.
        attention("attention-clips", 160, 13, 104, hq=14, hkv=14, d=64, causal=False),
        # One utterance's transcript and audio tokens, a step of batch one.
        attention("attention-1", 1, 420, 420),
        # A packed training batch of utterances.
        attention("attention-32", 32, 50, 450),
        # Four long recordings, few key heads of 64, in half precision.
        attention("attention-4-f16", 4, 600, 2000, hq=32, hkv=4, d=64, dtype="f16"),
        # Answers behind a prompt that gets no gradient rows of its own: fewer queries than keys.
        attention("attention-answers", 8, 40, 260, extra=700),
        # One long recording.
        attention("attention-long", 1, 8192, 8192),
        # The prologue of one utterance, and of the packed batch.
        prologue("prologue-420", 420),
        prologue("prologue-8561", 8561),
        # One token of each of 32 speakers, half of the head, pairs interleaved.
        rotary("rotary-32", 32, part=64, interleaved=True),
        # The packed batch, the whole head, a scaled table; and the gradient of the interleaved form.
        rotary("rotary-8561", 8561, scaled=True),
        rotary("rotary-grad-8561", 8561, part=64, interleaved=True, inverse=True),
    ]


def attention(name, seqs, lo, hi, *, hq=16, hkv=8, d=128, causal=True, extra=0, dtype="bf16", mix=0):
    return {"name": name, "kind": "attention", "seqs": seqs, "lo": lo, "hi": hi, "hq": hq, "hkv": hkv, "d": d,
            "causal": causal, "extra": extra, "dtype": dtype, "mix": mix}


def prologue(name, tokens, *, hq=16, hkv=8, d=128, dtype="bf16", weight="bf16", wide=True, mix=0):
    return {"name": name, "kind": "prologue", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "dtype": dtype,
            "weight": weight, "wide": wide, "mix": mix}


def rotary(name, tokens, *, hq=16, hkv=8, d=128, part=0, interleaved=False, scaled=False, inverse=False,
           dtype="bf16", wide=True, mix=0):
    return {"name": name, "kind": "rotary", "tokens": tokens, "hq": hq, "hkv": hkv, "d": d, "part": part or d,
            "interleaved": interleaved, "scaled": scaled, "inverse": inverse, "dtype": dtype, "wide": wide, "mix": mix}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(16, 8), (16, 8), (14, 14), (32, 8), (32, 4), (8, 1), (12, 4)]


def draw(rng):
    """One more case of the listed ranges; none multiplies more than attention-long or moves more than the batch's
    prologue."""
    kind = rng.choice(["attention", "attention", "attention", "prologue", "rotary"])
    mix = rng.randrange(1, 1 << 20)
    hq, hkv = rng.choice(HEADS)
    if kind == "attention":
        d = rng.choice([64, 128])
        causal = rng.random() < 0.7
        seqs = _log(rng, 1, 160)
        most = 8192 * (16 / hq) ** 0.5 / seqs ** 0.6
        hi = _log(rng, 8, max(16, most if causal else most / 2))
        extra = _log(rng, 1, hi // 2) if causal and rng.random() < 0.3 else 0
        hi -= extra
        # (A sequence of one key has no gradient of q and k: a case is not made of those alone.)
        least = 1 if seqs >= 4 else 2
        case = attention("", seqs, rng.randint(least, max(least, int(hi * rng.uniform(0.05, 1.0)))), hi, hq=hq,
                         hkv=hkv, d=d, causal=causal, extra=extra, dtype=rng.choice(["bf16", "bf16", "f16"]), mix=mix)
    elif kind == "prologue":
        d = rng.choice([64, 128, 128, 256])
        case = prologue("", _log(rng, 1, 8561 * 24 * 128 // ((hq + hkv) * d)), hq=hq, hkv=hkv, d=d,
                        dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), wide=rng.random() < 0.5, mix=mix)
        case["weight"] = rng.choice([case["dtype"], "f32"])
    else:
        d = rng.choice([64, 80, 96, 128, 128, 256])
        case = rotary("", _log(rng, 1, 8561 * 24 * 128 // ((hq + hkv) * d)), hq=hq, hkv=hkv, d=d,
                      part=rng.choice([d, d, d // 2, d // 4]), interleaved=rng.random() < 0.5,
                      scaled=rng.random() < 0.4, inverse=rng.random() < 0.4,
                      dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), wide=rng.random() < 0.5, mix=mix)
    if case["dtype"] == "f32":
        case["tokens"] = max(1, case["tokens"] // 2)
    del case["name"]
    return case


def lengths(case):
    """(query, key) lengths of the case's sequences, the same for every seed."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    new = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    more = [rng.randint(0, case["extra"]) for _ in new] if case["extra"] else [0] * len(new)
    return new, [n + m for n, m in zip(new, more)]


def work(case):
    """Bytes and operations of one pass: every input read once, every output written once; five products over the
    visible pairs."""
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "attention":
        new, lens = lengths(case)
        pairs = sum(m * (n - m) + m * (m + 1) // 2 if case["causal"] else m * n for m, n in zip(new, lens))
        rows = 4 * case["hq"] * sum(new) + 4 * case["hkv"] * sum(lens)  # q, out, dout, dq; k, v, dk, dv
        return {"bytes": rows * case["d"] * size, "flops": 10 * case["d"] * case["hq"] * pairs}
    elements = case["tokens"] * (case["hq"] + case["hkv"]) * case["d"]
    if case["kind"] == "prologue":
        return {"bytes": 3 * elements * size + case["tokens"] * (case["d"] * 4 + 8), "flops": 16 * elements}
    return {"bytes": 2 * elements * size + case["tokens"] * (case["part"] * 4 + 8), "flops": 3 * elements}


# ------------------------------------------------------------------------------------ the inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV)


def _table(gen, count, width, scaled):
    """[count, width] cosines and sines; scaled: angles four times slower where a turn is longer than the context, and
    all factors a little larger, as contexts beyond the trained ones are run."""
    freq = 1e6 ** (-torch.arange(0, width, 2, dtype=torch.float64, device=DEV) / width)
    if scaled:
        keep = ((count / 4) * freq / (2 * math.pi)).clamp(1, 32).sub(1).div(31)
        freq = freq * (keep + (1 - keep) / 4)
    angle = torch.arange(count, dtype=torch.float64, device=DEV)[:, None] * freq
    factor = 0.1 * math.log(4) + 1 if scaled else 1.0
    return torch.cat((angle.cos() * factor, angle.sin() * factor), -1).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dtype, hq, hkv, d = DTYPES[case["dtype"]], case["hq"], case["hkv"], case["d"]
    if case["kind"] == "attention":
        new, lens = lengths(case)
        cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device=DEV)  # noqa: E731
        gain = torch.ones(d, device=DEV)
        gain[5::37] = 3.0  # a few channels larger, as keys have them
        s = {"kind": "attention", "cu_q": cu(new), "cu_k": cu(lens), "most_q": max(new), "most_k": max(lens),
             "causal": case["causal"], "scale": d ** -0.5,
             "q": _normal(gen, sum(new), hq, d).to(dtype), "k": (_normal(gen, sum(lens), hkv, d) * gain).to(dtype),
             "v": _normal(gen, sum(lens), hkv, d).to(dtype),
             "dout": (_normal(gen, sum(new), hq, d) / 64).to(dtype)}
        s["out"] = _outputs(s).to(dtype)
        return s
    tokens = case["tokens"]
    s = {"kind": case["kind"],
         "positions": torch.randint(0, 32768, (tokens,), generator=gen, device=DEV).to(
             torch.int64 if case["wide"] else torch.int32),
         "q": _normal(gen, tokens, hq, d).to(dtype), "k": _normal(gen, tokens, hkv, d).to(dtype)}
    if case["kind"] == "prologue":
        weight = DTYPES[case["weight"]]
        s.update(table=_table(gen, 32768, d, False), dq=(_normal(gen, tokens, hq, d) / 64).to(dtype),
                 dk=(_normal(gen, tokens, hkv, d) / 64).to(dtype), qw=(1 + 0.2 * _normal(gen, d)).to(weight),
                 kw=(1 + 0.2 * _normal(gen, d)).to(weight))
    else:
        s.update(table=_table(gen, 32768, case["part"], case["scaled"]), interleaved=case["interleaved"],
                 inverse=case["inverse"])
    return s


# ------------------------------------------------------------------------------- the plain forms
def _padded(rows, cu, most, heads):
    """Packed rows [T, H, D] as [S, heads, most, D] in 32 bits, zeros behind each sequence; KV heads repeated."""
    cu = cu.long()
    at = torch.arange(most, device=DEV)
    here = at < (cu[1:] - cu[:-1])[:, None]
    x = rows.float()[(cu[:-1, None] + at).clamp(max=rows.shape[0] - 1)] * here[..., None, None]
    return x.repeat_interleave(heads // rows.shape[1], 2).transpose(1, 2).contiguous(), here


def _probabilities(s):
    """P [S, Hq, most_q, most_k], and what it was made of."""
    heads = s["q"].shape[1]
    q, rows = _padded(s["q"], s["cu_q"], s["most_q"], heads)
    k, cols = _padded(s["k"], s["cu_k"], s["most_k"], heads)
    live = rows[:, :, None] & cols[:, None, :]
    if s["causal"]:
        ahead = (s["cu_k"][1:] - s["cu_k"][:-1] - s["cu_q"][1:] + s["cu_q"][:-1])[:, None, None]
        at = torch.arange(max(s["most_q"], s["most_k"]), device=DEV)
        live = live & (at[None, None, :s["most_k"]] <= at[None, :s["most_q"], None] + ahead)
    x = torch.matmul(q * s["scale"], k.transpose(2, 3).contiguous()).masked_fill_(~live[:, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = x.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    return p, q, k, rows, cols


def _outputs(s):
    p, q, k, rows, _ = _probabilities(s)
    v, _ = _padded(s["v"], s["cu_k"], s["most_k"], s["q"].shape[1])
    return torch.matmul(p, v).transpose(1, 2)[rows]


def plain_attention(s):
    p, q, k, rows, cols = _probabilities(s)
    heads, kv = s["q"].shape[1], s["k"].shape[1]
    v, _ = _padded(s["v"], s["cu_k"], s["most_k"], heads)
    dout, _ = _padded(s["dout"], s["cu_q"], s["most_q"], heads)
    out, _ = _padded(s["out"], s["cu_q"], s["most_q"], heads)
    dv = torch.matmul(p.transpose(2, 3).contiguous(), dout)
    ds = torch.matmul(dout, v.transpose(2, 3).contiguous()).sub_((dout * out).sum(-1, keepdim=True)).mul_(p)
    del p
    dq = torch.matmul(ds, k) * s["scale"]
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q) * s["scale"]
    shared = lambda x: x.unflatten(1, (kv, heads // kv)).sum(2).transpose(1, 2)[cols]  # noqa: E731
    return {"dq": dq.transpose(1, 2)[rows].to(s["q"].dtype), "dk": shared(dk).to(s["k"].dtype),
            "dv": shared(dv).to(s["v"].dtype)}


def _turned_back(dz, rows):
    """The transposed half-split rotation of dz [T, H, D]."""
    c, s = rows[:, None].chunk(2, -1)
    a, b = dz.float().chunk(2, -1)
    return torch.cat((a * c + b * s, b * c - a * s), -1)


def plain_prologue(s):
    rows = s["table"][s["positions"].long()]

    def side(x, dz, w):
        x, dy, w32 = x.float(), _turned_back(dz, rows), w.float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        n, dn = x * r, dy * w32
        dx = r * (dn - n * (dn * n).mean(-1, keepdim=True))
        return dx.to(dz.dtype), (dy * n).sum((0, 1)).to(w.dtype)

    dq, dqw = side(s["q"], s["dq"], s["qw"])
    dk, dkw = side(s["k"], s["dk"], s["kw"])
    return {"dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}


def plain_rotary(s):
    part = s["table"].shape[-1]
    c, sn = s["table"][s["positions"].long()][:, None].chunk(2, -1)
    sn = -sn if s["inverse"] else sn

    def side(x):
        f = x.float()
        head, rest = f[..., :part], f[..., part:]
        if s["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack((a * c - b * sn, b * c + a * sn), -1).flatten(-2)
        else:
            a, b = head.chunk(2, -1)
            head = torch.cat((a * c - b * sn, b * c + a * sn), -1)
        return torch.cat((head, rest), -1).to(x.dtype)

    return {"q": side(s["q"]), "k": side(s["k"])}


# --------------------------------------------------------------------------------------- a pass
def run(s):
    if own:
        return own_run(s)
    if s["kind"] == "attention":
        return plain_attention(s)
    if s["kind"] == "prologue":
        return plain_prologue(s)
    return plain_rotary(s)


def own_run(s):
    from voiceagent_amd import ops

    if s["kind"] == "attention":
        dq, dk, dv = ops.varlen_attention_backward(
            s["dout"], s["q"], s["k"], s["v"], s["out"], s["cu_q"], s["cu_k"], s["most_q"], s["most_k"],
            scale=s["scale"], causal=s["causal"])
        return {"dq": dq, "dk": dk, "dv": dv}
    if s["kind"] == "prologue":
        pro = ops.QKPrologue(s["qw"], s["kw"], EPS, s["table"], s["positions"])
        dq, dk, dqw, dkw = ops.qk_norm_rope_backward(s["dq"], s["dk"], s["q"], s["k"], pro)
        return {"dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}
    q, k = ops.rotary_embedding(s["q"], s["k"], s["table"], s["positions"], interleaved=s["interleaved"],
                                inverse=s["inverse"])
    return {"q": q, "k": k}


# ----------------------------------------------------------------------- the definition, 64 bits
def exact(case, seed):
    """What the definitions give in 64 bits: attention one sequence and KV head at a time, rotations as products of
    complex numbers."""
    s = prepare(case, seed)
    if case["kind"] == "attention":
        new, lens = lengths(case)
        group = case["hq"] // case["hkv"]
        got = {n: torch.zeros(x.shape, dtype=torch.float64, device=DEV) for n, x in (("dq", s["q"]), ("dk", s["k"]), ("dv", s["v"]))}
        i0 = j0 = 0
        for m, n in zip(new, lens):
            i1, j1 = i0 + m, j0 + n
            for h in range(case["hkv"]):
                heads = slice(h * group, (h + 1) * group)
                k, v = s["k"][j0:j1, h].double(), s["v"][j0:j1, h].double()
                for g in range(heads.start, heads.stop):
                    q, do, o = (s[x][i0:i1, g].double() for x in ("q", "dout", "out"))
                    x = (q @ k.T.contiguous()) * s["scale"]
                    if case["causal"]:
                        x = x.masked_fill(torch.ones_like(x, dtype=torch.bool).triu(n - m + 1), -math.inf)
                    p = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                    ds = p * (do @ v.T.contiguous() - (do * o).sum(-1, keepdim=True)) * s["scale"]
                    got["dq"][i0:i1, g] = ds @ k
                    got["dk"][j0:j1, h] += ds.T.contiguous() @ q
                    got["dv"][j0:j1, h] += p.T.contiguous() @ do
            i0, j0 = i1, j1
        return got
    c, sn = s["table"][s["positions"].long()].double().chunk(2, -1)
    turn = torch.complex(c, sn)[:, None]

    def turned(x, factor, interleaved):
        z = torch.complex(x[..., 0::2], x[..., 1::2]) if interleaved else torch.complex(*(t.contiguous() for t in x.chunk(2, -1)))
        z = z * factor
        return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)

    if case["kind"] == "rotary":
        part, factor = case["part"], turn.conj() if case["inverse"] else turn
        return {n: torch.cat((turned(s[n][..., :part].double(), factor, case["interleaved"]), s[n][..., part:].double()), -1)
                for n in ("q", "k")}
    got = {}
    for n, w in (("q", s["qw"]), ("k", s["kw"])):
        x, dy = s[n].double(), turned(s["d" + n].double(), turn.conj(), False)
        size = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        g = dy * w.double()
        got["d" + n] = g / size - x * (g * x).sum(-1, keepdim=True) / (case["d"] * size ** 3)
        got["d%sw" % n] = (dy * x / size).flatten(0, 1).sum(0)
    return {n: got[n] for n in ("dq", "dk", "dqw", "dkw")}
