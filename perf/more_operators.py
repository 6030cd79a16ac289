"""The operators of a decoder's training step that stand between its packed layers (embedding, norm and rotation of
queries and keys, gated unit) and the activations that are kept in 8 bits for the backward pass (of the gated unit, and of a
packed layer's weight gradient), as cases to measure: what they are called with, their plain form in elementary torch
operations, and their definition in 64 bits.

Sizes are those of the repository's workloads (the char GPT: width 384, MLP 1536, 65 symbols, 16,384 tokens a step; the
Llama-style decoder: width 2048, 16 heads of 128, MLP 5504, vocabulary 32000, 8 x 2048 tokens; the UNet's transformers: width
1280, gated units of 5120), with grouped heads, ragged lengths and odd sizes beside them.

A value kept in 8 bits: 32 tokens of one feature share a power of two, the least with |x| <= 127 2^e, and each is
the whole number nearest to x / 2^e (ties to even).
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one short prompt into the char GPT, nothing learned: the smallest call, latency counts
        dict(name="embed_prompt", op="embed", tokens=77, vocab=65, dim=384, w="fp32", y="bf16", scale=1.0, train=False),
        # the char GPT's step: every symbol some 250 times, residual stream in 32 bits
        dict(name="embed_step_65", op="embed", tokens=16384, vocab=65, dim=384, w="fp32", y="fp32", scale=1.0,
             train=True),
        # the Llama-style decoder's step: tokens by a Zipf law, scaled by sqrt(width), weights in 32 bits
        dict(name="embed_step_32000", op="embed", tokens=16384, vocab=32000, dim=2048, w="fp32", y="bf16",
             scale=45.25, train=True),
        # a few sequences' next tokens at far positions, grouped heads: serving, latency counts
        dict(name="qk_tokens", op="qk", tokens=5, seqs=5, heads=16, kv_heads=4, dim=128, rot=128, x="bf16",
             interleaved=False, norm=True, far=30000, train=False),
        # the Llama-style decoder's step, pairs of neighbours as its model rotates them
        dict(name="qk_step_8x2048", op="qk", tokens=16384, seqs=8, heads=16, kv_heads=16, dim=128, rot=128, x="bf16",
             interleaved=True, norm=True, far=0, train=True),
        # packed documents, heads of 80 of which half is rotated, grouped heads
        dict(name="qk_ragged_80", op="qk", tokens=20011, seqs=37, heads=20, kv_heads=5, dim=80, rot=40, x="fp16",
             interleaved=False, norm=True, far=0, train=True),
        # one prompt through the char GPT's MLP width, forward alone
        dict(name="gated_prompt", op="gated", rows=77, dim=1536, x="bf16", act="gelu", halves=False, eight=False,
             train=False),
        # the UNet's gated unit: halves of one projection
        dict(name="gated_halves_5120", op="gated", rows=4096, dim=5120, x="fp16", act="gelu", halves=True, eight=True,
             train=True),
        # the Llama-style decoder's MLP
        dict(name="gated_step_5504", op="gated", rows=16384, dim=5504, x="bf16", act="silu", halves=False, eight=True,
             train=True),
        # the char GPT's MLP weight over packed tokens of an odd number: few output tiles, a long sum
        dict(name="dw_16381x1536x384", op="dw", rows=16381, out=1536, dim=384, x="bf16"),
        # a square projection of the decoder
        dict(name="dw_16384x2048x2048", op="dw", rows=16384, out=2048, dim=2048, x="bf16"),
        # the decoder's down projection, the widest input
        dict(name="dw_16384x2048x5504", op="dw", rows=16384, out=2048, dim=5504, x="bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["embed", "qk", "gated", "dw"])
        if op == "embed":
            case = dict(op=op, tokens=_log_int(rng, 1, 65536), vocab=_log_int(rng, 65, 150000),
                        dim=_log_int(rng, 64, 4096), w=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                        y=rng.choice(["bf16", "bf16", "fp16", "fp32"]), scale=rng.choice([1.0, 1.0, 8.0, 45.25]),
                        train=rng.random() < 0.7)
            if case["tokens"] * case["dim"] > 16384 * 2048 or case["vocab"] * case["dim"] > 32000 * 2048:
                continue
        elif op == "qk":
            heads = rng.choice([4, 6, 8, 10, 12, 16, 20])
            dim = rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128])
            seqs = _log_int(rng, 1, 64)
            case = dict(op=op, tokens=max(seqs, _log_int(rng, 1, 32768)), seqs=seqs, heads=heads,
                        kv_heads=rng.choice([h for h in (1, 2, 4, 5, 8, 10, 16, 20) if heads % h == 0]), dim=dim,
                        rot=rng.choice([dim, dim, dim, dim // 2]), x=rng.choice(["bf16", "bf16", "fp16"]),
                        interleaved=rng.random() < 0.4, norm=rng.random() < 0.8, far=rng.choice([0, 0, 1000, 30000]),
                        train=rng.random() < 0.7)
            if case["tokens"] * (heads + case["kv_heads"]) * dim > 16384 * 32 * 128:
                continue
        elif op == "gated":
            case = dict(op=op, rows=_log_int(rng, 1, 65536), dim=_log_int(rng, 64, 16384),
                        x=rng.choice(["bf16", "bf16", "fp16", "fp32"]), act=rng.choice(["silu", "silu", "gelu"]),
                        halves=rng.random() < 0.4, eight=rng.random() < 0.7, train=rng.random() < 0.8)
            if case["rows"] * case["dim"] > 16384 * 5504:
                continue
        else:
            case = dict(op=op, rows=_log_int(rng, 16, 65536), out=8 * _log_int(rng, 8, 1024),
                        dim=_log_int(rng, 64, 8192), x=rng.choice(["bf16", "bf16", "bf16", "fp32"]))
            if case["rows"] * case["out"] * case["dim"] > 16384 * 2048 * 5504 or \
                    case["rows"] * max(case["out"], case["dim"]) > 16384 * 8192:
                continue
        return case


def work(case):
    if case["op"] == "embed":
        t, v, d, bw, by = case["tokens"], case["vocab"], case["dim"], SIZE[case["w"]], SIZE[case["y"]]
        fwd = min(t, v) * d * bw + t * d * by + 8 * t
        if not case["train"]:
            return {"bytes": fwd, "flops": t * d}
        return {"bytes": fwd + t * d * by + v * d * bw, "flops": 3 * t * d}
    if case["op"] == "qk":
        n, b = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"], SIZE[case["x"]]
        return {"bytes": (4 if case["train"] else 2) * n * b, "flops": (25 if case["train"] else 8) * n}
    if case["op"] == "gated":
        n, b = case["rows"] * case["dim"], SIZE[case["x"]]
        return {"bytes": (6 if case["train"] else 3) * n * b, "flops": (30 if case["train"] else 10) * n}
    m, n, k = case["rows"], case["out"], case["dim"]
    return {"bytes": m * k * SIZE[case["x"]] + 2 * m * n + 2 * n * k, "flops": 2 * m * n * k}


# ---------------------------------------------------------------- inputs
def _lengths(case):
    """The lengths of the packed sequences: from the case alone, one token at least."""
    total, n = case["tokens"], case["seqs"]
    r = random.Random(total * 131 + n)
    share = [math.exp(r.gauss(0.0, 0.7)) for _ in range(n)]
    got = [1 + int((total - n) * s / sum(share)) for s in share]
    got[got.index(max(got))] += total - sum(got)
    return got


def _tables(length, rot):
    """cos and sin of position times 10000^(-2 i / rot), as a program keeps them: from 64 bits, held in 32."""
    at = torch.arange(length, dtype=torch.float64, device="cuda")
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = at[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "embed":
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        # a Zipf law over the vocabulary, its ranks scattered over the ids; a few places hold padding (-1)
        u = torch.rand(t, generator=g, device="cuda", dtype=torch.float64)
        rank = ((v + 1.0) ** u - 1.0).long().clamp_(0, v - 1)
        ids = torch.randperm(v, generator=g, device="cuda")[rank]
        ids = torch.where(torch.rand(t, generator=g, device="cuda") < 0.01, -1, ids)
        s = dict(case=case, ids=ids, w=(randn(v, d) * 0.02).to(DTYPES[case["w"]]))
        if case["train"]:
            s["dy"] = (randn(t, d) * 1e-2).to(DTYPES[case["y"]])
        return s
    if case["op"] == "qk":
        t, h, hk, d = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        dt = DTYPES[case["x"]]
        lens = _lengths(case)
        start = torch.tensor([0] + lens[:-1]).cumsum(0).cuda()
        doc = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), torch.tensor(lens).cuda())
        pos = (torch.arange(t, device="cuda") - start[doc] + case["far"]).to(torch.int32)
        cos, sin = _tables(case["far"] + max(lens), case["rot"])
        qkv = (randn(t, h + 2 * hk, d) * (0.5 + 2.0 * torch.rand(d, generator=g, device="cuda"))).to(dt)
        s = dict(case=case, q=qkv[:, :h], k=qkv[:, h:h + hk], pos=pos, cos=cos, sin=sin, qw=None, kw=None)
        if case["norm"]:
            s["qw"], s["kw"] = 1.0 + 0.2 * randn(d), 1.0 + 0.2 * randn(d)
        if case["train"]:
            s["dq"], s["dk"] = (randn(t, h, d) * 1e-2).to(dt), (randn(t, hk, d) * 1e-2).to(dt)
        return s
    if case["op"] == "gated":
        n, d, dt = case["rows"], case["dim"], DTYPES[case["x"]]
        if case["halves"]:                                     # one projection's output: value half, gate half
            both = randn(n, 2 * d).mul_(1.5).to(dt)
            up, gate = both[:, :d], both[:, d:]
        else:
            gate, up = randn(n, d).mul_(1.5).to(dt), randn(n, d).to(dt)
        s = dict(case=case, gate=gate, up=up)
        if case["train"]:
            s["dh"] = (randn(n, d) * 1e-2).to(dt)
        return s
    m, n, k = case["rows"], case["out"], case["dim"]
    # activations: features of different spread, a few of them far out
    spread = 0.3 + torch.rand(k, generator=g, device="cuda")
    spread = torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 20.0, spread)
    return dict(case=case, x=(randn(m, k) * spread).to(DTYPES[case["x"]]), dy=(randn(m, n) * 1e-2).bfloat16())


# ---------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _own_embed(s):
    import concord_b200
    c = s["case"]
    kw = dict(scale=c["scale"], out_dtype=DTYPES[c["y"]])
    if not c["train"]:
        with torch.no_grad():
            return concord_b200.embedding(s["ids"], s["w"], **kw)
    w = s["w"].detach().requires_grad_()
    y = concord_b200.embedding(s["ids"], w, **kw)
    return (y.detach(),) + torch.autograd.grad(y, (w,), s["dy"])


def _own_qk(s):
    import concord_b200
    c = s["case"]
    kw = dict(norm=c["norm"], eps=EPS, interleaved=c["interleaved"])
    if not c["train"]:
        with torch.no_grad():
            return concord_b200.qk_norm_rope(s["q"], s["k"], s["cos"], s["sin"], s["pos"], s["qw"], s["kw"], **kw)
    leaves = [t.detach().requires_grad_() for t in (s["q"], s["k"], s["qw"], s["kw"]) if t is not None]
    q, k = concord_b200.qk_norm_rope(leaves[0], leaves[1], s["cos"], s["sin"], s["pos"], *leaves[2:], **kw)
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))


def _own_gated(s):
    import concord_b200
    c = s["case"]
    kw = dict(act=c["act"], save8=c["eight"])
    if not c["train"]:
        with torch.no_grad():
            return concord_b200.gated_unit(s["gate"], s["up"], **kw)
    gate, up = s["gate"].detach().requires_grad_(), s["up"].detach().requires_grad_()
    h = concord_b200.gated_unit(gate, up, **kw)
    return (h.detach(),) + torch.autograd.grad(h, (gate, up), s["dh"])


def _own_dw(s):
    import concord_b200
    return concord_b200.grad_weight8(s["dy"], concord_b200.save8(s["x"]))


def _plain_embed(s):
    c = s["case"]
    ids, ok = s["ids"].clamp(min=0), (s["ids"] >= 0)[:, None]
    y = torch.where(ok, s["w"][ids].float() * c["scale"], 0.0).to(DTYPES[c["y"]])
    if not c["train"]:
        return y
    dw = torch.zeros(c["vocab"], c["dim"], device="cuda")
    dw.index_add_(0, ids, torch.where(ok, s["dy"].float() * c["scale"], 0.0))
    return y, dw.to(s["w"].dtype)


def _turn(x, cos, sin, rot, interleaved):
    if interleaved:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_qk(s):
    c = s["case"]
    at = s["pos"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    outs, grads, wgrads = [], [], []
    for x, w, dy in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        xf = x.float()
        n = xf
        if c["norm"]:
            r = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + EPS)
            n = xf * r * w
        outs.append(_turn(n, cos, sin, c["rot"], c["interleaved"]).to(x.dtype))
        if dy is None:
            continue
        dn = _turn(dy.float(), cos, -sin, c["rot"], c["interleaved"])
        if c["norm"]:
            xh = xf * r
            wgrads.append((dn * xh).sum((0, 1)))
            dn = dn * w
            dn = r * (dn - xh * (dn * xh).mean(-1, keepdim=True))
        grads.append(dn.to(x.dtype))
    return tuple(outs + grads + wgrads)


def _plain_eight(x):
    """The values that 8 bits keep of x [N, D], in 32 bits."""
    n, d = x.shape
    blocks = torch.nn.functional.pad(x.float(), (0, 0, 0, -n % 32)).view(-1, 32, d)
    m, e = torch.frexp(blocks.abs().amax(1, keepdim=True))
    e = e - torch.where(m * 128 > 127, 6, 7)
    return torch.ldexp(torch.round(torch.ldexp(blocks, -e)), e).view(-1, d)[:n]


def _plain_act(g, act):
    """act(g) and its derivative."""
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-g))
        return g * q, q * (1.0 + g * (1.0 - q))
    p = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * p, p + g * torch.exp(-0.5 * g * g) * (2.0 * math.pi) ** -0.5


def _plain_gated(s):
    c = s["case"]
    g, u, dt = s["gate"].float(), s["up"].float(), s["gate"].dtype
    h = (_plain_act(g, c["act"])[0] * u).to(dt)
    if not c["train"]:
        return h
    if c["eight"]:
        g, u = _plain_eight(g), _plain_eight(u)
    a, da = _plain_act(g, c["act"])
    dh = s["dh"].float()
    return h, (dh * u * da).to(dt), (dh * a).to(dt)


def _plain_dw(s):
    return (s["dy"].float().t() @ _plain_eight(s["x"])).bfloat16()


_run_own = {"embed": _own_embed, "qk": _own_qk, "gated": _own_gated, "dw": _own_dw}
_run_plain = {"embed": _plain_embed, "qk": _plain_qk, "gated": _plain_gated, "dw": _plain_dw}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_eight(x):
    n = x.shape[0]
    out = torch.zeros(-(-n // 32) * 32, x.shape[1], dtype=torch.float64, device="cuda")
    out[:n] = x.double()
    blocks = out.view(-1, 32, x.shape[1])
    most = blocks.abs().amax(1, keepdim=True)
    step = torch.exp2(torch.floor(torch.log2(most.clamp(min=2.0 ** -100))) - 6)
    step = torch.where(127 * (step / 2) >= most, step / 2, torch.where(127 * step >= most, step, 2 * step))
    return (blocks / step).round().mul(step).view(-1, x.shape[1])[:n]


def _exact_gated(s, case):
    outs = []
    for at in range(0, case["rows"], 4096):                    # blocks of 32 tokens stay whole
        g, u = s["gate"][at:at + 4096].double(), s["up"][at:at + 4096].double()
        cdf = torch.special.ndtr if case["act"] == "gelu" else torch.sigmoid
        part = [g * cdf(g) * u]
        if case["train"]:
            dh = s["dh"][at:at + 4096].double()
            if case["eight"]:
                g, u = _exact_eight(g), _exact_eight(u)
            p = cdf(g)
            if case["act"] == "gelu":
                slope = p + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
            else:
                slope = p + g * p * (1 - p)
            part += [dh * u * slope, dh * g * p]
        outs.append(part)
    cat = tuple(torch.cat(col) for col in zip(*outs))
    return cat if case["train"] else cat[0]


def _exact_qk(s, case):
    rot, t = case["rot"], case["tokens"]
    freq = torch.tensor([10000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float64, device="cuda")
    turn = torch.polar(torch.ones(t, 1, rot // 2, dtype=torch.float64, device="cuda"),
                       (s["pos"].double()[:, None] * freq)[:, None])

    def turned(x, by):
        first = x[..., :rot]
        pairs = first.unflatten(-1, (rot // 2, 2)) if case["interleaved"] else \
            first.unflatten(-1, (2, rot // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * by)
        z = z if case["interleaved"] else z.transpose(-1, -2)
        return torch.cat((z.flatten(-2), x[..., rot:]), -1)

    outs, grads, wgrads = [], [], []
    for x, w, dy in ((s["q"], s["qw"], s.get("dq")), (s["k"], s["kw"], s.get("dk"))):
        x = x.double()
        size = (x.square().mean(-1, keepdim=True) + EPS).sqrt()
        outs.append(turned(x / size * w.double() if case["norm"] else x, turn))
        if dy is None:
            continue
        back = turned(dy.double(), turn.conj())
        if case["norm"]:
            xh = x / size
            wgrads.append((back * xh).sum((0, 1)))
            back = back * w.double()
            back = (back - xh * (back * xh).mean(-1, keepdim=True)) / size
        grads.append(back)
    return tuple(outs + grads + wgrads)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embed":
        keep = s["ids"] >= 0
        y = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
        y[keep] = s["w"].double()[s["ids"][keep]] * case["scale"]
        if not case["train"]:
            return y
        dw = torch.zeros(case["vocab"], case["dim"], dtype=torch.float64, device="cuda")
        dw.index_put_((s["ids"][keep],), s["dy"][keep].double() * case["scale"], accumulate=True)
        return y, dw
    if case["op"] == "qk":
        return _exact_qk(s, case)
    if case["op"] == "gated":
        return _exact_gated(s, case)
    dw = torch.zeros(case["out"], case["dim"], dtype=torch.float64, device="cuda")
    for at in range(0, case["rows"], 8192):
        dw += s["dy"][at:at + 8192].double().t() @ _exact_eight(s["x"][at:at + 8192])
    return dw
