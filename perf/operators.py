"""The training operators around the packed layers (layer norm, packed attention, distillation from a teacher's top
logits), as cases to measure: what they are called with, their plain form in elementary torch operations, and their
definition in 64 bits.

Sizes are those of the repository's workloads (the char GPT: width 384, 6 heads of 64, 256 tokens, 65 symbols; the
Llama-style decoder: width 2048, 16 heads of 128, 2048 tokens, vocabulary 32000; the UNet's transformers: heads of 64,
1024 and 4096 tokens, 77 tokens of context), with ragged batches, grouped heads and odd sizes beside them.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
IGNORE = -100


# ---------------------------------------------------------------- the cases
def listed():
    return [
        # one short document through a narrow norm when nothing is learned: the smallest call, latency counts
        dict(name="norm_short_384", op="norm", rows=77, dim=384, x="bf16", y="bf16", train=False),
        # the char GPT's step: residual stream in 32 bits, the next GEMM's input in bf16
        dict(name="norm_step_384", op="norm", rows=16384, dim=384, x="fp32", y="bf16", train=True),
        # the largest: a Llama-width step of 65,533 packed tokens
        dict(name="norm_step_2048", op="norm", rows=65533, dim=2048, x="bf16", y="bf16", train=True),
        # the char GPT student: 65 symbols, logits in 32 bits, teacher's top 16, hard labels beside
        dict(name="distill_step_65", op="distill", rows=16384, vocab=65, top=16, x="fp32", temp=2.0, alpha=0.5,
             labels=True, fused=False),
        # a decoder's step: 16,384 tokens of vocabulary 32000, value and gradient in one call
        dict(name="distill_step_32000", op="distill", rows=16384, vocab=32000, top=32, x="bf16", temp=2.0, alpha=0.7,
             labels=True, fused=True),
        # a few answer tokens under a large odd vocabulary, teacher's distribution alone
        dict(name="distill_few_100003", op="distill", rows=9, vocab=100003, top=64, x="fp16", temp=1.0, alpha=1.0,
             labels=False, fused=False),
        # a handful of short prompts, forward only: latency
        dict(name="attend_short", op="attend", total=301, seqs=4, ragged=True, heads=6, kv_heads=6, dim=64, x="bf16",
             causal=True, cross=0, train=False),
        # ragged prompts with grouped heads, forward only
        dict(name="attend_prompts_gqa", op="attend", total=16000, seqs=13, ragged=True, heads=16, kv_heads=4, dim=128,
             x="bf16", causal=True, cross=0, train=False),
        # the char GPT's step: 64 windows of 256
        dict(name="attend_step_64x256", op="attend", total=16384, seqs=64, ragged=False, heads=6, kv_heads=6, dim=64,
             x="bf16", causal=True, cross=0, train=True),
        # the UNet's cross attention onto 77 tokens of context, heads of 64
        dict(name="attend_cross_77", op="attend", total=4096, seqs=4, ragged=False, heads=20, kv_heads=20, dim=64,
             x="fp16", causal=False, cross=77, train=True),
        # the Llama-style decoder's step: 8 sequences of 2048, heads of 128
        dict(name="attend_step_8x2048", op="attend", total=16384, seqs=8, ragged=False, heads=16, kv_heads=16, dim=128,
             x="bf16", causal=True, cross=0, train=True),
        # one long document with grouped heads, forward and backward
        dict(name="attend_long_8191", op="attend", total=8191, seqs=1, ragged=False, heads=16, kv_heads=4, dim=128,
             x="bf16", causal=True, cross=0, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["norm", "distill", "attend", "attend"])
        if op == "norm":
            case = dict(op=op, rows=_log_int(rng, 16, 65536), dim=_log_int(rng, 64, 8192),
                        x=rng.choice(["bf16", "fp16", "fp32"]), y=rng.choice(["bf16", "bf16", "fp32"]),
                        train=rng.random() < 0.7)
            if case["rows"] * case["dim"] > 65536 * 1024:
                continue
        elif op == "distill":
            labels = rng.random() < 0.6
            vocab = _log_int(rng, 65, 150000)
            case = dict(op=op, rows=_log_int(rng, 1, 16384), vocab=vocab,
                        top=min(_log_int(rng, 1, 128), vocab // 2),
                        x=rng.choice(["bf16", "bf16", "fp16", "fp32"]), temp=rng.choice([1.0, 1.5, 2.0, 4.0]),
                        alpha=rng.choice([0.3, 0.5, 0.9]) if labels else 1.0, labels=labels,
                        fused=rng.random() < 0.5)
            if case["rows"] * vocab > 16384 * 15000:
                continue
        else:
            heads = rng.choice([4, 6, 8, 10, 12, 16])
            cross = rng.choice([0, 0, 0, 77, 300])
            seqs = _log_int(rng, 1, 64)
            mean = _log_int(rng, 16, 4096)
            dim = rng.choice([32, 64, 64, 80, 96, 128, 128])
            case = dict(op=op, total=seqs * mean + rng.randrange(0, 8), seqs=seqs, ragged=rng.random() < 0.7,
                        heads=heads, kv_heads=rng.choice([h for h in (1, 2, 3, 4, 6, 8, 10, 12, 16) if heads % h == 0]),
                        dim=dim, x=rng.choice(["bf16", "bf16", "fp16"]),
                        causal=cross == 0 and rng.random() < 0.8, cross=cross, train=rng.random() < 0.6)
            longest = max(_lengths(case))
            # what the plain form holds: a padded score matrix for every sequence and head
            if seqs * heads * longest * (cross or longest) > 6e8:
                continue
        if work(case)["flops"] <= 0.5 * 14 * 128 * 16 * 8191 * 8192:
            return case


def _lengths(case):
    """The lengths of the packed sequences: from the case alone."""
    total, n = case["total"], case["seqs"]
    if not case["ragged"]:
        base = total // n
        return [base + (1 if i < total - base * n else 0) for i in range(n)]
    r = random.Random(total * 131 + n)
    share = [math.exp(r.gauss(0.0, 0.7)) for _ in range(n)]
    got = [int(total * s / sum(share)) for s in share]
    got[got.index(max(got))] += total - sum(got)
    return got


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "norm":
        n, d, bx, by = case["rows"], case["dim"], size[case["x"]], size[case["y"]]
        fwd = n * d * (bx + by) + 8 * d
        if not case["train"]:
            return {"bytes": fwd, "flops": 8 * n * d}
        return {"bytes": fwd + n * d * (by + bx) + 8 * d, "flops": 20 * n * d}
    if case["op"] == "distill":
        n, v, bx = case["rows"], case["vocab"], size[case["x"]]
        return {"bytes": 2 * n * v * bx + n * case["top"] * 8 + n * 8, "flops": 12 * n * v}
    lens = _lengths(case)
    if case["cross"]:
        pairs, keys = sum(lens) * case["cross"], len(lens) * case["cross"]
    else:
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        keys = case["total"]
    q, kv = case["total"] * case["heads"] * case["dim"] * 2, keys * case["kv_heads"] * case["dim"] * 2
    per = 14 if case["train"] else 4
    return {"bytes": (2 * q + 2 * kv) * (2 if case["train"] else 1), "flops": per * case["dim"] * case["heads"] * pairs}


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "norm":
        n, d = case["rows"], case["dim"]
        # a residual stream: channels of different spread, rows off centre
        x = randn(n, d) * (0.5 + 2.0 * torch.rand(d, generator=g, device="cuda")) + 0.3 * randn(n, 1)
        s = dict(case=case, x=x.to(DTYPES[case["x"]]), w=1.0 + 0.2 * randn(d), b=0.1 * randn(d))
        if case["train"]:
            s["dy"] = (randn(n, d) * 1e-2).to(DTYPES[case["y"]])
        return s
    if case["op"] == "distill":
        n, v, k = case["rows"], case["vocab"], case["top"]
        z = torch.empty(n, v, dtype=DTYPES[case["x"]], device="cuda")
        for at in range(0, n, 4096):
            z[at:at + 4096] = (randn(min(4096, n - at), v) * 2.0).to(z.dtype)
        start = torch.randint(0, v, (n, 1), generator=g, device="cuda")
        ids = (start + torch.arange(k, device="cuda") * (v // k)) % v
        t = 12.0 - torch.rand(n, k, generator=g, device="cuda").mul_(0.8).cumsum(1)
        have = torch.where(torch.rand(n, 1, generator=g, device="cuda") < 0.1,
                           torch.randint(0, k + 1, (n, 1), generator=g, device="cuda"), k)   # some rows have fewer
        have[0] = k
        ids = torch.where(torch.arange(k, device="cuda") < have, ids, -1)
        s = dict(case=case, z=z, ids=ids, t=t, labels=None)
        if case["labels"]:
            y = torch.randint(0, v, (n,), generator=g, device="cuda")
            s["labels"] = torch.where(torch.rand(n, generator=g, device="cuda") < 0.05, IGNORE, y)
            s["labels"][0] = y[0]
        return s
    lens = _lengths(case)
    total, h, hk, d, dt = case["total"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["x"]]
    cu = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
    if case["cross"]:
        cuk = torch.tensor([case["cross"] * i for i in range(len(lens) + 1)], dtype=torch.int32).cuda()
        q = randn(total, h, d).to(dt)
        kv = randn(len(lens) * case["cross"], 2, hk, d).to(dt)
        k, v = kv[:, 0], kv[:, 1]
    else:
        cuk = None
        qkv = randn(total, h + 2 * hk, d).to(dt)          # one projection's output, split by heads
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    s = dict(case=case, q=q, k=k, v=v, cu=cu, cuk=cuk, longest=max(lens), longest_k=case["cross"] or max(lens))
    if case["train"]:
        s["do"] = randn(total, h, d).to(dt)
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _own_norm(s):
    import concord_b200
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return concord_b200.layer_norm(s["x"], s["w"], s["b"], out_dtype=DTYPES[c["y"]])
    x, w, b = (s[n].detach().requires_grad_() for n in ("x", "w", "b"))
    y = concord_b200.layer_norm(x, w, b, out_dtype=DTYPES[c["y"]])
    return (y.detach(),) + torch.autograd.grad(y, (x, w, b), s["dy"])


def _own_distill(s):
    import concord_b200
    c = s["case"]
    kw = dict(labels=s["labels"], temperature=c["temp"], alpha=c["alpha"], ignore_index=IGNORE)
    if c["fused"]:
        return concord_b200.distill_loss_and_grad(s["z"], s["ids"], s["t"], **kw)
    z = s["z"].detach().requires_grad_()
    loss = concord_b200.distill_loss(z, s["ids"], s["t"], **kw)
    return (loss.detach(),) + torch.autograd.grad(loss, (z,))


def _own_attend(s):
    import concord_b200
    c = s["case"]
    if not c["train"]:
        with torch.no_grad():
            return concord_b200.packed_attention(s["q"], s["k"], s["v"], s["cu"], s["cuk"], causal=c["causal"],
                                                 return_lse=True)
    q, k, v = (s[n].detach().requires_grad_() for n in ("q", "k", "v"))
    o = concord_b200.packed_attention(q, k, v, s["cu"], s["cuk"], causal=c["causal"])
    return (o.detach(),) + torch.autograd.grad(o, (q, k, v), s["do"])


def _plain_norm(s):
    c = s["case"]
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + 1e-5)
    xh = xc * rstd
    y = (xh * s["w"] + s["b"]).to(DTYPES[c["y"]])
    if not c["train"]:
        return y
    dy = s["dy"].float()
    g = dy * s["w"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    return y, dx.to(s["x"].dtype), (dy * xh).sum(0), dy.sum(0)


def _plain_distill(s):
    c, z = s["case"], s["z"].float()
    n, v = z.shape
    temp, alpha = c["temp"], c["alpha"]
    ids, valid = s["ids"].clamp(min=0), s["ids"] >= 0
    has = valid.any(1, keepdim=True)
    t = torch.where(valid, s["t"] / temp, -math.inf)
    t = torch.where(has, t - t.amax(1, keepdim=True), t)
    p = torch.where(valid, torch.exp(t), 0.0)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
    top = z.amax(1, keepdim=True)
    e = torch.exp((z - top) / temp)
    total = e.sum(1, keepdim=True)
    logq = (z.gather(1, ids) - top) / temp - torch.log(total)
    kl = torch.where(p > 0, p * (torch.log(p.clamp(min=1e-30)) - logq), 0.0).sum(1)
    loss = alpha * temp * temp * kl
    dz = e * (alpha * temp * has / total)
    dz.scatter_add_(1, ids, -alpha * temp * p)
    counts = has[:, 0]
    if s["labels"] is not None:
        counts = s["labels"] != IGNORE
        y = torch.where(counts, s["labels"], 0)[:, None]
        e1 = torch.exp(z - top)
        total1 = e1.sum(1, keepdim=True)
        loss = loss + (1 - alpha) * (torch.log(total1) + top - z.gather(1, y))[:, 0]
        dz += e1 * ((1 - alpha) / total1)
        dz.scatter_add_(1, y, torch.full_like(total1, alpha - 1))
    number = counts.sum().clamp(min=1)
    loss = torch.where(counts, loss, 0.0).sum() / number
    dz *= counts[:, None] / number
    return loss, dz.to(s["z"].dtype)


def _plain_attend(s):
    c = s["case"]
    h, hk, d = c["heads"], c["kv_heads"], c["dim"]
    grp, scale = h // hk, d ** -0.5

    def padded(cu, longest, rows):
        pos = torch.arange(longest, device="cuda")
        valid = pos < (cu[1:] - cu[:-1])[:, None]
        return torch.where(valid, cu[:-1, None] + pos, rows), valid       # row `rows`: zeros, and what is dropped

    cuk = s["cu"] if s["cuk"] is None else s["cuk"]
    at, ok = padded(s["cu"], s["longest"], s["q"].shape[0])
    atk, okk = padded(cuk, s["longest_k"], s["k"].shape[0])

    def take(x, idx, heads):                                               # [T, H, D] -> [B, Hk, (g L), D]
        x = torch.cat([x.float(), x.new_zeros(1, *x.shape[1:], dtype=torch.float32)])[idx]
        return x.view(*idx.shape, hk, heads // hk, d).permute(0, 2, 3, 1, 4).reshape(len(idx), hk, -1, d)

    def back(x, idx, heads, rows):                                         # and back to [T, H, D]
        x = x.view(len(idx), hk, heads // hk, idx.shape[1], d).permute(0, 3, 1, 2, 4).reshape(*idx.shape, heads, d)
        out = x.new_zeros(rows + 1, heads, d)
        out[idx] = x
        return out[:rows]

    q, k, v = take(s["q"], at, h), take(s["k"], atk, hk), take(s["v"], atk, hk)
    mask = ok[:, :, None] & okk[:, None, :]
    if c["causal"]:
        more = ((cuk[1:] - cuk[:-1]) - (s["cu"][1:] - s["cu"][:-1]))[:, None, None]
        i, j = torch.arange(s["longest"], device="cuda"), torch.arange(s["longest_k"], device="cuda")
        mask = mask & (j[None, None, :] <= i[None, :, None] + more)
    mask = mask[:, None, None].expand(-1, -1, grp, -1, -1).reshape(len(at), 1, grp * s["longest"], s["longest_k"])
    p = (q @ k.transpose(2, 3)).mul_(scale).masked_fill_(~mask, -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    p = p.div_(torch.where(total > 0, total, 1.0))
    o = p @ v
    rows, dt = s["q"].shape[0], s["q"].dtype
    out = back(o, at, h, rows).to(dt)
    if not c["train"]:
        lse = lse.view(len(at), hk, grp, s["longest"]).permute(0, 3, 1, 2).reshape(*at.shape, h)
        flat = lse.new_zeros(rows + 1, h)
        flat[at] = lse
        return out, flat[:rows].t().contiguous()
    do = take(s["do"], at, h)
    delta = (do * o).sum(-1, keepdim=True)
    dv = p.transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3)).sub_(delta).mul_(p).mul_(scale)
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    rows_k = s["k"].shape[0]
    return out, back(dq, at, h, rows).to(dt), back(dk, atk, hk, rows_k).to(dt), back(dv, atk, hk, rows_k).to(dt)


_run_own = {"norm": _own_norm, "distill": _own_distill, "attend": _own_attend}
_run_plain = {"norm": _plain_norm, "distill": _plain_distill, "attend": _plain_attend}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        outs, dw, db = [], 0.0, 0.0
        for at in range(0, case["rows"], 8192):
            x = s["x"][at:at + 8192].double()
            var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
            sd = torch.sqrt(var + 1e-5)
            xh = (x - mean) / sd
            part = [xh * s["w"].double() + s["b"].double()]
            if case["train"]:
                dy = s["dy"][at:at + 8192].double()
                gw = dy * s["w"].double()
                part.append((gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True)) / sd)
                dw, db = dw + (dy * xh).sum(0), db + dy.sum(0)
            outs.append(part)
        cat = [torch.cat(col) for col in zip(*outs)]
        return cat[0] if not case["train"] else (cat[0], cat[1], dw, db)
    if case["op"] == "distill":
        n, v = s["z"].shape
        temp, alpha, loss = case["temp"], case["alpha"], 0.0
        keep = (s["ids"] >= 0).any(1) if s["labels"] is None else s["labels"] != IGNORE
        number = max(1, int(keep.sum()))
        dz = torch.zeros(n, v, dtype=torch.float64, device="cuda")
        for at in range(0, n, 2048):
            rows = torch.arange(at, min(n, at + 2048), device="cuda")
            rows = rows[keep[rows]]
            if not len(rows):
                continue
            z = s["z"][rows].double()
            target = torch.zeros_like(z)                                    # the teacher's distribution, dense
            t = s["t"][rows].double().div(temp).masked_fill(s["ids"][rows] < 0, -math.inf)
            some = (s["ids"][rows] >= 0).any(1)
            p = torch.zeros_like(t)
            p[some] = torch.softmax(t[some], 1)
            target.scatter_add_(1, s["ids"][rows].clamp(min=0), p)
            logq = torch.log_softmax(z / temp, 1)
            kl = (torch.xlogy(target, target) - target * logq).sum(1)
            grad = alpha * temp * (logq.exp() * some[:, None] - target)
            each = alpha * temp * temp * kl
            if s["labels"] is not None:
                y = s["labels"][rows]
                logp = torch.log_softmax(z, 1)
                each = each - (1 - alpha) * logp.gather(1, y[:, None])[:, 0]
                hot = torch.zeros_like(z).scatter_(1, y[:, None], 1.0)
                grad = grad + (1 - alpha) * (logp.exp() - hot)
            loss = loss + each.sum() / number
            dz[rows] = grad / number
        return loss, dz
    lens = _lengths(case)
    h, hk, d, total = case["heads"], case["kv_heads"], case["dim"], case["total"]
    f64 = dict(dtype=torch.float64, device="cuda")
    o, lse, dq = torch.zeros(total, h, d, **f64), torch.zeros(h, total, **f64), torch.zeros(total, h, d, **f64)
    dk, dv = torch.zeros(s["k"].shape[0], hk, d, **f64), torch.zeros(s["k"].shape[0], hk, d, **f64)
    first, first_k = 0, 0
    for n in lens:
        nk = case["cross"] or n
        a, b = slice(first, first + n), slice(first_k, first_k + nk)
        first, first_k = first + n, first_k + nk
        if n == 0:
            continue
        hidden = torch.ones(n, nk, dtype=torch.bool, device="cuda").triu_(nk - n + 1) if case["causal"] else None
        for head in range(h):
            kvh = head // (h // hk)
            q, k, v = s["q"][a, head].double(), s["k"][b, kvh].double(), s["v"][b, kvh].double()
            score = (q @ k.T) / math.sqrt(d)
            if hidden is not None:
                score.masked_fill_(hidden, -math.inf)
            lse[head, a] = torch.logsumexp(score, 1)
            p = score.sub_(lse[head, a][:, None]).exp_()
            o[a, head] = p @ v
            if case["train"]:
                g = s["do"][a, head].double()
                dv[b, kvh] += p.T @ g
                ds = p * (g @ v.T - (g * o[a, head]).sum(1, keepdim=True)) / math.sqrt(d)
                dq[a, head] = ds @ k
                dk[b, kvh] += ds.T @ q
    return (o, dq, dk, dv) if case["train"] else (o, lse)
