"""Cases of the attention operators that keep the log-sum-exp and of the layer-norm operators, forward and backward.

    attn      out, lse = attention_lse(q, k, v)            softmax(scale q k^T + mask) v and the log-sum-exp of every row
    attn_bwd  dq, dk, dv = attention_lse_bwd(dout, ...)    its gradient; the probabilities are recomputed from lse
    ln        y, stats = layer_norm(x, gamma, beta, eps)
    ln_bwd    dx, dgamma, dbeta = layer_norm_bwd(dy, ...)  the gradient, with the reduction of the weights' over the rows

`own = False`: elementary torch operations in 32 bits.  `own = True`: the framework's kernels, as torch operators.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6


def _attn(op, dtype, b, tq, tk, hq, hkv, d, causal=False, ragged=False, layout="separate"):
    return dict(op=op, dtype=dtype, B=b, Tq=tq, Tk=tk, Hq=hq, Hkv=hkv, D=d, causal=causal, ragged=ragged, layout=layout)


def _ln(op, dtype, rows, c, wtype="f32", addend=False):
    return dict(op=op, dtype=dtype, rows=rows, C=c, wtype=wtype, addend=addend)


def listed():
    return [
        # a transformer classifier behind the purifier: 14 x 14 patches and a class token, 12 heads, q / k / v in one projection
        dict(name="attn_patches", **_attn("attn", "bf16", 64, 197, 197, 12, 12, 64, layout="split")),
        # the guided UNet's 32 x 32 attention level (512 channels, heads of 64) at the headline batch of 64
        dict(name="attn_32x32", **_attn("attn", "f16", 64, 1024, 1024, 8, 8, 64, layout="legacy")),
        # one pooling query over a long token axis, heads sharing their keys: few rows, a long sum
        dict(name="attn_one_query", **_attn("attn", "bf16", 4, 1, 50001, 16, 4, 128)),
        # the guided UNet's 16 x 16 level for one image at full precision: the small call of an attack step
        dict(name="attn_bwd_16x16_f32", **_attn("attn_bwd", "f32", 1, 256, 256, 16, 16, 64, layout="legacy")),
        # the classifier's gradient over a padded batch of token sequences (dropped patches), one of them empty
        dict(name="attn_bwd_patches_padded", **_attn("attn_bwd", "bf16", 32, 197, 197, 12, 12, 64, ragged=True, layout="split")),
        # the gradient of the 32 x 32 level at the adjoint workload's batch of 32
        dict(name="attn_bwd_32x32", **_attn("attn_bwd", "f16", 32, 1024, 1024, 8, 8, 64, layout="legacy")),
        # NCSN++'s 16 x 16 level: one head of 256 channels, the CIFAR adjoint's batch of 128
        dict(name="attn_bwd_one_wide_head", **_attn("attn_bwd", "f16", 128, 256, 256, 1, 1, 256, layout="split")),
        # a long causal sequence of odd length, four query heads to a key head
        dict(name="attn_bwd_long_causal", **_attn("attn_bwd", "bf16", 1, 8191, 8191, 16, 4, 128, causal=True)),
        # the last norm of a classifier, over the class tokens of a batch only
        dict(name="ln_class_tokens", **_ln("ln", "f32", 64, 768)),
        # the norm of a block of a classifier, over a batch of 256 images
        dict(name="ln_patches", **_ln("ln", "bf16", 256 * 197, 768)),
        # its gradient in a pre-norm block: the residual branch's gradient is added to dx
        dict(name="ln_bwd_patches", **_ln("ln_bwd", "bf16", 256 * 197, 768, addend=True)),
        # an odd width and an odd number of rows
        dict(name="ln_bwd_odd", **_ln("ln_bwd", "f32", 5003, 1001)),
    ]


#: most score elements, score elements x head dimension, and norm elements of a listed case
_MOST_SCORES, _MOST_WORK, _MOST_NORM = 16 * 8191 * 8191, 16 * 8191 * 8191 * 128, 256 * 197 * 768


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn_bwd", "attn_bwd", "ln", "ln_bwd"])
    dtype = rng.choice(["f32", "f16", "bf16", "f16", "bf16"])
    if op in ("ln", "ln_bwd"):
        c = _log(rng, 64, 5000)
        c = c if rng.random() < 0.4 else max(64, c // 64 * 64)
        rows = _log(rng, 1, max(2, min(60000, _MOST_NORM // c)))
        return _ln(op, dtype, rows, c, wtype=rng.choice(["f32", dtype]), addend=op == "ln_bwd" and rng.random() < 0.5)
    d = rng.choice([32, 64, 64, 64, 80, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 1, 1, 2, 4])
    causal, ragged = rng.random() < 0.3, rng.random() < 0.3
    while True:
        b, tq = _log(rng, 1, 64), _log(rng, 1, 8000)
        tk = tq if rng.random() < 0.7 else _log(rng, 1, 8000)
        if op == "attn_bwd" and tk < 8:   # the gradient of a softmax over one key is zero: nothing to compare but rounding
            continue
        scores = b * hq * tq * tk
        if scores <= _MOST_SCORES // 4 and scores * d <= _MOST_WORK // (8 if dtype == "f32" else 1) and b * max(tq, tk) * hq * d <= 2 ** 28:
            break
    layout = rng.choice(["legacy", "split", "separate"]) if tq == tk and hq == hkv else "separate"
    return _attn(op, dtype, b, tq, tk, hq, hkv, d, causal, ragged, layout)


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] in ("ln", "ln_bwd"):
        n, c, rows = case["rows"] * case["C"], case["C"], case["rows"]
        w = BYTES[case["wtype"]] * c
        if case["op"] == "ln":
            return {"bytes": 2 * n * e + 2 * w + 8 * rows, "flops": 8 * n}
        return {"bytes": (4 if case["addend"] else 3) * n * e + 3 * w + 8 * rows, "flops": 14 * n}
    b, tq, tk, hq, hkv, d = (case[x] for x in ("B", "Tq", "Tk", "Hq", "Hkv", "D"))
    q, kv, rows = b * tq * hq * d, b * tk * hkv * d, b * hq * tq
    # a ragged batch: lengths spread over nothing to everything leave half the inputs and, for both lengths together, a third of the scores;
    # a causal diagonal leaves half of a square
    share = (0.5 if case["causal"] and tq == tk else 1.0) * (1 / 3 if case["ragged"] else 1.0)
    half = 0.5 if case["ragged"] else 1.0
    scores = share * b * hq * tq * tk
    if case["op"] == "attn":
        return {"bytes": half * (q + 2 * kv) * e + q * e + 4 * rows, "flops": 4 * scores * d}
    return {"bytes": half * ((3 * q + 2 * kv) * e + 4 * rows) + (q + 2 * kv) * e, "flops": 10 * scores * d}


# ---- inputs --------------------------------------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _keep(s):
    """[B, 1, Tq, Tk] truth values: which scores count.  Lengths are per sample; the causal diagonal ends at the last valid key."""
    tq, tk = s["q"].shape[1], s["k"].shape[1]
    i, j = torch.arange(tq, device="cuda")[None, :, None], torch.arange(tk, device="cuda")[None, None, :]
    n = s["q_lens"][:, None, None] if s["q_lens"] is not None else tq
    m = s["kv_lens"][:, None, None] if s["kv_lens"] is not None else tk
    keep = (i < n) & (j < m)
    if s["causal"]:
        keep = keep & (j <= i + (m - n))
    return keep[:, None]


def _heads_first(t, heads):
    """[B, T, H, D] of any type -> [B, heads, T, D] in 32 bits, key heads repeated for the query heads that share them"""
    t = t.float().permute(0, 2, 1, 3)
    return t.repeat_interleave(heads // t.shape[1], dim=1) if t.shape[1] != heads else t.contiguous()


def _scores(s):
    hq = s["q"].shape[2]
    return torch.matmul(_heads_first(s["q"], hq) * s["scale"], _heads_first(s["k"], hq).transpose(2, 3).contiguous())


def _attention(s):
    hq, x = s["q"].shape[2], _scores(s)
    if s["masked"]:
        x.masked_fill_(~_keep(s), -math.inf)
    top = x.amax(dim=3, keepdim=True)
    if s["masked"]:
        top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = x.sub_(top).exp_()
    total = p.sum(dim=3, keepdim=True)
    out = torch.matmul(p, _heads_first(s["v"], hq)) / (total if not s["masked"] else total.clamp(min=1e-30))
    return out.permute(0, 2, 1, 3).contiguous().to(s["q"].dtype), (top + total.log())[..., 0]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["dtype"]]
    if case["op"] in ("ln", "ln_bwd"):
        rows, c = case["rows"], case["C"]
        # activations of a residual stream: an offset and a spread of their own per row, a few strong channels
        x = _randn(g, rows, c) * (0.5 + torch.rand(rows, 1, generator=g, device="cuda")) + 0.3 * _randn(g, rows, 1)
        x[:, :: max(1, c // 7)] *= 4.0
        s = dict(case, x=x.to(t), gamma=(1 + 0.2 * _randn(g, c)).to(TYPES[case["wtype"]]), beta=(0.2 * _randn(g, c)).to(TYPES[case["wtype"]]))
        if case["op"] == "ln_bwd":
            xf = s["x"].float()
            mean = xf.mean(dim=1, keepdim=True)
            s["stats"] = torch.cat([mean, (xf - mean).square().mean(dim=1, keepdim=True).add(EPS).rsqrt()], dim=1)
            s["dy"] = _randn(g, rows, c).mul_(0.1).to(t)
            s["addend"] = _randn(g, rows, c).mul_(0.1).to(t) if case["addend"] else None
        return s
    b, tq, tk, hq, hkv, d = (case[x] for x in ("B", "Tq", "Tk", "Hq", "Hkv", "D"))
    if case["layout"] == "legacy":        # heads x [q | k | v]
        q, k, v = (1.3 * _randn(g, b, tq, hq, 3, d)).to(t).unbind(3)
    elif case["layout"] == "split":       # [q of all heads | k | v]
        q, k, v = (1.3 * _randn(g, b, tq, 3, hq, d)).to(t).unbind(2)
    else:
        q, k, v = ((1.3 * _randn(g, b, n, h, d)).to(t) for n, h in ((tq, hq), (tk, hkv), (tk, hkv)))
    s = dict(case, q=q, k=k, v=v, scale=1 / math.sqrt(d), q_lens=None, kv_lens=None, masked=case["causal"] or case["ragged"])
    if case["ragged"]:                    # sequences of every length, the whole one and none among them
        share = torch.rand(b, generator=g, device="cuda")
        share[0] = 1.0
        if b > 2:
            share[b // 2] = 0.0
        s["q_lens"], s["kv_lens"] = ((share * n).round().to(torch.int32) for n in (tq, tk))
    if case["op"] == "attn_bwd":          # what the forward pass left
        s["out"], s["lse"] = _attention(s)
        s["dout"] = _randn(g, b, tq, hq, d).mul_(0.1).to(t)
    return s


# ---- one pass ------------------------------------------------------------------------------------------------------
def _attention_bwd(s):
    hq, hkv = s["q"].shape[2], s["k"].shape[2]
    p = _scores(s)
    if s["masked"]:
        keep = _keep(s)
        p = p.sub_(s["lse"][..., None]).masked_fill_(~keep, -math.inf).exp_()
    else:
        p = p.sub_(s["lse"][..., None]).exp_()
    do = _heads_first(s["dout"], hq)
    if s["q_lens"] is not None:           # rows behind a sequence's end carry no gradient, whatever they hold
        do = do * (torch.arange(do.shape[2], device="cuda") < s["q_lens"][:, None])[:, None, :, None]
    dv = torch.matmul(p.transpose(2, 3), do)
    delta = (do * _heads_first(s["out"], hq)).sum(dim=3, keepdim=True)
    ds = torch.matmul(do, _heads_first(s["v"], hq).transpose(2, 3).contiguous()).sub_(delta).mul_(p).mul_(s["scale"])
    dq = torch.matmul(ds, _heads_first(s["k"], hq))
    dk = torch.matmul(ds.transpose(2, 3), _heads_first(s["q"], hq))
    if hq != hkv:                         # the gradient of a shared head is the sum over the heads that share it
        dk, dv = (x.unflatten(1, (hkv, hq // hkv)).sum(dim=2) for x in (dk, dv))
    return tuple(x.permute(0, 2, 1, 3).contiguous().to(s["q"].dtype) for x in (dq, dk, dv))


def _layer_norm(s):
    x = s["x"].float()
    mean = x.mean(dim=1, keepdim=True)
    x = x - mean
    rstd = x.square().mean(dim=1, keepdim=True).add(EPS).rsqrt()
    return (x * rstd * s["gamma"].float() + s["beta"].float()).to(s["x"].dtype), torch.cat([mean, rstd], dim=1)


def _layer_norm_bwd(s):
    dy = s["dy"].float()
    xhat = (s["x"].float() - s["stats"][:, :1]) * s["stats"][:, 1:]
    g = dy * s["gamma"].float()
    dx = (g - g.mean(dim=1, keepdim=True) - xhat * (g * xhat).mean(dim=1, keepdim=True)) * s["stats"][:, 1:]
    if s["addend"] is not None:
        dx = dx + s["addend"].float()
    return dx.to(s["x"].dtype), (dy * xhat).sum(dim=0).to(s["gamma"].dtype), dy.sum(dim=0).to(s["gamma"].dtype)


def run(s):
    op = s["op"]
    if own:
        import diffpure_amd.torch_ops  # noqa: F401
        fw = torch.ops.diffpure_hip
        if op == "attn":
            return fw.attention_lse(s["q"], s["k"], s["v"], s["scale"], s["causal"], s["q_lens"], s["kv_lens"])
        if op == "attn_bwd":
            return fw.attention_lse_bwd(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["scale"], s["causal"], s["q_lens"], s["kv_lens"])
        if op == "ln":
            return fw.layer_norm(s["x"], s["gamma"], s["beta"], EPS)
        return fw.layer_norm_bwd(s["dy"], s["x"], s["gamma"], s["stats"], s["addend"])
    return {"attn": _attention, "attn_bwd": _attention_bwd, "ln": _layer_norm, "ln_bwd": _layer_norm_bwd}[op](s)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------
def _softmax_rows(q, k, v, scale, causal):
    """one sample and one head, cut to its lengths: [n, D], [m, D], [m, D] -> out [n, D], lse [n]; rows without a key give 0 and -inf"""
    n, m = q.shape[0], k.shape[0]
    if m == 0:
        return q * 0.0, q.sum(dim=1) * 0.0 - math.inf
    z = (q @ k.T) * scale
    if causal:
        z = z + torch.full((n, m), -math.inf, device=z.device, dtype=z.dtype).triu(m - n + 1)
    empty = max(0, n - m) if causal else 0          # the first rows of a sequence that is longer than its keys
    lse = torch.logsumexp(z[empty:], dim=1)
    out = torch.exp(z[empty:] - lse[:, None]) @ v
    return torch.cat([q[:empty] * 0.0, out]), torch.cat([q[:empty].sum(dim=1) * 0.0 - math.inf, lse])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("ln", "ln_bwd"):
        grad = case["op"] == "ln_bwd"
        x, w, z = (s[n].double().requires_grad_(grad) for n in ("x", "gamma", "beta"))
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + z
        if not grad:
            return y, torch.cat([mean, 1 / torch.sqrt(var + EPS)], dim=1)
        dx, dw, dz = torch.autograd.grad(y, (x, w, z), s["dy"].double())
        return (dx if s["addend"] is None else dx + s["addend"].double()), dw, dz
    b, hq, hkv = case["B"], case["Hq"], case["Hkv"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    grad = case["op"] == "attn_bwd"
    if grad:
        res = [torch.zeros_like(x) for x in (q, k, v)]
    else:
        res = [torch.zeros_like(q), torch.full((b, hq, case["Tq"]), -math.inf, device="cuda", dtype=torch.float64)]
    ends = [(case["Tq"], case["Tk"])] * b if s["q_lens"] is None else list(zip(s["q_lens"].tolist(), s["kv_lens"].tolist()))
    for i, (n, m) in enumerate(ends):
        for h in range(hq):
            if n == 0:
                continue
            a = [q[i, :n, h], k[i, :m, h // (hq // hkv)], v[i, :m, h // (hq // hkv)]]
            if not grad:
                res[0][i, :n, h], res[1][i, h, :n] = _softmax_rows(*a, s["scale"], case["causal"])
                continue
            if m == 0:
                continue
            a = [x.detach().requires_grad_(True) for x in a]
            got = torch.autograd.grad(_softmax_rows(*a, s["scale"], case["causal"])[0], a, s["dout"][i, :n, h].double())
            res[0][i, :n, h] += got[0]
            res[1][i, :m, h // (hq // hkv)] += got[1]
            res[2][i, :m, h // (hq // hkv)] += got[2]
    return tuple(res)
