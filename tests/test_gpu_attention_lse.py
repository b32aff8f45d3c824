"""attention_lse / attention_lse_bwd (csrc/attention_lse*.hip) against the definition in 64 bits, element by element.

Tolerances are sums of the roundings that the kernels make, weighted by what each rounding multiplies (u = eps / 2 of the type, e = 2^-24):
  scores    |ds| <= (D + 4) e |scale| |q| |k|^T                               fp32 products and sums
  P         |dP| <= P (2 ds + 4 e (1 + |lse|) + 8 e)  =: P ep                 the exponent's argument, exp2 (1 ulp)
  out       u (W |v|) [P as operand] + u |out| + W |v| (ep + (Tk + 8) e)      fp16: + Tk 2^-25 max|v| (probabilities below the normal range; the sum is >= 1)
  dV        u P^T |dO| + u |dV| + P^T |dO| (ep + (Tq Hq/Hkv + 8) e)           fp16: + Tq 2^-31 max|dO| (2^6 P)
  dS        E = u |dS| + P (|dO| . tol(out)) [delta is formed from the forward pass's own out, off by as much as `out` may be] + P (|dP| + |delta|)(ep + (D + 8) e) + P (D + 4) e (|dO| |v|^T + |dO| . |out|)
  dQ, dK    |scale| E |k|, |scale| E^T |q| + u |result| + (T + 8) e |scale| |dS| |k|,  fp16: + 2^-31 per element of dS
exp2 gives 0 below 2^-126 (the range of normal numbers): every P may be off by that much, an absolute term that only probabilities of 1e-38 meet.
fp32 operands are not rounded: u = 0 in the P and dS terms, 2^-24 in the others.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
E = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def keep_mask(b, tq, tk, causal, ql, kl):
    n = torch.full((b,), tq) if ql is None else ql.cpu().clamp(0, tq)
    m = torch.full((b,), tk) if kl is None else kl.cpu().clamp(0, tk)
    i, j = torch.arange(tq)[None, :, None], torch.arange(tk)[None, None, :]
    keep = (i < n[:, None, None]) & (j < m[:, None, None])
    if causal:
        keep = keep & (j <= i + (m - n)[:, None, None])
    return keep[:, None]


def clean(t, lens):
    """64-bit copy on the host with what lies behind the lengths (NaN, say) set to zero: the definition does not look at it"""
    t = t.detach().double().cpu().clone()
    if lens is not None:
        for i, n in enumerate(lens.cpu().clamp(0, t.shape[1]).tolist()):
            t[i, n:] = 0
    return t


class Ref:
    """the definition: forward, and gradients by its formulas; heads first, key heads repeated"""

    def __init__(self, q, k, v, scale, causal, ql, kl):
        self.u = torch.finfo(q.dtype).eps / 2
        self.up = 0.0 if q.dtype == torch.float32 else self.u         # rounding of P / dS as operands
        self.tiny = q.dtype == torch.float16
        self.b, self.tq, self.hq, self.d = q.shape
        self.tk, self.hkv = k.shape[1], k.shape[2]
        self.g = self.hq // self.hkv
        self.scale = 1 / math.sqrt(self.d) if scale is None else scale
        self.q, self.k, self.v = (self.first(clean(t, le)) for t, le in ((q, ql), (k, kl), (v, kl)))
        self.keep = keep_mask(self.b, self.tq, self.tk, causal, ql, kl)
        s = (self.q @ self.k.transpose(2, 3) * self.scale).masked_fill(~self.keep, -math.inf)
        top = s.amax(3, keepdim=True)
        top = torch.where(top.isinf(), torch.zeros_like(top), top)
        p = torch.exp(s - top)
        tot = p.sum(3, keepdim=True)
        self.p = torch.where(tot > 0, p / tot.clamp(min=1e-300), torch.zeros_like(p))
        self.lse = (top + tot.log())[..., 0]
        self.o = self.p @ self.v
        ds = (self.d + 4) * E * abs(self.scale) * (self.q.abs() @ self.k.abs().transpose(2, 3))
        self.ep = torch.where(self.keep, 2 * ds + 12 * E + 4 * E * self.lse.abs().nan_to_num(0, 0, 0)[..., None], torch.zeros_like(ds))
        w = self.p @ self.v.abs()
        self.tout = self.u * self.o.abs() + w * self.up + (self.p * self.ep) @ self.v.abs() + w * (self.ep.amax(3, keepdim=True) + (self.tk + 8) * E)
        if self.tiny:
            self.tout = self.tout + self.tk * 2.0 ** -25 * self.v.abs().amax() + 2.0 ** -25
        self.eps = (self.ep.amax(3) + 4 * E * (1 + self.lse.abs().nan_to_num(0, 0, 0)) + (self.tk + 8) * E)

    def first(self, t):
        t = t.permute(0, 2, 1, 3)
        return t.repeat_interleave(self.hq // t.shape[1], 1)

    def back(self, t):
        return t.permute(0, 2, 1, 3)

    def fold(self, t):
        return t.unflatten(1, (self.hkv, self.g)).sum(2).permute(0, 2, 1, 3)

    def out_tol(self):
        return self.back(self.tout)

    def bwd(self, dout, ql):
        do = self.first(clean(dout, ql))
        self.do = do
        dp = do @ self.v.transpose(2, 3)
        delta = (do * self.o).sum(3, keepdim=True)
        ds = self.p * (dp - delta)
        ado, ao = do.abs(), (do.abs() * self.o.abs()).sum(3, keepdim=True)
        adp = ado @ self.v.abs().transpose(2, 3)
        err = self.up * ds.abs() + self.p * ((ado * self.tout).sum(3, keepdim=True) + (dp.abs() + delta.abs()) * (self.ep + (self.d + 8) * E) + (self.d + 4) * E * (adp + ao))
        err = err * (1 + self.up) + 2.0 ** -126 * self.keep * (dp.abs() + delta.abs())
        if self.tiny:
            err = err + 2.0 ** -31 * self.keep
        sc, n = abs(self.scale), self.tq * self.g
        dv, dk, dq = self.p.transpose(2, 3) @ do, self.scale * ds.transpose(2, 3) @ self.q, self.scale * ds @ self.k
        aq, ak = self.q.abs(), self.k.abs()
        tdq = sc * (err + (self.tk + 8) * E * ds.abs()) @ ak
        tdk = sc * (err + (n + 8) * E * ds.abs()).transpose(2, 3) @ aq
        pv = self.p * (self.up + self.ep + (n + 8) * E) + 2.0 ** -126 * self.keep
        if self.tiny:
            pv = pv + 2.0 ** -31 * self.keep
        tdv = pv.transpose(2, 3) @ ado
        res = [self.back(dq), self.fold(dk), self.fold(dv)]
        # the last rounding; fp16 results below the normal range: half of 2^-24
        low = 2.0 ** -25 if self.tiny else 1e-37
        tol = [t + self.u * r.abs() * (1 + 2 * self.u) + low for t, r in zip((self.back(tdq), self.fold(tdk), self.fold(tdv)), res)]
        return res, tol


def close(got, want, tol, name):
    got = got.detach().double().cpu()
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{name}: not finite where it should be (or the reverse)"
    fin = torch.isfinite(want)
    assert torch.equal(got[~fin], want[~fin]), name
    off, tol = (got - want).abs()[fin], tol[fin]
    assert (off <= tol).all(), f"{name}: {(off / tol)[off > tol].max().item():.3f} of the tolerance"


def make(dtype, b, tq, tk, hq, hkv, d, layout="separate", amp=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s):
        return (amp * torch.randn(*s, generator=g, device="cuda")).to(dtype)
    if layout == "legacy":
        q, k, v = rnd(b, tq, hq, 3, d).unbind(3)
    elif layout == "split":
        q, k, v = rnd(b, tq, 3, hq, d).unbind(2)
    elif layout == "heads":               # [B, H, T, D] memory, a wider row, an offset
        q, k, v = (rnd(b, h, t + 1, d + 16)[:, :, 1:, 8:8 + d].transpose(1, 2) for h, t in ((hq, tq), (hkv, tk), (hkv, tk)))
    else:
        q, k, v = rnd(b, tq, hq, d), rnd(b, tk, hkv, d), rnd(b, tk, hkv, d)
    return q, k, v, rnd(b, tq, hq, d)


def lens_of(*v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


SHAPES = [      # b, tq, tk, hq, hkv, d, causal, q_lens, kv_lens, layout
    (1, 1, 1, 1, 1, 8, False, None, None, "separate"),
    (2, 1, 77, 4, 2, 64, False, None, None, "separate"),
    (1, 77, 1, 2, 2, 64, False, None, None, "separate"),
    (2, 33, 33, 3, 3, 40, False, None, None, "legacy"),
    (2, 31, 65, 2, 1, 32, True, None, None, "heads"),
    (2, 65, 31, 2, 1, 32, True, None, None, "heads"),              # more rows than keys: the first 34 see nothing
    (3, 197, 197, 2, 2, 64, False, None, None, "split"),
    (2, 128, 128, 2, 2, 64, False, None, None, "legacy"),
    (2, 300, 257, 6, 2, 64, True, None, None, "separate"),
    (4, 130, 90, 2, 2, 72, False, (130, 0, 33, 64), (90, 17, 0, 64), "separate"),
    (4, 100, 100, 4, 1, 128, True, (100, 1, 64, 37), (100, 1, 64, 80), "separate"),
    (3, 64, 200, 2, 2, 96, True, (64, 500, -3), (10, 200, 70), "heads"),      # lengths outside 0 .. T are clamped
    (1, 150, 150, 1, 1, 256, False, None, None, "split"),
    (2, 70, 140, 2, 1, 200, True, None, None, "separate"),
    (2, 40, 50, 2, 2, 64, True, (40, 7), None, "separate"),
    (2, 40, 50, 2, 2, 64, False, None, (50, 9), "separate"),
    (1, 513, 513, 1, 1, 128, True, None, None, "legacy"),
    (1, 5, 1030, 8, 1, 16, False, None, None, "separate"),
    (1, 1030, 5, 8, 1, 16, True, None, None, "separate"),
    # more than 256 blocks: every wave has columns of its own
    (8, 130, 130, 40, 40, 64, False, None, None, "split"),
    (5, 100, 133, 60, 20, 32, True, (100, 3, 0, 64, 77), (133, 133, 9, 0, 40), "heads"),
    (6, 97, 65, 48, 48, 128, True, None, None, "legacy"),
    (9, 33, 70, 32, 32, 256, False, None, None, "separate"),
    (9, 80, 40, 32, 32, 96, True, None, None, "separate"),
    # a few rows over a long axis, both ways: ranges of their own, joined
    (2, 1, 3001, 8, 2, 64, False, None, None, "separate"),
    (2, 3, 2500, 6, 2, 128, True, (3, 1), (2500, 700), "heads"),
    (1, 2, 1500, 2, 2, 256, False, None, None, "separate"),
    (1, 3001, 3, 4, 2, 64, False, None, None, "separate"),
    (2, 1500, 40, 2, 1, 128, True, (1500, 900), (40, 40), "separate"),
    (1, 1400, 1400, 2, 1, 40, True, None, None, "separate"),
]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=[f"{s[0]}x{s[1]}x{s[2]}x{s[3]}h{s[4]}x{s[5]}{'c' if s[6] else ''}{'l' if s[7] else ''}_{s[9]}" for s in SHAPES])
def test_forward_and_gradients(dtype, shape):
    from diffpure_amd import ops
    b, tq, tk, hq, hkv, d, causal, ql, kl, layout = shape
    q, k, v, dout = make(dtype, b, tq, tk, hq, hkv, d, layout)
    ql, kl = (None if x is None else lens_of(*x) for x in (ql, kl))
    for t, le in ((q, ql), (k, kl), (v, kl), (dout, ql)):           # what lies behind the lengths may be anything
        if le is not None:
            for i, n in enumerate(le.clamp(0, t.shape[1]).tolist()):
                t[i, n:] = float("nan")
    ref = Ref(q, k, v, None, causal, ql, kl)
    out, lse = ops.attention_lse(q, k, v, None, causal, ql, kl)
    close(out, ref.back(ref.o), ref.out_tol(), "out")
    close(lse, ref.lse, ref.eps, "lse")
    grads = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl)
    res, tol = ref.bwd(dout, ql)
    for name, g, r, t in zip(("dq", "dk", "dv"), grads, res, tol):
        close(g, r, t, name)


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [-0.3, 2.0])
def test_scales_and_peaked_rows(dtype, scale):
    """negative and large scales: rows whose probabilities are 0 and 1, maxima that move from tile to tile"""
    from diffpure_amd import ops
    q, k, v, dout = make(dtype, 1, 70, 300, 2, 2, 64, amp=2.0, seed=3)
    k = (k.float() * torch.linspace(0.1, 2.0, 300, device="cuda")[None, :, None, None]).to(dtype)
    ref = Ref(q, k, v, scale, False, None, None)
    out, lse = ops.attention_lse(q, k, v, scale)
    close(out, ref.back(ref.o), ref.out_tol(), "out")
    close(lse, ref.lse, ref.eps, "lse")
    res, tol = ref.bwd(dout, None)
    for name, g, r, t in zip(("dq", "dk", "dv"), ops.attention_lse_bwd(dout, q, k, v, out, lse, scale), res, tol):
        close(g, r, t, name)


def test_float16_small_cotangents_keep_their_precision():
    """dout of 1e-3 over 600 keys: dS around 1e-6, below fp16's normal range, is carried as 2^6 dS"""
    from diffpure_amd import ops
    q, k, v, dout = make(torch.float16, 1, 200, 600, 2, 2, 64, seed=5)
    dout = (dout.float() * 1e-3).half()
    ref = Ref(q, k, v, None, False, None, None)
    out, lse = ops.attention_lse(q, k, v)
    res, tol = ref.bwd(dout, None)
    for name, g, r, t in zip(("dq", "dk", "dv"), ops.attention_lse_bwd(dout, q, k, v, out, lse), res, tol):
        close(g, r, t, name)


def test_gradient_against_differences():
    """<grad, x> of the kernels in fp32 against central differences of the 64-bit forward pass (step 1e-4: truncation below 1e-7 of the sum)"""
    from diffpure_amd import ops
    q, k, v, dout = make(torch.float32, 2, 20, 37, 4, 2, 24, seed=7)
    ql, kl = lens_of(20, 11), lens_of(37, 15)
    out, lse = ops.attention_lse(q, k, v, None, True, ql, kl)
    grads = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, True, ql, kl)
    _, tol = Ref(q, k, v, None, True, ql, kl).bwd(dout, ql)
    w = clean(dout, ql)

    def loss(*x):
        r = Ref(*x, None, True, ql, kl)
        return (r.back(r.o) * w).sum().item()
    gen = torch.Generator().manual_seed(1)
    base = [t.detach().cpu().double() for t in (q, k, v)]
    for i, name in enumerate(("q", "k", "v")):
        step = torch.randn(base[i].shape, generator=gen, dtype=torch.float64)
        plus, minus = (loss(*[t + sg * 1e-4 * step if j == i else t for j, t in enumerate(base)]) for sg in (1, -1))
        want, got = (plus - minus) / 2e-4, (grads[i].cpu().double() * step).sum().item()
        assert abs(want - got) <= (tol[i] * step.abs()).sum().item() + 1e-6 * (1 + abs(want)), (name, want, got)


def test_same_results_twice_on_another_stream_and_in_a_graph():
    from diffpure_amd import ops
    q, k, v, dout = make(torch.bfloat16, 2, 197, 197, 4, 2, 64, seed=9)

    def step():
        out, lse = ops.attention_lse(q, k, v, None, True)
        return (out, lse) + tuple(ops.attention_lse_bwd(dout, q, k, v, out, lse, None, True))
    first = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs = []
    for _ in range(2):                        # two graphs of the same call, replayed in turn
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            res = step()
        graphs.append((gr, res))
    for k_ in range(4):
        q.copy_(torch.randn_like(q, dtype=torch.float32).to(q.dtype))
        for gr, _ in graphs:
            gr.replay()
        eager = step()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(eager, res)), k_


def test_offsets_beyond_32_bits():
    """tokens 128 KB apart, 40 000 of them: 5 GB between the first and the last; the same results as from dense tensors"""
    from diffpure_amd import ops
    t, d = 40000, 64
    far = torch.empty(t, 65536, device="cuda", dtype=torch.float16)
    dense = [(0.7 * torch.randn(1, t, 1, d, device="cuda")).half() for _ in range(2)]
    views = [far[:, i * 1024:i * 1024 + d].view(1, t, 1, d) for i in range(4)]
    for v, x in zip(views, dense):
        v.copy_(x)
    q, _, _, dout = make(torch.float16, 1, 70, 1, 1, 1, d)
    want = ops.attention_lse(q, *dense)
    got = ops.attention_lse(q, *views[:2])
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    want = ops.attention_lse_bwd(dout, q, *dense, *want)
    got = ops.attention_lse_bwd(dout, q, *views[:2], *got, grads=(torch.empty_like(q), views[2], views[3]))
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # and as queries: the streamed operand of dK and dV
    qs, do = views[0], views[1]
    k, v = (0.7 * torch.randn(2, 1, 33, 1, d, device="cuda")).half().unbind(0)
    out, lse = ops.attention_lse(qs, k, v)
    for a, b in zip(ops.attention_lse_bwd(dense[1], dense[0], k, v, out, lse), ops.attention_lse_bwd(do, qs, k, v, out, lse)):
        assert torch.equal(a, b)


def test_gradients_into_views_and_nothing_beside_them():
    """grads= views of one dqkv tensor in the reference's head order, inside a larger buffer that keeps its values around them"""
    from diffpure_amd import ops
    b, t, h, d = 2, 77, 3, 64
    q, k, v, dout = make(torch.float16, b, t, t, h, h, d, "legacy", seed=11)
    out, lse = ops.attention_lse(q, k, v)
    want = ops.attention_lse_bwd(dout, q, k, v, out, lse)
    buf = torch.full((b, t + 2, h, 3, d + 8), 7.0, device="cuda", dtype=torch.float16)
    views = buf[:, 1:t + 1, :, :, :d].unbind(3)
    got = ops.attention_lse_bwd(dout, q, k, v, out, lse, grads=views)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    buf[:, 1:t + 1, :, :, :d] = 7.0
    assert (buf == 7.0).all()


def test_autograd_shared_heads_expanded_inputs_and_refusals():
    import diffpure_amd.torch_ops  # noqa: F401
    att = torch.ops.diffpure_hip.attention_lse
    q, k, v, dout = make(torch.float32, 3, 40, 50, 4, 2, 32, seed=13)
    k1 = k[:1].clone().requires_grad_(True)               # one key tensor for the whole batch
    q, v = q.requires_grad_(True), v.requires_grad_(True)
    out, lse = att(q, k1.expand(3, -1, -1, -1), v)
    assert not lse.requires_grad
    gq, gk, gv = torch.autograd.grad(out, (q, k1, v), dout, retain_graph=True)
    ref = Ref(q, k1.expand(3, -1, -1, -1), v, None, False, None, None)
    (rq, rk, rv), (tq, tk, tv) = ref.bwd(dout, None)
    close(gq, rq, tq, "dq")
    close(gk, rk.sum(0, keepdim=True), tk.sum(0, keepdim=True) + 4 * E * rk.abs().sum(0, keepdim=True), "dk")
    close(gv, rv, tv, "dv")
    out.sum().backward()                                  # an expanded cotangent
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(att(q, k1.expand(3, -1, -1, -1), v)[0].sum(), q, create_graph=True)
    for bad, what in ((dict(k=k.half()), "k must be"), (dict(q_lens=torch.zeros(3, device="cuda")), "q_lens"), (dict(scale=0.0), "scale"), (dict(v=v[..., :24]), "v must be")):
        kw = dict(q=q, k=k, v=v) | bad
        with pytest.raises(RuntimeError, match=what):
            att(kw["q"], kw["k"], kw["v"], kw.get("scale"), False, kw.get("q_lens"))


def test_refusals_of_the_python_entry_points():
    from diffpure_amd import ops
    from diffpure_amd._lib import DiffpureHipError
    q, k, v, dout = make(torch.float16, 2, 8, 8, 2, 2, 16)
    out, lse = ops.attention_lse(q, k, v)
    cases = [
        (dict(q=q[..., 0]), "expected a"), (dict(q=q.double()), "expected a"), (dict(k=k.float()), "expected torch.float16"), (dict(v=v[:, :4]), "expected"),
        (dict(q=q.transpose(2, 3).contiguous().transpose(2, 3)), "contiguous"), (dict(scale=float("nan")), "scale"), (dict(scale=0.0), "scale"),
        (dict(kv_lens=torch.zeros(2, dtype=torch.int64, device="cuda")), "int32"), (dict(q_lens=torch.zeros(3, dtype=torch.int32, device="cuda")), "int32"),
        (dict(q=q[..., :12], k=k[..., :12], v=v[..., :12]), "multiple of 8"), (dict(k=k[:, :, :1], v=v[:, :, :1], q=q), None),
        (dict(q=torch.zeros(2, 8, 3, 16, device="cuda", dtype=torch.float16)), "multiple of"),
        (dict(q=torch.zeros(2 * 8 * 2 * 16 + 1, device="cuda", dtype=torch.float16)[1:].view(2, 8, 2, 16)), "aligned"),
        (dict(q=torch.zeros(2, 8, 2, 20, device="cuda", dtype=torch.float16)[..., :16]), "strides"),
    ]
    for kw, what in cases:
        a = dict(q=q, k=k, v=v) | kw
        if what is None:
            ops.attention_lse(**a)
            continue
        with pytest.raises(DiffpureHipError, match=what):
            ops.attention_lse(**a)
    for kw, what in [(dict(lse=lse[:, :1]), "lse"), (dict(lse=lse.double()), "lse"), (dict(dout=dout[:, :4]), "dout"), (dict(out=out.float()), "out"),
                     (dict(grads=(q.expand(2, 8, 2, 16), k[:1].expand(2, 8, 2, 16), v)), "also positive")]:
        a = dict(dout=dout, q=q, k=k, v=v, out=out, lse=lse) | kw
        with pytest.raises(DiffpureHipError, match=what):
            ops.attention_lse_bwd(**a)
