"""layer_norm / layer_norm_bwd (csrc/layer_norm.hip) against the definition in 64 bits, element by element, and a transformer block of the new operators.

Tolerances (u = eps / 2 of the type, e = 2^-24; every sum over a row has at most S = 48 fp32 additions in a chain: 32 per thread, 6 + 10 to join):
  mean      M = S e mean|x|
  xhat      X = rstd (M + 2 e |x - mean|) + |xhat| (R + 4 e),   R = S e + M^2 rstd^2 (relative error of rstd: half of the variance's, and the mean's)
  y         X |gamma| + 2 e (|xhat gamma| + |y|) + u |y|
  dx        rstd [ X-weighted terms of the two means ] + (S + 8) e of every product + u |dx|,  written out below
  dgamma    sum_rows |dy| X + (rows / blocks' share + 80) e sum_rows |dy xhat| + u' |dgamma|;  dbeta alike
"""
import pytest
import torch

pytestmark = pytest.mark.gpu
E, S = 2.0 ** -24, 48
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def u_of(t):
    return torch.finfo(t).eps / 2


def low_of(t):
    return 2.0 ** -25 if t == torch.float16 else 1e-37


class Ref:
    def __init__(self, x, gamma, beta, eps):
        self.x, self.c = x.detach().double().cpu().reshape(-1, x.shape[-1]), x.shape[-1]
        self.ga = torch.ones(self.c, dtype=torch.float64) if gamma is None else gamma.detach().double().cpu()
        self.be = torch.zeros(self.c, dtype=torch.float64) if beta is None else beta.detach().double().cpu()
        self.t = x.dtype
        self.mean = self.x.mean(1, keepdim=True)
        dev = self.x - self.mean
        self.rstd = 1 / torch.sqrt(dev.square().mean(1, keepdim=True) + eps)
        self.xhat = dev * self.rstd
        self.y = self.xhat * self.ga + self.be
        self.tm = S * E * self.x.abs().mean(1, keepdim=True)
        self.tr = S * E + 4 * E + (self.tm * self.rstd).square()
        self.tx = self.rstd * (self.tm + 2 * E * dev.abs()) + self.xhat.abs() * (self.tr + 4 * E)

    def y_tol(self):
        return self.tx * self.ga.abs() + 2 * E * ((self.xhat * self.ga).abs() + self.y.abs()) + u_of(self.t) * self.y.abs() * (1 + 2 * E) + low_of(self.t)

    def bwd(self, dy, addend, wtype):
        dy = dy.detach().double().cpu().reshape(-1, self.c)
        g = dy * self.ga
        m1, m2 = g.mean(1, keepdim=True), (g * self.xhat).mean(1, keepdim=True)
        dx = (g - m1 - self.xhat * m2) * self.rstd
        # the kernel's xhat comes from the given stats: rounded mean and rstd, (x - mean) rstd
        tx = self.tx
        t1, t2 = (S + 4) * E * g.abs().mean(1, keepdim=True), (g.abs() * tx).mean(1, keepdim=True) + (S + 4) * E * (g * self.xhat).abs().mean(1, keepdim=True)
        inner = 2 * E * g.abs() + t1 + tx * m2.abs() + self.xhat.abs() * t2 + 4 * E * (g.abs() + m1.abs() + (self.xhat * m2).abs())
        tdx = inner * self.rstd + dx.abs() * (self.tr + 2 * E)
        if addend is not None:
            a = addend.detach().double().cpu().reshape(-1, self.c)
            tdx = tdx + 2 * E * (dx.abs() + a.abs())
            dx = dx + a
        tdx = tdx * (1 + 4 * E) + u_of(self.t) * dx.abs() + low_of(self.t)
        chain = dy.shape[0] / 1024 + 16 + 1024 / 16 + 16 + 8         # a thread's rows, the rows of a workgroup, a wave's share of the partials, the waves
        dg, db = (dy * self.xhat).sum(0), dy.sum(0)
        tdg = (dy.abs() * (tx + 2 * E * self.xhat.abs())).sum(0) + chain * E * (dy * self.xhat).abs().sum(0) + u_of(wtype) * dg.abs() + low_of(wtype)
        tdb = chain * E * dy.abs().sum(0) + u_of(wtype) * db.abs() + low_of(wtype)
        return (dx, dg, db), (tdx, tdg, tdb)


def close(got, want, tol, name):
    got = got.detach().double().cpu().reshape(want.shape)
    over = ((got - want).abs() / tol).max().item()
    assert over <= 1, f"{name}: {over:.3f} of the tolerance"


def rnd(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


# widths on both sides of every thread plan's border (16-bit and fp32), odd ones, the widest
WIDTHS = [1, 2, 7, 64, 65, 128, 130, 257, 384, 512, 513, 768, 1001, 1024, 1281, 2048, 2050, 4096, 4099, 8192, 8200, 16384]


@pytest.mark.parametrize("dtype", TYPES, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("c", WIDTHS)
def test_widths_and_types(dtype, c):
    from diffpure_amd import ops
    rows = 37 if c < 3000 else 5
    x = (rnd(c, rows, c) * 1.5 + rnd(c + 1, rows, 1)).to(dtype)
    dy, add = rnd(c + 2, rows, c).to(dtype), rnd(c + 3, rows, c).to(dtype)
    for wtype in {torch.float32, dtype}:
        ga, be = (1 + 0.3 * rnd(c + 4, c)).to(wtype), rnd(c + 5, c).to(wtype)
        ref = Ref(x, ga, be, 1e-5)
        y, stats = ops.layer_norm(x, ga, be, 1e-5)
        close(y, ref.y, ref.y_tol(), "y")
        close(stats[:, :1], ref.mean, ref.tm + E * ref.mean.abs() + 1e-37, "mean")
        close(stats[:, 1:], ref.rstd, ref.rstd * (ref.tr + 8 * E), "rstd")
        for a in (None, add):
            want, tol = ref.bwd(dy, a, wtype)
            for name, g, w, t in zip(("dx", "dgamma", "dbeta"), ops.layer_norm_bwd(dy, x, ga, stats, a), want, tol):
                close(g, w, t, name)


@pytest.mark.parametrize("rows", [1, 3, 4, 1025, 20011])
def test_row_counts(rows):
    """one row, ragged last workgroups, more rows than the persistent grid has threads for"""
    from diffpure_amd import ops
    c = 200
    x, dy = (rnd(rows, rows, c) + 3.0).bfloat16(), rnd(rows + 1, rows, c).bfloat16()
    ga, be = 1 + 0.3 * rnd(1, c), rnd(2, c)
    ref = Ref(x, ga, be, 1e-6)
    y, stats = ops.layer_norm(x, ga, be, 1e-6)
    close(y, ref.y, ref.y_tol(), "y")
    want, tol = ref.bwd(dy, None, torch.float32)
    got = ops.layer_norm_bwd(dy, x, ga, stats)
    for name, g, w, t in zip(("dx", "dgamma", "dbeta"), got, want, tol):
        close(g, w, t, name)
    again = ops.layer_norm_bwd(dy, x, ga, stats)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_pitches_missing_weights_and_offsets():
    """rows inside wider rows at odd addresses, expanded rows, no gamma / beta, a large common offset, constant rows"""
    from diffpure_amd import ops
    wide = rnd(1, 2, 9, 131).half()
    x = wide[:, :, 1:102]                                   # 101 columns at an odd address, pitch 131
    dy = rnd(2, 101).half().expand(2, 9, 101)
    ref = Ref(x, None, None, 1e-5)
    y, stats = ops.layer_norm(x)
    assert y.is_contiguous() and y.shape == x.shape and stats.shape == (18, 2)
    close(y, ref.y, ref.y_tol(), "y")
    want, tol = ref.bwd(dy, x, torch.float32)
    got = ops.layer_norm_bwd(dy, x, None, stats, addend=x)
    assert got[1].dtype == torch.float32
    for name, g, w, t in zip(("dx", "dgamma", "dbeta"), got, want, tol):
        close(g, w, t, name)
    dx, dg, db = ops.layer_norm_bwd(dy, x, None, stats, addend=x, weights=False)
    assert dg is None and db is None and torch.equal(dx, got[0])
    x = rnd(3, 8, 333) + 1000.0                             # fp32: the deviations carry 2^-14 of the offset's rounding and no more
    ref = Ref(x, None, None, 1e-5)
    close(ops.layer_norm(x)[0], ref.y, ref.y_tol(), "offset")
    y, stats = ops.layer_norm(torch.full((3, 50), 0.7, device="cuda"))
    assert (y.abs() <= 1e-4).all() and torch.isfinite(stats).all()


def test_autograd_graph_and_refusals():
    import diffpure_amd.torch_ops  # noqa: F401
    from diffpure_amd import ops
    from diffpure_amd._lib import DiffpureHipError
    ln = torch.ops.diffpure_hip.layer_norm
    x, ga, be = rnd(1, 4, 5, 96).requires_grad_(True), (1 + rnd(2, 96)).requires_grad_(True), rnd(3, 96).requires_grad_(True)
    dy = rnd(4, 5, 4, 96).transpose(0, 1)                   # not contiguous
    y, stats = ln(x, ga, be, 1e-5)
    assert not stats.requires_grad
    want, tol = Ref(x, ga, be, 1e-5).bwd(dy.contiguous(), None, torch.float32)
    for name, g, w, t in zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(y, (x, ga, be), dy), want, tol):
        close(g, w, t, name)
    ln(x, None, be)[0].sum().backward()
    assert ga.grad is None and be.grad is not None
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ln(x, ga, be)[0].sum(), x, create_graph=True)
    xs, dys = rnd(5, 300, 96), rnd(6, 300, 96)

    def step():
        y, st = ops.layer_norm(xs, ga.detach(), be.detach())
        return (y, st) + ops.layer_norm_bwd(dys, xs, ga.detach(), st)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for k in range(3):
        xs.copy_(rnd(10 + k, 300, 96))
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, held)), k
    z = torch.zeros(4, 32, device="cuda")
    st = torch.zeros(4, 2, device="cuda")
    for call, what in ((lambda: ops.layer_norm(z.double()), "expected a"), (lambda: ops.layer_norm(z.t()), "contiguous"), (lambda: ops.layer_norm(z, z[0, :16]), "gamma"),
                       (lambda: ops.layer_norm(z, z[0], z[0].half()), "beta"), (lambda: ops.layer_norm(z.half(), z[0].bfloat16()), "gamma"),
                       (lambda: ops.layer_norm(z.half(), z[0].half(), z[0]), "one type"), (lambda: ops.layer_norm(z, eps=-1.0), "eps"), (lambda: ops.layer_norm(z[:0]), "at least one"),
                       (lambda: ops.layer_norm(torch.zeros(1, 16385, device="cuda")), "16384"), (lambda: ops.layer_norm(z.view(2, 2, 32).transpose(0, 1)), "one pitch"),
                       (lambda: ops.layer_norm_bwd(z, z, None, st[:3]), "stats"), (lambda: ops.layer_norm_bwd(z[:2], z, None, st), "dy"),
                       (lambda: ops.layer_norm_bwd(z, z, None, st, addend=z.half()), "addend")):
        with pytest.raises(DiffpureHipError, match=what):
            call()


def block_weights(c, heads, seed):
    g = torch.Generator().manual_seed(seed)

    def w(*s, sc=1.0):
        return sc * torch.randn(*s, generator=g, dtype=torch.float64)
    return dict(g1=1 + 0.1 * w(c), b1=0.1 * w(c), wqkv=w(c, 3 * c, sc=c ** -0.5), wp=w(c, c, sc=c ** -0.5), g2=1 + 0.1 * w(c), b2=0.1 * w(c), wh=w(c, 10, sc=c ** -0.5))


def test_a_classifier_block_behind_the_purifier_forward_and_backward():
    """norm -> attention -> residual -> norm -> class scores over a padded batch, as a classifier behind the purifier runs it: loss gradients w.r.t. the
    tokens and every weight through the operators (fp32) against torch's autograd of the same block in 64 bits.  Tolerance: the block is a chain of about
    ten fp32 operators of relative error below 1e-6 each on values of order one; 1e-4 of the largest gradient element bounds their sum."""
    import diffpure_amd.torch_ops  # noqa: F401
    fw = torch.ops.diffpure_hip
    b, t, c, heads = 3, 50, 96, 3
    lens = torch.tensor([50, 21, 1], dtype=torch.int32)
    x = torch.randn(b, t, c, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    weights = block_weights(c, heads, 2)
    label = torch.tensor([3, 1, 7])

    def head(tok, w):                  # class scores of the first token, cross entropy
        z = tok[:, 0] @ w["wh"]
        return (torch.logsumexp(z, 1) - z.gather(1, label.to(z.device)[:, None])[:, 0]).sum()

    def plain(x, w):
        def norm(x, g, be):
            v, m = torch.var_mean(x, -1, unbiased=False, keepdim=True)
            return (x - m) / torch.sqrt(v + 1e-6) * g + be
        q, k, v = (norm(x, w["g1"], w["b1"]) @ w["wqkv"]).view(b, t, 3, heads, c // heads).permute(2, 0, 3, 1, 4)
        s = (q @ k.transpose(2, 3)) * (c // heads) ** -0.5
        valid = torch.arange(t)[None, :] < lens[:, None]
        a = torch.softmax(s.masked_fill(~valid[:, None, None, :], -float("inf")), -1) @ v
        a = a.permute(0, 2, 1, 3) * valid[:, :, None, None]
        return head(norm(x + a.reshape(b, t, c) @ w["wp"], w["g2"], w["b2"]), w)

    def kernels(x, w):
        n = lens.cuda()
        y, _ = fw.layer_norm(x, w["g1"], w["b1"], 1e-6)
        q, k, v = (y.view(b * t, c) @ w["wqkv"]).view(b, t, 3, heads, c // heads).unbind(2)
        a, _ = fw.attention_lse(q, k, v, None, False, n, n)
        x = x + (a.reshape(b * t, c) @ w["wp"]).view(b, t, c)
        return head(fw.layer_norm(x, w["g2"], w["b2"], 1e-6)[0], w)

    res = []
    for fn, dev, dt in ((plain, "cpu", torch.float64), (kernels, "cuda", torch.float32)):
        leaves = {n: v.to(dev, dt).requires_grad_(True) for n, v in (weights | {"x": x}).items()}
        loss = fn(leaves["x"], leaves)
        names = sorted(leaves)
        res.append((loss.item(), dict(zip(names, torch.autograd.grad(loss, [leaves[n] for n in names])))))
    assert abs(res[0][0] - res[1][0]) <= 1e-5 * abs(res[0][0])
    for n, want in res[0][1].items():
        got = res[1][1][n].double().cpu()
        assert (got - want).abs().max() <= 1e-4 * want.abs().max(), n
