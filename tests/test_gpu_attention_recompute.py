"""DIFFPURE_ATTN_RECOMPUTE=1 beyond the engines' usual layers: head dimensions that attention_lse does not take."""
import pytest
import torch

from conftest import load_golden
from diffpure_amd.synth import synth_state_dict

DEV = "cuda:0"


def test_which_layers_are_recomputed(monkeypatch):
    from diffpure_amd import ops
    monkeypatch.setenv("DIFFPURE_ATTN_RECOMPUTE", "1")
    assert [d for d in (4, 8, 12, 20, 64, 250, 256, 264, 384, 512) if ops.attention_recompute_wanted(d)] == [8, 64, 256]
    for off in ("0", ""):
        monkeypatch.setenv("DIFFPURE_ATTN_RECOMPUTE", off)
        assert not ops.attention_recompute_wanted(64)
    monkeypatch.delenv("DIFFPURE_ATTN_RECOMPUTE")
    assert not ops.attention_recompute_wanted(64)


def guided(heads, precision):
    from diffpure_amd import guided_unet as pg
    g = load_golden("guided_small.pt")
    cfg = pg.parse_config(dict(g["cfg"], num_head_channels=-1, num_heads=heads))
    return pg.GuidedUNet(cfg, DEV, precision).load_state_dict(synth_state_dict(pg.param_shapes(cfg), 7)), g["x"], g["t"].float()


def wide_ncsnpp(precision):
    from diffpure_amd import ncsnpp as pn
    g = load_golden("ncsnpp_full.pt")
    model = dict(g["cfg"]["model"], nf=256, num_res_blocks=1)              # its attention level: one head of 512 channels
    cfg = pn.parse_config(dict(g["cfg"], model=model))
    return pn.NCSNpp(cfg, DEV, precision).load_state_dict(synth_state_dict(pn.param_shapes(cfg), 7)), g["x"], g["labels"]


@pytest.mark.gpu
@pytest.mark.parametrize("precision", ["f32", "f16sr"])
@pytest.mark.parametrize("net", [lambda p: guided(64, p), wide_ncsnpp], ids=["heads_of_4", "head_of_512"])
def test_layers_that_it_does_not_take_keep_the_stored_form(net, precision, monkeypatch):
    """the same gradient, bit for bit, as without the switch"""
    from test_gpu_grad import nhwc
    net, x, lab = net(precision)
    u = torch.randn(x.shape, generator=torch.Generator().manual_seed(1))
    res = []
    for on in ("0", "1"):
        monkeypatch.setenv("DIFFPURE_ATTN_RECOMPUTE", on)
        tape = []
        net.forward(nhwc(x).to(DEV), lab.to(DEV), tape=tape)
        res.append(net.vjp(tape, nhwc(u).to(DEV)).cpu())
    assert torch.isfinite(res[0]).all() and res[0].abs().max() > 0 and torch.equal(*res)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["f16", "bf16"])
def test_fp32_gradients_are_the_16_bit_ones_before_their_last_rounding(dtype):
    """every form of a launch (own and shared columns, packed heads, ranges, masks): the same sums, so rounding them gives the other call's bits; and fp32 views of
    one tensor, whose surroundings stay as they were"""
    from diffpure_amd import ops
    from test_gpu_attention_lse import SHAPES, lens_of, make
    for n, (b, tq, tk, hq, hkv, d, causal, ql, kl, layout) in enumerate(SHAPES):
        q, k, v, dout = make(dtype, b, tq, tk, hq, hkv, d, layout, seed=n)
        ql, kl = (None if x is None else lens_of(*x) for x in (ql, kl))
        out, lse = ops.attention_lse(q, k, v, None, causal, ql, kl)
        want = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl)
        bufs = [torch.full((t.shape[0], t.shape[1], t.shape[2], d + 8), 7.0, device=DEV) for t in (q, k, v)]
        got = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl, grads=tuple(t[..., 4:4 + d] for t in bufs))
        for name, a, w, t in zip(("dq", "dk", "dv"), got, want, bufs):
            assert a.dtype == torch.float32 and torch.equal(a.to(dtype), w), (n, name)
            assert (t[..., :4] == 7).all() and (t[..., 4 + d:] == 7).all(), (n, name)


@pytest.mark.gpu
def test_fp32_gradients_beyond_fp16():
    """fp16 operands whose gradients pass 65504, and a dS that does: finite in fp32, and their rounding to fp16 is the fp16 call's (infinite where they do not fit)"""
    from diffpure_amd import ops
    from test_gpu_attention_range import FORMS, expected, inputs
    from test_gpu_attention_lse import Ref, close
    for form in FORMS:
        q, k, v, dout, causal = inputs(form, (6e4, 300.0))
        ref = Ref(q, k, v, None, causal, None, None)
        res, tol = expected(ref, dout)
        q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
        out, lse = ops.attention_lse(q, k, v, None, causal)
        got = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, grads=tuple(torch.empty(t.shape, device=DEV) for t in (q, k, v)))
        assert max(r.abs().max() for r in res) > 1e5
        for name, g, r, t in zip(("dq", "dk", "dv"), got, res, tol):
            close(g, r, t, name)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -30, 2.0 ** -12, 1.0, 2.0 ** 14, 2.0 ** 60], ids=lambda s: f"{s:.0e}")
@pytest.mark.parametrize("layout", ["legacy", "split"])
def test_recompute_from_an_fp16_tape_at_every_size_of_the_cotangent(size, layout):
    """1024 tokens, heads of 64, an fp32 cotangent of elements that fp16 holds times a power of two: within the tolerances of fp16 operands without a last rounding of the
    results to fp16 (that is in fp32: 2^-23 of them), each scaled by the power.  (dQ and dK of such rows are 1e-2 of the cotangent and below.)"""
    from diffpure_amd import ops
    from test_gpu_attention_lse import Ref, close
    b, t, h, d = 2, 1024, 2, 64
    g = torch.Generator().manual_seed(43)
    qkv, dout = torch.randn(b, t, 3 * h * d, generator=g).half(), torch.randn(b, t, h, d, generator=g).clamp(-3.9, 3.9).half()
    q, k, v = qkv.view(b, t, h, 3, d).unbind(3) if layout == "legacy" else qkv.view(b, t, 3, h, d).unbind(2)
    ref = Ref(q, k, v, None, False, None, None)
    res, tol = ref.bwd(dout, None)
    got = ops.attention_recompute_bwd(qkv.cuda(), (dout.float() * size).view(b, t, h * d).cuda(), h, layout)
    assert got.dtype == torch.float32
    got = got.view(b, t, h, 3, d).unbind(3) if layout == "legacy" else got.view(b, t, 3, h, d).unbind(2)
    for name, a, r, w in zip(("dq", "dk", "dv"), got, res, tol):
        w = w - ref.u * r.abs() * (1 + 2 * ref.u) - 2.0 ** -25 + 2.0 ** -23 * r.abs()
        close(a.double().cpu() / size, r, w, name)


@pytest.mark.gpu
def test_recompute_scales_each_sample_by_itself():
    """a sample's gradient keeps its bits whatever the other's cotangent, 0 stays 0, and one that is not finite stays visible"""
    from diffpure_amd import ops
    b, t, h, d = 2, 100, 2, 64
    qkv, dout = torch.randn(b, t, 3 * h * d, device=DEV).half(), torch.randn(b, t, h * d, device=DEV)
    want = ops.attention_recompute_bwd(qkv, dout, h, "split")
    for fill in (0.0, 1e-30, 1e30, float("nan"), float("inf")):
        do = dout.clone()
        do[1] = fill
        got = ops.attention_recompute_bwd(qkv, do, h, "split")
        assert torch.equal(got[0], want[0]), fill
        assert (got[1] == 0).all() if fill == 0 else torch.isfinite(got[1]).all() == (abs(fill) < 1e38), fill


@pytest.mark.gpu
def test_recompute_in_a_graph():
    """captured and replayed, with other work between: the reductions and the scaling follow the inputs"""
    from diffpure_amd import ops
    b, t, h, d = 2, 256, 2, 64
    qkv, dout = torch.randn(b, t, 3 * h * d, device=DEV).half(), torch.randn(b, t, h * d, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.attention_recompute_bwd(qkv, dout, h, "split")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = ops.attention_recompute_bwd(qkv, dout, h, "split")
    for i in range(4):
        dout.copy_(torch.randn(b, t, h * d, device=DEV) * 10.0 ** (3 - 2 * i))
        graph.replay()
        want = ops.attention_recompute_bwd(qkv, dout, h, "split")
        torch.cuda.synchronize()
        assert torch.equal(res, want), i


@pytest.mark.gpu
def test_refusals_of_fp32_gradients():
    from diffpure_amd import ops
    from diffpure_amd._lib import DiffpureHipError
    q = torch.randn(1, 8, 2, 16, device=DEV).half()
    k, v, dout = q.clone(), q.clone(), q.clone()
    out, lse = ops.attention_lse(q, k, v)
    f = [torch.empty(q.shape, device=DEV) for _ in range(3)]
    half = [torch.empty_like(q) for _ in range(3)]
    for grads in ((f[0], half[1], f[2]), (half[0], f[1], half[2]), (f[0], f[1], half[2]), (f[0], f[1], f[2].double())):
        with pytest.raises(DiffpureHipError, match="expected"):
            ops.attention_lse_bwd(dout, q, k, v, out, lse, grads=grads)
    wide = torch.empty(1, 8, 2, 17, device=DEV)
    with pytest.raises(DiffpureHipError, match="strides"):
        ops.attention_lse_bwd(dout, q, k, v, out, lse, grads=(wide[..., :16], f[1], f[2]))


@pytest.mark.gpu
def test_sample_scale_is_a_factor_of_the_gradients():
    """powers of two: the bits of the unscaled call times the factor, in every form of a launch and for fp32 operands too; what else it is is refused"""
    from diffpure_amd import ops
    from diffpure_amd._lib import DiffpureHipError
    from test_gpu_attention_lse import SHAPES, lens_of, make
    for dtype in (torch.float16, torch.float32):
        for n, (b, tq, tk, hq, hkv, d, causal, ql, kl, layout) in enumerate(SHAPES):
            q, k, v, dout = make(dtype, b, tq, tk, hq, hkv, d, layout, seed=n)
            ql, kl = (None if x is None else lens_of(*x) for x in (ql, kl))
            out, lse = ops.attention_lse(q, k, v, None, causal, ql, kl)
            factor = torch.tensor([2.0 ** (11 * i - 20) for i in range(b)], device=DEV)        # (made on the host: the GPU's pow(2, 24) is 16777215)
            grads = lambda: tuple(torch.empty(t.shape, device=DEV) for t in (q, k, v))
            want = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl, grads=grads())
            got = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl, grads=grads(), sample_scale=factor)
            for a, w in zip(got, want):
                assert torch.equal(a, w * factor.view(b, 1, 1, 1)), (dtype, n)
    q = torch.randn(2, 8, 2, 16, device=DEV).half()
    k, v, dout = q.clone(), q.clone(), q.clone()
    out, lse = ops.attention_lse(q, k, v)
    f = [torch.empty(q.shape, device=DEV) for _ in range(3)]
    for bad in (torch.ones(3, device=DEV), torch.ones(2, device=DEV, dtype=torch.float64), torch.ones(2), torch.ones(2, 1, device=DEV), torch.ones(4, device=DEV)[::2], 2.0):
        with pytest.raises(DiffpureHipError, match="sample_scale"):
            ops.attention_lse_bwd(dout, q, k, v, out, lse, grads=f, sample_scale=bad)
    with pytest.raises(DiffpureHipError, match="sample_scale"):
        ops.attention_lse_bwd(dout, q, k, v, out, lse, sample_scale=torch.ones(2, device=DEV))
    with pytest.raises(DiffpureHipError, match="sample_scale"):                       # on what the call writes
        ops.attention_lse_bwd(dout, q, k, v, out, lse, grads=f, sample_scale=f[1].view(-1)[:2])
