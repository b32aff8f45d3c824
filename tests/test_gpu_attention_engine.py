"""DIFFPURE_ATTN_RECOMPUTE=1: the engines' attention backward on attention_lse / attention_lse_bwd (no stored probabilities)."""
import pytest
import torch

import refops  # noqa: F401
from conftest import load_golden
from diffpure_amd.synth import synth_state_dict
from test_gpu_grad import DEV, nchw, nhwc, relerr, rnd

pytestmark = pytest.mark.gpu


def ncsnpp(precision):
    from diffpure_amd import ncsnpp as pn
    from oracle import ncsnpp as on
    g = load_golden("ncsnpp_full.pt")
    cfg = pn.parse_config(g["cfg"])
    sd = synth_state_dict(pn.param_shapes(cfg), g["seed"])
    return pn.NCSNpp(cfg, DEV, precision).load_state_dict(sd), g["x"], g["labels"], lambda x: on.ncsnpp_forward(sd, on.parse_ncsnpp_config(g["cfg"]), x, g["labels"])


def guided(precision):
    from diffpure_amd import guided_unet as pg
    from oracle import guided_unet as og
    g = load_golden("guided_small.pt")
    cfg = pg.parse_config(g["cfg"])
    sd = synth_state_dict(pg.param_shapes(cfg), g["seed"])
    return pg.GuidedUNet(cfg, DEV, precision).load_state_dict(sd), g["x"], g["t"].float(), lambda x: og.guided_unet_forward(sd, og.parse_guided_config(g["cfg"]), x, g["t"])[:, :3]


def vjp(net, x, lab, u):
    tape = []
    net.forward(nhwc(x).to(DEV), lab.to(DEV), tape=tape)
    return nchw(net.vjp(tape, nhwc(u).to(DEV))).cpu()


@pytest.mark.parametrize("engine", [ncsnpp, guided])
def test_engine_gradient_without_stored_probabilities(engine, monkeypatch):
    """fp32: against the oracle's autograd within the bound of the stored form's own test.  f16sr: against the stored form of the same engine; the two differ by
    the fp16 roundings of the attention's gradient only - operands of five products and its result, 2^-11 each: 6 * 2^-11 of a gradient that
    the attention blocks make a part of."""
    for precision in ("f32", "f16sr"):
        net, x, lab, forward = engine(precision)
        u = rnd(*x.shape, seed=1)
        monkeypatch.setenv("DIFFPURE_ATTN_RECOMPUTE", "0")
        stored = vjp(net, x, lab, u)
        monkeypatch.setenv("DIFFPURE_ATTN_RECOMPUTE", "1")
        got = vjp(net, x, lab, u)
        assert not torch.equal(got, stored)              # the other path ran
        if precision == "f32":
            xr = x.clone().requires_grad_(True)
            (ref,) = torch.autograd.grad(forward(xr), xr, u)
            assert relerr(got, ref) < 2e-3, relerr(got, ref)
            assert relerr(got, stored) < 1e-4, relerr(got, stored)
        else:
            assert relerr(got, stored) < 6 * 2.0 ** -11, relerr(got, stored)


@pytest.mark.parametrize("layout", ["legacy", "split"])
def test_recomputing_backward_against_the_stored_one(layout):
    """ops level, fp32: attention_recompute_bwd against attention_bwd on the same qkv (both fp32 matrix products; sums of at most 196 terms of order one,
    reordered: 1e-5 of the largest element bounds the difference)"""
    from diffpure_amd import ops
    from diffpure_amd._lib import DiffpureHipError
    b, t, h, d = 3, 196, 4, 64          # (the stored form takes token counts that are multiples of 4)
    qkv, dout = (torch.randn(b, t, n * h * d, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n)) for n in (3, 1))
    _, probs = ops.attention(qkv, h, layout, probs_only=True)
    want = ops.attention_bwd(qkv, probs, dout, h, layout)
    got = ops.attention_recompute_bwd(qkv, dout, h, layout)
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()
    assert ops.attention_recompute_bwd(qkv.half(), dout, h, layout).dtype == torch.float32
    with pytest.raises(ValueError):
        ops.attention_recompute_bwd(qkv, dout, h, "other")
    with pytest.raises(DiffpureHipError):
        ops.attention_recompute_bwd(qkv.transpose(0, 1), dout, h, layout)
