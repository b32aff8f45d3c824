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
