"""attention_lse_bwd in fp16 over the whole range of cotangents and values: a dS that fits fp16 or not, a result that does.  Inputs are made on the CPU.

Tolerances are those of test_gpu_attention_lse.Ref; its term for fp16's smallest steps, 2^-31 per element of dS, stands for the factor 2^6 that P and dS are carried with.
Where 2^6 dS does not fit, the factor falls in steps of 2^12, so that the largest |dS| of a query or key is still carried as more than 2^3 (65504 / 2^12): half a step of 2^-24
is 2^-28 of that largest one, and |dS| <= max|dout_i| max|v_j|, the largest row norms."""
import math

import pytest
import torch

from test_gpu_attention_lse import Ref, close, lens_of

pytestmark = pytest.mark.gpu

# b, tq, tk, hq, hkv, d, causal: heads of 64 (dK and dV together) with columns of their own and shared ones; 128 and 256 (apart); shared heads; ranges
FORMS = {"own": (8, 130, 130, 40, 40, 64, False), "shared": (1, 70, 90, 2, 2, 64, False), "causal": (2, 100, 100, 4, 2, 128, True), "wide": (1, 150, 150, 1, 1, 256, False),
         "odd": (3, 65, 61, 6, 2, 40, True), "few_keys": (1, 801, 24, 4, 2, 64, False), "few_queries": (1, 5, 1500, 2, 2, 96, False)}
# largest dout, size of v
SIZES = [(66.0, 1.0), (400.0, 1.0), (1e3, 30.0), (2e4, 1.0), (3.0, 1e4), (2e-3, 1.0), (2e-5, 1.0), (1.0, 1e-4), (50.0, 1e-3)]


def inputs(form, size, seed=41):
    b, tq, tk, hq, hkv, d, causal = FORMS[form]
    g = torch.Generator().manual_seed(seed)
    q, k, v, dout = (torch.randn(b, t, h, d, generator=g) for t, h in ((tq, hq), (tk, hkv), (tk, hkv), (tq, hq)))
    return q.half(), k.half(), (v * size[1]).half(), (dout * (size[0] / dout.abs().max())).half(), causal


def expected(ref, dout, ql=None):
    res, tol = ref.bwd(dout, ql)
    norms = (ref.do.norm(dim=3).amax() * ref.v.norm(dim=3).amax()).item()
    step = abs(ref.scale) * 2.0 ** -28 * norms
    tol[0] = tol[0] + ref.back(step * ref.keep.double() @ ref.k.abs())
    tol[1] = tol[1] + ref.fold(step * ref.keep.double().transpose(2, 3) @ ref.q.abs())
    return res, tol


@pytest.mark.parametrize("size", SIZES, ids=[f"dout{a:g}_v{c:g}" for a, c in SIZES])
@pytest.mark.parametrize("form", FORMS)
def test_float16_gradients_at_every_size(form, size):
    from diffpure_amd import ops
    q, k, v, dout, causal = inputs(form, size)
    ref = Ref(q, k, v, None, causal, None, None)
    res, tol = expected(ref, dout)
    assert all(r.abs().max() < 65000 for r in res), "the results themselves have to fit"
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    out, lse = ops.attention_lse(q, k, v, None, causal)
    for name, g, r, t in zip(("dq", "dk", "dv"), ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal), res, tol):
        close(g, r, t, name)


def test_two_keys_by_hand():
    """two keys of weight 1/2, dout 66 in 64 channels, values 0 and 1: dP = 0 and 4224, dS = -+1056, dq = scale * 1056 = 132"""
    from diffpure_amd import ops
    k = torch.tensor([0.0, 1.0], device="cuda").half().view(1, 2, 1, 1).expand(1, 2, 1, 64)
    q, dout = torch.zeros(1, 1, 1, 64, device="cuda", dtype=torch.float16), torch.full((1, 1, 1, 64), 66.0, device="cuda", dtype=torch.float16)
    out, lse = ops.attention_lse(q, k.contiguous(), k.contiguous())
    dq, dk, dv = ops.attention_lse_bwd(dout, q, k.contiguous(), k.contiguous(), out, lse)
    assert ((dq.float() - 132).abs() <= 132 * 2.0 ** -10).all() and (dk == 0).all() and ((dv.float() - 33).abs() <= 33 * 2.0 ** -10).all()


def test_samples_and_heads_do_not_meet():
    """one sample's cotangent, and the rows behind the lengths, may be anything: the other samples' gradients keep their bits"""
    from diffpure_amd import ops
    q, k, v, dout, causal = inputs("causal", (1.0, 1.0))
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    ql, kl = lens_of(100, 77), lens_of(100, 80)
    out, lse = ops.attention_lse(q, k, v, None, causal, ql, kl)
    want = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl)
    for fill in (3e4, 1e-6, 0.0, math.inf, math.nan):
        do, vv = dout.clone(), v.clone()
        do[0], do[1, 77:], vv[1, 80:] = fill, 6e4, math.inf
        got = ops.attention_lse_bwd(do, q, k, vv, out, lse, None, causal, ql, kl)
        assert all(torch.equal(a[1], c[1]) for a, c in zip(got, want)), fill
        if fill == 0:
            assert all((a[0] == 0).all() for a in got)


def test_rows_that_are_not_finite_do_not_choose_the_factor():
    """an infinite dout in one row (its own gradients are lost) leaves dq of the others within the tolerances of theirs"""
    from diffpure_amd import ops
    q, k, v, dout, causal = inputs("shared", (400.0, 1.0))
    ref = Ref(q, k, v, None, causal, None, None)
    res, tol = expected(ref, dout)
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    dout[0, 9, 0, 3] = math.inf
    out, lse = ops.attention_lse(q, k, v)
    dq = ops.attention_lse_bwd(dout, q, k, v, out, lse)[0]
    assert not torch.isfinite(dq[0, 9, 0]).any()
    rest = torch.ones(70, dtype=torch.bool)
    rest[9] = False
    close(dq[:, rest.cuda(), 0], res[0][:, rest, 0], tol[0][:, rest, 0], "dq")
    close(dq[:, :, 1], res[0][:, :, 1], tol[0][:, :, 1], "dq of the other head")


@pytest.mark.parametrize("form", ["own", "causal", "wide", "few_keys"])
def test_lost_and_ordinary_calls_in_turn(form):
    """eager twice, on another stream, and replayed from two graphs: ordinary cotangents, ones whose dS overflow, and NaN follow one another in the same buffers; every
    result has the bits of the eager call"""
    from diffpure_amd import ops
    q, k, v, dout, causal = inputs(form, (1.0, 1.0))
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    b, tq, tk = q.shape[0], q.shape[1], k.shape[1]
    ql, kl = lens_of(*[tq - 3 * i for i in range(b)]), lens_of(*[tk - 2 * i for i in range(b)])
    out, lse = ops.attention_lse(q, k, v, None, causal, ql, kl)
    base = dout.clone()

    def step():
        return ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal, ql, kl)
    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = step()
        graphs.append((g, res))
    side = torch.cuda.Stream()
    for size in (1.0, 2e4, 1.0, math.nan, 2e4, 1e-3, 2e4):
        dout.copy_(base)
        if size == size:
            dout.copy_((base.float() * size).half())
        else:
            dout[0, 0, 0] = size
        for g, _ in graphs:
            g.replay()
        want = step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        if size == size:
            assert all(torch.isfinite(t).all() for t in want), size
        for res in [other] + [r for _, r in graphs]:
            assert all(torch.equal(a.view(torch.int16), c.view(torch.int16)) for a, c in zip(res, want)), size


@pytest.mark.parametrize("form", ["own", "shared", "causal", "wide", "odd", "few_queries"])
@pytest.mark.parametrize("channel", [0, 4, -1])
@pytest.mark.parametrize("size", [1.0, 2e4])
def test_a_key_that_is_infinite_in_one_channel(form, channel, size):
    """its score is -inf: weight 0, and 0 * inf in that channel of dq alone.  The other channels are what they are without the key, whether dS overflows on the way or not; dk and
    dv of every key too (0 of this one)"""
    from diffpure_amd import ops
    q, k, v, dout, causal = inputs(form, (size, 1.0))
    if channel == -1 and q.shape[3] not in (64, 96, 128, 256):
        pytest.skip("the last channels also fill a narrower head up to the kernel's width: its scores are NaN")
    channel %= q.shape[3]
    q[..., channel], k[..., channel] = 1.0, 0.0
    at = k.shape[1] // 2
    z = k.clone()
    z[:, at, :, channel] = -100 * q.shape[3] ** 0.5                  # the definition's: exp(-100) is nothing beside the others
    ref = Ref(q, z, v, None, causal, None, None)
    res, tol = expected(ref, dout)
    k[:, at, :, channel] = -math.inf
    q, k, v, dout = (t.cuda() for t in (q, k, v, dout))
    out, lse = ops.attention_lse(q, k, v, None, causal)
    close(out, ref.back(ref.o), ref.out_tol(), "out")
    dq, dk, dv = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal)
    rest = [c for c in range(q.shape[3]) if c != channel]
    close(dq[..., rest], res[0][..., rest], tol[0][..., rest], "dq")
    seen = (ref.keep[0, 0, :, at]).cuda()
    assert torch.isnan(dq[:, seen][..., channel]).all()
    close(dk, res[1], tol[1], "dk")
    close(dv, res[2], tol[2], "dv")
