"""Scores that are not finite, inside the lengths, in attention_lse and attention_lse_bwd: a row that meets one is not finite in the results either - in
every form of a launch (waves with columns of their own, waves that share columns, ranges of keys that are joined) - and every other row is as if it
were not there.  A row is 0 with a log-sum-exp of -inf only where the lengths and the causal diagonal leave it no key."""
import math

import pytest
import torch

from test_gpu_attention_lse import Ref, close, lens_of, make

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
# b, tq, tk, hq, hkv, d, causal: more blocks than the chip takes at once; shared columns; ranges (heads packed, and a diagonal over one range's end)
FORMS = [(9, 33, 70, 32, 32, 64, False), (2, 97, 97, 40, 40, 128, True), (1, 40, 300, 2, 2, 40, False), (2, 1, 3001, 8, 2, 64, False),
         (2, 3, 2500, 6, 2, 128, True), (1, 2, 1500, 2, 2, 256, False)]
FORM_IDS = ["own", "own_causal", "shared", "packed_ranges", "causal_ranges", "wide_ranges"]


def splits(dtype, b, tq, tk, hq, hkv, d):
    from diffpure_amd import _lib
    return _lib.load().dp_attention_lse_workspace({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype], b, tq, tk, hq, hkv, d) > 0


def seen(b, tq, tk, causal):
    i, j = torch.arange(tq)[:, None], torch.arange(tk)[None, :]
    return (j <= i + tk - tq if causal else torch.ones(tq, tk, dtype=torch.bool)).expand(b, tq, tk)


def check(got, lse, ref, bad):
    """bad [B, Hq, Tq]: rows that must not be finite; the others within the tolerances of the definition"""
    got, lse = got.detach().double().cpu().transpose(1, 2), lse.detach().double().cpu()
    assert torch.isnan(got[bad]).all(), "a row that met a non-finite score came out finite"
    assert not torch.isfinite(lse[bad]).any(), "its log-sum-exp came out finite"
    close(got[~bad], ref.o[~bad], ref.tout[~bad], "out")
    close(lse[~bad], ref.lse[~bad], ref.eps[~bad], "lse")


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("where", ["key", "query"])
def test_nan_in_a_key_or_a_query(dtype, form, where):
    from diffpure_amd import ops
    b, tq, tk, hq, hkv, d, causal = form
    q, k, v, dout = make(dtype, b, tq, tk, hq, hkv, d, seed=17)
    ref = Ref(q, k, v, None, causal, None, None)
    group, bad = hq // hkv, torch.zeros(b, hq, tq, dtype=torch.bool)
    if where == "key":
        at = tk // 2 if not causal else tk - 2
        k[b - 1, at, hkv - 1, d - 3] = float("nan")
        bad[b - 1, (hkv - 1) * group:] = seen(b, tq, tk, causal)[0, :, at]
    else:
        q[b - 1, tq // 2, hq - 1, 5] = float("nan")
        bad[b - 1, hq - 1, tq // 2] = True
    out, lse = ops.attention_lse(q, k, v, None, causal)
    check(out, lse, ref, bad)
    if "ranges" in FORM_IDS[FORMS.index(form)]:
        assert splits(dtype, b, tq, tk, hq, hkv, d), "this form no longer cuts the keys: choose another"


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("form", FORMS, ids=FORM_IDS)
def test_scores_beyond_the_range(dtype, form):
    """one key's score is +inf (finite inputs whose product overflows; fp16, whose products cannot: an infinite input): NaN.  One key's is -inf: it has weight 0 and the
    others theirs.  Every score of a row is -inf: 0 / 0, NaN, and log 0 = -inf - not the 0 of a row without keys."""
    from diffpure_amd import ops
    b, tq, tk, hq, hkv, d, causal = form
    big = math.inf if dtype == torch.float16 else 1e30
    q, k, v, _ = make(dtype, b, tq, tk, hq, hkv, d, seed=19)
    q[..., 0], k[..., 0] = 1.0, 0.0
    if big != math.inf:
        q[..., 0] = big
    group, at = hq // hkv, tk - 2
    vis = seen(b, tq, tk, causal)[0, :, at]
    for sign in (1, -1):
        kk = k.clone()
        kk[0, at, 0, 0] = sign * big
        out, lse = ops.attention_lse(q, kk, v, None, causal)
        bad = torch.zeros(b, hq, tq, dtype=torch.bool)
        if sign > 0:
            bad[0, :group] = vis
            check(out, lse, Ref(q, k, v, None, causal, None, None), bad)
        else:                                                # the definition with this key's score at about -100: exp(-100) is nothing beside the others
            z = k.clone()
            z[0, at, 0, 0] = -100 / abs(q[0, 0, 0, 0].item()) * d ** 0.5
            check(out, lse, Ref(q, z, v, None, causal, None, None), bad)
    if dtype != torch.float16:
        kk = k.clone()
        kk[0, :, 0, 0] = -big
        out, lse = ops.attention_lse(q, kk, v, None, causal)
        some = seen(b, tq, tk, causal)[0].any(1)
        assert torch.isnan(out[0, some.to(out.device), :group]).all()
        assert (lse[0, :group] == -math.inf).all()


def test_rows_without_a_key_stay_zero():
    """lengths and the diagonal, one form with ranges: 0 and -inf, also beside rows that are NaN"""
    from diffpure_amd import ops
    for dtype in TYPES:
        for b, tq, tk, ql, kl in ((4, 100, 100, (100, 1, 64, 37), (60, 1, 0, 80)), (3, 40, 2500, (40, 0, 3), (20, 2500, 1))):
            q, k, v, _ = make(dtype, b, tq, tk, 4, 2, 64, seed=23)
            k[0, 3, 0] = float("nan")
            out, lse = ops.attention_lse(q, k, v, None, True, lens_of(*ql), lens_of(*kl))
            for i, (n, m) in enumerate(zip(ql, kl)):
                t = torch.arange(tq)
                none = ((t >= n) | (t + m - n < 0)).cuda()
                assert (out[i, none] == 0).all() and (lse[i][:, none] == -math.inf).all()
            met = ((torch.arange(tq) < ql[0]) & (torch.arange(tq) + kl[0] - ql[0] >= 3)).cuda()
            assert torch.isnan(out[0, met, :2]).all() and torch.isfinite(out[0, :, 2:]).all()


BACK = FORMS + [(1, 3001, 3, 4, 2, 64, False), (2, 1500, 40, 2, 1, 128, True), (9, 33, 70, 32, 32, 256, False)]


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("form", BACK, ids=FORM_IDS + ["few_keys", "few_keys_causal", "wide_heads"])
@pytest.mark.parametrize("what", ["statistics", "query"])
def test_gradients_of_a_row_that_is_nan(dtype, form, what):
    """One row of one head is NaN - its log-sum-exp alone (scores, out and dout finite), or as the forward pass leaves it for a NaN query: its dq, and dk and dv of every
    key it sees, are NaN, not the 0 of a row without keys.  Other heads of the sample and other samples do not notice."""
    from diffpure_amd import ops
    b, tq, tk, hq, hkv, d, causal = form
    q, k, v, dout = make(dtype, b, tq, tk, hq, hkv, d, seed=29)
    ref, group = Ref(q, k, v, None, causal, None, None), hq // hkv
    i, h, s = tq - 1, hq - 1, b - 1                                  # the last row of the last head sees a key under a diagonal too
    if what == "query":
        q[s, i, h, 5] = float("nan")
    out, lse = ops.attention_lse(q, k, v, None, causal)
    if what == "statistics":
        lse[s, h, i] = float("nan")
    dq, dk, dv = ops.attention_lse_bwd(dout, q, k, v, out, lse, None, causal)
    assert torch.isnan(dq[s, i, h]).all(), "dq of the row"
    at = torch.arange(tk)[seen(b, tq, tk, causal)[0, i]].cuda()
    assert torch.isnan(dk[s, at, hkv - 1]).all() and torch.isnan(dv[s, at, hkv - 1]).all(), "dk and dv of the keys that it sees"
    (rq, rk, rv), (uq, uk, uv) = ref.bwd(dout, None)
    fq, fk = torch.ones(b, hq, dtype=torch.bool), torch.ones(b, hkv, dtype=torch.bool)
    fq[s, (hkv - 1) * group:] = False
    fk[s, hkv - 1] = False
    for name, g, r, t, f in (("dq", dq, rq, uq, fq), ("dk", dk, rk, uk, fk), ("dv", dv, rv, uv, fk)):
        g, r, t = (x.detach().double().cpu().transpose(1, 2)[f] for x in (g, r, t))
        close(g, r, t, name)


def test_gradients_of_rows_without_a_key_stay_zero():
    """by the lengths or the diagonal: dq 0 and nothing added to dk and dv, whatever the log-sum-exp that is handed in says"""
    from diffpure_amd import ops
    for dtype in TYPES:
        q, k, v, dout = make(dtype, 3, 90, 40, 4, 2, 64, seed=31)
        ql, kl = lens_of(90, 50, 7), lens_of(40, 0, 12)
        ref = Ref(q, k, v, None, True, ql, kl)
        out, lse = ops.attention_lse(q, k, v, None, True, ql, kl)
        assert (lse == -math.inf).any()
        for fill in (-math.inf, math.inf, 3.0, float("nan")):
            given = torch.where(lse == -math.inf, torch.full_like(lse, fill), lse)
            grads = ops.attention_lse_bwd(dout, q, k, v, out, given, None, True, ql, kl)
            res, tol = ref.bwd(dout, ql)
            for name, g, r, t in zip(("dq", "dk", "dv"), grads, res, tol):
                close(g, r, t, name)
