"""Refusals of the C entry points of the log-sum-exp attention and of layer norm: every argument check answers before anything is launched (no GPU)."""
import ctypes as C

import pytest


def lib():
    from diffpure_amd import _lib
    return _lib.load()


PTR = 1 << 20          # never read: each call is refused


def attn_fwd(q=PTR, k=PTR, v=PTR, out=PTR, lse=PTR, strides=None, dtype=1, b=2, tq=8, tk=8, hq=2, hkv=2, d=16, scale=0.25, strides_null=False, work=None, nbytes=0):
    st = (C.c_longlong * 12)(*(strides or [h * t * d if i == 0 else (h * d if i == 1 else d) for h, t in ((hq, tq), (hkv, tk), (hkv, tk), (hq, tq)) for i in range(3)]))
    return lib().dp_attention_lse(q, k, v, None if strides_null else C.addressof(st), dtype, b, tq, tk, hq, hkv, d, None, None, scale, 0, out, lse, work, nbytes, None)


@pytest.mark.parametrize("kw,what", [
    (dict(q=0), b"q is null"), (dict(k=PTR + 8), b"k is null or not 16-byte"), (dict(out=0), b"out is null"), (dict(lse=0), b"lse"), (dict(strides_null=True), b"strides"),
    (dict(dtype=3), b"dtype"), (dict(dtype=-1), b"dtype"), (dict(b=0), b"positive"), (dict(tq=0), b"positive"), (dict(tk=-4), b"positive"), (dict(hkv=0), b"positive"),
    (dict(hq=3), b"multiple"), (dict(d=12), b"multiple of 8"), (dict(d=264), b"multiple of 8"), (dict(d=0), b"multiple of 8"), (dict(scale=0.0), b"scale"),
    (dict(scale=float("inf")), b"scale"), (dict(scale=float("nan")), b"scale"), (dict(tq=(1 << 30) + 1), b"tokens"), (dict(b=1 << 20, hq=1 << 12, hkv=1 << 12), b"too many"),
    (dict(strides=[256, 32, 16] * 3 + [0, 32, 16]), b"also positive"), (dict(strides=[256, 32, 12] + [256, 32, 16] * 3), b"multiples"),
    (dict(strides=[-256, 32, 16] + [256, 32, 16] * 3), b"multiples"), (dict(strides=[256, 1 << 24, 16] + [256, 32, 16] * 3), b"apart"),
    (dict(b=1, tq=1, tk=8000, hq=1, hkv=1), b"workspace"), (dict(b=1, tq=1, tk=8000, hq=1, hkv=1, work=PTR, nbytes=16), b"workspace"),
])
def test_attention_lse_refuses(kw, what):
    assert attn_fwd(**kw) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


def attn_bwd(work=PTR, nbytes=1 << 30, lse=PTR, dq=PTR, dout=PTR, dk_st=None):
    st = [256, 32, 16] * 8
    if dk_st:
        st[18:21] = dk_st
    st = (C.c_longlong * 24)(*st)
    return lib().dp_attention_lse_bwd(dout, PTR, PTR, PTR, PTR, lse, C.addressof(st), 1, 2, 8, 8, 2, 2, 16, None, None, 0.25, 0, dq, PTR, PTR, work, nbytes, None)


@pytest.mark.parametrize("kw,what", [(dict(work=0), b"workspace"), (dict(work=PTR + 4), b"workspace"), (dict(nbytes=16), b"workspace"), (dict(lse=0), b"lse"),
                                     (dict(dq=0), b"dq"), (dict(dout=PTR + 2), b"dout"), (dict(dk_st=[0, 32, 16]), b"dk")])
def test_attention_lse_bwd_refuses(kw, what):
    assert attn_bwd(**kw) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


@pytest.mark.parametrize("off,what", [(0, b"out overlaps q"), (2 * 8 * 2 * 16 * 2 - 16, b"out overlaps q"), (-16, b"out overlaps q"), (1 << 20, b"out overlaps k"), (2 << 20, b"out overlaps v")])
def test_attention_lse_refuses_outputs_on_inputs(off, what):
    q = 1 << 24
    assert attn_fwd(q=q, k=q + (1 << 20), v=q + (2 << 20), out=q + off) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


def test_attention_lse_columns_of_one_row_are_apart():
    """q and out as columns of rows of 128: 32 columns to the right they pass that check (and are refused for the next tensor), nearer or beyond the row's end not"""
    for tq, b in ((1, 2), (6, 1), (6, 2)):
        st = [128 * tq, 128, 16, 256, 32, 16, 256, 32, 16, 128 * tq, 128, 16]
        for col, what in ((0, b"q"), (16, b"q"), (24, b"q"), (112, b"q"), (32, b"k"), (96, b"k")):
            out = (1 << 24) + 2 * col
            assert attn_fwd(q=1 << 24, k=out, v=1 << 27, out=out, b=b, tq=tq, strides=st) != 0
            assert b"out overlaps " + what in lib().dp_last_error(), (tq, b, col, lib().dp_last_error())


@pytest.mark.parametrize("grads,what", [((0, 10, 11), b"dq overlaps q"), ((10, 0, 11), b"dk overlaps q"), ((10, 11, 2), b"dv overlaps v"), ((10, 4, 11), b"dk overlaps dout"),
                                        ((3, 10, 11), b"dq overlaps out"), ((10, 10, 11), b"one address"), ((10, 11, 11), b"one address"), ((11, 10, 11), b"one address")])
def test_attention_lse_bwd_refuses_gradients_on_inputs(grads, what):
    at = lambda i: (1 << 24) + (i << 20)                  # q, k, v, out, dout lie at 0 .. 4, lse at 5, the workspace at 6
    st = (C.c_longlong * 24)(*[256, 32, 16] * 8)
    assert lib().dp_attention_lse_bwd(at(4), at(0), at(1), at(2), at(3), at(5), C.addressof(st), 1, 2, 8, 8, 2, 2, 16, None, None, 0.25, 0, *map(at, grads), at(6), 1 << 30,
                                      None) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


def test_attention_workspace_sizes():
    fwd, bwd = lib().dp_attention_lse_workspace, lib().dp_attention_lse_bwd_workspace
    for ws in (fwd, bwd):
        assert ws(1, 0, 4, 4, 1, 1, 64) == 0 and ws(1, 1, 0, 4, 1, 1, 64) == 0 and ws(1, 1, 4, 4, 3, 2, 64) == 0 and ws(3, 1, 4, 4, 1, 1, 64) == 0 and ws(1, 1, 4, 4, 1, 1, 300) == 0
    assert fwd(1, 64, 1024, 1024, 8, 8, 64) == 0                       # the queries fill the chip
    assert fwd(2, 1, 1, 50000, 4, 1, 128) > 4 * 4 * 129                # a few rows over a long axis: partial results
    assert bwd(1, 2, 65, 65, 3, 3, 64) >= 2 * 2 * 3 * 128 * 4
    assert bwd(1, 64, 1 << 20, 8, 64, 64, 64) >= 2 * 64 * 64 * (1 << 20) * 4          # beyond 32 bits


@pytest.mark.parametrize("kw,what", [
    (dict(x=0), b"missing"), (dict(y=0), b"missing"), (dict(dt=3), b"dtype"), (dict(wt=2), b"weights are"), (dict(rows=0), b"rows of"), (dict(rows=-1), b"rows of"),
    (dict(c=0), b"rows of"), (dict(c=16385), b"rows of"), (dict(eps=-1.0), b"eps"), (dict(eps=float("inf")), b"eps"), (dict(xs=-1), b"pitch"), (dict(ys=63), b"pitch"),
])
def test_layer_norm_refuses(kw, what):
    a = dict(x=PTR, dt=1, rows=4, c=64, xs=64, wt=0, eps=1e-5, y=PTR, ys=64) | kw
    assert lib().dp_layer_norm(a["x"], a["dt"], a["rows"], a["c"], a["xs"], None, None, a["wt"], a["eps"], a["y"], a["ys"], None, None) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


@pytest.mark.parametrize("kw,what", [
    (dict(dy=0), b"missing"), (dict(stats=0), b"missing"), (dict(dx=0), b"missing"), (dict(dxs=63), b"pitch"), (dict(dys=-1), b"pitch"), (dict(work=0), b"workspace"),
    (dict(work=PTR + 2), b"workspace"), (dict(nbytes=8), b"workspace"), (dict(c=20000), b"rows of"),
])
def test_layer_norm_bwd_refuses(kw, what):
    a = dict(dy=PTR, dys=64, rows=4, c=64, stats=PTR, dx=PTR, dxs=64, work=PTR, nbytes=1 << 20) | kw
    assert lib().dp_layer_norm_bwd(a["dy"], a["dys"], PTR, 64, 1, a["rows"], a["c"], None, 0, a["stats"], None, 0, a["dx"], a["dxs"], PTR, PTR, a["work"], a["nbytes"], None) != 0
    assert what in lib().dp_last_error(), lib().dp_last_error()


def test_layer_norm_workspace_sizes():
    ws = lib().dp_layer_norm_bwd_workspace
    assert ws(0, 64, 0) == 0 and ws(5, 0, 0) == 0 and ws(5, 20000, 0) == 0
    assert ws(1, 64, 0) == 2 * 64 * 4
    assert ws(1 << 40, 16384, 1) == ws(1 << 20, 16384, 1)              # a persistent grid: bounded
