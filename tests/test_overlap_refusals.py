"""Arguments that share memory, at the C entry points of the log-sum-exp attention and of layer norm: whatever a call writes lies apart from everything that it reads and from
everything else that it writes, or the call is refused before anything is launched (no GPU; every call here is refused).  Which of two views share a byte is known by
listing their bytes."""
import ctypes as C
import itertools
import random

import pytest

MB = 1 << 20


def lib():
    from diffpure_amd import _lib
    return _lib.load()


def error():
    return lib().dp_last_error().decode()


B, T, H, D = 2, 8, 2, 16
DENSE = [T * H * D, H * D, D]
AT = {n: (i + 16) * MB for i, n in enumerate(("q", "k", "v", "out", "dout", "lse", "work", "dq", "dk", "dv", "q_lens", "kv_lens"))}


def bwd(f32=False, strides=None, **at):
    a = {n: at.pop(n, p) for n, p in AT.items()}
    st = {n: DENSE for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv")} | (strides or {})
    arr = (C.c_longlong * 24)(*[x for n in ("q", "k", "v", "out", "dout", "dq", "dk", "dv") for x in st[n]])
    fn = lib().dp_attention_lse_bwd_f32 if f32 else lib().dp_attention_lse_bwd
    need = lib().dp_attention_lse_bwd_workspace(1, B, T, T, H, H, D)
    assert fn(a["dout"], a["q"], a["k"], a["v"], a["out"], a["lse"], C.addressof(arr), 1, B, T, T, H, H, D, a["q_lens"], a["kv_lens"], 0.25, 0, a["dq"], a["dk"],
              a["dv"], *([None] if f32 else []), a["work"], need, None) != 0
    return error()


@pytest.mark.parametrize("written,other", [(w, o) for w in ("dq", "dk", "dv") for o in ("q", "k", "v", "out", "dout", "lse", "q_lens", "kv_lens")])
def test_a_gradient_on_an_input(written, other):
    size = {"lse": B * H * T * 4, "q_lens": B * 4, "kv_lens": B * 4}.get(other, B * T * H * D * 2)
    for off in {0, (size - 1) // 16 * 16, -(B * T * H * D * 2 - 16)}:
        assert bwd(**{written: AT[other] + off}).endswith(f"{written} overlaps {other}"), error()


@pytest.mark.parametrize("first,second", [("dq", "dk"), ("dq", "dv"), ("dk", "dv")])
@pytest.mark.parametrize("f32", [False, True])
def test_two_gradients(first, second, f32):
    size = B * T * H * D * (4 if f32 else 2)
    assert "one address" in bwd(f32, **{second: AT[first]})
    for off in (16, size - 16, -16, 16 - size):
        e = bwd(f32, **{second: AT[first] + off})
        assert "overlaps" in e and first in e and second in e, e


def test_fp32_gradients_cover_twice_the_bytes():
    end = B * T * H * D * 2                               # where a 16-bit one ends
    assert "dk" in bwd(True, dk=AT["dq"] + end) and "overlaps" in error()
    assert bwd(True, dq=AT["q"] - end).endswith("dq overlaps q"), error()


@pytest.mark.parametrize("other", ["q", "k", "v", "out", "dout", "lse", "dq", "dk", "dv", "q_lens", "kv_lens"])
def test_the_workspace_on_anything(other):
    e = bwd(work=AT[other])
    assert ("work" in e and other in e), e


@pytest.mark.parametrize("strides", [[T * H * D, H * D, 8], [T * H * D, 24, 16], [128, 32, 16], [8, 32, 16], [T * 16, 16, 16]])
def test_rows_of_a_gradient_that_overlap_one_another(strides):
    for name in ("dq", "dk", "dv"):
        assert bwd(strides={name: strides}).endswith(f"the rows of {name} overlap"), error()


def fwd(strides=None, work_bytes=0, tk=T, **at):
    a = {n: at.get(n, AT[n]) for n in ("q", "k", "v", "out", "lse", "work", "q_lens", "kv_lens")}
    st = {"q": DENSE, "k": [tk * H * D, H * D, D], "v": [tk * H * D, H * D, D], "out": DENSE} | (strides or {})
    arr = (C.c_longlong * 12)(*[x for n in ("q", "k", "v", "out") for x in st[n]])
    assert lib().dp_attention_lse(a["q"], a["k"], a["v"], C.addressof(arr), 1, B, T, tk, H, H, D, a["q_lens"], a["kv_lens"], 0.25, 0, a["out"], a["lse"], a["work"], work_bytes,
                                  None) != 0
    return error()


@pytest.mark.parametrize("other", ["q", "k", "v", "q_lens", "kv_lens"])
@pytest.mark.parametrize("written", ["out", "lse"])
def test_forward_results_on_an_input(written, other):
    assert fwd(**{written: AT[other]}).endswith(f"{written} overlaps {other}"), error()


def test_forward_results_on_each_other_and_out_on_itself():
    assert "one address" in fwd(lse=AT["out"])
    assert "overlaps" in fwd(lse=AT["out"] + B * T * H * D * 2 - 16)
    assert fwd(strides={"out": [T * H * D, 24, 16]}).endswith("the rows of out overlap")


def test_forward_workspace_on_anything():
    tk = 8000
    need = lib().dp_attention_lse_workspace(1, B, T, tk, H, H, D)
    assert need > 0
    for other in ("q", "k", "v", "out", "lse", "q_lens", "kv_lens"):
        e = fwd(tk=tk, work=AT[other], work_bytes=need)
        assert "work" in e and other in e, e


def bytes_of(at, dims, strides, row):
    return {at + sum(i * s for i, s in zip(idx, strides)) + j for idx in itertools.product(*map(range, dims)) for j in range(0, row, 16)}


def views(rng):
    """two gradients as views of one tensor, or of two that meet: axes in any order, heads side by side or apart, padded rows"""
    d = 16                                                # 32 bytes
    b, t, h = rng.choice([1, 2, 3]), rng.choice([1, 2, 5]), rng.choice([1, 2, 3])
    order = rng.sample(range(3), 3)
    inner = rng.choice([32, 32, 48, 96, 128])
    strides, step = [0, 0, 0], inner
    for ax in order:
        strides[ax] = step
        step *= (b, t, h)[ax]
        if rng.random() < 0.3:
            step += rng.choice([16, 32, 64, 96])
    return (b, t, h), strides, d


def test_the_rule_against_listed_bytes():
    """dq and dk of random related layouts, and a dv that begins where dq does, which is compared last: it is what the call is refused for if dq and dk pass.  Whatever shares
    a byte is refused; what is refused without need is little."""
    rng, refused = random.Random(5), 0
    for _ in range(1500):
        dims, s1, d = views(rng)
        s2 = s1 if rng.random() < 0.7 else views(rng)[1]
        at1 = 64 * MB
        at2 = at1 + 16 * rng.choice([0, 1, 2, 3, 4, 6, 8, 12, 40, -2, -3, -6, 200])
        share = bytes_of(at1, dims, s1, 32) & bytes_of(at2, dims, s2, 32)
        own2 = len(bytes_of(at2, dims, s2, 32)) == 2 * dims[0] * dims[1] * dims[2]
        b, t, h = dims
        el = lambda s: [x // 2 for x in s]
        dense = [t * h * d, h * d, d]
        st = (C.c_longlong * 24)(*[x for s in (dense, dense, dense, dense, dense, el(s1), el(s2), dense) for x in s])
        need = lib().dp_attention_lse_bwd_workspace(1, b, t, t, h, h, d)
        # dv begins at dq's first byte: it is compared with dq and dk after they were with each other
        assert lib().dp_attention_lse_bwd(AT["dout"], AT["q"], AT["k"], AT["v"], AT["out"], AT["lse"], C.addressof(st), 1, b, t, t, h, h, d, None, None, 0.25, 0, at1, at2, at1,
                                          AT["work"], need, None) != 0
        e = error()
        about_two = ("dq" in e and "dk" in e) or "the rows of dk" in e
        if share or not own2:
            assert about_two, (dims, s1, s2, at2 - at1, e)
        elif about_two:
            refused += 1
            assert s1 != s2, ("equal layouts, apart, refused", dims, s1, at2 - at1, e)
        else:
            assert "dv" in e, e
    assert refused < 15, refused


def test_usual_views_pass():
    """heads x [q | k | v], [q | k | v] x heads, batch inside tokens, one padded buffer: dq and dk pass (and dv, which begins where dq does, is compared last and refused)"""
    d3 = 3 * H * D
    for s, step in (([T * d3, d3, 3 * D], D), ([T * d3, d3, D], H * D), ([d3, B * d3, D], H * D), ([T * 3 * H * (D + 8), 3 * H * (D + 8), 3 * (D + 8)], D + 8),
                    ([T * (d3 + 8), d3 + 8, 3 * D], D), ([T * (d3 + 8) + 16, d3 + 8, 3 * D], D), ([D, B * H * 3 * D, 3 * B * D], B * D)):
        e = bwd(strides={"dq": s, "dk": s, "dv": s}, dk=AT["dq"] + 2 * step, dv=AT["dq"])
        assert e.endswith("dq and dv begin at one address"), e
    # query heads and the key heads that they share in one projection's gradient: [dq of 4 heads | dk of 2 | dv of 2], and dv one head short of its place
    w = 8 * D
    for at, e in ((AT["dq"] + 2 * 6 * D, None), (AT["dq"] + 2 * 5 * D, "dk overlaps dv")):
        st = (C.c_longlong * 24)(*([T * 4 * D, 4 * D, D] + [T * 2 * D, 2 * D, D] * 2 + [T * 4 * D, 4 * D, D] * 2 + [T * w, w, D] * 3))
        dout = AT["dout"] if e else AT["work"]             # (on the workspace: refused for that if nothing before it is)
        assert lib().dp_attention_lse_bwd(dout, AT["q"], AT["k"], AT["v"], AT["out"], AT["lse"], C.addressof(st), 1, B, T, T, 4, 2, D, None, None, 0.25, 0, AT["dq"],
                                          AT["dq"] + 2 * 4 * D, at, AT["work"], MB, None) != 0
        assert error().endswith(e or "work overlaps dout"), error()
    # one sample, one token, heads apart
    st = (C.c_longlong * 24)(*([H * D, H * D, D] * 5 + [0, 0, 3 * D] * 3))
    assert lib().dp_attention_lse_bwd(AT["dout"], AT["q"], AT["k"], AT["v"], AT["out"], AT["lse"], C.addressof(st), 1, 1, 1, 1, H, H, D, None, None, 0.25, 0, AT["dq"],
                                      AT["dq"] + 2 * D, AT["dq"], AT["work"], MB, None) != 0
    assert error().endswith("dq and dv begin at one address"), error()


ROWS, WIDTH, PITCH = 6, 32, 40
LN = {n: (i + 64) * MB for i, n in enumerate(("x", "gamma", "beta", "y", "stats", "dy", "addend", "dx", "dgamma", "dbeta", "work"))}
SIZE = {n: ((ROWS - 1) * PITCH + WIDTH) * 2 for n in ("x", "y", "dy", "addend", "dx")} | {n: WIDTH * 4 for n in ("gamma", "beta", "dgamma", "dbeta")} | {"stats": ROWS * 8, "work": 8}


def ln(**at):
    a = LN | at
    assert lib().dp_layer_norm(a["x"], 1, ROWS, WIDTH, PITCH, a["gamma"], a["beta"], 0, 1e-6, a["y"], PITCH, a["stats"], None) != 0
    return error()


def ln_bwd(**at):
    a = LN | at
    need = lib().dp_layer_norm_bwd_workspace(ROWS, WIDTH, 1)
    assert lib().dp_layer_norm_bwd(a["dy"], PITCH, a["x"], PITCH, 1, ROWS, WIDTH, a["gamma"], 0, a["stats"], a["addend"], PITCH, a["dx"], PITCH, a["dgamma"], a["dbeta"], a["work"],
                                   need, None) != 0
    return error()


@pytest.mark.parametrize("call,written,other", [(ln, w, o) for w in ("y", "stats") for o in ("x", "gamma", "beta")] +
                         [(ln_bwd, w, o) for w in ("dx", "dgamma", "dbeta", "work") for o in ("dy", "x", "gamma", "stats", "addend")])
def test_layer_norm_results_on_an_input(call, written, other):
    """the whole, its last bytes, and its first (a row's part counts, the gap behind it does not: see below)"""
    for off in (0, SIZE[other] - 4, -(SIZE[written] - 4)):
        assert call(**{written: LN[other] + off}).endswith(f"{written} overlaps {other}"), (off, error())


@pytest.mark.parametrize("call,first,second", [(ln, "y", "stats")] + [(ln_bwd, *p) for p in itertools.combinations(("dx", "dgamma", "dbeta", "work"), 2)])
def test_two_results_of_layer_norm(call, first, second):
    assert "one address" in call(**{second: LN[first]}) and first in error() and second in error()
    e = call(**{second: LN[first] + SIZE[first] - 4})
    assert "overlaps" in e and first in e and second in e, e


def test_layer_norm_columns_of_one_row_are_apart():
    """two parts of rows of one pitch: y in the columns behind x's (then refused for the statistics, which are put onto x)"""
    a = LN | dict(y=LN["x"] + 2 * WIDTH, stats=LN["x"])
    for c, ok in ((WIDTH, True), (WIDTH - 1, False), (WIDTH + 1, True)):
        assert lib().dp_layer_norm(a["x"], 1, ROWS, WIDTH, 2 * WIDTH + 4, a["gamma"], a["beta"], 0, 1e-6, a["x"] + 2 * c, 2 * WIDTH + 4, a["stats"], None) != 0
        assert error().endswith("stats overlaps x" if ok else "y overlaps x"), (c, error())


def test_layer_norm_pitches_have_a_limit():
    far = (1 << 40) + 1
    for xs, ys in ((far, PITCH), (PITCH, far), (1 << 62, PITCH)):
        assert lib().dp_layer_norm(LN["x"], 1, ROWS, WIDTH, xs, None, None, 0, 1e-6, LN["y"], ys, None, None) != 0 and "pitch" in error()
    for i in range(4):
        p = [PITCH] * 4
        p[i] = far
        assert lib().dp_layer_norm_bwd(LN["dy"], p[0], LN["x"], p[1], 1, ROWS, WIDTH, None, 0, LN["stats"], LN["addend"], p[2], LN["dx"], p[3], None, None, None, 0, None) != 0
        assert "pitch" in error()
