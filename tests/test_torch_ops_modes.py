"""torch.ops.diffpure_hip.attention_lse / layer_norm below autograd: what a dispatch mode (tracing, fake tensors, counting) and forward-mode differentiation see (no GPU:
the kernels are answered by the mode)."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


def fw():
    import diffpure_amd.torch_ops  # noqa: F401
    return torch.ops.diffpure_hip


class Answer(TorchDispatchMode):
    """records this library's operators and answers them with tensors of the right shapes"""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        name = func.name()
        if not name.startswith("diffpure_hip::"):
            return func(*args, **(kwargs or {}))
        self.seen.append(name.split("::")[1])
        if name.endswith("attention_lse"):
            q = args[0]
            return torch.full_like(q, 2.0), torch.zeros(q.shape[0], q.shape[2], q.shape[1])
        if name.endswith("attention_lse_bwd"):
            return tuple(torch.full_like(t, 3.0 + i) for i, t in enumerate(args[1:4]))
        if name.endswith("layer_norm"):
            return torch.full_like(args[0], 2.0), torch.zeros(args[0].numel() // args[0].shape[-1], 2)
        assert name.endswith("layer_norm_bwd"), name
        c = args[1].shape[-1]
        return torch.full_like(args[1], 3.0), torch.full((c,), 4.0), torch.full((c,), 5.0)


def qkv(grad):
    return [torch.randn(2, 5, 3, 8, requires_grad=grad) for _ in range(3)]


@pytest.mark.parametrize("grad", [False, True])
def test_a_dispatch_mode_sees_attention(grad):
    q, k, v = qkv(grad)
    with Answer() as mode:
        out, lse = fw().attention_lse(q, k, v)
        assert mode.seen == ["attention_lse"] and (out == 2).all() and out.requires_grad == grad and not lse.requires_grad
        if grad:
            got = torch.autograd.grad(out.sum(), (q, k, v))
            assert mode.seen == ["attention_lse", "attention_lse_bwd"]
            assert [g.unique().item() for g in got] == [3.0, 4.0, 5.0]


@pytest.mark.parametrize("grad", [False, True])
def test_a_dispatch_mode_sees_layer_norm(grad):
    x, g, b = torch.randn(2, 5, 16, requires_grad=grad), torch.randn(16, requires_grad=grad), torch.randn(16, requires_grad=grad)
    with Answer() as mode:
        y, stats = fw().layer_norm(x, g, b, 1e-6)
        assert mode.seen == ["layer_norm"] and (y == 2).all() and y.requires_grad == grad and not stats.requires_grad
        if grad:
            got = torch.autograd.grad(y.sum(), (x, g, b))
            assert mode.seen == ["layer_norm", "layer_norm_bwd"]
            assert [t.unique().item() for t in got] == [3.0, 4.0, 5.0]


def test_optional_arguments_reach_the_mode():
    """what the caller gave, in the schema's order: scale, causal and lengths; eps; weights left out"""
    lens = torch.tensor([5, 2], dtype=torch.int32)
    calls = []

    class Args(Answer):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.name().startswith("diffpure_hip::"):
                calls.append((func.name().split("::")[1], args, kwargs or {}))
            return super().__torch_dispatch__(func, types, args, kwargs)

    for grad in (False, True):
        q, k, v = qkv(grad)
        x = torch.randn(4, 16, requires_grad=grad)
        with Args():
            out, _ = fw().attention_lse(q, k, v, 0.25, True, lens, lens)
            y, _ = fw().layer_norm(x, None, None, 1e-3)
            if grad:
                (out.sum() + y.sum()).backward()
    att = [a for n, a, _ in calls if n == "attention_lse"]
    assert len(att) == 2 and all(a[3] == 0.25 and a[4] is True and torch.equal(a[5], lens) and torch.equal(a[6], lens) for a in att)
    ln = [a for n, a, _ in calls if n == "layer_norm"]
    assert len(ln) == 2 and all((a[1] if len(a) > 1 else None) is None and a[3] == 1e-3 for a in ln)
    (bwd,) = [a for n, a, _ in calls if n == "attention_lse_bwd"]
    assert bwd[6] == 0.25 and bwd[7] is True and torch.equal(bwd[8], lens) and torch.equal(bwd[9], lens)
    (lb,) = [a for n, a, _ in calls if n == "layer_norm_bwd"]
    assert lb[2] is None and (lb[5] if len(lb) > 5 else True) is False          # no weights: their gradients are not formed


def test_a_fake_tensor_does_not_reach_the_kernels():
    """no shape rule is registered for these operators (nor for the older ones): a fake tensor is refused, not handed to the library"""
    from torch._subclasses.fake_tensor import FakeTensorMode, UnsupportedOperatorException
    with FakeTensorMode():
        for grad in (False, True):
            q, k, v = qkv(grad)
            with pytest.raises((NotImplementedError, UnsupportedOperatorException)):
                fw().attention_lse(q, k, v)
            with pytest.raises((NotImplementedError, UnsupportedOperatorException)):
                fw().layer_norm(torch.randn(4, 16, requires_grad=grad), None, None, 1e-6)


def test_without_a_mode_a_cpu_tensor_is_refused():
    for grad in (False, True):
        with pytest.raises((RuntimeError, NotImplementedError), match="GPU tensor|CPU"):
            fw().attention_lse(*qkv(grad))
        with pytest.raises((RuntimeError, NotImplementedError), match="GPU tensor|CPU"):
            fw().layer_norm(torch.randn(4, 16, requires_grad=grad))


@pytest.mark.parametrize("which", range(6))
@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused_not_lost(which, grad_mode):
    """a dual tensor in any place, without requires_grad: there is no formula for its tangent (nor has the older operators'), and the call says so"""
    from torch.autograd import forward_ad as fa
    a = qkv(False) + [torch.randn(2, 5, 16), torch.randn(16), torch.randn(16)]
    with fa.dual_level(), Answer(), torch.set_grad_enabled(grad_mode):
        a[which] = fa.make_dual(a[which], torch.ones_like(a[which]))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp|forward"):
            if which < 3:
                fw().attention_lse(*a[:3])
            else:
                fw().layer_norm(a[3], a[4], a[5], 1e-6)


def test_a_cotangent_is_handed_on_as_the_kernel_takes_it():
    """whatever its strides (autograd passes a view on as it is): expanded, transposed, beside a 16-byte border, tokens further apart than the kernel takes"""
    q = torch.randn(1, 3, 2, 8, requires_grad=True)
    k, v = torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8)
    wide = torch.zeros(3 * 4500000)                       # 18 MB between two tokens
    cases = [torch.ones(1).expand(1, 3, 2, 8), torch.randn(1, 3, 8, 2).transpose(2, 3), torch.randn(49)[1:].view(1, 3, 2, 8), torch.randn(1, 3, 2, 9)[..., :8],
             wide.as_strided((1, 3, 2, 8), (0, 4500000, 8, 1)), torch.randn(1, 2, 3, 8).transpose(1, 2), torch.randn(1, 1, 2, 8).expand(1, 3, 2, 8)]
    got = []

    class Look(Answer):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            if func.name().endswith("attention_lse_bwd"):
                got.append(args[0])
            return super().__torch_dispatch__(func, types, args, kwargs)

    for c in cases:
        with Look():
            torch.autograd.grad(fw().attention_lse(q, k, v)[0], q, c)
        g = got.pop()
        assert torch.equal(g, c)
        assert g.stride(3) == 1 and g.data_ptr() % 16 == 0 and all(g.stride(i) * 4 % 16 == 0 for i in range(3) if g.shape[i] > 1), g.stride()
        assert g.stride(1) * 4 <= 1 << 24, g.stride()
    for c in cases[5:]:                                   # what it takes is not copied
        with Look():
            torch.autograd.grad(fw().attention_lse(q, k, v)[0], q, c)
        assert got.pop().data_ptr() == c.data_ptr()
