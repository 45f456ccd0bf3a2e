"""Calls of the residual-trunk operators that torch cannot follow are refused, not answered with a constant: forward-mode tangents and
tracing.  An empty batch reaches the autograd nodes without a GPU."""
import pytest
import torch
import torch.autograd.forward_ad as fw

from scpair_amd import _lib


def calls(x, W, b):
    """name, argument that carries the tangent, call"""
    T = _lib.trunk()
    norm = lambda h, *rest: T.residual_norm(x, h, *rest, 2, 1, 0, 0, 0, 1.0, 1e-5, False)
    none = [None] * 6
    return [("linear8", "x", lambda: T.linear8(x, W, b, False)), ("linear8", "W", lambda: T.linear8(x, W, b, False)),
            ("linear8", "b", lambda: T.linear8(x, W, b, False)), ("act8", "x", lambda: T.act8(x, 0, 0.0)),
            ("norm", "x", lambda: norm(x, *none)), ("norm", "h", lambda: norm(x + 0, *none)),
            ("norm", "b", lambda: norm(x.detach().clone(), None, None, b, None, None, None))]


@pytest.mark.parametrize("tracked", [False, True])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", range(7))
def test_forward_mode_derivatives_are_refused(which, grad, tracked):
    leaf = lambda *shape: torch.zeros(*shape).requires_grad_(tracked)
    with fw.dual_level(), torch.set_grad_enabled(grad):
        x, W, b = leaf(0, 8), leaf(8, 8), leaf(8)
        dual = lambda t: fw.make_dual(t, torch.zeros_like(t))
        _, arg, _ = calls(x, W, b)[which]
        x, W, b = (dual(x) if arg in ("x", "h") else x), (dual(W) if arg == "W" else W), (dual(b) if arg == "b" else b)
        with pytest.raises(RuntimeError, match="forward-mode derivatives are not implemented"):
            calls(x, W, b)[which][2]()


@pytest.mark.parametrize("tracked", [False, True])
def test_tracing_is_refused(tracked):
    W, b = torch.zeros(8, 8), torch.zeros(8)
    for which in (0, 3, 4):
        x = torch.zeros(0, 8).requires_grad_(tracked)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(lambda v: calls(v, W, b)[which][2](), (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(lambda v: _lib.trunk().pack8(v), (torch.zeros(0, 8),), check_trace=False)


def test_plain_calls_still_run():
    x, W, b = torch.zeros(0, 8, requires_grad=True), torch.zeros(8, 8, requires_grad=True), torch.zeros(8)
    for which in (0, 4, 6):
        out = calls(x, W, b)[which][2]()
        assert out.requires_grad if which == 0 else out[1].requires_grad


def test_linear8_module_takes_the_arguments_of_its_base():
    import scpair_amd as S
    layer = S.HipLinear8(8, 3)
    for args in ((), (False,), (True,)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            layer(torch.zeros(2, 8), *args)
