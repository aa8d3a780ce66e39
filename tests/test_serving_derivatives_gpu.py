"""The serving operators have no derivatives: what asks for one is refused, in reverse and in forward mode."""
import pytest
import torch
import torch.autograd.forward_ad as forward

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def calls(ops):
    """(name, call of a tensor) for every tensor of 16-bit values that a call reads."""
    z = lambda *s: torch.zeros(*s, dtype=torch.float16, device=DEV)  # noqa: E731
    q, x = ops.mx4_quantize(z(32, 64)), z(2, 64)
    wr, w1, w2 = z(4, 64), z(4, 32, 64), z(4, 64, 32)
    plan = ops.MoeLayerPlan((wr, None), w1, w2)
    return [("quantize", x, ops.mx4_quantize), ("linear", x, lambda t: ops.mx4_linear(t, q)), ("bias", z(32), lambda t: ops.mx4_linear(x, q, t)),
            ("log probs", x, lambda t: ops.token_log_probs(t)), ("layer", x, plan.forward), ("layer, 70 tokens", z(70, 64), plan.forward),
            ("router", wr, lambda t: ops.MoeLayerPlan((t, None), w1, w2)), ("w1", w1, lambda t: ops.MoeLayerPlan((wr, None), t, w2)),
            ("b2", z(4, 64), lambda t: ops.MoeLayerPlan((wr, None), w1, w2, None, t))]


def test_tangents_and_gradients_are_refused(ops):
    for name, t, call in calls(ops):
        call(t)
        with pytest.raises(ops.NNRuntimeException):
            call(t.clone().requires_grad_())
        with torch.no_grad():
            call(t.clone().requires_grad_())
        with forward.dual_level():
            call(t)
            dual = forward.make_dual(t, torch.ones_like(t))
            for mode in (torch.enable_grad(), torch.no_grad()):
                with mode, pytest.raises(ops.NNRuntimeException):
                    call(dual)
            call(forward.unpack_dual(dual).primal)


def test_transforms_end_in_an_error(ops):
    for name, t, call in calls(ops)[:6]:
        def f(v):
            out = call(v)
            return out.dequantize(torch.float32).sum() if name == "quantize" else out[-1].float().sum() if isinstance(out, tuple) else out.float().sum()
        for transform in (lambda: torch.func.jvp(f, (t,), (torch.ones_like(t),)), lambda: torch.func.grad(f)(t)):
            with pytest.raises(Exception):
                transform()
