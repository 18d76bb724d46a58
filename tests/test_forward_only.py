"""The dense-block operators have no derivatives: a call that autograd would have to follow is refused, in either mode."""
import pytest
import torch
import torch.autograd.forward_ad as fwd


def _ask(t, *more):
    from omni_infer_amd import hip_ops as ops
    ops._forward_only("op", t, None, *more)


def test_reverse_mode():
    x, y = torch.ones(3), torch.ones(3, requires_grad=True)
    _ask(x)
    for a in ((y,), (x, y)):
        with pytest.raises(RuntimeError, match="no backward"):
            _ask(*a)
        with torch.no_grad():
            _ask(*a)


def test_forward_mode():
    x = torch.ones(3)
    with fwd.dual_level():
        d = fwd.make_dual(x, torch.ones(3))
        _ask(x)
        for a in ((d,), (x, d)):
            with pytest.raises(RuntimeError, match="tangent"):
                _ask(*a)
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):   # tangents flow there all the same
                _ask(*a)
        _ask(x, torch.ones(3, dtype=torch.int32), fwd.unpack_dual(d).primal)
    with pytest.raises(RuntimeError, match="tangent"):
        torch.func.jvp(lambda v: (_ask(v), v)[1], (x,), (torch.ones(3),))
    _ask(x)


@pytest.mark.gpu
def test_the_operators_refuse_tangents():
    from omni_infer_amd import hip_ops as ops
    x = torch.randn(4, 64, device="cuda").to(torch.bfloat16)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    a, b = torch.zeros(2, 8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 64, 8, device="cuda", dtype=torch.bfloat16)
    plan = ops.adapter_plan(torch.zeros(4, dtype=torch.int32, device="cuda"), 2)
    calls = (lambda v: ops.npu_swiglu(v), lambda v: ops.swiglu_quant(v, want_quant=True),
             lambda v: ops.sandwich_norm(v, x, w, w, 1e-6, 1e-6), lambda v: ops.sandwich_norm(x, v, w, w, 1e-6, 1e-6),
             lambda v: ops.sandwich_norm(x, x, w, w, 1e-6, 1e-6, gate=v), lambda v: ops.adapter_linear(v, x, a, b, plan),
             lambda v: ops.adapter_linear(x, v, a, b, plan), lambda v: ops.adapter_linear(x, x.clone(), a, b, plan, out=v))
    for call in calls:
        call(x.clone())
        with fwd.dual_level(), pytest.raises(RuntimeError, match="tangent"):
            call(fwd.make_dual(x.clone(), torch.ones_like(x)))
