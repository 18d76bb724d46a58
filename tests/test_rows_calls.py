"""Calls of the sandwich norm and of the SwiGLU of rows beside the tests of their formulas."""
import pytest
import torch

from tests.test_rows import BF16, FP16, FP32, norm_inputs


# ------------------------------------------------------------------ one order of operations for every kind of gate
@pytest.mark.gpu
@pytest.mark.parametrize("dt", [FP32, BF16, FP16])
@pytest.mark.parametrize("T,H", [(1, 264), (37, 265), (600, 2056), (3, 8200)])
def test_norm_gives_the_same_bits_for_every_kind_of_gate(T, H, dt):
    """r' = residual + (residual_scale * gate) * t in that order: a gate per token or per channel is the full gate spread out."""
    from omni_infer_amd import hip_ops as ops
    d = norm_inputs(T, H, dt, seed=T + H)
    g = torch.Generator().manual_seed(H)
    args = (d["x"], d["residual"], d["post_weight"], d["pre_weight"], 1e-6, 1e-5)
    for shape in ((T, 1), (H,)):
        gate = torch.randn(*shape, generator=g).to(dt).cuda()
        a = ops.sandwich_norm(*args, gate=gate, residual_scale=0.3, want_quant=True)
        b = ops.sandwich_norm(*args, gate=gate.expand(T, H).contiguous(), residual_scale=0.3, want_quant=True)
        assert all(torch.equal(u, v) for u, v in zip(a, b)), shape
    one = torch.ones(T, H, dtype=dt, device="cuda")
    a, b = (ops.sandwich_norm(*args, gate=v, residual_scale=0.3, want_quant=True) for v in (None, one))
    assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_norm_rounds_in_the_stated_order():
    """In fp32 t is what comes out over a residual of zeros, so the residual can be redone on the host to the last bit."""
    from omni_infer_amd import hip_ops as ops
    T, H, c = 50, 1000, 0.3
    d = norm_inputs(T, H, FP32, seed=7)
    w = (d["post_weight"], d["pre_weight"], 1e-6, 1e-6)
    t = ops.sandwich_norm(d["x"], torch.zeros_like(d["x"]), *w)[1].cpu()
    g = torch.Generator().manual_seed(8)
    for shape in ((T, 1), (H,), (T, H)):
        gate = torch.randn(*shape, generator=g)
        r = ops.sandwich_norm(d["x"], d["residual"], *w, gate=gate.cuda(), residual_scale=c)[1].cpu()
        assert torch.equal(r, d["residual"].cpu() + (torch.tensor(c) * gate) * t), shape
