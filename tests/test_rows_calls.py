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


# ------------------------------------------------------------------ a residual written in place over another input
@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 5])
def test_norm_in_place_refuses_weights_and_gates_inside_the_residual(rows):
    """Rows are worked on by blocks of their own, in no order: one would read a weight that another has written over."""
    from omni_infer_amd import hip_ops as ops
    H = 64
    d = norm_inputs(rows, H, BF16, seed=1)
    buf = torch.ones(rows + 1, H, dtype=BF16, device="cuda")
    res, inside, behind = buf[:rows], buf[0], buf[rows]
    for key in ("post_weight", "pre_weight", "gate"):
        with pytest.raises(ValueError, match="overlaps"):
            ops.sandwich_norm(**{**d, "residual": res, key: inside}, post_eps=1e-6, pre_eps=1e-6, inplace_residual=True)
        with pytest.raises(ValueError, match="overlaps"):
            ops.sandwich_norm(**{**d, "residual": res, key: buf.view(-1)[(rows - 1) * H + 8:rows * H + 8]}, post_eps=1e-6, pre_eps=1e-6,
                              inplace_residual=True)
        buf.fill_(1)
        want = ops.sandwich_norm(**{**d, "residual": res.clone(), key: behind.clone()}, post_eps=1e-6, pre_eps=1e-6)
        got = ops.sandwich_norm(**{**d, "residual": res, key: behind}, post_eps=1e-6, pre_eps=1e-6, inplace_residual=True)
        assert torch.equal(got[0], want[0]) and torch.equal(res, want[1]) and bool((behind == 1).all())
        ops.sandwich_norm(**{**d, "residual": res, key: inside}, post_eps=1e-6, pre_eps=1e-6)     # not in place: fine


def test_where_rows_share_memory():
    from omni_infer_amd.hip_ops import _overlap
    buf = torch.zeros(8, 32)
    left, right, row = buf[:, :16], buf[:, 16:], buf.view(-1)
    assert not _overlap(left, right) and not _overlap(right, left) and _overlap(left, buf[:, 15:20]) and _overlap(buf[:, 8:], left)
    one = lambda at, n: row[at:at + n].view(1, -1)  # noqa: E731
    for at, n, shared in ((0, 16, True), (16, 16, False), (48, 16, False), (48, 17, True), (47, 4, True), (40, 8, True), (240, 16, False),
                          (16, 48, True), (8, 16, True)):
        assert _overlap(left, one(at, n)) == shared and _overlap(one(at, n), left) == shared, (at, n)
    assert not _overlap(one(0, 16), one(16, 16)) and _overlap(one(0, 17), one(16, 16)) and not _overlap(left, torch.zeros(8, 32))
    assert _overlap(buf.view(16, 16)[1:4], left)     # other pitches: taken for shared
    assert not _overlap(left[:0], left)
