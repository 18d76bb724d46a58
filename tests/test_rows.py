"""The sandwich norm and the SwiGLU of rows in memory: refusals (CPU), the kernels against the formulas in 64 bits (GPU).

Tolerances.  Sums of squares have no cancellation: a thread adds at most 64 squares, the rest is a tree, so a sum is
off by less than 100 * 2^-24 of itself, its root by half of that, and with the division, the products and eps a norm's
factor by less than 2^-17; what comes out is rounded once to its type (eps / 2).  The activation is off by a few units in
the last place of fp32: 2^-20."""
import ctypes
import os

import pytest
import torch

from oracle import moe_oracle as O

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
NORM, ACT = 2.0 ** -17, 2.0 ** -20


def half(dt):
    return torch.finfo(dt).eps / 2


def least(dt):  # half a step of the type's subnormals
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


# ------------------------------------------------------------------ CPU
@pytest.fixture(scope="module")
def lib():
    from omni_infer_amd import _lib
    if not os.path.exists(_lib.LIB_PATH):
        from omni_infer_amd import _build
        _build.build(verbose=False)
    return _lib.lib()


def test_refusals_of_the_library(lib):
    buf = ctypes.create_string_buffer(256)
    p = (ctypes.addressof(buf) + 63) // 64 * 64

    def norm(x=p, dtype=0, ldx=64, res=p, ldr=64, w1=p, w2=p, gate=None, mode=0, ldg=0, rows=2, H=64, out=p, ldo=64, y=p, q=None,
             scale=None):
        return lib.omni_sandwich_norm(x, dtype, ldx, res, ldr, w1, w2, gate, mode, ldg, rows, H, 1e-6, 1e-6, 1.0, out, ldo, y, q,
                                      scale, None)

    assert norm(dtype=3) == -1 and norm(rows=-1) == -1 and norm(H=0) == -1
    assert norm(ldx=63) == -1 and norm(ldr=63) == -1 and norm(ldo=63) == -1
    assert norm(mode=4) == -1 and norm(mode=1) == -1 and norm(gate=p) == -1
    assert norm(gate=p, mode=2, ldg=0) == -1 and norm(gate=p, mode=3, ldg=63) == -1
    for null in ("x", "res", "w1", "w2", "out"):
        assert norm(**{null: None}) == -1
    assert norm(q=p) == -1 and norm(scale=p) == -1
    assert norm(H=16392, ldx=16392, ldr=16392, ldo=16392) == -2 and norm(rows=1 << 22) == -2
    assert norm(x=p + 1) == -1 and norm(dtype=1, x=p + 2) == -1 and norm(q=p, scale=p + 2) == -1
    assert norm(rows=0, x=None) == 0

    def act(x=p, dtype=0, ld=128, rows=2, I=64, h=p, q=None, scale=None):
        return lib.omni_swiglu_quant(x, dtype, ld, rows, I, h, q, scale, None)

    assert act(dtype=3) == -1 and act(rows=-1) == -1 and act(I=0) == -1 and act(ld=127) == -1
    assert act(x=None) == -1 and act(h=None) == -1 and act(q=p) == -1 and act(scale=p) == -1
    assert act(I=32769, ld=65538) == -2 and act(rows=1 << 22) == -2
    assert act(x=p + 1) == -1 and act(dtype=1, x=p + 2) == -1
    assert act(rows=0, x=None) == 0


def test_cpu_tensors_are_refused():
    from omni_infer_amd import hip_ops as ops
    z, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.sandwich_norm(z, z, w, w, 1e-6, 1e-6)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.swiglu_quant(z)


# ------------------------------------------------------------------ the norm (GPU)
GATES = {"none": None, "channel": lambda T, H: (H,), "token": lambda T, H: (T, 1), "full": lambda T, H: (T, H)}


def norm_inputs(T, H, dt, gate="none", seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    d = {"x": rnd(T, H) * 2, "residual": rnd(T, H) * 3, "post_weight": 1 + 0.1 * rnd(H), "pre_weight": 1 + 0.1 * rnd(H)}
    if GATES[gate]:
        d["gate"] = rnd(*GATES[gate](T, H)) * 0.7
    return {k: v.to(dt).cuda() for k, v in d.items()}


def norm_formula(d, e1, e2, c):
    x, res, w1, w2 = (d[k].double().cpu() for k in ("x", "residual", "post_weight", "pre_weight"))
    gate = d["gate"].double().cpu() if "gate" in d else torch.ones(())
    cgt = float(torch.tensor(c, dtype=FP32)) * gate * (x / (x.square().mean(1, keepdim=True) + e1).sqrt() * w1)
    r = res + cgt
    f = 1 / (r.square().mean(1, keepdim=True) + e2).sqrt()
    dr = NORM * cgt.abs() + 2.0 ** -24 * r.abs()
    y = r * f * w2
    # the error of r goes into y directly and through the second norm's factor
    dy = dr * (f * w2).abs() + y.abs() * (NORM + dr.norm(dim=1, keepdim=True) / r.norm(dim=1, keepdim=True).clamp(min=1e-300))
    return r, dr, y, dy


def norm_check(d, got, e1, e2, c):
    y, r, q, s = got
    dt = d["x"].dtype
    wr, dr, wy, dy = norm_formula(d, e1, e2, c)
    for name, v, w, off in (("residual", r, wr, dr), ("y", y, wy, dy)):
        if v is not None:
            assert v.dtype == dt
            assert bool(((v.double().cpu() - w).abs() <= half(dt) * (w.abs() + off) + off + least(dt)).all()), name
    if q is not None and y is not None:
        wq, ws = O.dynamic_quant(y.cpu().float())
        assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)


SIZES = [(1, 1), (1, 7), (2, 8), (3, 9), (1, 7168), (5, 2047), (5, 2048), (4, 2049), (64, 7680), (3, 8192), (3, 8193),
         (2, 8200), (2, 16383), (2, 16384), (37, 130), (700, 264), (300, 7168)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,H", SIZES)
def test_norm_against_the_formula(T, H, dt):
    from omni_infer_amd import hip_ops as ops
    e1, e2, c = 1e-5, 1e-6, 0.7
    for gate in GATES:
        d = norm_inputs(T, H, dt, gate, seed=H)
        args = (d["x"], d["residual"], d["post_weight"], d["pre_weight"], e1, e2)
        got = ops.sandwich_norm(*args, gate=d.get("gate"), residual_scale=c, want_quant=True)
        norm_check(d, got, e1, e2, c)
        y, r, q, s = got
        # the forms with fewer outputs and in place give the same bits
        y2, r2, q2, s2 = ops.sandwich_norm(*args, gate=d.get("gate"), residual_scale=c)
        assert torch.equal(y, y2) and torch.equal(r, r2) and q2 is None and s2 is None
        kept = d["residual"].clone()
        y3, r3, q3, s3 = ops.sandwich_norm(d["x"], kept, *args[2:], gate=d.get("gate"), residual_scale=c, want_y=False,
                                           want_quant=True, inplace_residual=True)
        assert y3 is None and r3 is kept and torch.equal(kept, r) and torch.equal(q3, q) and torch.equal(s3, s)
        y4, r4, q4, _ = ops.sandwich_norm(*args, gate=d.get("gate"), residual_scale=c, want_y=False)
        assert y4 is None and q4 is None and torch.equal(r4, r)


@pytest.mark.gpu
@pytest.mark.parametrize("H", [264, 265])
def test_norm_strides(H):
    """Rows out of wider buffers, at odd places, gates with strides; what lies between the rows stays."""
    from omni_infer_amd import hip_ops as ops
    T, dt = 21, BF16
    d = norm_inputs(T, H, dt, "full", seed=2)
    args = dict(post_eps=1e-6, pre_eps=1e-6, residual_scale=0.3)
    want = ops.sandwich_norm(d["x"], d["residual"], d["post_weight"], d["pre_weight"], gate=d["gate"], **args)
    for pad, at in ((8, 8), (7, 3)):
        wide = {k: torch.full((T, H + pad + at), 5.0, dtype=dt, device="cuda") for k in ("x", "residual", "gate")}
        view = {k: v[:, at:at + H] for k, v in wide.items()}
        for k in view:
            view[k].copy_(d[k])
        got = ops.sandwich_norm(view["x"], view["residual"], d["post_weight"], d["pre_weight"], gate=view["gate"], **args)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        got = ops.sandwich_norm(view["x"], view["residual"], d["post_weight"], d["pre_weight"], gate=view["gate"],
                                inplace_residual=True, **args)
        assert torch.equal(got[0], want[0]) and torch.equal(view["residual"], want[1])
        assert bool((wide["residual"][:, :at] == 5).all()) and bool((wide["residual"][:, at + H:] == 5).all())
    tok = torch.randn(T, 3, device="cuda").to(dt)
    a = ops.sandwich_norm(d["x"], d["residual"], d["post_weight"], d["pre_weight"], gate=tok[:, 1:2], **args)
    b = ops.sandwich_norm(d["x"], d["residual"], d["post_weight"], d["pre_weight"], gate=tok[:, 1:2].expand(T, H), **args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a = ops.sandwich_norm(d["x"].view(3, 7, H), d["residual"].view(3, 7, H), d["post_weight"], d["pre_weight"],
                          gate=d["gate"].view(3, 7, H), want_quant=True, **args)
    assert a[0].shape == (3, 7, H) and a[2].shape == (3, 7, H) and a[3].shape == (3, 7)
    assert torch.equal(a[0].view(T, H), want[0])
    one = ops.sandwich_norm(d["x"][0], d["residual"][0], d["post_weight"], d["pre_weight"], gate=d["gate"][0], **args)
    assert one[0].shape == (H,) and torch.equal(one[0], want[0][0])
    same = d["x"].clone()   # the block's output is the residual itself
    got = ops.sandwich_norm(same, same, d["post_weight"], d["pre_weight"], inplace_residual=True, **args)
    ref = ops.sandwich_norm(d["x"], d["x"].clone(), d["post_weight"], d["pre_weight"], **args)
    assert torch.equal(same, ref[1]) and torch.equal(got[0], ref[0])


@pytest.mark.gpu
@pytest.mark.parametrize("H", [264, 265])
def test_norm_of_special_rows(H):
    """Rows of zeros, a residual that the block undoes, infinities and NaN in one row, sums beyond fp16."""
    from omni_infer_amd import hip_ops as ops
    d = norm_inputs(8, H, FP16, seed=5)
    d["x"][1] = 0
    d["residual"][1] = 0
    d["x"][2] = 0
    d["residual"][3, 4] = float("inf")
    d["x"][4, 0] = float("nan")
    d["residual"][5] = 60000.0
    y, r, q, s = ops.sandwich_norm(d["x"], d["residual"], d["post_weight"], d["pre_weight"], 1e-6, 1e-6, residual_scale=30000.0,
                                   want_quant=True)
    assert not bool(y[1].any()) and not bool(r[1].any()) and not bool(q[1].any()) and float(s[1]) == 0
    assert torch.equal(r[2], d["residual"][2])
    for row in (3, 4):
        assert not bool(torch.isfinite(s[row])) and not bool(q[row].any())
    assert bool(torch.isinf(r[5]).any()) and bool(torch.isfinite(y[5]).all())     # y goes by the unrounded sum
    ok = [0, 6, 7]
    fine = {k: (v[ok] if v.dim() == 2 else v) for k, v in d.items()}
    norm_check(fine, (y[ok], None, q[ok], s[ok]), 1e-6, 1e-6, 30000.0)
    # -residual + block: what is left is small against both
    x = torch.randn(4, H, device="cuda")
    w = torch.ones(H, device="cuda")
    t = ops.sandwich_norm(x, torch.zeros_like(x), w, w, 0.0, 1e-6)[1]
    r = ops.sandwich_norm(x, -t, w, w, 0.0, 1e-6)[1]
    assert float(r.abs().max()) <= NORM * float(t.abs().max())


@pytest.mark.gpu
def test_norm_refusals():
    from omni_infer_amd import hip_ops as ops
    d = norm_inputs(4, 64, BF16, "full")
    call = lambda **kw: ops.sandwich_norm(**{**dict(d, post_eps=1e-6, pre_eps=1e-6), **kw})  # noqa: E731
    call()
    for bad in (dict(x=d["x"].float()), dict(residual=d["residual"][:3]), dict(post_weight=d["post_weight"][:8]),
                dict(pre_weight=d["pre_weight"].to(FP16)), dict(gate=d["gate"][:3]), dict(gate=d["gate"][:1, :1]),
                dict(gate=d["gate"].float()), dict(x=d["x"].to(torch.int8)), dict(residual=d["residual"].view(2, 2, 64))):
        with pytest.raises(ValueError):
            call(**bad)
    with pytest.raises(ValueError, match="in place"):
        call(residual=d["residual"].t().contiguous().t(), inplace_residual=True)
    buf = torch.zeros(5, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        call(x=buf[1:], residual=buf[:4], inplace_residual=True)
    with pytest.raises(RuntimeError, match="16384"):
        big = norm_inputs(1, 16385, BF16)
        ops.sandwich_norm(**big, post_eps=1e-6, pre_eps=1e-6)
    with pytest.raises(RuntimeError, match="no backward"):
        call(post_weight=d["post_weight"].clone().requires_grad_())
    e = ops.sandwich_norm(d["x"][:0], d["residual"][:0], d["post_weight"], d["pre_weight"], 1e-6, 1e-6, want_quant=True)
    assert e[0].shape == (0, 64) and e[3].shape == (0,)


# ------------------------------------------------------------------ SwiGLU (GPU)
def swiglu_check(x, h, dt):
    I = x.shape[1] // 2
    g, u = x[:, :I].double().cpu(), x[:, I:].double().cpu()
    want = g * torch.sigmoid(g) * u
    # a value of at least the largest number plus half its step rounds to an infinity: 3e38 * 1.5 does in fp32
    over = want.abs() >= torch.finfo(dt).max * (1 + torch.finfo(dt).eps / 4)
    assert torch.equal(h.double().cpu()[over], torch.sign(want[over]) * float("inf"))
    off = torch.where(over, 0.0, (h.double().cpu() - want).abs())
    assert bool((off <= (ACT + half(dt)) * want.abs() + least(dt) + 2.0 ** -126 * u.abs()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [BF16, FP16, FP32])
@pytest.mark.parametrize("T,I", [(1, 1), (1, 7), (2, 8), (3, 9), (64, 2048), (5, 2047), (4, 2049), (3, 8192), (3, 8193), (2, 16392),
                                 (2, 32767), (2, 32768), (700, 136), (300, 1003)])
def test_swiglu_against_the_formula(T, I, dt):
    from omni_infer_amd import hip_ops as ops
    g = torch.Generator().manual_seed(I)
    x = (torch.randn(T, 2 * I, generator=g) * 3).to(dt).cuda()
    h, q, s = ops.swiglu_quant(x, want_quant=True)
    swiglu_check(x, h, dt)
    wq, ws = O.dynamic_quant(h.cpu().float())
    assert torch.equal(q.cpu(), wq) and torch.equal(s.cpu(), ws)
    assert torch.equal(ops.npu_swiglu(x), h)
    _, q2, s2 = ops.swiglu_quant(x, want_y=False, want_quant=True)
    assert torch.equal(q2, q) and torch.equal(s2, s)
    wide = torch.full((T, 2 * I + 5), 9.0, device="cuda", dtype=dt)
    wide[:, 3:2 * I + 3] = x
    assert torch.equal(ops.npu_swiglu(wide[:, 3:2 * I + 3]), h)
    assert torch.equal(ops.npu_swiglu(x.view(T, 1, 2 * I)), h.view(T, 1, I))
    assert torch.equal(ops.npu_swiglu(x.t().contiguous().t()), h)


@pytest.mark.gpu
def test_swiglu_of_special_values():
    from omni_infer_amd import hip_ops as ops
    inf, nan = float("inf"), float("nan")
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 79.0, -79.0, -81.0, -90.0, -103.0, -150.0, -300.0, -3e38, 88.0, 89.0, 1e4, 3e38])
    x = torch.cat([g, torch.full((16,), 1.5)]).view(1, 32).cuda()
    swiglu_check(x, ops.npu_swiglu(x), FP32)
    rows = torch.ones(5, 32, device="cuda")
    rows[0, 3], rows[1, 4], rows[2, 20], rows[3, 6] = inf, -inf, nan, nan
    h, q, s = ops.swiglu_quant(rows, want_quant=True)
    assert float(h[0, 3]) == inf and bool(torch.isnan(h[1, 4])) and bool(torch.isnan(h[2, 4])) and bool(torch.isnan(h[3, 6]))
    assert int(torch.isfinite(h).sum()) == 76
    assert not bool(torch.isfinite(s[:4]).any()) and not bool(q[:4].any()) and bool(torch.isfinite(s[4]))
    z, zq, zs = ops.swiglu_quant(torch.zeros(2, 32, device="cuda", dtype=BF16), want_quant=True)
    assert not bool(z.any()) and not bool(zq.any()) and not bool(zs.any())


@pytest.mark.gpu
def test_swiglu_refusals():
    from omni_infer_amd import hip_ops as ops
    with pytest.raises(ValueError):
        ops.swiglu_quant(torch.zeros(2, 7, device="cuda"))
    with pytest.raises(ValueError):
        ops.swiglu_quant(torch.zeros(2, 8, device="cuda", dtype=torch.int8))
    with pytest.raises(ValueError):
        ops.swiglu_quant(torch.zeros(2, 8, device="cuda"), want_y=False)
    with pytest.raises(RuntimeError, match="32768"):
        ops.swiglu_quant(torch.zeros(1, 2 * 32776, device="cuda"))
    with pytest.raises(RuntimeError, match="no backward"):
        ops.swiglu_quant(torch.zeros(2, 8, device="cuda", requires_grad=True))
    assert ops.npu_swiglu(torch.zeros(0, 8, device="cuda")).shape == (0, 4)


# ------------------------------------------------------------------ both, captured and on two streams (GPU)
@pytest.mark.gpu
def test_captured_replayed_and_beside_each_other():
    from omni_infer_amd import hip_ops as ops
    def both(d, gu):
        y, r, q, s = ops.sandwich_norm(d["x"], d["residual"], d["post_weight"], d["pre_weight"], 1e-6, 1e-6, gate=d["gate"],
                                       want_quant=True)
        return (y, r, q, s) + ops.swiglu_quant(gu, want_quant=True)

    made = []
    for T, H in ((5, 264), (300, 1001)):
        d, gu = norm_inputs(T, H, BF16, "channel", seed=T), torch.randn(T, 2 * H, device="cuda").to(BF16)
        both(d, gu)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = both(d, gu)
        made.append((d, gu, graph, got))
    for k in range(3):
        for d, gu, graph, _ in made:
            for v in (*d.values(), gu):
                v.copy_(torch.randn(v.shape, device="cuda"))
            graph.replay()
        for d, gu, _, got in made:
            assert all(torch.equal(a, b) for a, b in zip(got, both(d, gu)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    want = [both(d, gu) for d, gu, _, _ in made]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for s, (d, gu, _, _) in zip(streams, made):
            with torch.cuda.stream(s):
                got.append(both(d, gu))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % 2]))
