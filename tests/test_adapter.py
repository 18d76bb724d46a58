"""Low-rank adapters beside a shared projection: refusals and launch shapes (CPU), the kernels against the formula in
64 bits (GPU).

Tolerance of an output, with p = |x|.|A|^T and v = x.A^T in 64 bits: an addition or product in fp32 is off by at most
2^-23 of the sums of magnitudes (the matrix cores may cut where they could round), the first product has H + 16 of
them, its result goes on with 16 bits (2^-16 of it; 22 in fp16, and no less than 2^-24 of the largest of its row), the
second product has 2r + 8, the result is rounded once (eps / 2)."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP16 = torch.bfloat16, torch.float16


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
    w = (ctypes.c_int32 * 5)(64, 64, 64, 64, 64)

    def call(x=p, dtype=0, ldx=64, base=p, ldb=64, a=p, b=p, scale=p, src=p, off=p, T=4, n=2, H=64, r=16, S=1, widths=w,
             out=p, ldo=64, ws=p, ws_bytes=1 << 30):
        return lib.omni_adapter_linear(x, dtype, ldx, base, ldb, a, b, scale, src, off, T, n, H, r, S, widths, out, ldo, ws,
                                       ws_bytes, None)

    assert call(dtype=1) == -1 and b"bf16" in lib.omni_moe_last_error()
    for bad in (dict(T=-1), dict(n=0), dict(H=0), dict(r=0), dict(S=0)):
        assert call(**bad) == -1
    assert call(S=5) == -2 and call(widths=None) == -1
    assert call(widths=(ctypes.c_int32 * 1)(0)) == -1
    assert call(widths=(ctypes.c_int32 * 1)(60)) == -2 and b"multiple of 8" in lib.omni_moe_last_error()
    assert call(H=60) == -2 and call(r=12) == -2 and call(r=264) == -2 and call(n=257) == -2
    assert call(T=(1 << 24) + 1) == -2
    assert call(T=1 << 24, widths=(ctypes.c_int32 * 1)(1 << 20), ldb=1 << 20, ldo=1 << 20) == -2    # more blocks than a grid holds
    assert call(ldx=56) == -1 and call(ldb=56) == -1 and call(ldo=56) == -1
    for null in ("x", "base", "a", "b", "src", "off", "out"):
        assert call(**{null: None}) == -1
    assert call(x=p + 8) == -1 and b"misaligned" in lib.omni_moe_last_error()
    assert call(ldx=68) == -1 and call(src=p + 2) == -1
    assert call(ldo=72) == -1                                    # out is base with another stride
    assert call(r=128, ws_bytes=8) == -3 and call(r=128, ws=None) == -3
    assert call(T=0, x=None, ws=None) == 0                       # nothing to do
    assert lib.omni_adapter_linear_workspace_bytes(0, 2, 64, 128, 1, 64) == 0
    assert lib.omni_adapter_linear_workspace_bytes(4, 2, 64, 128, 2, 64) >= 4 * 256 * 4


def test_cpu_tensors_are_refused():
    from omni_infer_amd import hip_ops as ops
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.adapter_plan(torch.zeros(4, dtype=torch.int32), 2)
    z = torch.zeros(4, 8, dtype=BF16)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.adapter_linear(z, z, z.view(1, 4, 8), z.view(1, 8, 4), None)


def test_launch_shape_holds_every_spread_of_tokens(tmp_path):
    """The host's bound on row blocks against spreads of the tokens over the adapters, under the sanitizers."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    exe = str(tmp_path / "adapter_plan_test")
    subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    os.path.join(ROOT, "tests", "host", "adapter_plan_test.cpp"), "-o", exe], check=True)
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr


# ------------------------------------------------------------------ GPU
def make(T, n, r, H, widths, dtype, seed=0, none=0.2, dev="cuda"):
    g = torch.Generator().manual_seed(seed)
    R, N = len(widths) * r, sum(widths)
    d = {"x": torch.randn(T, H, generator=g), "base": torch.randn(T, N, generator=g),
         "a": torch.randn(n, R, H, generator=g) * H ** -0.5, "b": torch.randn(n, N, r, generator=g) * r ** -0.5}
    d = {k: v.to(dtype).to(dev) for k, v in d.items()}
    d["scale"] = (0.5 + torch.rand(n, generator=g)).to(dev)
    ids = torch.randint(0, n, (T,), generator=g, dtype=torch.int32)
    ids[torch.rand(T, generator=g) < none] = -1
    d["ids"] = ids.to(dev)
    d["widths"] = list(widths)
    return d


def formula(d):
    """(value, bound) in 64 bits, adapter by adapter."""
    x, a, b = (d[k].double().cpu() for k in ("x", "a", "b"))
    out = d["base"].double().cpu()
    dt, r, H = d["x"].dtype, b.shape[2], x.shape[1]
    err = torch.zeros_like(out)
    eps16, floor = (2.0 ** -16, 0.0) if dt == BF16 else (2.0 ** -22, 2.0 ** -24)
    ids = d["ids"].cpu()
    for g in range(a.shape[0]):
        rows = (ids == g).nonzero().flatten()
        s = 1.0 if d["scale"] is None else float(d["scale"][g])
        n0 = 0
        for j, w in enumerate(d["widths"]):
            A, B = a[g, j * r:(j + 1) * r], b[g, n0:n0 + w]
            v, p = x[rows] @ A.T, x[rows].abs() @ A.abs().T
            off = 2.0 ** -23 * (H + 16) * p + eps16 * v.abs() + floor * v.abs().amax(1, keepdim=True)
            err[rows, n0:n0 + w] = s * (off @ B.abs().T + 2.0 ** -23 * (2 * r + 8) * (v.abs() @ B.abs().T))
            out[rows, n0:n0 + w] += s * (v @ B.T)
            n0 += w
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    return out, err * 1.01 + (torch.finfo(dt).eps / 2) * (out.abs() + err) + tiny


def check(got, d, what=""):
    want, bound = formula(d)
    off = (got.double().cpu() - want).abs()
    assert bool(torch.isfinite(got.double()).all()), what
    assert bool((off <= bound).all()), f"{what}: {float((off / bound).max())} times the bound"
    none = (d["ids"] < 0) | (d["ids"] >= d["a"].shape[0])
    assert torch.equal(got[none], d["base"][none]), "rows without an adapter"


def run(d, **kw):
    from omni_infer_amd import hip_ops as ops
    plan = ops.adapter_plan(d["ids"], d["a"].shape[0])
    return ops.adapter_linear(d["x"], d["base"], d["a"], d["b"], plan, d["scale"], slices=d["widths"], **kw)


CASES = [  # T, n, r, H, widths
    (1, 1, 8, 8, [8]),
    (1, 4, 16, 7168, [2048, 2048]),
    (2, 3, 8, 64, [16]),
    (3, 5, 40, 72, [24]),
    (15, 2, 16, 128, [64]),
    (16, 1, 16, 56, [64]),
    (17, 2, 24, 200, [72, 8, 200]),
    (64, 64, 16, 2048, [7168]),
    (65, 200, 8, 320, [136]),
    (333, 12, 24, 1992, [1048]),
    (130, 3, 256, 136, [264]),
    (40, 2, 128, 1024, [64, 64, 128, 72]),
    (1024, 3, 16, 264, [1000]),
    (1500, 3, 64, 520, [136, 136]),
    (2047, 2, 8, 64, [40]),
    (1100, 2, 128, 192, [328]),
    (1030, 1, 72, 4104, [64, 72]),
    (1300, 2, 256, 328, [200]),
    (1025, 3, 40, 4096, [128, 24]),
    (33, 2, 56, 136, [200]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,n,r,H,widths", CASES)
def test_against_the_formula(T, n, r, H, widths, dtype):
    d = make(T, n, r, H, widths, dtype, seed=T + r)
    got = run(d)
    check(got, d)
    assert torch.equal(got, run(d)), "two calls differ"
    out = d["base"].clone()
    d2 = dict(d, base=out)
    assert run(d2, out=out) is out
    assert torch.equal(out, got), "in place"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [0, 1, 20, 1200])
def test_spreads_of_the_tokens(T):
    """Nobody has an adapter, all have the same one, ids that name none of the adapters, no scale."""
    d = make(T, 6, 16, 136, [72], BF16, seed=T)
    for ids in (torch.full((T,), -1), torch.full((T,), 3), torch.full((T,), 6), torch.full((T,), 2 ** 31 - 1),
                torch.full((T,), 2 ** 33 + 1), torch.arange(T) % 2 * 5):
        d["ids"] = (ids if int(ids.abs().max() if T else 0) >= 2 ** 31 else ids.to(torch.int32)).cuda()
        for scale in (d["scale"], None):
            got = run(dict(d, scale=scale))
            if T:
                check(got, dict(d, scale=scale))
            else:
                assert got.shape == d["base"].shape


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 45, 1100])
def test_strides_and_what_lies_around_the_output(T):
    d = make(T, 4, 16, 264, [120, 64], FP16, seed=9)
    want = run(d)
    wide = torch.randn(T, 264 + 64, device="cuda").to(FP16)
    wide[:, 32:296] = d["x"]
    both = torch.full((T + 3, 2 * 184 + 16), 7.0, device="cuda", dtype=FP16)
    both[:T, :184] = d["base"]
    out = both[:T, 192:376]
    got = run(dict(d, x=wide[:, 32:296], base=both[:T, :184]), out=out)   # base and out side by side in one buffer
    assert got is out and torch.equal(out, want)
    assert torch.equal(both[:T, :184], d["base"]) and bool((both[T:] == 7).all()) and bool((both[:, 376:] == 7).all())
    assert bool((both[:, 184:192] == 7).all())
    # elements at odd places, transposed rows, more dimensions
    odd = torch.randn(T, 265, device="cuda").to(FP16)
    odd[:, 1:] = d["x"]
    assert torch.equal(run(dict(d, x=odd[:, 1:])), want)
    assert torch.equal(run(dict(d, base=d["base"].t().contiguous().t())), want)
    from omni_infer_amd import hip_ops as ops
    plan = ops.adapter_plan(d["ids"], 4)
    got = ops.adapter_linear(d["x"].view(T, 1, -1), d["base"].view(T, 1, -1), d["a"], d["b"], plan, d["scale"], [120, 64])
    assert got.shape == (T, 1, 184) and torch.equal(got.view(T, -1), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T", [20, 1200])
def test_values_that_are_not_finite_stay_in_their_rows(T, dtype):
    d = make(T, 4, 24, 136, [72], dtype, seed=3, none=0.0)
    want = run(d)
    d2 = dict(d, x=d["x"].clone(), a=d["a"].clone(), b=d["b"].clone())
    d2["x"][5, 7] = float("nan")
    d2["x"][9, 1] = float("inf")
    bad = int(d["ids"][2])
    d2["b"][bad] = float("nan")
    got = run(d2)
    touched = d["ids"] == bad
    touched[5] = touched[9] = True
    assert torch.equal(got[~touched], want[~touched])
    assert not bool(torch.isfinite(got[touched].float()).any())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [3, 1200])
def test_first_products_beyond_the_range_of_fp16(T):
    """x . A^T far above 65504 and far below the smallest fp16, brought back by B and by the scale."""
    d = make(T, 2, 16, 512, [64], FP16, seed=4)
    d["x"] = d["x"] * 2000
    d["a"] = torch.sign(d["a"].float()).to(FP16) * 500
    d["scale"] = torch.tensor([1e-6, 3e-7], device="cuda")
    check(run(d), d, "large")
    d["x"] = (d["x"].float() * 1e-10).to(FP16)      # fp16 subnormals
    d["a"] = (d["a"].float() / 500 * 2e-5).to(FP16)
    d["base"] = torch.zeros_like(d["base"])
    d["scale"] = torch.tensor([3e7, 1e7], device="cuda")
    check(run(d), d, "small")


@pytest.mark.gpu
def test_long_batches():
    """More than 2^31 bytes of rows: offsets past 32 bits."""
    T, H, N = 150000, 8192, 64
    x = torch.zeros(T, H, dtype=BF16, device="cuda")
    d = make(8, 2, 8, H, [N], BF16, seed=8)
    pos = torch.tensor([0, 1, 77777, 131071, 131072, 149990, 149998, 149999], device="cuda")
    x[pos] = d["x"]
    ids = torch.full((T,), -1, dtype=torch.int32, device="cuda")
    ids[pos] = d["ids"]
    base = torch.zeros(T, N, dtype=BF16, device="cuda")
    base[pos] = d["base"]
    got = run(dict(d, x=x, base=base, ids=ids))
    check(got[pos], d)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[pos] = False
    assert not bool(got[rest].any())


@pytest.mark.gpu
def test_captured_and_replayed_on_two_graphs():
    """Plan and product recorded twice into graphs of different sizes, replayed in turn with new inputs and eager calls
    in between."""
    from omni_infer_amd import hip_ops as ops
    made = []
    for T, seed in ((37, 1), (1200, 2)):
        d = make(T, 5, 16, 264, [72, 72], BF16, seed=seed)
        run(d)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(d)
        made.append((d, graph, got))
    for k in range(3):
        for d, graph, got in made:
            new = make(d["x"].shape[0], 5, 16, 264, [72, 72], BF16, seed=50 + k)
            for key in ("x", "base", "ids", "a", "b", "scale"):
                d[key].copy_(new[key])
            graph.replay()
        for d, graph, got in made:
            assert torch.equal(got, run(d))


@pytest.mark.gpu
def test_two_streams_at_once():
    d1, d2 = make(700, 5, 16, 2048, [512], BF16, seed=1), make(900, 3, 32, 1024, [768], BF16, seed=2)
    want1, want2 = run(d1), run(d2)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(s1):
            got.append((run(d1), want1))
        with torch.cuda.stream(s2):
            got.append((run(d2), want2))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in got)


@pytest.mark.gpu
def test_refusals():
    from omni_infer_amd import hip_ops as ops
    d = make(12, 3, 16, 64, [40, 24], BF16)
    plan = ops.adapter_plan(d["ids"], 3)
    call = lambda **kw: ops.adapter_linear(**{**dict(x=d["x"], base=d["base"], a=d["a"], b=d["b"], plan=plan,  # noqa: E731
                                                     scale=d["scale"], slices=[40, 24]), **kw})
    call()
    for bad in (dict(x=d["x"].float()), dict(b=d["b"].to(FP16)), dict(x=d["x"][:5]), dict(base=d["base"][:, :8]),
                dict(a=d["a"][:2]), dict(slices=[40, 25]), dict(slices=[64]), dict(slices=None), dict(scale=d["scale"][:2]),
                dict(scale=d["scale"].double()), dict(plan=ops.adapter_plan(d["ids"], 4)),
                dict(plan=ops.adapter_plan(d["ids"][:5], 3)), dict(a=d["a"].transpose(1, 2).contiguous().transpose(1, 2)),
                dict(out=d["base"][:, :8]), dict(out=d["base"].float())):
        with pytest.raises(ValueError):
            call(**bad)
    buf = torch.zeros(13, 64, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        call(base=buf[:12], out=buf[1:])
    with pytest.raises(ValueError, match="overlaps"):
        call(x=buf[:12], out=buf[:12])
    with pytest.raises(ValueError):
        call(out=torch.zeros(12, 65, dtype=BF16, device="cuda")[:, 1:])
    with pytest.raises(RuntimeError, match="multiple of 8"):
        e = make(4, 2, 8, 60, [8], BF16)
        run(e)
    e = make(12, 3, 128, 64, [40, 24], BF16)
    with pytest.raises(RuntimeError, match="workspace"):
        run(e, workspace=torch.zeros(16, dtype=torch.uint8, device="cuda"))
    assert torch.equal(run(e, workspace=torch.zeros(1 << 20, dtype=torch.uint8, device="cuda")), run(e))
    with pytest.raises(RuntimeError, match="no backward"):
        call(x=d["x"].clone().requires_grad_())
    with torch.no_grad():
        call(x=d["x"].clone().requires_grad_())
    with pytest.raises(ValueError):
        ops.adapter_plan(d["ids"].view(3, 4), 3)
    with pytest.raises(ValueError):
        ops.adapter_plan(d["ids"].float(), 3)
    with pytest.raises(ValueError):
        ops.adapter_plan(d["ids"], 0)
    with pytest.raises(RuntimeError):
        ops.adapter_plan(d["ids"], 257)
