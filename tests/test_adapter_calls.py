"""Calls of the adapters beside the tests of their formula: slots that hold nothing, batches on other streams, every kernel the
dispatch can choose."""
import os
import re
import shutil
import subprocess

import pytest
import torch

from tests.test_adapter import BF16, FP16, ROOT, check, make, run

# tokens, adapters, rank, H, widths: one launch; two launches with 16-row blocks; with 128-row blocks
FORMS = [(20, 4, 24, 136, [72]), (65, 3, 128, 264, [136, 64]), (1200, 4, 40, 264, [72, 128])]


# ------------------------------------------------------------------ a scale of zero
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,n,r,H,widths", FORMS)
def test_a_scale_of_zero_adds_nothing(T, n, r, H, widths, dtype):
    """Rows of such an adapter are their base rows to the bit, whatever the rows and its matrices hold."""
    d = make(T, n, r, H, widths, dtype, seed=T)
    d["scale"][1], d["scale"][2] = 0.0, -0.0
    d["base"][::3] = -0.0
    want = run(d)
    off = (d["ids"] == 1) | (d["ids"] == 2)
    assert int(off.sum()) > 2
    assert torch.equal(want[off].view(torch.int16), d["base"][off].view(torch.int16))
    check(want, d)
    bad = dict(d, x=d["x"].clone(), a=d["a"].clone(), b=d["b"].clone(), base=d["base"].clone())
    rows = off.nonzero().flatten()
    bad["x"][rows[0], 3], bad["x"][rows[1], 0], bad["x"][rows[2]] = float("nan"), float("inf"), -float("inf")
    bad["a"][1], bad["b"][2] = float("nan"), float("inf")
    got = run(bad)
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    got = run(bad, out=bad["base"])
    assert torch.equal(got.view(torch.int16), want.view(torch.int16)), "in place"


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 1100])
def test_a_slot_that_holds_nothing(T):
    from omni_infer_amd.layers.adapters import AdapterBatch, AdapterSlots
    g = torch.Generator().manual_seed(T)
    slots = AdapterSlots(136, [72, 64], 3, 16, device="cuda")
    for slot in (0, 1):
        slots.set_adapter(slot, [torch.randn(16, 136, generator=g)] * 2, [torch.randn(72, 16, generator=g), torch.randn(64, 16, generator=g)])
    slots.clear(1)
    ids = torch.randint(-1, 3, (T,), generator=g, dtype=torch.int32)
    ids[:4] = torch.tensor([0, 1, 2, -1])
    x = torch.randn(T, 136, generator=g).to(BF16)
    x[1, 5], x[2, 0], x[3, 7] = float("inf"), float("nan"), float("inf")
    base = torch.randn(T, 136, generator=g).to(BF16).cuda()
    got = slots.add_to(base.clone(), x.cuda(), AdapterBatch(ids.cuda(), 3))
    held = ids.cuda() == 0
    assert torch.equal(got[~held], base[~held]) and not torch.equal(got[held], base[held])


# ------------------------------------------------------------------ a plan on another stream than its own
class _Recorded:
    def __init__(self):
        self.log = []

    def record_stream(self, s):
        self.log.append(("record", s.cuda_stream))


class _FakeStream:
    def __init__(self, handle, log):
        self.cuda_stream, self.log = handle, log

    def wait_stream(self, s):
        self.log.append(("wait", s))


@pytest.mark.parametrize("capturing", [False, True])
def test_a_plan_joins_the_stream_that_uses_it(capturing, monkeypatch):
    """The first use of a plan on another stream waits until the plan is made and holds its memory for that stream; a stream being
    captured cannot wait for what happened outside."""
    from omni_infer_amd import hip_ops as ops
    plan, buf = ops.AdapterPlan(), _Recorded()
    plan.buffer, plan.stream, plan.joined = buf, "its stream", {7}
    monkeypatch.setattr(ops, "_capturing", lambda device: capturing)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: _FakeStream(9, buf.log))
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 7, raising=False)
    ops._join_plan(plan, 0)
    assert buf.log == []                      # its own stream
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: 9, raising=False)
    ops._join_plan(plan, 0)
    want = [("record", 9)] if capturing else [("wait", "its stream"), ("record", 9)]
    assert buf.log == want
    ops._join_plan(plan, 0)
    assert buf.log == (want * 2 if capturing else want)      # once for a stream
    plan.stream, plan.joined = None, {7}                       # made inside a capture: its streams are joined by whoever captures
    del buf.log[:]
    if capturing:
        ops._join_plan(plan, 0)
        assert buf.log == [("record", 9)]
        return
    for raw in (7, 9):                                        # before a replay its places could be anywhere
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda device: raw, raising=False)
        with pytest.raises(RuntimeError, match="capture"):
            ops._join_plan(plan, 0)
    assert buf.log == []


@pytest.mark.gpu
@pytest.mark.parametrize("T,n,r,H,widths", FORMS)
def test_a_plan_made_on_one_stream_and_used_on_another(T, n, r, H, widths):
    """Without a word about streams from the caller: the plan lies behind long work of its stream, and its memory is given away
    while the other stream still has work to do with it."""
    from omni_infer_amd import hip_ops as ops
    d = make(T, n, r, H, widths, BF16, seed=T)
    want = run(d)
    m = torch.randn(4096, 4096, device="cuda").to(BF16)
    out = torch.empty_like(m)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(s1):
            for _ in range(20):
                torch.mm(m, m, out=out)
            plan = ops.adapter_plan(d["ids"], n)
        with torch.cuda.stream(s2):
            got = ops.adapter_linear(d["x"], d["base"], d["a"], d["b"], plan, d["scale"], slices=d["widths"])
        size = plan.buffer.numel()
        del plan
        with torch.cuda.stream(s1):
            waste = [torch.full((size,), 255, dtype=torch.uint8, device="cuda") for _ in range(4)]
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del waste


@pytest.mark.gpu
def test_a_plan_made_before_a_capture_is_used_in_it():
    from omni_infer_amd import hip_ops as ops
    for T, n, r, H, widths in FORMS:
        d = make(T, n, r, H, widths, BF16, seed=T)
        plan = ops.adapter_plan(d["ids"], n)
        call = lambda: ops.adapter_linear(d["x"], d["base"], d["a"], d["b"], plan, d["scale"], slices=d["widths"])  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = call()
        for k in range(3):
            d["x"].copy_(torch.randn(T, H, device="cuda"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, call())


# ------------------------------------------------------------------ slots filled from slots
def test_a_slot_is_set_from_its_own_matrices():
    """To change its scale, to take off its last ranks, to move it to the other shard."""
    from omni_infer_amd.layers.adapters import AdapterSlots
    s = AdapterSlots(24, [16, 16], 2, 8)
    a, b = torch.randn(6, 24).to(BF16), torch.randn(16, 6).to(BF16)
    s.set_adapter(1, [a, None], [b, None], 0.5)
    s.set_adapter(1, [s.a.data[1, :6], None], [s.b.data[1, :16, :6], None], 0.25)
    assert torch.equal(s.a[1, :6], a) and torch.equal(s.b[1, :16, :6], b) and float(s.scale[1]) == 0.25
    s.set_adapter(1, [s.a.data[1, 2:6], None], [s.b.data[1, :16, 2:6], None])
    assert torch.equal(s.a[1, :4], a[2:]) and torch.equal(s.b[1, :16, :4], b[:, 2:]) and not bool(s.a[1, 4:].any())
    s.set_adapter(1, [None, s.a.data[1, :4]], [None, s.b.data[1, :16, :4]])
    assert torch.equal(s.a[1, 8:12], a[2:]) and torch.equal(s.b[1, 16:, :4], b[:, 2:])
    assert not bool(s.a[1, :8].any()) and not bool(s.b[1, :16].any()) and not bool(s.a[1, 12:].any()) and not bool(s.b[1, :, 4:].any())
    s.set_adapter(0, [s.a.data[1, 8:12]] * 2, [s.b.data[1, 16:, :4]] * 2)
    assert torch.equal(s.a[0, :4], a[2:]) and torch.equal(s.a[0, 8:12], a[2:]) and torch.equal(s.b[0, 16:, :4], b[:, 2:])


# ------------------------------------------------------------------ every kernel the dispatch can choose
# What one launch does not take: prompts of many adapters, ranks above 16 at wide H, ranks above 64; odd numbers of tokens
# and widths that fill no tile; sums in one part and in many; more adapters than a wavefront has lanes
DISPATCH = [  # T, n, r, H, widths
    (1024, 64, 16, 4096, [4096]),
    (1024, 64, 16, 4096, [2048, 2048]),
    (64, 32, 64, 4096, [4096]),
    (64, 32, 16, 16384, [5120]),
    (512, 256, 16, 7168, [2048, 2048]),
    (1, 4, 32, 7168, [2048, 2048]),
    (1, 4, 64, 7168, [2048, 2048]),
    (1031, 66, 8, 4104, [1048]),
    (1025, 100, 16, 1992, [200, 72]),
    (2040, 256, 32, 520, [72]),
    (77, 9, 56, 5000, [136, 1032]),
    (3, 2, 40, 7176, [264]),
    (1100, 64, 64, 328, [72]),
    (1040, 100, 32, 520, [40, 72, 24]),
    (65, 3, 128, 264, [136, 64]),
    (130, 3, 256, 136, [264]),
    (1200, 5, 16, 136, [72]),
    (1200, 5, 40, 264, [200]),
    (1111, 3, 24, 1992, [40, 72, 24]),
    (1025, 3, 64, 4104, [128, 24]),
    (1030, 1, 72, 4104, [64, 72]),
    (1300, 2, 256, 328, [200]),
    (1, 4, 16, 7168, [2048, 2048]),
    (333, 12, 24, 1992, [1048]),
    (33, 2, 56, 136, [200]),
]


def _chosen(tmp_path, cases):
    exe = str(tmp_path / "adapter_dispatch")
    subprocess.run([shutil.which("g++"), "-std=c++17", "-O1", os.path.join(ROOT, "tests", "host", "adapter_dispatch.cpp"), "-o", exe], check=True)
    lines = "".join(f"{T} {n} {H} {r} {len(w)} {sum(w)}\n" for T, n, r, H, w in cases)
    at = subprocess.run([exe, "-"], input=lines, capture_output=True, text=True, check=True, timeout=60).stdout.splitlines()
    every = subprocess.run([exe], capture_output=True, text=True, check=True, timeout=60).stdout.splitlines()
    return [tuple(a.split(" parts ")) for a in at], set(every)


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_the_cases_reach_every_kernel_of_the_dispatch(tmp_path):
    """A rule that is changed later must not leave a kernel without a case; and no kernel is there that no shape reaches."""
    at, every = _chosen(tmp_path, DISPATCH)
    assert {k for k, _ in at} == every
    assert {int(parts) for _, parts in at} >= {1, 3, 8, 14}
    text = open(os.path.join(ROOT, "omni_infer_amd", "csrc", "adapter.hip")).read()
    seconds = {k.split()[1] for k in every if " " in k}
    assert seconds == {"out1_32", "out1_64", "out1_256", "out2_64", "out2_256"}
    assert len(set(re.findall(r"EXPAND\((\d), (\d), (\d)\);", text))) == len(seconds)
    assert {k.split()[0] for k in every} == {"one_launch_16", "one_launch_32", "one_launch_64", "rows_16", "rows_32", "rows_64",
                                             "rows_128", "tile_64", "tile_128"}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T,n,r,H,widths", DISPATCH)
def test_every_kernel_against_the_formula(T, n, r, H, widths, dtype):
    d = make(T, n, r, H, widths, dtype, seed=T + r + n)
    got = run(d)
    check(got, d)
    assert torch.equal(got, run(d)), "two calls differ"
    out = d["base"].clone()
    assert run(dict(d, base=out), out=out) is out
    assert torch.equal(out, got), "in place"


# ------------------------------------------------------------------ two calls at once, each with partial sums in memory
@pytest.mark.gpu
def test_two_streams_with_workspaces():
    """Two launches with sums of their own between them (workspaces of different sizes, some in many parts), one launch beside."""
    from omni_infer_amd import _lib as L
    shapes = [(1200, 5, 16, 2048, [512]), (1100, 3, 128, 1024, [768]), (40, 6, 64, 7168, [1024, 1024]), (700, 5, 16, 2048, [512])]
    need = [L.lib().omni_adapter_linear_workspace_bytes(T, n, H, r, len(w), sum(w)) for T, n, r, H, w in shapes]
    assert len(set(need[:3])) == 3 and min(need[:3]) > 0 and need[3] == 0
    ds = [make(*s, BF16, seed=k) for k, s in enumerate(shapes)]
    want = [run(d) for d in ds]
    for d, w in zip(ds, want):
        check(w, d)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for k in range(12):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                i = (k + j) % len(ds) if k < 8 else k % len(ds)     # different ones beside each other, then twice the same
                got.append((i, run(ds[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i, g in got)


@pytest.mark.gpu
def test_two_graphs_with_workspaces():
    """Recorded and replayed beside each other on two streams: a graph's partial sums are its own."""
    shapes = [(1200, 5, 16, 2048, [512]), (40, 6, 64, 7168, [1024, 1024])]
    made = []
    for k, s in enumerate(shapes):
        d = make(*s, BF16, seed=k)
        run(d)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = run(d)
        made.append((d, graph, got))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for k in range(4):
        for d, _, _ in made:
            d["x"].copy_(torch.randn(d["x"].shape, generator=torch.Generator().manual_seed(k)))
        torch.cuda.synchronize()
        for s, (_, graph, _) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for d, _, got in made:
            assert torch.equal(got, run(d)), k


@pytest.mark.gpu
def test_a_plan_of_a_capture_stays_in_captures():
    """Refused outside, on the capture's own stream too; used on a second stream that the capture forks to and joins."""
    from omni_infer_amd import hip_ops as ops
    T, n, r, H, widths = FORMS[2]
    d = make(T, n, r, H, widths, BF16, seed=2)
    want = run(d)
    call = lambda plan: ops.adapter_linear(d["x"], d["base"], d["a"], d["b"], plan, d["scale"], slices=d["widths"])  # noqa: E731
    main, side = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        plan = ops.adapter_plan(d["ids"], n)
        here = call(plan)
        side.wait_stream(main)
        with torch.cuda.stream(side):
            there = call(plan)
        main.wait_stream(side)
    for s in (torch.cuda.current_stream(), main, side):
        with torch.cuda.stream(s), pytest.raises(RuntimeError, match="capture"):
            call(plan)
    for k in range(3):
        d["ids"].copy_(torch.randint(-1, n, (T,), dtype=torch.int32, generator=torch.Generator().manual_seed(k)))
        want = run(d)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(here, want) and torch.equal(there, want)
