"""Calls of the adapters beside the tests of their formula: slots that hold nothing, batches on other streams, every kernel the
dispatch can choose."""
import pytest
import torch

from tests.test_adapter import BF16, FP16, check, make, run

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
    ops._join_plan(plan, 0)
    assert buf.log == [("record", 9)]


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
