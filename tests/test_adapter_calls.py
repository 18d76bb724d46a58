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
