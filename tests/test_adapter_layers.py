"""Adapters and sandwich norms where the layers use them: the linears, the dense MLP, the MoE block's shared expert, and
the whole run norm -> MLP with adapters -> norm."""
import types

import pytest
import torch

from tests.helpers import gen, rel_err

BF16 = torch.bfloat16


# ------------------------------------------------------------------ CPU
def test_slots_hold_what_checkpoints_hold():
    from omni_infer_amd.layers.adapters import AdapterSlots
    s = AdapterSlots(24, [16, 8], 3, 10)
    assert s.rank == 16 and s.a.shape == (3, 32, 24) and s.b.shape == (3, 24, 16) and s.scale.shape == (3,)
    a, b = torch.randn(10, 24).to(BF16), torch.randn(8, 10).to(BF16)
    s.set_adapter(1, [None, a], [None, b], 0.25)
    assert torch.equal(s.a[1, 16:26], a) and torch.equal(s.b[1, 16:24, :10], b) and float(s.scale[1]) == 0.25
    assert not bool(s.a[1, :16].any()) and not bool(s.a[1, 26:].any()) and not bool(s.b[1, :16].any()) and not bool(s.b[1, :, 10:].any())
    assert not bool(s.a[0].any()) and not bool(s.a[2].any())
    s.set_adapter(1, [a[:4], None], [torch.ones(16, 4), None])          # another adapter in the same slot: nothing of the first is left
    assert not bool(s.a[1, 16:].any()) and not bool(s.b[1, 16:].any()) and float(s.scale[1]) == 1.0
    s.clear(1)
    assert not bool(s.a.any()) and not bool(s.b.any()) and not bool(s.scale.any())
    assert not any(p.requires_grad for p in s.parameters())


def test_slot_refusals():
    from omni_infer_amd.layers.adapters import AdapterSlots
    for bad in (dict(input_size=20), dict(output_sizes=[12]), dict(max_adapters=0), dict(max_rank=0), dict(max_rank=257),
                dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            AdapterSlots(**{**dict(input_size=24, output_sizes=[16], max_adapters=2, max_rank=8), **bad})
    s = AdapterSlots(24, [16], 2, 8)
    a, b = torch.zeros(8, 24), torch.zeros(16, 8)
    for slot, x, y in ((2, a, b), (-1, a, b), (0, a[:, :8], b), (0, a, b[:8]), (0, a[:4], b), (0, torch.zeros(9, 24), torch.zeros(16, 9)),
                       (0, [a, a], [b, b]), (0, [a], [None])):
        with pytest.raises(ValueError):
            s.set_adapter(slot, x, y)
    from omni_infer_amd.layers.layernorm import RMSNorm, SandwichNorm
    with pytest.raises(ValueError):
        SandwichNorm(RMSNorm(16), RMSNorm(24))


# ------------------------------------------------------------------ GPU
def _mlp(H, I, quant=True, n=4, r=16, seed=1, dtype=BF16):
    """A dense MLP with adapters in three of four slots; returns it with its weights in 64 bits."""
    from omni_infer_amd.layers.deepseek_moe import ReplicatedDeepseekMLP
    from omni_infer_amd.quantization.compressed_tensors import AscendCompressedTensorsConfig
    g = gen(seed)
    old = torch.get_default_dtype()
    torch.set_default_dtype(dtype)
    try:
        m = ReplicatedDeepseekMLP(H, I, "silu", AscendCompressedTensorsConfig() if quant else None, prefix="mlp", device="cuda")
    finally:
        torch.set_default_dtype(old)
    w = []
    for lin, (N, K) in ((m.gate_up_proj, (2 * I, H)), (m.down_proj, (H, I))):
        if quant:
            q = torch.randint(-127, 128, (N, K), generator=g).to(torch.int8)
            sc = (0.7 + torch.rand(N, generator=g)).mul(K ** -0.5 / 73.0).to(BF16)
            lin.weight.data.copy_(q)
            lin.weight_scale.data.copy_(sc.view(-1, 1))
            lin.quant_method.process_weights_after_loading(lin)
            w.append(q.double() * sc.double().view(-1, 1))
        else:
            lin.weight.data.copy_(torch.randn(N, K, generator=g) * K ** -0.5)
            w.append(lin.weight.data.double().cpu())
    m.enable_adapters(n, r)
    for slot in range(n - 1):
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        k = (r, r // 2, 3)[slot % 3]
        m.gate_up_proj.adapters.set_adapter(slot, [rnd(k, H) * H ** -0.5, None if slot == 1 else rnd(k, H) * H ** -0.5],
                                            [rnd(I, k) * k ** -0.5, None if slot == 1 else rnd(I, k) * k ** -0.5], 0.5 + slot)
        m.down_proj.adapters.set_adapter(slot, rnd(k, I) * I ** -0.5, rnd(H, k) * k ** -0.5, 0.75)
    return m, w


def _linear64(x, w, slots, ids):
    y = x @ w.T
    a, b, s = (t.data.double().cpu() for t in (slots.a, slots.b, slots.scale))
    for g in range(slots.max_adapters):
        rows, n0 = (ids == g).nonzero().flatten(), 0
        for j, width in enumerate(slots.output_sizes):
            y[rows, n0:n0 + width] += s[g] * (x[rows] @ a[g, j * slots.rank:(j + 1) * slots.rank].T) @ b[g, n0:n0 + width].T
            n0 += width
    return y


def _mlp64(x, w, m, ids):
    g, u = _linear64(x, w[0], m.gate_up_proj.adapters, ids).chunk(2, dim=1)
    return _linear64(g * torch.sigmoid(g) * u, w[1], m.down_proj.adapters, ids)


def _ids(T, n, seed):
    ids = torch.randint(-1, n, (T,), generator=gen(seed), dtype=torch.int32)
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 23, 1500])
def test_mlp_with_adapters(T):
    """Against the formula in 64 bits: int8 activations carry about max/127/sqrt(12) of a row's largest value as noise, 1 % of
    the root mean square before the first product, which the gated product doubles, and 2 % (heavier tails) before the
    second: 3 % together, held to twice that.  And bit for bit against its own operators in a row."""
    from omni_infer_amd import hip_ops as ops
    from omni_infer_amd.layers.adapters import AdapterBatch
    H, I = 1024, 512
    m, w = _mlp(H, I)
    x = torch.randn(T, H, generator=gen(T)).to(BF16)
    ids = _ids(T, 4, T + 1)
    batch = AdapterBatch(ids.cuda(), 4)
    y = m(x.cuda(), batch)
    assert rel_err(y.cpu(), _mlp64(x.double(), w, m, ids)) < 0.06
    if T > 1:   # the adapters are a good part of it
        assert rel_err(m(x.cuda()).cpu(), _mlp64(x.double(), w, m, ids)) > 0.2
    xq, xs = ops.npu_dynamic_quant(x.cuda())
    gu, dn = m.gate_up_proj, m.down_proj
    off = ops.dense_offsets(T, "cuda")
    h = ops.grouped_gemm2_dequant(xq, xs, gu.weight, gu.weight_scale, off, 2 * I, H)[0]
    h = ops.adapter_linear(x.cuda(), h, gu.adapters.a.data, gu.adapters.b.data, batch.plan, gu.adapters.scale.data, [I, I])
    h, hq, hs = ops.swiglu_quant(h, want_quant=True)
    want = ops.grouped_gemm2_dequant(hq, hs, dn.weight, dn.weight_scale, off, H, I)[0]
    want = ops.adapter_linear(h, want, dn.adapters.a.data, dn.adapters.b.data, batch.plan, dn.adapters.scale.data)
    assert torch.equal(y, want)
    assert torch.equal(m({"x": x.cuda(), "x_int8": xq, "pertoken_scale": xs}, batch), want)
    with pytest.raises(ValueError, match="before their quantisation"):
        m({"x_int8": xq, "pertoken_scale": xs}, batch)
    with pytest.raises(ValueError, match="4"):
        m(x.cuda(), AdapterBatch(ids.cuda(), 5))
    # a batch that uses no adapter: nothing but the rounding of the stacked product differs from the shared path
    none = AdapterBatch(torch.full((T,), -1, dtype=torch.int32, device="cuda"), 4)
    assert rel_err(m(x.cuda(), none).cpu(), m(x.cuda()).cpu()) < 0.02


@pytest.mark.gpu
def test_shared_path_is_untouched_by_empty_room_for_adapters():
    from omni_infer_amd.layers.deepseek_moe import ReplicatedDeepseekMLP
    m, _ = _mlp(512, 256, seed=2)
    x = torch.randn(40, 512, generator=gen(3)).to(BF16).cuda()
    y = m(x)
    m.gate_up_proj.adapters = m.down_proj.adapters = None
    from omni_infer_amd.layers.adapters import AdapterBatch
    assert torch.equal(m(x), y)
    assert torch.equal(m(x, AdapterBatch(torch.zeros(40, dtype=torch.int32, device="cuda"), 4)), y)
    assert isinstance(m, ReplicatedDeepseekMLP) and not m.has_adapters


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, torch.float16])
def test_mlp_without_quantisation(dtype):
    """Projections of a checkpoint's ``ignore`` list.  Two products of 16-bit operands with results rounded to 16 bits, an
    activation between them: a few half steps, held to eight."""
    from omni_infer_amd.layers.adapters import AdapterBatch
    m, w = _mlp(512, 328, quant=False, seed=5, dtype=dtype)
    x = torch.randn(300, 512, generator=gen(6)).to(dtype)
    ids = _ids(300, 4, 7)
    tol = 8 * torch.finfo(dtype).eps / 2
    y = m(x.cuda(), AdapterBatch(ids.cuda(), 4))
    assert y.dtype == dtype and rel_err(y.cpu(), _mlp64(x.double(), w, m, ids)) < tol
    assert rel_err(m(x.cuda()).cpu(), _mlp64(x.double(), w, m, torch.full((300,), -1))) < tol


@pytest.mark.gpu
def test_moe_block_with_adapters_on_its_shared_expert():
    from omni_infer_amd import config, distributed
    from omni_infer_amd.layers.adapters import AdapterBatch
    from omni_infer_amd.layers.layernorm import RMSNorm, SandwichNorm
    from tests.test_gpu_layer import _dsv3_block
    env = types.SimpleNamespace(config=config, dist=distributed)
    H, I, T = 1024, 512, 50
    blk, *_ = _dsv3_block(env, 4, 8, 2, H=H, I=I, seed=4)
    g = gen(11)
    x = torch.randn(T, H, generator=g).to(BF16).cuda()
    ids = _ids(T, 3, 12)
    batch = AdapterBatch(ids.cuda(), 3)
    plain, _ = blk(x, None, None, 3)
    assert torch.equal(blk(x, None, None, 3, adapters=batch)[0], plain)      # no room for adapters yet
    blk.shared_experts.enable_adapters(3, 8)
    for slot in range(3):
        blk.shared_experts.gate_up_proj.adapters.set_adapter(slot, [torch.randn(8, H, generator=g) * H ** -0.5] * 2,
                                                             [torch.randn(I, 8, generator=g)] * 2, 0.5)
        blk.shared_experts.down_proj.adapters.set_adapter(slot, torch.randn(8, I, generator=g) * I ** -0.5,
                                                          torch.randn(H, 8, generator=g), 0.5)
    assert torch.equal(blk(x, None, None, 3)[0], plain)
    out, _ = blk(x, None, None, 3, adapters=batch)
    assert not torch.equal(out, plain)
    shared = blk.shared_experts
    blk.shared_experts = None
    routed, _ = blk(x, None, None, 3)
    blk.shared_experts = shared
    assert torch.equal(out, routed + shared(x, batch))
    blk.fused = False
    assert torch.equal(blk(x, None, None, 3, adapters=batch)[0], out)        # operator by operator: the same bits
    blk.fused = True
    post, pre = (RMSNorm(H, 1e-6, params_dtype=BF16, device="cuda") for _ in range(2))
    norm = SandwichNorm(post, pre, residual_scale=0.5)
    res = torch.randn(T, H, generator=g).to(BF16).cuda()
    handed, r = norm.forward_moe_input(x, res)
    y, r2 = norm(x, res)
    assert torch.equal(handed["x"], y) and torch.equal(r, r2)
    assert torch.equal(blk(handed, None, None, 3, adapters=batch)[0], blk(y, None, None, 3, adapters=batch)[0])
    d, _ = norm(x, res, quant_symbol=True)
    assert set(d) == {"x_int8", "pertoken_scale"} and torch.equal(d["x_int8"], handed["x_int8"])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 64, 1100])
def test_run_of_norm_mlp_norm(T):
    """The three operators as a dense layer uses them: norms around an MLP with adapters, eager and as a graph that is replayed
    with new tokens, new adapters of the requests and new adapter weights."""
    from omni_infer_amd.layers.adapters import AdapterBatch
    from omni_infer_amd.layers.layernorm import RMSNorm, SandwichNorm
    H, I = 1024, 512
    m, w = _mlp(H, I, seed=T)
    g = gen(T + 9)
    norms = [RMSNorm(H, 1e-6, params_dtype=BF16, device="cuda") for _ in range(4)]
    for v in norms:
        v.weight.data.copy_(1 + 0.1 * torch.randn(H, generator=g))
    before, after = SandwichNorm(norms[0], norms[1], 0.5), SandwichNorm(norms[2], norms[3], 0.5)
    gate = (1 + 0.2 * torch.randn(H, generator=g)).to(BF16).cuda()
    state = {"x": torch.randn(T, H, generator=g).to(BF16).cuda(), "res": torch.randn(T, H, generator=g).to(BF16).cuda(),
             "ids": _ids(T, 4, T + 2).cuda()}

    def step():
        handed, res = before.forward_moe_input(state["x"], state["res"], gate)
        y = m(handed, AdapterBatch(state["ids"], 4))
        return (handed["x"], y) + after(y, res, gate)

    h, y, out, res = step()
    # a norm rounds once (2^-8); the second one also reads an input that was rounded before
    def norm64(v, weight):
        v = v.double()
        return v / (v.square().mean(1, keepdim=True) + 1e-6).sqrt() * weight.data.double()
    gg = gate.double() * 0.5
    r1 = state["res"].double() + gg * norm64(state["x"], norms[0].weight)
    assert rel_err(h, norm64(r1, norms[1].weight)) < 2.0 ** -8
    assert rel_err(y.cpu(), _mlp64(h.double().cpu(), w, m, state["ids"].cpu())) < 0.06
    r2 = r1 + gg * norm64(y, norms[2].weight)
    assert rel_err(res, r2) < 2.0 ** -7 and rel_err(out, norm64(r2, norms[3].weight)) < 2.0 ** -7
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for k in range(3):
        state["x"].copy_(torch.randn(T, H, generator=gen(100 + k)))
        state["ids"].copy_(_ids(T, 4, 200 + k))
        m.gate_up_proj.adapters.scale.data[0] = 0.1 * k
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {k}"
