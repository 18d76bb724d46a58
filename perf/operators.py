"""Cases, plain forms and 64-bit values of the operators around a dense MLP that is served with low-rank adapters.

``adapter``  a projection's rows plus the low-rank update of each token's own adapter,
``norm``     the norm after a block, its gate and residual scale, the residual sum and the norm before the next block,
``swiglu``   the gated activation between the two projections; both of the last also as int8 rows with a scale per row.
"""
import math

import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one token of one request through stacked gate and up projections: nothing but latency
        {"name": "adapter one token", "op": "adapter", "T": 1, "n": 8, "r": 16, "H": 7168, "N": 2048, "slices": 2,
         "requests": 1, "type": "bf16"},
        # a decode step in which no two requests share an adapter
        {"name": "adapter decode", "op": "adapter", "T": 64, "n": 64, "r": 16, "H": 2048, "N": 7168, "slices": 1,
         "requests": 64, "type": "bf16"},
        # a batch of short prompts and single tokens, an odd number of rows, widths that fill no tile
        {"name": "adapter mixed", "op": "adapter", "T": 333, "n": 12, "r": 24, "H": 1992, "N": 1048, "slices": 1,
         "requests": 40, "type": "fp16"},
        # prompts through gate and up projections, adapters of a high rank
        {"name": "adapter prompts gate_up", "op": "adapter", "T": 8192, "n": 4, "r": 64, "H": 7168, "N": 2048,
         "slices": 2, "requests": 8, "type": "bf16"},
        # prompts of many requests through a down projection
        {"name": "adapter prompts down", "op": "adapter", "T": 8192, "n": 16, "r": 16, "H": 2048, "N": 7168,
         "slices": 1, "requests": 24, "type": "bf16"},
        # one token between two blocks, handed on as int8
        {"name": "norm one token", "op": "norm", "T": 1, "H": 7168, "gate": "none", "quant": True, "type": "bf16"},
        # a decode step, a learned factor for each channel, handed on as int8
        {"name": "norm decode", "op": "norm", "T": 64, "H": 7680, "gate": "channel", "quant": True, "type": "bf16"},
        # a width that no vector divides, a gate for each token
        {"name": "norm odd width", "op": "norm", "T": 1021, "H": 5121, "gate": "token", "quant": False, "type": "fp16"},
        # a long prompt
        {"name": "norm prompt", "op": "norm", "T": 8192, "H": 7168, "gate": "none", "quant": False, "type": "bf16"},
        # a decode step, handed on as rows for the adapters and as int8 for the shared projection
        {"name": "swiglu decode", "op": "swiglu", "T": 64, "H": 2048, "quant": True, "type": "bf16"},
        # an odd width in 32 bits
        {"name": "swiglu odd width", "op": "swiglu", "T": 777, "H": 1003, "quant": False, "type": "fp32"},
        # a long prompt
        {"name": "swiglu prompt", "op": "swiglu", "T": 8192, "H": 8192, "quant": True, "type": "bf16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["adapter", "adapter", "norm", "swiglu"])
    if op == "adapter":
        slices = rng.choice([1, 1, 2])
        H, N, r = 8 * spread(16, 960), 8 * spread(16, 960 // slices), 8 * rng.randint(1, 8)
        T = min(spread(1, 8192), 8192 * 16384 // (H + 2 * slices * N))
        n = min(spread(1, 64), max(1, 2 ** 24 // (max(T, 256) * r)))
        return {"op": op, "T": T, "n": n, "r": r, "H": H, "N": N, "slices": slices,
                "requests": min(T, spread(1, 64)) if rng.random() < 0.7 else T, "type": rng.choice(["bf16", "bf16", "fp16"])}
    case = {"op": op, "H": spread(64, 8192) if rng.random() < 0.5 else 8 * spread(8, 1024)}
    case["T"] = min(spread(1, 8192), 8192 * 7168 // case["H"])
    if op == "norm":
        case["gate"] = rng.choice(["none", "channel", "token", "full"])
    case["quant"] = rng.random() < 0.5
    case["type"] = rng.choice(["bf16", "bf16", "fp16"] if case["quant"] else ["bf16", "bf16", "fp16", "fp32"])
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dt, T, H = TYPES[case["type"]], case["T"], case["H"]

    def normal(*shape, scale=1.0, add=0.0, dtype=dt):
        return (torch.randn(*shape, device=DEVICE, generator=gen) * scale + add).to(dtype)

    if case["op"] == "adapter":
        n, r, S, N, requests = case["n"], case["r"], case["slices"], case["N"], case["requests"]
        # requests of uneven lengths lie one after the other; one in eight uses no adapter
        of_request = torch.randperm(n, device=DEVICE, generator=gen)[torch.arange(requests, device=DEVICE) % n]
        of_request = of_request[torch.randperm(requests, device=DEVICE, generator=gen)]
        if requests > 1:
            of_request[torch.rand(requests, device=DEVICE, generator=gen) < 0.125] = -1
        if requests < T:
            cuts = torch.sort(torch.rand(requests - 1, device=DEVICE, generator=gen)).values * T
            of_token = torch.bucketize(torch.arange(T, device=DEVICE) + 0.5, cuts)
        else:
            of_token = torch.arange(T, device=DEVICE)
        return {"x": normal(T, H), "base": normal(T, S * N), "a": normal(n, S * r, H, scale=H ** -0.5),
                "b": normal(n, S * N, r, scale=0.5 * r ** -0.5), "scale": 0.5 + torch.rand(n, device=DEVICE, generator=gen),
                "ids": of_request[of_token].to(torch.int32)}
    if case["op"] == "norm":
        shape = {"none": None, "channel": (H,), "token": (T, 1), "full": (T, H)}[case["gate"]]
        return {"x": normal(T, H, scale=2.0), "residual": normal(T, H, scale=3.0),
                "post_weight": normal(H, scale=0.1, add=1.0), "pre_weight": normal(H, scale=0.1, add=1.0),
                "gate": None if shape is None else normal(*shape, scale=0.5)}
    return {"gate_up": normal(T, 2 * H, scale=1.5)}


POST_EPS, PRE_EPS, RESIDUAL_SCALE = 1e-5, 1e-6, 0.7


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case)
    if case.get("quant"):
        state["values"] = torch.empty(case["T"], case["H"], dtype=TYPES[case["type"]], device=DEVICE)
    if own and case["op"] == "adapter":
        from omni_infer_amd import hip_ops
        state["plan"] = hip_ops.adapter_plan(state["ids"], case["n"])  # once for a batch, for all its projections
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    case = s["case"]
    if own:
        return _own(s, case)
    return {"adapter": _adapter, "norm": _norm, "swiglu": _swiglu}[case["op"]](s, case)


def _own(s, case):
    from omni_infer_amd import hip_ops
    if case["op"] == "adapter":
        return hip_ops.adapter_linear(s["x"], s["base"], s["a"], s["b"], s["plan"], s["scale"],
                                      slices=[case["N"]] * case["slices"])
    quant = case["quant"]
    if case["op"] == "norm":
        y, residual, q, scale = hip_ops.sandwich_norm(
            s["x"], s["residual"], s["post_weight"], s["pre_weight"], POST_EPS, PRE_EPS, gate=s["gate"],
            residual_scale=RESIDUAL_SCALE, want_y=not quant, want_quant=quant)
        return (_values(q, scale, s) if quant else y), residual
    h, q, scale = hip_ops.swiglu_quant(s["gate_up"], want_quant=quant)
    return (h, _values(q, scale, s)) if quant else h


def _values(q, scale, s):
    """What int8 rows stand for, in a tensor of each pass's own, as the plain form gives them."""
    return torch.mul(q, scale.unsqueeze(-1), out=torch.empty_like(s["values"]))


def _adapter(s, case):
    """Few tokens: each token's own matrices. Else the products with all adapters at once, those of other adapters zero."""
    n, r, S, N, T = case["n"], case["r"], case["slices"], case["N"], case["T"]
    x, a, b, ids = s["x"].float(), s["a"], s["b"], s["ids"].long()
    if T <= n:
        kept = (ids >= 0).unsqueeze(-1)
        at = ids.clamp(min=0)
        v = torch.bmm(a[at].float(), x.unsqueeze(-1)).view(T, S, r) * s["scale"][at].view(T, 1, 1)
        delta = torch.matmul(b[at].float().view(T, S, N, r), v.unsqueeze(-1)).view(T, S * N)
        return (s["base"].float() + torch.where(kept, delta, torch.zeros_like(delta))).to(s["base"].dtype)
    v = (x @ a.float().view(n * S * r, -1).t()).view(T, n, S, r) * s["scale"].view(1, n, 1, 1)
    mine = (ids.unsqueeze(-1) == torch.arange(n, device=ids.device)).view(T, n, 1, 1)
    v = torch.where(mine, v, torch.zeros_like(v)).permute(2, 0, 1, 3).reshape(S, T, n * r)
    w = b.float().view(n, S, N, r).permute(1, 0, 3, 2).reshape(S, n * r, N)
    delta = torch.bmm(v, w).transpose(0, 1).reshape(T, S * N)
    return (s["base"].float() + delta).to(s["base"].dtype)


def _int8_values(s, y):
    """The int8 rows of `y` (as it is rounded) as the values they stand for."""
    y = y.float()
    scale = y.abs().amax(dim=-1, keepdim=True) / 127.0
    q = torch.where(scale > 0, torch.round(y / scale).clamp(-128, 127), torch.zeros_like(y))
    return (q * scale).to(s["values"].dtype)


def _norm(s, case):
    x = s["x"].float()
    t = x * torch.rsqrt(x.square().mean(dim=-1, keepdim=True) + POST_EPS) * s["post_weight"].float()
    if s["gate"] is not None:
        t = t * s["gate"].float()
    r = s["residual"].float() + t * RESIDUAL_SCALE
    y = (r * torch.rsqrt(r.square().mean(dim=-1, keepdim=True) + PRE_EPS) * s["pre_weight"].float()).to(s["x"].dtype)
    return (_int8_values(s, y) if case["quant"] else y), r.to(s["x"].dtype)


def _swiglu(s, case):
    g, u = s["gate_up"].float().chunk(2, dim=-1)
    h = (g / (1.0 + torch.exp(-g)) * u).to(s["gate_up"].dtype)
    return (h, _int8_values(s, h)) if case["quant"] else h


# ------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    size, T, H = (4 if case["type"] == "fp32" else 2), case["T"], case["H"]
    if case["op"] == "adapter":
        n, r, out = case["n"], case["r"], case["slices"] * case["N"]
        used = min(n, case["requests"])
        return {"bytes": size * (T * (H + 2 * out) + used * r * (case["slices"] * H + out)) + 4 * T,
                "flops": 2 * T * r * (case["slices"] * H + out) + T * out}
    if case["op"] == "norm":
        gate = {"none": 0, "channel": H, "token": T, "full": T * H}[case["gate"]]
        y = T * (H + 4) if case["quant"] else size * T * H
        return {"bytes": size * (3 * T * H + 2 * H + gate) + y, "flops": 10 * T * H}
    return {"bytes": size * 3 * T * H + (T * (H + 4) if case["quant"] else 0), "flops": 6 * T * H}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "adapter":
        out, r, N = s["base"].double(), case["r"], case["N"]
        for g in range(case["n"]):
            rows = torch.nonzero(s["ids"] == g).flatten()
            x = s["x"][rows].double()
            for j in range(case["slices"]):
                down, up = s["a"][g, j * r:(j + 1) * r].double(), s["b"][g, j * N:(j + 1) * N].double()
                out[rows, j * N:(j + 1) * N] += s["scale"][g].double() * ((x @ down.T) @ up.T)
        return out

    def int8_values(y):  # of the rows as their type holds them
        y = y.to(TYPES[case["type"]]).double()
        step = y.abs().max(dim=1).values[:, None] / 127
        return torch.where(step == 0, step, (y / step.where(step != 0, torch.ones_like(step))).round() * step)

    if case["op"] == "norm":
        x, r = s["x"].double(), s["residual"].double()
        t = x / ((x ** 2).sum(1, keepdim=True) / case["H"] + POST_EPS).sqrt() * s["post_weight"].double()
        r = r + RESIDUAL_SCALE * (1 if s["gate"] is None else s["gate"].double()) * t
        y = r / ((r ** 2).sum(1, keepdim=True) / case["H"] + PRE_EPS).sqrt() * s["pre_weight"].double()
        return (int8_values(y) if case["quant"] else y), r
    g, u = s["gate_up"][:, :case["H"]].double(), s["gate_up"][:, case["H"]:].double()
    h = g * torch.sigmoid(g) * u
    return (h, int8_values(h)) if case["quant"] else h
