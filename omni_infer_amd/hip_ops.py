"""Operator boundary: torch-tensor wrappers over the C ABI of libomni_moe_hip.so.

Each function stands where the reference calls a ``torch_npu.npu_*`` operator on the MoE
path and keeps that operator's argument meaning; the arithmetic is done by the gfx950 HIP
kernels.  torch is used for device memory and the current stream only.  Nothing here has a
CPU or eager fallback: tensors must live on the GPU and the library must be built.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib as L


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _need_gpu(*tensors: torch.Tensor) -> None:
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise RuntimeError("omni_infer_amd operators run on the GPU only (got a CPU tensor)")


_DT = {torch.bfloat16: L.OMNI_DT_BF16, torch.float32: L.OMNI_DT_F32, torch.float16: L.OMNI_DT_F16}


# ----------------------------------------------------------------------------- routing
def moe_route(logits: torch.Tensor, bias: Optional[torch.Tensor], top_k: int, n_group: int, topk_group: int,
              score_fn: str, group_mode: int, masked_fill_zero: bool, weight_from_c: bool, renorm: bool,
              scale: float, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    _need_gpu(logits, bias)
    if logits.dim() != 2:
        raise ValueError("router logits must be [T, E]")
    logits = logits.float().contiguous()
    T, E = logits.shape
    if bias is not None:
        bias = bias.float().contiguous()
        if bias.numel() != E:
            raise ValueError("bias must have one entry per expert")
    w = torch.empty(T, top_k, dtype=torch.float32, device=logits.device)
    ids = torch.empty(T, top_k, dtype=torch.int32, device=logits.device)
    fn = {"softmax": L.OMNI_SCORE_SOFTMAX, "sigmoid": L.OMNI_SCORE_SIGMOID}.get(score_fn)
    if fn is None:
        raise ValueError(f"Unsupported scoring function: {score_fn}")
    rc = L.lib().omni_moe_route(_ptr(logits), _ptr(bias), T, E, int(n_group), int(topk_group), int(top_k), fn,
                                int(group_mode), int(masked_fill_zero), int(weight_from_c), int(renorm),
                                float(scale), float(eps), _ptr(w), _ptr(ids), _stream())
    L.check(rc, "omni_moe_route")
    return w, ids


_GATE_WS = {}


def moe_gate_route(x: torch.Tensor, gate_w: torch.Tensor, bias: Optional[torch.Tensor], top_k: int, n_group: int,
                   topk_group: int, score_fn: str, group_mode: int, masked_fill_zero: bool, weight_from_c: bool,
                   renorm: bool, scale: float, eps: float, want_logits: bool = False, round_logits_bf16: bool = False):
    """Gate projection and router in one library call: ``self.gate.forward(hidden_states.float())`` +
    ``FusedMoE.select_experts`` (deepseek_moe.py:147-152,253-256).  ``x`` [T,H] bf16 or fp32 is read as it
    is (no fp32 copy), ``gate_w`` [E,H] fp32 or bf16.  ``top_k`` = 0 computes the logits only.
    Returns (topk_w, topk_ids, logits or None)."""
    _need_gpu(x, gate_w, bias)
    if x.dim() != 2 or gate_w.dim() != 2 or x.shape[1] != gate_w.shape[1]:
        raise ValueError("gate: x must be [T, H] and the gate weight [E, H]")
    if x.dtype not in (torch.bfloat16, torch.float32) or gate_w.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("gate: tokens and gate weight must be bf16 or fp32")
    x = x.contiguous()
    gate_w = gate_w.contiguous()
    T, H = x.shape
    E = gate_w.shape[0]
    dev = x.device
    if bias is not None:
        bias = bias.float().contiguous()
        if bias.numel() != E:
            raise ValueError("bias must have one entry per expert")
    fn = {"softmax": L.OMNI_SCORE_SOFTMAX, "sigmoid": L.OMNI_SCORE_SIGMOID}.get(score_fn)
    if fn is None:
        raise ValueError(f"Unsupported scoring function: {score_fn}")
    need = L.lib().omni_moe_gate_route_workspace_bytes(T, H, E)
    key = str(dev)
    ws = _GATE_WS.get(key)   # one scratch per device, grown on demand; calls on one stream are ordered
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        _GATE_WS[key] = ws
    w = torch.empty(T, top_k, dtype=torch.float32, device=dev) if top_k > 0 else None
    ids = torch.empty(T, top_k, dtype=torch.int32, device=dev) if top_k > 0 else None
    logits = torch.empty(T, E, dtype=torch.float32, device=dev) if (want_logits or top_k == 0) else None
    rc = L.lib().omni_moe_gate_route(_ptr(x), _DT[x.dtype], _ptr(gate_w), _DT[gate_w.dtype], _ptr(bias), T, H, E,
                                     int(n_group), int(topk_group), int(top_k), fn, int(group_mode),
                                     int(masked_fill_zero), int(weight_from_c), int(renorm), float(scale), float(eps),
                                     int(round_logits_bf16), _ptr(logits), _ptr(w), _ptr(ids), _ptr(ws), ws.numel(),
                                     _stream())
    L.check(rc, "omni_moe_gate_route")
    return w, ids, logits


def gate_logits(x: torch.Tensor, gate_w: torch.Tensor, round_logits_bf16: bool = False) -> torch.Tensor:
    """``ReplicatedLinear.forward`` of the gate (deepseek_moe.py:147-152): fp32 logits [T, E] in the
    library's fixed summation order."""
    return moe_gate_route(x, gate_w, None, 0, 1, 1, "softmax", L.OMNI_GROUP_MAX, False, False, False, 1.0, 0.0,
                          round_logits_bf16=round_logits_bf16)[2]


_ROW_IDX = {}


def _row_idx(T: int, K: int, device) -> torch.Tensor:
    """row_idx[n, k] = k*T + n (fused_moe.py:80-81, layer.py:352-353).  A constant of (T, K): made once per
    shape and device, so that the routing wrappers launch nothing but the router."""
    key = (int(T), int(K), str(device))
    t = _ROW_IDX.get(key)
    if t is None:
        if len(_ROW_IDX) > 256:
            _ROW_IDX.clear()
        t = torch.arange(T * K, device=device, dtype=torch.int32).view(K, T).transpose(0, 1)
        _ROW_IDX[key] = t
    return t


def npu_moe_gating_top_k(x: torch.Tensor, k: int, bias: Optional[torch.Tensor], k_group: int, group_count: int,
                         group_select_mode: int = 1, renorm: int = 0, norm_type: int = 1,
                         routed_scaling_factor: float = 1.0, eps: float = 1e-20):
    """Stands in for ``torch_npu.npu_moe_gating_top_k`` as called at
    omni/models/common/layers/moe/fused_moe/layer.py:341-351."""
    if renorm != 0:
        raise ValueError("npu_moe_gating_top_k: only renorm=0 (score, then top-k) is supported")
    w, ids = moe_route(x, bias, k, group_count, k_group, "sigmoid" if norm_type == 1 else "softmax",
                       L.OMNI_GROUP_TOP2SUM if group_select_mode == 1 else L.OMNI_GROUP_MAX,
                       masked_fill_zero=False, weight_from_c=False, renorm=True,
                       scale=routed_scaling_factor, eps=eps)
    return w, ids, None


def npu_moe_gating_top_k_softmax(x: torch.Tensor, k: int):
    """Stands in for ``torch_npu.npu_moe_gating_top_k_softmax`` (fused_moe.py:29)."""
    w, ids = moe_route(x, None, k, 1, 1, "softmax", L.OMNI_GROUP_MAX, False, False, False, 1.0, 0.0)
    return w, ids, _row_idx(x.shape[0], k, x.device)


# ----------------------------------------------------------------------------- quant
def npu_dynamic_quant(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Stands in for ``torch_npu.npu_dynamic_quant`` (deepseek_moe.py:247,323;
    compressed_tensors_moe.py:241,247; schemes/compressed_tensors_w8a8_int8.py:97)."""
    _need_gpu(x)
    if x.dtype not in _DT:
        raise ValueError(f"npu_dynamic_quant: unsupported dtype {x.dtype}")
    shape = x.shape
    x2 = x.reshape(-1, shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    rows, cols = x2.shape
    q = torch.empty(rows, cols, dtype=torch.int8, device=x.device)
    s = torch.empty(rows, dtype=torch.float32, device=x.device)
    rc = L.lib().omni_dynamic_quant(_ptr(x2), _DT[x.dtype], rows, cols, x2.stride(0) if rows > 1 else cols,
                                    _ptr(q), _ptr(s), _stream())
    L.check(rc, "omni_dynamic_quant")
    return q.view(shape), s.view(shape[:-1])


def add_rms_norm_quant(x: torch.Tensor, residual: Optional[torch.Tensor], weight: torch.Tensor, eps: float,
                       want_y: bool = True, want_quant: bool = False, inplace_residual: bool = False):
    """Stands in for ``npu_add_rms_norm`` / ``npu_rms_norm`` and, with ``want_quant``, the
    ``npu_dynamic_quant`` that follows it (omni/models/common/layers/layernorm.py:13-32).
    Returns (y or None, residual_out or None, x_int8 or None, pertoken_scale or None)."""
    _need_gpu(x, weight)
    if x.dtype != torch.bfloat16 or weight.dtype != torch.bfloat16 or (residual is not None and residual.dtype != torch.bfloat16):
        raise ValueError("add_rms_norm_quant: bf16 tensors only")
    shape = x.shape
    H = shape[-1]
    x2 = x.reshape(-1, H).contiguous()
    rows = x2.shape[0]
    r2 = residual.reshape(-1, H).contiguous() if residual is not None else None
    res_out = None
    if r2 is not None:
        res_out = r2 if inplace_residual else torch.empty_like(r2)
    y = torch.empty_like(x2) if want_y else None
    q = torch.empty(rows, H, dtype=torch.int8, device=x.device) if want_quant else None
    sc = torch.empty(rows, dtype=torch.float32, device=x.device) if want_quant else None
    rc = L.lib().omni_add_rms_norm_quant(_ptr(x2), _ptr(r2), _ptr(weight.contiguous()), rows, H, float(eps),
                                         _ptr(res_out), _ptr(y), _ptr(q), _ptr(sc), _stream())
    L.check(rc, "omni_add_rms_norm_quant")
    return (y.view(shape) if y is not None else None, res_out.view(shape) if res_out is not None else None,
            q.view(shape) if q is not None else None, sc.view(shape[:-1]) if sc is not None else None)



# ----------------------------------------------------------------------------- rows of dense blocks
# The calls below are short on the GPU (a few microseconds for a decode step), so what they ask of torch is counted:
# the raw handle of the current stream instead of a Stream object, no views where shapes agree, one pass over the checks.
def _forward_only(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """The operators have no derivatives: a call that autograd would have to record is refused instead of cutting the
    graph silently, and so is one whose inputs carry tangents (which flow under ``torch.no_grad()`` too)."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f"{what}: no backward pass is built (call it under torch.no_grad() or detach the inputs)")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{what}: no forward-mode derivative is built (an input carries a tangent)")


def _one_device(what: str, x: torch.Tensor, *tensors: Optional[torch.Tensor]) -> int:
    """Index of the GPU that holds all of the tensors."""
    device = x.get_device()   # -1 on the CPU
    if device < 0:
        _need_gpu(x)
    for t in tensors:
        if t is not None and t.get_device() != device:
            _need_gpu(t)
            raise ValueError(f"{what}: tensors on {x.device} and {t.device}")
    return device


def _launch(device: int, what: str, fn, *args) -> None:
    """Calls a library entry on the current stream of ``device``, which is made current where it is not."""
    if device == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        L.check(rc, what)


def _rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``t`` [..., cols] as [rows, cols] with elements of a row side by side and rows that do not overlap; a copy
    only where its strides cannot say that."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    if t.is_contiguous():
        return t
    if (cols > 1 and t.stride(1) != 1) or (t.shape[0] > 1 and t.stride(0) < cols):
        t = t.contiguous()
    return t


def _like(t: torch.Tensor, dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """New rows without gaps of t's shape."""
    if t.is_contiguous():
        return torch.empty_like(t, dtype=dtype)
    return torch.empty(t.shape, dtype=dtype or t.dtype, device=t.device)


def _ld(t: torch.Tensor) -> int:
    """Row stride of a [rows, cols] tensor; a single row's stride says nothing."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two [rows, cols] tensors of one device share an element (columns side by side in one buffer do not)."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    ea, eb = a.element_size(), b.element_size()
    pa, pb = a.data_ptr(), b.data_ptr()
    end_a = pa + ((a.shape[0] - 1) * _ld(a) + a.shape[1]) * ea
    end_b = pb + ((b.shape[0] - 1) * _ld(b) + b.shape[1]) * eb
    if end_a <= pb or end_b <= pa:
        return False
    pitches = {_ld(t) * e for t, e in ((a, ea), (b, eb)) if t.shape[0] > 1}   # a single row has none
    if len(pitches) == 1:
        pitch = pitches.pop()
        at = (pb - pa) % pitch
        return not (at >= a.shape[1] * ea and at + b.shape[1] * eb <= pitch)
    return True


def sandwich_norm(x: torch.Tensor, residual: torch.Tensor, post_weight: torch.Tensor, pre_weight: torch.Tensor,
                  post_eps: float, pre_eps: float, gate: Optional[torch.Tensor] = None, residual_scale: float = 1.0,
                  want_y: bool = True, want_quant: bool = False, inplace_residual: bool = False):
    """The norm after a block, its gate and residual scale, the residual sum and the norm before the next block, in
    one launch: with ``t = rms_norm(x, post_weight)`` and ``r = residual + residual_scale * gate * t``, returns
    (rms_norm(r, pre_weight) or None, r, x_int8 or None, pertoken_scale or None), as ``add_rms_norm_quant`` does.

    ``x``, ``residual`` [..., H], the weights [H] and ``gate`` are of one type (bf16, fp16 or fp32).  ``gate`` is [H] (a
    factor per channel), [..., 1] (per token) or of x's shape.  The sums are fp32 and every output is rounded once: the
    second norm goes by the unrounded r, the int8 rows by the rounded first result.  A row that holds an infinity or a
    NaN has it as its scale and zeros as its int8 values.  ``inplace_residual`` writes r over ``residual``."""
    what = "sandwich_norm"
    device = _one_device(what, x, residual, post_weight, pre_weight, gate)
    _forward_only(what, x, residual, post_weight, pre_weight, gate)
    dt = x.dtype
    if dt not in _DT or residual.dtype != dt or post_weight.dtype != dt or pre_weight.dtype != dt or (
            gate is not None and gate.dtype != dt):
        raise ValueError(f"{what}: all tensors must be of one type out of bf16, fp16 and fp32")
    shape = x.shape
    if len(shape) == 0:
        raise ValueError(f"{what}: x must have at least one dimension")
    H = shape[-1]
    if residual.shape != shape:
        raise ValueError(f"{what}: x and residual differ in shape")
    if post_weight.shape != (H,) or pre_weight.shape != (H,):
        raise ValueError(f"{what}: the weights must be [{H}]")
    x2, r2 = _rows(x, H), _rows(residual, H)
    rows = x2.shape[0]
    mode, ldg, g2 = L.OMNI_GATE_NONE, 0, None
    if gate is not None:
        if gate.shape == (H,):
            mode, g2 = L.OMNI_GATE_CHANNEL, gate.contiguous()
        elif gate.shape == shape:
            g2 = _rows(gate, H)
            mode, ldg = L.OMNI_GATE_FULL, _ld(g2)
        elif gate.shape == (*shape[:-1], 1):
            g2 = gate.reshape(-1, 1)
            g2 = g2.contiguous() if rows > 1 and g2.stride(0) < 1 else g2
            mode, ldg = L.OMNI_GATE_TOKEN, _ld(g2)
        else:
            raise ValueError(f"{what}: the gate must be [{H}], [..., 1] or of x's shape")
    if not (post_weight.is_contiguous() and pre_weight.is_contiguous()):
        post_weight, pre_weight = post_weight.contiguous(), pre_weight.contiguous()
    if inplace_residual:
        if r2.data_ptr() != residual.data_ptr():
            raise ValueError(f"{what}: a residual with these strides cannot be written in place")
        out, res_out = r2, residual
        same = x2.data_ptr() == r2.data_ptr() and _ld(x2) == _ld(r2)
        # rows are worked on in no order: one may read what another has written
        if (not same and _overlap(x2, out)) or (g2 is not None and _overlap(g2 if g2.dim() == 2 else g2.view(1, -1), out)) or (
                _overlap(post_weight.view(1, -1), out) or _overlap(pre_weight.view(1, -1), out)):
            raise ValueError(f"{what}: the residual written in place overlaps another input")
    else:
        out = _like(x2)
        res_out = out if len(shape) == 2 else out.view(shape)
    y = _like(x2) if want_y else None
    q = sc = None
    if want_quant:
        q = _like(x2, torch.int8)
        sc = torch.empty((rows,), dtype=torch.float32, device=x.device)
    _launch(device, "omni_sandwich_norm", L.lib().omni_sandwich_norm, x2.data_ptr(), _DT[dt], _ld(x2), r2.data_ptr(), _ld(r2),
            post_weight.data_ptr(), pre_weight.data_ptr(), _ptr(g2), mode, ldg, rows, H, post_eps, pre_eps, residual_scale,
            out.data_ptr(), _ld(out), _ptr(y), _ptr(q), _ptr(sc))
    if len(shape) != 2:
        y = y.view(shape) if want_y else None
        q, sc = (q.view(shape), sc.view(shape[:-1])) if want_quant else (None, None)
    return y, res_out, q, sc


def swiglu_quant(gate_up: torch.Tensor, want_y: bool = True, want_quant: bool = False):
    """``silu(gate) * up`` of rows [..., 2I] (gate channels first; bf16, fp16 or fp32), rounded once, and with
    ``want_quant`` the ``npu_dynamic_quant`` of the rounded result in the same launch.  Returns (h [..., I] or None,
    x_int8 or None, pertoken_scale or None); a row that holds an infinity or a NaN has it as its scale and zeros as its
    int8 values."""
    what = "swiglu_quant"
    device = _one_device(what, gate_up)
    _forward_only(what, gate_up)
    dt, shape = gate_up.dtype, gate_up.shape
    if dt not in _DT:
        raise ValueError(f"{what}: unsupported dtype {dt}")
    if len(shape) == 0 or shape[-1] % 2 or shape[-1] == 0:
        raise ValueError(f"{what}: rows must hold a gate and an up half")
    I = shape[-1] // 2
    g2 = _rows(gate_up, 2 * I)
    rows = g2.shape[0]
    h = torch.empty((rows, I), dtype=dt, device=gate_up.device) if want_y else None
    q = sc = None
    if want_quant:
        q = torch.empty((rows, I), dtype=torch.int8, device=gate_up.device)
        sc = torch.empty((rows,), dtype=torch.float32, device=gate_up.device)
    _launch(device, "omni_swiglu_quant", L.lib().omni_swiglu_quant, g2.data_ptr(), _DT[dt], _ld(g2), rows, I, _ptr(h), _ptr(q),
            _ptr(sc))
    if len(shape) != 2:
        h = h.view(*shape[:-1], I) if want_y else None
        q, sc = (q.view(*shape[:-1], I), sc.view(shape[:-1])) if want_quant else (None, None)
    return h, q, sc


def npu_swiglu(x: torch.Tensor) -> torch.Tensor:
    """Stands in for ``torch_npu.npu_swiglu`` (omni/models/common/layers/activation.py:29)."""
    return swiglu_quant(x)[0]


# ----------------------------------------------------------------------------- permutation
class Permutation:
    """Result of sorting the (token, k) assignments by local expert."""
    __slots__ = ("sorted_src", "src_to_dst", "counts", "offsets", "T", "K", "n_local", "idx_mode")


def moe_permute(topk_ids: torch.Tensor, lo: int, hi: int, idx_mode: int = L.OMNI_IDX_TOKEN_MAJOR) -> Permutation:
    _need_gpu(topk_ids)
    if topk_ids.dtype != torch.int32:
        topk_ids = topk_ids.to(torch.int32)
    topk_ids = topk_ids.contiguous()
    T, K = topk_ids.shape
    G = hi - lo
    dev = topk_ids.device
    p = Permutation()
    p.T, p.K, p.n_local, p.idx_mode = T, K, G, idx_mode
    p.sorted_src = torch.empty(max(T * K, 1), dtype=torch.int32, device=dev)
    p.src_to_dst = torch.empty(max(T * K, 1), dtype=torch.int32, device=dev)
    p.counts = torch.empty(G, dtype=torch.int32, device=dev)
    p.offsets = torch.empty(G + 1, dtype=torch.int32, device=dev)
    ws_bytes = L.lib().omni_moe_permute_workspace_bytes(T, K, G)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    rc = L.lib().omni_moe_permute(_ptr(topk_ids), T, K, lo, hi, idx_mode, _ptr(p.sorted_src), _ptr(p.src_to_dst),
                                  _ptr(p.counts), _ptr(p.offsets), _ptr(ws), ws_bytes, _stream())
    L.check(rc, "omni_moe_permute")
    return p


def moe_gather_rows(x: torch.Tensor, x_scale: Optional[torch.Tensor], p: Permutation):
    _need_gpu(x)
    x = x.contiguous()
    T, H = x.shape
    rows = torch.zeros(T * p.K, H, dtype=x.dtype, device=x.device)
    sc = torch.zeros(T * p.K, dtype=torch.float32, device=x.device) if x_scale is not None else None
    rc = L.lib().omni_moe_gather_rows(_ptr(x), x.element_size(), H, _ptr(x_scale), _ptr(p.sorted_src),
                                      _ptr(p.offsets), p.n_local, T, p.K, p.idx_mode, _ptr(rows), _ptr(sc), _stream())
    L.check(rc, "omni_moe_gather_rows")
    return rows, sc


def npu_moe_init_routing_v2(x: torch.Tensor, expert_idx: torch.Tensor, scale: Optional[torch.Tensor] = None,
                            active_expert_range=None, expert_num: int = 0, **_unused):
    """Stands in for ``torch_npu.npu_moe_init_routing_v2`` with ``row_idx_type=1``,
    ``expert_tokens_num_type=1``, ``quant_mode=-1`` (fused_moe.py:514-515): returns
    (sorted rows, expanded_x_idx, per-expert counts int64, gathered scale)."""
    lo, hi = active_expert_range if active_expert_range is not None else (0, expert_num)
    p = moe_permute(expert_idx, lo, hi, L.OMNI_IDX_TOKEN_MAJOR)
    rows, sc = moe_gather_rows(x, scale, p)
    return rows, p.sorted_src, p.counts.to(torch.int64), sc


def npu_moe_init_routing(x: torch.Tensor, row_idx: torch.Tensor, expert_idx: torch.Tensor, active_num: int,
                         num_experts: int = 256):
    """Stands in for ``torch_npu.npu_moe_init_routing`` (compressed_tensors_moe.py:235-236):
    returns (sorted rows, expanded_src_to_dst_row indexed by k*T+n, sorted expert ids).
    ``row_idx`` must be the reference's k*T+n numbering (the only one it ever builds,
    compressed_tensors_moe.py:186-187); ``num_experts`` bounds the expert ids (no host sync)."""
    T, K = expert_idx.shape
    p = moe_permute(expert_idx, 0, num_experts, L.OMNI_IDX_K_MAJOR)
    rows, _ = moe_gather_rows(x, None, p)
    sorted_ids = torch.repeat_interleave(torch.arange(p.n_local, device=x.device, dtype=torch.int32),
                                         p.counts.to(torch.int64), output_size=T * K)
    return rows, p.src_to_dst, sorted_ids


def group_offsets(counts: torch.Tensor) -> torch.Tensor:
    """int32 [G+1] row offsets of the groups from their sizes (int32 or int64 [G]): what the reference's grouped
    operators make of ``group_list`` with ``group_list_type=1`` inside (fused_moe.py:531-536)."""
    _need_gpu(counts)
    if counts.dtype not in (torch.int32, torch.int64):
        counts = counts.to(torch.int64)
    counts = counts.contiguous()
    G = counts.numel()
    offsets = torch.empty(G + 1, dtype=torch.int32, device=counts.device)
    rc = L.lib().omni_moe_group_offsets(_ptr(counts), int(counts.dtype == torch.int64), G, _ptr(offsets), _stream())
    L.check(rc, "omni_moe_group_offsets")
    return offsets


def npu_moe_compute_expert_tokens(sorted_expert_idx: torch.Tensor, num_experts: int) -> torch.Tensor:
    """Stands in for ``torch_npu.npu_moe_compute_expert_tokens`` (compressed_tensors_moe.py:237):
    cumulative number of rows up to and including each expert."""
    return group_offsets(torch.bincount(sorted_expert_idx.to(torch.int64), minlength=num_experts))[1:]


_DENSE_OFFSETS = {}


def dense_offsets(M: int, device) -> torch.Tensor:
    """[0, M] int32 on the device: the row grouping of a dense (one group) GEMM.  Cached so that
    the steady state issues no host-to-device copy."""
    key = (int(M), str(device))
    t = _DENSE_OFFSETS.get(key)
    if t is None:
        t = torch.tensor([0, int(M)], dtype=torch.int32, device=device)
        _DENSE_OFFSETS[key] = t
    return t


# ----------------------------------------------------------------------------- adapters
class AdapterPlan:
    """The tokens of a batch sorted by adapter: one buffer with what ``omni_moe_permute`` makes of them."""
    __slots__ = ("T", "n", "buffer", "sorted_src", "offsets",   # the last two: addresses inside the buffer
                 "stream", "joined")   # the stream it was made on (None inside a capture), streams that are behind the sort


def _capturing(device: int) -> bool:
    if device == torch._C._cuda_getDevice():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _join_plan(plan: AdapterPlan, device: int) -> None:
    """Lets the current stream use a plan that was made on another one: what the kernels read from it are places in
    memory, so neither a sort that has not run yet nor memory that was given to someone else may be read.  A stream being
    captured cannot wait for work outside; the capture's own start lies behind the plan."""
    raw = torch._C._cuda_getCurrentRawStream(device)
    if plan.stream is None and not _capturing(device):
        raise RuntimeError("adapter_linear: the plan was made inside a graph capture and holds nothing outside of it")
    if raw in plan.joined:
        return
    stream = torch.cuda.current_stream(device)
    if plan.stream is None:
        plan.joined.add(raw)
    elif not _capturing(device):
        stream.wait_stream(plan.stream)
        plan.joined.add(raw)
    plan.buffer.record_stream(stream)


def adapter_plan(adapter_ids: torch.Tensor, n_adapters: int) -> AdapterPlan:
    """The tokens of a batch sorted by adapter, for ``adapter_linear``: ``adapter_ids`` [T] integers, the adapter of each
    token; a value outside [0, n_adapters) (-1, say) means none.  Made once for a batch and used by all its
    projections, also on other streams: the first use there waits for what the plan's stream has been given so far.  A
    graph that uses a plan made outside of it reads the plan's memory at every replay, so the plan has to live as long
    as the graph; one made inside is made anew by every replay and refused outside of a capture: before the first replay
    it would name places anywhere."""
    device = _one_device("adapter_plan", adapter_ids)
    if adapter_ids.dim() != 1 or adapter_ids.dtype not in (torch.int32, torch.int64):
        raise ValueError("adapter_plan: adapter_ids must be [T], int32 or int64")
    n = int(n_adapters)
    if n < 1:
        raise ValueError("adapter_plan: at least one adapter")
    if adapter_ids.dtype == torch.int64:  # what int32 cannot hold is no adapter either
        adapter_ids = torch.where((adapter_ids >= 0) & (adapter_ids < n), adapter_ids, -1).to(torch.int32)
    adapter_ids = adapter_ids.contiguous()
    lib, p = L.lib(), AdapterPlan()
    p.T, p.n = adapter_ids.shape[0], n
    ws_bytes = lib.omni_moe_permute_workspace_bytes(p.T, 1, n)
    # sorted_src [T], src_to_dst [T], counts [n], offsets [n + 1], then the sort's workspace
    ws_at = (8 * p.T + 8 * n + 4 + 255) // 256 * 256
    p.buffer = torch.empty((ws_at + ws_bytes,), dtype=torch.uint8, device=adapter_ids.device)
    at = p.buffer.data_ptr()
    p.sorted_src, p.offsets = at, at + 8 * p.T + 4 * n
    _launch(device, "omni_moe_permute", lib.omni_moe_permute, adapter_ids.data_ptr(), p.T, 1, 0, n, L.OMNI_IDX_TOKEN_MAJOR, at,
            at + 4 * p.T, at + 8 * p.T, p.offsets, at + ws_at, ws_bytes)
    p.joined = {torch._C._cuda_getCurrentRawStream(device)}
    p.stream = None if _capturing(device) else torch.cuda.current_stream(device)
    return p


def _vector_rows(t: torch.Tensor, cols: int) -> torch.Tensor:
    """``_rows`` for kernels that move 16 bytes at a time: a copy where an alignment forbids that."""
    t = _rows(t, cols)
    if t.data_ptr() % 16 or _ld(t) * t.element_size() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


_WIDTHS = {}


def _widths(slices: tuple):
    """The C array of a projection's slice widths: a constant of the widths, made once."""
    arr = _WIDTHS.get(slices)
    if arr is None:
        if len(_WIDTHS) > 256:
            _WIDTHS.clear()
        arr = _WIDTHS[slices] = (ctypes.c_int32 * len(slices))(*slices)
    return arr


def adapter_linear(x: torch.Tensor, base: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: AdapterPlan,
                   scale: Optional[torch.Tensor] = None, slices=None, out: Optional[torch.Tensor] = None,
                   workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """A shared projection's rows with the low-rank update of each token's adapter:
    ``out[t] = base[t] + scale[g] * (x[t] @ a[g].T) @ b[g].T`` for the adapter g of token t, ``base[t]`` without one.

    ``x`` [..., H] went into the projection, ``base`` [..., N] came out of it.  ``a`` [n, S*r, H] and ``b`` [n, N, r] hold n
    adapters; ``slices`` are the S output widths of a stacked projection (gate and up; default: one slice), whose
    columns take rows j*r..(j+1)*r of ``a``.  ``scale`` [n] fp32 (default 1; an adapter of scale 0 adds nothing, whatever
    the rows and its matrices hold).  bf16 or fp16; H, r and the widths are multiples of 8, r at most 256 (shorter ranks
    are filled up with zeros).  ``out`` may be ``base``.  Both products are summed in fp32 and the result is rounded
    once."""
    what = "adapter_linear"
    device = _one_device(what, x, base, a, b, scale, plan.buffer if plan is not None else None, out, workspace)
    _forward_only(what, x, base, a, b, scale, out)
    dt = x.dtype
    if dt not in (torch.bfloat16, torch.float16) or base.dtype != dt or a.dtype != dt or b.dtype != dt:
        raise ValueError(f"{what}: x, base, a and b must be of one type, bf16 or fp16")
    xs, bs = x.shape, base.shape
    if a.dim() != 3 or b.dim() != 3 or len(xs) == 0 or len(bs) != len(xs):
        raise ValueError(f"{what}: x [..., H], base [..., N], a [n, S*r, H] and b [n, N, r]")
    n, R, H = a.shape
    nb, N, r = b.shape
    if nb != n or xs[-1] != H or bs[-1] != N or xs[:-1] != bs[:-1]:
        raise ValueError(f"{what}: x [..., H], base [..., N], a [n, S*r, H] and b [n, N, r] do not fit")
    widths = (N,) if slices is None else tuple(slices)
    S = len(widths)
    if sum(widths) != N or S * r != R:
        raise ValueError(f"{what}: slices {widths} do not fit {N} columns and {R} = S * {r} rows of a")
    if not (a.is_contiguous() and b.is_contiguous()):
        raise ValueError(f"{what}: a and b must be contiguous")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != (n,) or not scale.is_contiguous()):
        raise ValueError(f"{what}: scale must be a contiguous fp32 [{n}] tensor")
    x2, base2 = _vector_rows(x, H), _vector_rows(base, N)
    T = x2.shape[0]
    if plan.T != T or plan.n != n:
        raise ValueError(f"{what}: the plan is for {plan.T} tokens and {plan.n} adapters, not {T} and {n}")
    _join_plan(plan, device)
    if out is None:
        out2 = _like(base2)
        out = out2 if len(bs) == 2 else out2.view(bs)
    else:
        if out.dtype != dt or out.shape != bs:
            raise ValueError(f"{what}: out must have base's shape and type")
        out2 = _rows(out, N)
        if out2.data_ptr() != out.data_ptr() or out2.data_ptr() % 16 or _ld(out2) % 8:
            raise ValueError(f"{what}: out must have rows of 16-byte aligned, adjacent elements")
        if out2.data_ptr() == base2.data_ptr() and _ld(out2) != _ld(base2) or (
                out2.data_ptr() != base2.data_ptr() and _overlap(out2, base2)) or _overlap(out2, x2):
            raise ValueError(f"{what}: out overlaps an input (it may be base itself)")
    lib = L.lib()
    if workspace is None:
        need = lib.omni_adapter_linear_workspace_bytes(T, n, H, r, S, N)
        if need:
            workspace = torch.empty((need,), dtype=torch.uint8, device=x.device)
    elif not workspace.is_contiguous():
        raise ValueError(f"{what}: the workspace must be contiguous")
    _launch(device, "omni_adapter_linear", lib.omni_adapter_linear, x2.data_ptr(), _DT[dt], _ld(x2), base2.data_ptr(), _ld(base2),
            a.data_ptr(), b.data_ptr(), _ptr(scale), plan.sorted_src, plan.offsets, T, n, H, r, S,
            _widths(widths), out2.data_ptr(), _ld(out2), _ptr(workspace), 0 if workspace is None else workspace.nbytes)
    return out


# ----------------------------------------------------------------------------- weights
def pack_weight(w: torch.Tensor, src_layout: int) -> torch.Tensor:
    """One-off re-layout of int8 weights into the frag16 format the GEMM kernels stream
    (the analogue of ``npu_format_cast(w, 29)``, compressed_tensors_moe.py:97-99).
    src_layout 0: w is [G, Kdim, N]; 1: w is [G, N, Kdim]."""
    _need_gpu(w)
    if w.dtype != torch.int8:
        raise ValueError("pack_weight expects int8 weights")
    if w.dim() == 2:
        w = w.unsqueeze(0)
    w = w.contiguous()
    G = w.shape[0]
    Kdim, N = (w.shape[1], w.shape[2]) if src_layout == 0 else (w.shape[2], w.shape[1])
    out = torch.empty(G, Kdim * N, dtype=torch.int8, device=w.device)
    rc = L.lib().omni_moe_pack_weight(_ptr(w), src_layout, G, Kdim, N, _ptr(out), _stream())
    L.check(rc, "omni_moe_pack_weight")
    return out


# ----------------------------------------------------------------------------- GEMMs
def _quant_scale(quant_scale: Optional[torch.Tensor], G: int, I: int) -> Optional[torch.Tensor]:
    """The ``quant_scale`` of ``npu_dequant_swiglu_quant`` as the library takes it: contiguous fp32 [G, I]."""
    if quant_scale is None:
        return None
    _need_gpu(quant_scale)
    if tuple(quant_scale.shape) != (G, I):
        raise ValueError(f"quant_scale must be [{G}, {I}] (one factor per expert and intermediate channel)")
    return quant_scale.float().contiguous()


def grouped_gemm1_swiglu_quant(x_q: torch.Tensor, x_scale: torch.Tensor, sorted_src: Optional[torch.Tensor],
                               idx_mode: int, K: int, w13_packed: torch.Tensor, w13_scale: torch.Tensor,
                               offsets: torch.Tensor, H: int, I: int, M_cap: int,
                               extra: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, extra_rows: int = 0,
                               bf16_intermediate: bool = False, want_acc: bool = False, flags: int = 0,
                               workspace: Optional[torch.Tensor] = None, out=None,
                               quant_scale: Optional[torch.Tensor] = None):
    """GEMM1 + dequant + SwiGLU + requant: ``npu_grouped_matmul(int32)`` +
    ``npu_dequant_swiglu_quant`` (fused_moe.py:531-534, :670-677).  Returns (h_q, h_scale, acc)."""
    _need_gpu(x_q, x_scale, w13_packed, w13_scale, offsets)
    dev = x_q.device
    T = x_q.shape[0]
    G = offsets.numel() - 1
    if out is None:
        h_q = torch.empty(M_cap, I, dtype=torch.int8, device=dev)
        h_s = torch.empty(M_cap, dtype=torch.float32, device=dev)
    else:
        h_q, h_s = out
    acc = torch.zeros(M_cap, 2 * I, dtype=torch.int32, device=dev) if want_acc else None
    ws_bytes = L.lib().omni_moe_gemm1_workspace_bytes(T, K, G, extra_rows, M_cap, H, I)
    ws = workspace if workspace is not None else torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    ew, es = extra if extra is not None else (None, None)
    quant_scale = _quant_scale(quant_scale, G, I)
    rc = L.lib().omni_moe_gemm1_swiglu_quant(
        _ptr(x_q), _ptr(x_scale), _ptr(sorted_src), idx_mode, T, K, _ptr(w13_packed), _ptr(w13_scale), _ptr(ew),
        _ptr(es), extra_rows, _ptr(offsets), G, H, I, M_cap,
        flags | (L.OMNI_GEMM1_BF16_INTERMEDIATE if bf16_intermediate else 0), _ptr(quant_scale),
        _ptr(h_q), _ptr(h_s), _ptr(acc), _ptr(ws), ws_bytes, _stream())
    L.check(rc, "omni_moe_gemm1_swiglu_quant")
    return h_q, h_s, acc


def grouped_gemm2_dequant(h_q: torch.Tensor, h_scale: torch.Tensor, w2_packed: torch.Tensor, w2_scale: torch.Tensor,
                          offsets: torch.Tensor, H: int, I: int, out_dtype: torch.dtype = torch.bfloat16,
                          extra: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, extra_rows: int = 0,
                          want_acc: bool = False, out: Optional[torch.Tensor] = None,
                          workspace: Optional[torch.Tensor] = None):
    """GEMM2 + dequant: ``npu_grouped_matmul(scale=, per_token_scale=, output_dtype=bf16)``
    (fused_moe.py:570-574, :681-685).  Returns (rows [M_cap, H], acc)."""
    _need_gpu(h_q, h_scale, w2_packed, w2_scale, offsets)
    dev = h_q.device
    M_cap = h_q.shape[0]
    G = offsets.numel() - 1
    # rows past the kept total are never written and never read by a consumer that goes by the offsets
    rows = out if out is not None else torch.empty(M_cap, H, dtype=out_dtype, device=dev)
    acc = torch.zeros(M_cap, H, dtype=torch.int32, device=dev) if want_acc else None
    ew, es = extra if extra is not None else (None, None)
    need = L.lib().omni_moe_gemm2_workspace_bytes(G, extra_rows, M_cap, H, I)
    if workspace is None and need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    rc = L.lib().omni_moe_gemm2_dequant(_ptr(h_q), _ptr(h_scale), _ptr(w2_packed), _ptr(w2_scale), _ptr(ew), _ptr(es),
                                        extra_rows, _ptr(offsets), G, H, I, M_cap, _DT[out_dtype], _ptr(rows),
                                        _ptr(acc), _ptr(workspace), workspace.numel() if workspace is not None else 0,
                                        _stream())
    L.check(rc, "omni_moe_gemm2_dequant")
    return rows, acc


def gemm_kernel_name(kind: int, T: int, K: int, G: int, extra_rows: int, M_cap: int, H: int, I: int) -> str:
    """Template name of the GEMM kernel the library launches for a call of these sizes (diagnostic)."""
    import ctypes
    buf = ctypes.create_string_buffer(64)
    rc = L.lib().omni_moe_gemm_kernel_name(kind, T, K, G, extra_rows, M_cap, H, I, ctypes.addressof(buf), 64)
    L.check(rc, "omni_moe_gemm_kernel_name")
    return buf.value.decode()


def moe_combine(rows: torch.Tensor, topk_w: torch.Tensor, src_to_dst: torch.Tensor, idx_mode: int, order: int,
                init: Optional[torch.Tensor] = None, post_add: Optional[torch.Tensor] = None,
                post_add_row0: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Weighted un-permute: ``npu_moe_finalize_routing`` (compressed_tensors_moe.py:253;
    deepseek_moe.py:292-301) and the routing half of ``npu_grouped_matmul_finalize_routing``
    (fused_moe.py:536).  Returns bf16 [T, H]."""
    _need_gpu(rows, topk_w, src_to_dst)
    T, K = topk_w.shape
    H = rows.shape[1]
    topk_w = topk_w.float().contiguous()
    if init is not None:
        init = init.to(torch.bfloat16).contiguous()
    out = torch.empty(T, H, dtype=torch.bfloat16, device=rows.device)
    rc = L.lib().omni_moe_combine(_ptr(rows), _DT[rows.dtype], _ptr(topk_w), _ptr(src_to_dst), idx_mode, order, T, K, H,
                                  _ptr(init), _ptr(post_add), _ptr(post_add_row0), _ptr(out), _stream())
    L.check(rc, "omni_moe_combine")
    return out


def moe_w8a8_layer(x: torch.Tensor, x_scale: Optional[torch.Tensor], topk_w: torch.Tensor, topk_ids: torch.Tensor,
                   lo: int, hi: int, w13_packed, w13_scale, w2_packed, w2_scale, shared=None, H: int = 0, I: int = 0,
                   workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   rows_dtype: torch.dtype = torch.float32, quant_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The whole local-share layer in one library call (quant if x is bf16, permute, GEMM1
    epilogue, GEMM2, combine), the shared expert carried as an extra group.

    ``rows_dtype`` is how the expert rows travel from GEMM2 to the weighted sum.  ``torch.float32``
    (default) keeps them fp32 and rounds once after the sum: the numerics of
    ``npu_grouped_matmul_finalize_routing`` (fused_moe.py:536).  ``torch.bfloat16`` rounds every row
    first: the numerics of the bf16 ``npu_grouped_matmul`` + ``npu_moe_finalize_routing`` pair
    (fused_moe.py:570-574, deepseek_moe.py:292-301), half the bytes of the largest intermediate."""
    _need_gpu(x, topk_w, topk_ids)
    T, K = topk_ids.shape
    dev = x.device
    x = x.contiguous()
    topk_w = topk_w.float().contiguous()
    topk_ids = topk_ids.to(torch.int32).contiguous()
    x_dtype = -1 if x.dtype == torch.int8 else _DT[x.dtype]
    sh = shared if shared is not None else (None, None, None, None)
    if rows_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("rows_dtype must be torch.float32 or torch.bfloat16")
    need = L.lib().omni_moe_w8a8_layer_workspace_bytes(T, K, hi - lo, H, I, int(shared is not None), _DT[rows_dtype])
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    quant_scale = _quant_scale(quant_scale, hi - lo, I)
    rc = L.lib().omni_moe_w8a8_layer(_ptr(x), x_dtype, _ptr(x_scale), _ptr(topk_w), _ptr(topk_ids), T, K, lo, hi,
                                     _ptr(w13_packed), _ptr(w13_scale), _ptr(w2_packed), _ptr(w2_scale), _ptr(sh[0]),
                                     _ptr(sh[1]), _ptr(sh[2]), _ptr(sh[3]), _ptr(quant_scale), H, I, _DT[rows_dtype],
                                     _ptr(out), _ptr(workspace), workspace.numel(), _stream())
    L.check(rc, "omni_moe_w8a8_layer")
    return out


def moe_w8a8_layer_routed(x: torch.Tensor, x_scale: Optional[torch.Tensor], logits: torch.Tensor,
                          bias: Optional[torch.Tensor], top_k: int, n_group: int, topk_group: int, score_fn: str,
                          group_mode: int, masked_fill_zero: bool, weight_from_c: bool, renorm: bool, scale: float,
                          eps: float, lo: int, hi: int, w13_packed, w13_scale, w2_packed, w2_scale, shared=None,
                          H: int = 0, I: int = 0, workspace: Optional[torch.Tensor] = None,
                          out: Optional[torch.Tensor] = None, rows_dtype: torch.dtype = torch.float32,
                          topk_w: Optional[torch.Tensor] = None, topk_ids: Optional[torch.Tensor] = None):
    """``moe_route`` followed by ``moe_w8a8_layer`` in one library call (``FusedMoE.select_experts`` and the
    quant method's ``apply``: deepseek_moe.py:253-263; layer.py:301-365), the same bits as the two calls.  Small
    calls route, quantise and sort in a single launch.  Returns (out, topk_w, topk_ids)."""
    _need_gpu(x, logits, bias)
    if logits.dim() != 2:
        raise ValueError("router logits must be [T, E]")
    logits = logits.float().contiguous()
    T, E = logits.shape
    if x.shape[0] != T:
        raise ValueError("one row of logits per token")
    if bias is not None:
        bias = bias.float().contiguous()
        if bias.numel() != E:
            raise ValueError("bias must have one entry per expert")
    fn = {"softmax": L.OMNI_SCORE_SOFTMAX, "sigmoid": L.OMNI_SCORE_SIGMOID}.get(score_fn)
    if fn is None:
        raise ValueError(f"Unsupported scoring function: {score_fn}")
    if rows_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("rows_dtype must be torch.float32 or torch.bfloat16")
    dev = x.device
    x = x.contiguous()
    K = int(top_k)
    if topk_w is None:
        topk_w = torch.empty(T, K, dtype=torch.float32, device=dev)
    if topk_ids is None:
        topk_ids = torch.empty(T, K, dtype=torch.int32, device=dev)
    if (topk_w.dtype != torch.float32 or topk_ids.dtype != torch.int32 or tuple(topk_w.shape) != (T, K) or
            tuple(topk_ids.shape) != (T, K) or not topk_w.is_contiguous() or not topk_ids.is_contiguous()):
        raise ValueError("topk_w must be a contiguous fp32 [T, K] tensor and topk_ids a contiguous int32 one")
    x_dtype = -1 if x.dtype == torch.int8 else _DT[x.dtype]
    sh = shared if shared is not None else (None, None, None, None)
    need = L.lib().omni_moe_w8a8_layer_workspace_bytes(T, K, hi - lo, H, I, int(shared is not None), _DT[rows_dtype])
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev)
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    rc = L.lib().omni_moe_w8a8_layer_routed(_ptr(x), x_dtype, _ptr(x_scale), _ptr(logits), _ptr(bias), E, int(n_group),
                                            int(topk_group), fn, int(group_mode), int(masked_fill_zero),
                                            int(weight_from_c), int(renorm), float(scale), float(eps), _ptr(topk_w),
                                            _ptr(topk_ids), T, K, lo, hi, _ptr(w13_packed), _ptr(w13_scale),
                                            _ptr(w2_packed), _ptr(w2_scale), _ptr(sh[0]), _ptr(sh[1]), _ptr(sh[2]),
                                            _ptr(sh[3]), H, I, _DT[rows_dtype], _ptr(out), _ptr(workspace),
                                            workspace.numel(), _stream())
    L.check(rc, "omni_moe_w8a8_layer_routed")
    return out, topk_w, topk_ids


def moe_w8a8_block(x: torch.Tensor, gate_w: torch.Tensor, bias: Optional[torch.Tensor], top_k: int, n_group: int,
                   topk_group: int, score_fn: str, group_mode: int, masked_fill_zero: bool, weight_from_c: bool,
                   renorm: bool, scale: float, eps: float, lo: int, hi: int, w13_packed, w13_scale, w2_packed, w2_scale,
                   shared=None, H: int = 0, I: int = 0, x_int8: Optional[torch.Tensor] = None,
                   pertoken_scale: Optional[torch.Tensor] = None, round_logits_bf16: bool = False,
                   workspace: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                   rows_dtype: torch.dtype = torch.float32, topk_w: Optional[torch.Tensor] = None,
                   topk_ids: Optional[torch.Tensor] = None):
    """The whole block in one library call: ``self.gate.forward(hidden_states.float())``, ``FusedMoE.select_experts``,
    the quant method's ``apply`` and the sum with the shared expert (deepseek_moe.py:147-152, 244-263, 303).  The same
    bits as ``moe_gate_route`` followed by ``moe_w8a8_layer``.  ``x`` [T,H] bf16 (or fp32 together with ``x_int8`` /
    ``pertoken_scale``, the tokens already quantised).  Returns (out, topk_w, topk_ids)."""
    _need_gpu(x, gate_w, bias, x_int8, pertoken_scale)
    if x.dim() != 2 or gate_w.dim() != 2 or x.shape[1] != gate_w.shape[1]:
        raise ValueError("block: x must be [T, H] and the gate weight [E, H]")
    if x.dtype not in (torch.bfloat16, torch.float32) or gate_w.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("block: tokens and gate weight must be bf16 or fp32")
    if (x_int8 is None) != (pertoken_scale is None):
        raise ValueError("block: quantised tokens and their scales come together")
    x = x.contiguous()
    gate_w = gate_w.contiguous()
    T, E, K, dev = x.shape[0], gate_w.shape[0], int(top_k), x.device
    if x_int8 is not None:
        x_int8 = x_int8.contiguous()
        pertoken_scale = pertoken_scale.float().reshape(-1).contiguous()
    if bias is not None:
        bias = bias.float().contiguous()
        if bias.numel() != E:
            raise ValueError("bias must have one entry per expert")
    fn = {"softmax": L.OMNI_SCORE_SOFTMAX, "sigmoid": L.OMNI_SCORE_SIGMOID}.get(score_fn)
    if fn is None:
        raise ValueError(f"Unsupported scoring function: {score_fn}")
    if rows_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("rows_dtype must be torch.float32 or torch.bfloat16")
    if topk_w is None:
        topk_w = torch.empty(T, K, dtype=torch.float32, device=dev)
    if topk_ids is None:
        topk_ids = torch.empty(T, K, dtype=torch.int32, device=dev)
    sh = shared if shared is not None else (None, None, None, None)
    need = L.lib().omni_moe_w8a8_block_workspace_bytes(T, K, hi - lo, H, I, E, int(shared is not None), _DT[rows_dtype])
    if workspace is None or workspace.numel() < need:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=dev)
    rc = L.lib().omni_moe_w8a8_block(_ptr(x), _DT[x.dtype], _ptr(x_int8), _ptr(pertoken_scale), _ptr(gate_w),
                                     _DT[gate_w.dtype], _ptr(bias), E, int(n_group), int(topk_group), fn, int(group_mode),
                                     int(masked_fill_zero), int(weight_from_c), int(renorm), float(scale), float(eps),
                                     int(round_logits_bf16), _ptr(topk_w), _ptr(topk_ids), T, K, lo, hi, _ptr(w13_packed),
                                     _ptr(w13_scale), _ptr(w2_packed), _ptr(w2_scale), _ptr(sh[0]), _ptr(sh[1]), _ptr(sh[2]),
                                     _ptr(sh[3]), H, I, _DT[rows_dtype], _ptr(out), _ptr(workspace), workspace.numel(),
                                     _stream())
    L.check(rc, "omni_moe_w8a8_block")
    return out, topk_w, topk_ids


def moe_w8a8_layer_static(x: torch.Tensor, x_scale: Optional[torch.Tensor], topk_w: torch.Tensor, topk_ids: torch.Tensor,
                          lo: int, hi: int, w13_packed, w13_scale, w2_packed, w2_scale, shared=None, H: int = 0,
                          I: int = 0, out: Optional[torch.Tensor] = None,
                          rows_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """``moe_w8a8_layer`` on the library's static scratch: the call allocates nothing on the device
    when ``out`` is given and the inputs are already fp32 / int32 / contiguous.  Sizes that need more
    than ``OMNI_STATIC_SCRATCH_BYTES`` of scratch raise RuntimeError.  Calls that overlap in time on
    one GPU share the scratch and race; calls on one stream are safe."""
    _need_gpu(x, topk_w, topk_ids)
    T, K = topk_ids.shape
    if not (x.is_contiguous() and topk_w.is_contiguous() and topk_ids.is_contiguous() and
            topk_w.dtype == torch.float32 and topk_ids.dtype == torch.int32):
        raise ValueError("moe_w8a8_layer_static: contiguous inputs, fp32 weights and int32 ids only (no conversion "
                         "copies are made here)")
    if rows_dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("rows_dtype must be torch.float32 or torch.bfloat16")
    x_dtype = -1 if x.dtype == torch.int8 else _DT[x.dtype]
    sh = shared if shared is not None else (None, None, None, None)
    if out is None:
        out = torch.empty(T, H, dtype=torch.bfloat16, device=x.device)
    rc = L.lib().omni_moe_w8a8_layer_static(_ptr(x), x_dtype, _ptr(x_scale), _ptr(topk_w), _ptr(topk_ids), T, K, lo, hi,
                                            _ptr(w13_packed), _ptr(w13_scale), _ptr(w2_packed), _ptr(w2_scale),
                                            _ptr(sh[0]), _ptr(sh[1]), _ptr(sh[2]), _ptr(sh[3]), H, I, _DT[rows_dtype],
                                            _ptr(out), _stream())
    L.check(rc, "omni_moe_w8a8_layer_static")
    return out


# ----------------------------------------------------------------------------- expert placement
def placement_tables(pattern: torch.Tensor, rank: int, devices_per_host: int, num_deploy: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Host tables of a placement pattern [world, layers, experts] (0/1, CPU): ``position_to_expert``
    [layers, num_deploy] (-1: unused position) and ``selector`` [layers, experts], the position ``rank`` routes
    each logical expert to (placement_mapping.cpp:223-257, :374-427).  Both are CPU int32 tensors."""
    if pattern.is_cuda or pattern.dim() != 3:
        raise ValueError("placement pattern must be a CPU tensor [world, layers, experts]")
    pat = pattern.to(torch.int32).contiguous()
    world, layers, experts = pat.shape
    pos = torch.empty(layers, max(int(num_deploy), 0), dtype=torch.int32)
    sel = torch.empty(layers, experts, dtype=torch.int32)
    rc = L.lib().omni_placement_tables(pat.data_ptr(), world, layers, experts, int(rank), int(devices_per_host),
                                       int(num_deploy), pos.data_ptr(), sel.data_ptr())
    L.check(rc, "omni_placement_tables")
    return pos, sel


def remap_ids(ids: torch.Tensor, expert_map: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``embedding(ids, expert_map).squeeze(-1)`` of OmniPlanner.plan (omni_planner.py:273): every id becomes
    ``expert_map[id]``; int32 in, int32 out (``out`` may be ``ids``)."""
    _need_gpu(ids, expert_map)
    if ids.dtype != torch.int32:
        ids = ids.to(torch.int32)
    ids = ids.contiguous()
    expert_map = expert_map.reshape(-1)
    if expert_map.dtype != torch.int32 or not expert_map.is_contiguous():
        expert_map = expert_map.to(torch.int32).contiguous()
    if out is None:
        out = torch.empty_like(ids)
    elif out.dtype != torch.int32 or not out.is_contiguous() or out.numel() != ids.numel():
        raise ValueError("remap_ids: out must be a contiguous int32 tensor of the ids' size")
    rc = L.lib().omni_moe_remap_ids(_ptr(ids), ids.numel(), _ptr(expert_map), expert_map.numel(), _ptr(out), _stream())
    L.check(rc, "omni_moe_remap_ids")
    return out


def record_activation(counts: torch.Tensor, tokens_per_expert: torch.Tensor, modulus: int) -> torch.Tensor:
    """``counts = (counts + tokens_per_expert) % modulus`` in place (omni_planner.py:337-343): int64 counters of
    one layer, int32 token counts of the rank's deployed experts."""
    _need_gpu(counts, tokens_per_expert)
    if counts.dtype != torch.int64 or not counts.is_contiguous():
        raise ValueError("record_activation: counts must be a contiguous int64 tensor (it is updated in place)")
    n = counts.numel()
    if tokens_per_expert.numel() != n:
        raise ValueError("record_activation: one token count per counter")
    if tokens_per_expert.dtype != torch.int32 or not tokens_per_expert.is_contiguous():
        tokens_per_expert = tokens_per_expert.to(torch.int32).contiguous()
    rc = L.lib().omni_moe_record_activation(_ptr(counts), _ptr(tokens_per_expert), n, int(modulus), _stream())
    L.check(rc, "omni_moe_record_activation")
    return counts
