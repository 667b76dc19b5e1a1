"""Dense / elementwise building blocks of the prefill layer loop behind the reference's function names
(python/krasis/weight_loader.py: quantize_to_int8, int8_linear; python/krasis/layer.py: norms, shared expert).
Every function launches libkrasis_b200 kernels; torch only owns the buffers."""
from typing import Optional, Tuple

import torch

from . import capi
from .streams import stream_of as _s, stream_on


def _dev(t):
    return t.device.index or 0


def _chk_bf16(t, name):
    if not t.is_cuda or t.dtype != torch.bfloat16 or t.dim() != 2 or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous 2-D CUDA bf16 tensor (krasis_b200 has no CPU path)")


def rmsnorm(x: torch.Tensor, weight_f32: torch.Tensor, eps: float, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """flashinfer.norm.rmsnorm(x, w, eps) (layer.py:163-165)."""
    _chk_bf16(x, "x")
    out = torch.empty_like(x) if out is None else out
    capi.check(capi.load().kb2_rmsnorm(x.data_ptr(), None, weight_f32.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1],
                                       float(eps), _dev(x), _s(x)))
    return out


def fused_add_rmsnorm(x: torch.Tensor, residual: torch.Tensor, weight_f32: torch.Tensor, eps: float) -> None:
    """flashinfer.norm.fused_add_rmsnorm — IN PLACE: residual += x; x = rmsnorm(residual) * w (layer.py:283-285)."""
    _chk_bf16(x, "x")
    _chk_bf16(residual, "residual")
    capi.check(capi.load().kb2_rmsnorm(x.data_ptr(), residual.data_ptr(), weight_f32.data_ptr(), x.data_ptr(), x.shape[0],
                                       x.shape[1], float(eps), _dev(x), _s(x)))


def fused_add_rmsnorm_q8(x: torch.Tensor, residual: torch.Tensor, weight_f32: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """fused_add_rmsnorm that also returns the INT8 row quantisation (q int8 [M,H], scale f32 [M]) of the normed rows — exactly what
    int8_linear (weight_loader.py:46-99) would compute from them, so the shared expert's first GEMM skips its quantisation pass."""
    _chk_bf16(x, "x")
    _chk_bf16(residual, "residual")
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    qs = torch.empty(x.shape[0], dtype=torch.float32, device=x.device)
    capi.check(capi.load().kb2_rmsnorm_q8(x.data_ptr(), residual.data_ptr(), weight_f32.data_ptr(), x.data_ptr(), q.data_ptr(), qs.data_ptr(),
                                          x.shape[0], x.shape[1], float(eps), _dev(x), _s(x)))
    return q, qs


def sum_slots(slots_ptr: int, world: int, rows: int, hidden: int, device: torch.device) -> torch.Tensor:
    """bf16(sum over the `world` partial rows of every token) from a peer-filled receive buffer [rows][world][hidden] bf16."""
    out = torch.empty((rows, hidden), dtype=torch.bfloat16, device=device)
    capi.check(capi.load().kb2_sum_slots_bf16(slots_ptr, world, out.data_ptr(), rows, hidden, device.index or 0,
                                              stream_on(device)))
    return out


def quantize_to_int8(weight_bf16: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """weight_loader.py:25-43: per-row symmetric INT8; returns (int8 [N,K], scale bf16 [N])."""
    _chk_bf16(weight_bf16, "weight")
    n, k = weight_bf16.shape
    q = torch.empty((n, k), dtype=torch.int8, device=weight_bf16.device)
    s = torch.empty(n, dtype=torch.bfloat16, device=weight_bf16.device)
    capi.check(capi.load().kb2_quantize_rows_int8(weight_bf16.data_ptr(), q.data_ptr(), None, s.data_ptr(), n, k,
                                                  _dev(weight_bf16), _s(weight_bf16)))
    return q, s


def int8_linear(x: torch.Tensor, weight_int8: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """weight_loader.py:46-99 (W8A8, bias-free)."""
    _chk_bf16(x, "x")
    m, k = x.shape
    n = weight_int8.shape[0]
    out = torch.empty((m, n), dtype=torch.bfloat16, device=x.device)
    xq = torch.empty((m, k), dtype=torch.int8, device=x.device)
    xs = torch.empty(m, dtype=torch.float32, device=x.device)
    capi.check(capi.load().kb2_int8_linear(x.data_ptr(), weight_int8.data_ptr(), scale.data_ptr(), out.data_ptr(),
                                           xq.data_ptr(), xs.data_ptr(), m, n, k, _dev(x), _s(x)))
    return out


def int8_linear_q8(xq: torch.Tensor, xs: torch.Tensor, weight_int8: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """int8_linear on an activation that is already row-quantised (xq int8 [M,K], xs f32 [M])."""
    m, k = xq.shape
    n = weight_int8.shape[0]
    out = torch.empty((m, n), dtype=torch.bfloat16, device=xq.device)
    capi.check(capi.load().kb2_int8_linear_q8(xq.data_ptr(), xs.data_ptr(), weight_int8.data_ptr(), scale.data_ptr(), out.data_ptr(),
                                              m, n, k, _dev(xq), _s(xq)))
    return out


def silu_mul_int8_linear(gate_up: torch.Tensor, weight_int8: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """int8_linear(silu(gate) * up, W) with the activation quantised straight from the [M, 2K] gate|up rows (bit-identical to
    silu_and_mul followed by int8_linear)."""
    _chk_bf16(gate_up, "gate_up")
    m, k = gate_up.shape[0], gate_up.shape[1] // 2
    n = weight_int8.shape[0]
    out = torch.empty((m, n), dtype=torch.bfloat16, device=gate_up.device)
    xq = torch.empty((m, k), dtype=torch.int8, device=gate_up.device)
    xs = torch.empty(m, dtype=torch.float32, device=gate_up.device)
    act = None if k in (256, 512, 1024, 2048) else torch.empty((m, k), dtype=torch.bfloat16, device=gate_up.device)
    capi.check(capi.load().kb2_silu_mul_int8_linear(gate_up.data_ptr(), weight_int8.data_ptr(), scale.data_ptr(), out.data_ptr(),
                                                    act.data_ptr() if act is not None else None, xq.data_ptr(), xs.data_ptr(), m, n, k,
                                                    _dev(gate_up), _s(gate_up)))
    return out


def silu_and_mul(x: torch.Tensor) -> torch.Tensor:
    _chk_bf16(x, "x")
    out = torch.empty((x.shape[0], x.shape[1] // 2), dtype=torch.bfloat16, device=x.device)
    capi.check(capi.load().kb2_silu_and_mul(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1] // 2, _dev(x), _s(x)))
    return out


# ------------------------------------------------------------------------------------------------ 8-bit floating-point products, a scale per block of 128

FP8_BLOCK = 128
_fp8_sizes = {}        # workspace bytes of fp8_linear by (rows, numbers of a row)


def _fp8_blocks(n: int) -> int:
    return (n + FP8_BLOCK - 1) // FP8_BLOCK


def _rows_of(m, k, dtype, device):
    """torch.empty((m, k)) in 1.6 us instead of 2.4."""
    return torch.empty_strided((m, k), (k, 1), dtype=dtype, device=device)


def _f32_code(t, name) -> int:
    if t.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError(f"{name}: {t.dtype}, expected bfloat16 or float32")
    return int(t.dtype is torch.float32)


def _fp8_device(name, first, *others) -> int:
    """The CUDA device that all tensors (None: not given) are on."""
    dev = first.get_device()
    for t in others:
        if t is not None and t.get_device() != dev:
            dev = -1
    if dev < 0:
        raise ValueError(f"{name}: the tensors belong on one CUDA device (krasis_b200 has no CPU path)")
    return dev


def _fp8_input(name, x):
    if x.dim() != 2 or (x.stride(1) != 1 and x.shape[1] != 1):
        raise ValueError(f"{name}: rows [M, K] whose numbers lie side by side, got {tuple(x.shape)} with strides {x.stride()}")
    m, k = x.shape
    if k == 0 or k % 16:
        raise ValueError(f"{name}: rows of {k} numbers, a multiple of 16 is needed")
    return m, k


def _fp8_matrix(name, w, scales, *shape):
    """Codes of `shape` and a scale per block of 128 x 128 of its last two axes."""
    want = (*shape[:-2], (shape[-2] + 127) // 128, (shape[-1] + 127) // 128)
    if w.dtype is not torch.float8_e4m3fn or w.shape != shape or not w.is_contiguous():
        raise ValueError(f"{name}: contiguous float8_e4m3fn weights {shape}, got {w.dtype} {tuple(w.shape)}")
    if scales.dtype is not torch.float32 or scales.shape != want or not scales.is_contiguous():
        raise ValueError(f"{name}: contiguous float32 scales {want}, got {scales.dtype} {tuple(scales.shape)}")


def quantize_fp8_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (bfloat16 or float32, any row stride, K a multiple of 16) in 8 bits: (codes [M, K] float8_e4m3fn, scales [M, ceil(K / 128)] float32, one for
    each 128 numbers of a row).  A block's scale is the least 2^k, k >= -126, that its largest magnitude is at most 448 times of; a block of zeros has scale 0, one
    with a number that is not finite scale NaN and codes 0.  The scales of one block of all rows lie side by side: strides (1, rows rounded up to 4)."""
    m, k = _fp8_input("quantize_fp8_rows", x)
    f32, dev, device, ld = _f32_code(x, "quantize_fp8_rows"), _fp8_device("quantize_fp8_rows", x), x.device, (m + 3) // 4 * 4
    codes = _rows_of(m, k, torch.float8_e4m3fn, device)
    scales = torch.empty_strided((m, _fp8_blocks(k)), (1, ld), dtype=torch.float32, device=device)
    capi.check(capi.load().kb2_fp8_quantize_rows(x.data_ptr(), f32, x.stride(0), m, k, codes.data_ptr(), scales.data_ptr(), ld, dev, stream_on(dev)))
    return codes, scales


def quantize_fp8_blocks(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """A matrix [N, K] or a stack of them [E, N, K] (bfloat16 or float32, contiguous, K a multiple of 16) in 8 bits: codes of that shape, and a scale for each block of
    128 x 128 by the rule of quantize_fp8_rows."""
    if w.dim() not in (2, 3) or not w.is_contiguous() or w.shape[-1] == 0 or w.shape[-2] == 0 or w.shape[-1] % 16:
        raise ValueError(f"quantize_fp8_blocks: contiguous [N, K] or [E, N, K] with K a multiple of 16, got {tuple(w.shape)}")
    f32, dev, (n, k) = _f32_code(w, "quantize_fp8_blocks"), _fp8_device("quantize_fp8_blocks", w), w.shape[-2:]
    e, nn, kk, device = w.shape[0] if w.dim() == 3 else 1, _fp8_blocks(n), _fp8_blocks(k), w.device
    if w.dim() == 2:
        codes, scales = _rows_of(n, k, torch.float8_e4m3fn, device), _rows_of(nn, kk, torch.float32, device)
    else:
        codes = torch.empty(w.shape, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty((e, nn, kk), dtype=torch.float32, device=device)
    capi.check(capi.load().kb2_fp8_quantize_blocks(w.data_ptr(), f32, e, n, k, codes.data_ptr(), scales.data_ptr(), dev, stream_on(dev)))
    return codes, scales


def _fp8_out(name, x, n, bias, out_dtype):
    if bias is not None and (bias.dtype is not torch.float32 or tuple(bias.shape) != (n,) or not bias.is_contiguous()):
        raise ValueError(f"{name}: a float32 bias [{n}]")
    out = _rows_of(x.shape[0], n, out_dtype, x.device)
    return out, _f32_code(out, name)


def fp8_linear(x: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None, out_dtype=None) -> torch.Tensor:
    """x [M, K] (bfloat16 or float32) times a matrix that is held in 8 bits, weight [N, K] float8_e4m3fn with any fp32 scales [ceil(N / 128), ceil(K / 128)], plus bias
    [N] float32: [M, N] in out_dtype (x's own).  The rows are quantised as by quantize_fp8_rows; sums are fp32."""
    m, k = _fp8_input("fp8_linear", x)
    n = weight.shape[0]
    _fp8_matrix("fp8_linear", weight, weight_scales, n, k)
    f32, dev = _f32_code(x, "fp8_linear"), _fp8_device("fp8_linear", x, weight, weight_scales, bias)
    out, o32 = _fp8_out("fp8_linear", x, n, bias, x.dtype if out_dtype is None else out_dtype)
    lib, size = capi.load(), _fp8_sizes.get((m, k))
    if size is None:
        if len(_fp8_sizes) >= 4096:
            _fp8_sizes.clear()
        size = _fp8_sizes[m, k] = lib.kb2_fp8_linear_workspace(m, k)
    work = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=x.device)
    capi.check(lib.kb2_fp8_linear(x.data_ptr(), f32, x.stride(0), weight.data_ptr(), weight_scales.data_ptr(), None if bias is None else bias.data_ptr(), out.data_ptr(), o32,
                                  m, n, k, work.data_ptr(), size, dev, stream_on(dev)))
    return out


def fp8_linear_rows(codes: torch.Tensor, scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                    out_dtype=torch.bfloat16) -> torch.Tensor:
    """fp8_linear on rows that are quantised already: codes [M, K] float8_e4m3fn and scales [M, ceil(K / 128)] float32 (in the order that quantize_fp8_rows leaves them;
    others are copied into it)."""
    m, k = _fp8_input("fp8_linear_rows", codes)
    n = weight.shape[0]
    if codes.dtype is not torch.float8_e4m3fn or not codes.is_contiguous() or scales.dtype is not torch.float32 or tuple(scales.shape) != (m, _fp8_blocks(k)):
        raise ValueError(f"fp8_linear_rows: contiguous float8_e4m3fn codes [M, K] and float32 scales [M, {_fp8_blocks(k)}]")
    _fp8_matrix("fp8_linear_rows", weight, weight_scales, n, k)
    dev = _fp8_device("fp8_linear_rows", codes, scales, weight, weight_scales, bias)
    out, o32 = _fp8_out("fp8_linear_rows", codes, n, bias, out_dtype)
    if scales.stride(0) != 1 or scales.stride(1) % 4 or scales.stride(1) < m or scales.data_ptr() % 16:
        kept = torch.empty((scales.shape[1], (m + 3) // 4 * 4), dtype=torch.float32, device=codes.device)
        scales = kept.t()[:m].copy_(scales)
    capi.check(capi.load().kb2_fp8_linear_rows(codes.data_ptr(), scales.data_ptr(), scales.stride(1), weight.data_ptr(), weight_scales.data_ptr(),
                                               None if bias is None else bias.data_ptr(), out.data_ptr(), o32, m, n, k, dev, stream_on(dev)))
    return out


def fp8_experts(h: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, w_gate_up: torch.Tensor, s_gate_up: torch.Tensor, w_down: torch.Tensor, s_down: torch.Tensor,
                out_dtype=None) -> torch.Tensor:
    """Routed experts whose matrices are held in 8 bits: out[t] = sum_j weights[t, j] down_e(q(silu(gate_e q(h[t])) * up_e q(h[t]))) with e = ids[t, j] and q the
    quantisation of quantize_fp8_rows.  h [T, W] bfloat16 or float32; ids [T, top] int32, those outside [0, E) bring nothing; weights [T, top] float32; w_gate_up
    [E, 2 F, W] = [gate ; up] and w_down [E, W, F] float8_e4m3fn, with a scale for each block of 128 x 128; W a multiple of 16, F of 128, at most 1024 experts.
    [T, W] in out_dtype (h's own); sums are fp32 and a bfloat16 result is rounded once."""
    T, W = _fp8_input("fp8_experts", h)
    if w_gate_up.dim() != 3 or w_gate_up.shape[1] % 256 or w_gate_up.shape[1] == 0:
        raise ValueError(f"fp8_experts: gate and up projections [E, 2 F, W] with F a multiple of 128, got {tuple(w_gate_up.shape)}")
    E, F = w_gate_up.shape[0], w_gate_up.shape[1] // 2
    _fp8_matrix("fp8_experts", w_gate_up, s_gate_up, E, 2 * F, W)
    _fp8_matrix("fp8_experts", w_down, s_down, E, W, F)
    if ids.dtype is not torch.int32 or ids.dim() != 2 or ids.shape[0] != T or ids.shape[1] == 0 or not ids.is_contiguous():
        raise ValueError(f"fp8_experts: contiguous int32 ids [{T}, top]")
    if weights.dtype is not torch.float32 or weights.shape != ids.shape or not weights.is_contiguous():
        raise ValueError(f"fp8_experts: contiguous float32 weights {tuple(ids.shape)}")
    dev = _fp8_device("fp8_experts", h, ids, weights, w_gate_up, s_gate_up, w_down, s_down)
    out = _rows_of(T, W, h.dtype if out_dtype is None else out_dtype, h.device)
    f32, o32, top, lib = _f32_code(h, "fp8_experts"), _f32_code(out, "fp8_experts"), ids.shape[1], capi.load()
    size = lib.kb2_fp8_experts_workspace(T, top, E, W, F, o32)
    work = torch.empty_strided((size,), (1,), dtype=torch.uint8, device=h.device)
    capi.check(lib.kb2_fp8_experts(h.data_ptr(), f32, h.stride(0), ids.data_ptr(), weights.data_ptr(), w_gate_up.data_ptr(), s_gate_up.data_ptr(), w_down.data_ptr(),
                                   s_down.data_ptr(), out.data_ptr(), o32, T, top, E, W, F, work.data_ptr(), size, dev, stream_on(dev)))
    return out


class SharedExpert:
    """TransformerLayer._shared_expert_forward (layer.py:508-524): INT8 gate_up / down + optional sigmoid gate."""

    def __init__(self, gate_up_proj_bf16: torch.Tensor, down_proj_bf16: torch.Tensor, shared_expert_gate: Optional[torch.Tensor] = None):
        self.gate_up = quantize_to_int8(gate_up_proj_bf16.contiguous())
        self.down = quantize_to_int8(down_proj_bf16.contiguous())
        self.gate = shared_expert_gate.reshape(-1).contiguous() if shared_expert_gate is not None else None

    def forward(self, hidden: torch.Tensor, hidden_q8=None) -> torch.Tensor:
        """hidden_q8 = (q, scale) from fused_add_rmsnorm_q8 when the caller's norm already quantised these rows."""
        gu = int8_linear_q8(hidden_q8[0], hidden_q8[1], *self.gate_up) if hidden_q8 is not None else int8_linear(hidden, *self.gate_up)
        out = silu_mul_int8_linear(gu, *self.down)
        if self.gate is not None:
            capi.check(capi.load().kb2_sigmoid_gate_mul(hidden.data_ptr(), self.gate.data_ptr(), out.data_ptr(), hidden.shape[0],
                                                         hidden.shape[1], out.shape[1], _dev(hidden), _s(hidden)))
        return out
