"""PyTorch-facing wrapper of the C ABI: tensors in, bf16 tensor out, work enqueued on the current
CUDA stream.  PyTorch supplies device memory and streams only; the arithmetic is the library's.

Mirrors the call the reference backends make,
`triton_fp8_row(xq, wq, x_scale, w_scale, bias=...)` / `torch.ops.fbgemm.f8f8bf16_rowwise(...)`
(tritonbench/operators/fp8_gemm_rowwise/operator.py:187-217): same argument order and meaning,
a fresh bf16 [M, N] tensor as the result.
"""
from typing import Callable, Dict, Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad as _forward_ad

from . import lib as _lib

_workspaces: Dict[Tuple[int, int], torch.Tensor] = {}


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the library has no CPU path)")


def get_workspace(device: torch.device, nbytes: int, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Zero-initialised workspace for (device, stream); grown, never shrunk.  Calls that share a
    workspace must be ordered on one stream, which is why it is keyed by stream."""
    stream = stream or torch.cuda.current_stream(device)
    key = (device.index if device.index is not None else torch.cuda.current_device(), stream.cuda_stream)
    ws = _workspaces.get(key)
    if ws is None or ws.numel() < nbytes:
        size = max(nbytes, _lib.WORKSPACE_HEADER_BYTES)
        ws = torch.zeros(size, dtype=torch.uint8, device=device)
        _workspaces[key] = ws
    return ws


def workspace_bytes(m: int, n: int, k: int, flags: int = 0) -> int:
    nbytes = _lib.load().b200fp8_workspace_bytes(m, n, k, flags)
    if nbytes == 0:
        raise ValueError(f"no plan for M={m} N={n} K={k} flags={flags:#x}")
    return nbytes


def _flags(variant: str, tma_store: bool, overlap: bool = False, split_config: Optional[Tuple[int, int]] = None) -> int:
    if variant not in _lib.VARIANTS:
        raise ValueError(f"unknown variant {variant!r}; one of {sorted(_lib.VARIANTS)}")
    flags = _lib.VARIANTS[variant] | (0 if tma_store else _lib.FLAG_NO_TMA_STORE) | (_lib.FLAG_PDL if overlap else 0)
    if split_config is not None:
        flags |= _lib.flag_splitk_config(*split_config)
    return flags


def fp8_gemm_rowwise(
    xq: torch.Tensor,
    wq: torch.Tensor,
    x_scale: torch.Tensor,
    w_scale: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    variant: str = "auto",
    tma_store: bool = True,
    workspace: Optional[torch.Tensor] = None,
    overlap: bool = False,
    out_dtype: torch.dtype = torch.bfloat16,
    split_config: Optional[Tuple[int, int]] = None,
) -> torch.Tensor:
    """Y = bf16((xq @ wq.T) * x_scale[:, None] * w_scale[None, :] (+ bias)), fp32 accumulation.
    out_dtype=torch.float16 rounds the result to IEEE fp16 instead of bf16.

    overlap=True (decode shapes): the kernel may start before the previous kernel on the stream has
    finished and reads wq - nothing else - that early; pass it only when nothing in flight writes wq.
    split_config=(block_n, split) forces the tile width and cluster size of the tc_splitk kernel.

    xq [M, K] and wq [N, K] are float8_e4m3fn (or uint8 holding e4m3 bytes) with K contiguous;
    x_scale [M], w_scale [N] float32; bias [N] bfloat16 or None.  Asynchronous on the current stream.
    """
    for t, name in ((xq, "xq"), (wq, "wq"), (x_scale, "x_scale"), (w_scale, "w_scale")):
        _require_cuda(t, name)
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"xq {tuple(xq.shape)} and wq {tuple(wq.shape)} must be [M, K] and [N, K]")
    if xq.element_size() != 1 or wq.element_size() != 1:
        raise ValueError("xq and wq must hold one byte per element (float8_e4m3fn)")
    if xq.stride(1) != 1 or wq.stride(1) != 1:
        raise ValueError("xq and wq must have K contiguous")
    m, k = xq.shape
    n = wq.shape[0]
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise ValueError("scales must be float32")
    if x_scale.numel() != m or w_scale.numel() != n:
        raise ValueError("x_scale must have M elements and w_scale N elements")
    x_scale = x_scale.contiguous()
    w_scale = w_scale.contiguous()
    if bias is not None:
        _require_cuda(bias, "bias")
        if bias.dtype != torch.bfloat16 or bias.numel() != n:
            raise ValueError("bias must be bfloat16 with N elements")
        bias = bias.contiguous()
    if out_dtype not in (torch.bfloat16, torch.float16):
        raise ValueError("out_dtype must be bfloat16 or float16")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=xq.device)
    elif out.dtype != out_dtype or tuple(out.shape) != (m, n) or out.stride(1) != 1:
        raise ValueError(f"out must be {out_dtype} [M, N] with N contiguous")

    flags = _flags(variant, tma_store, overlap, split_config) | (_lib.FLAG_OUT_FP16 if out_dtype == torch.float16 else 0)
    lib = _lib.load()
    if workspace is None:
        workspace = get_workspace(xq.device, workspace_bytes(m, n, k, flags))
    stream = torch.cuda.current_stream(xq.device).cuda_stream
    status = lib.b200fp8_gemm_rowwise(
        xq.data_ptr(), wq.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(),
        bias.data_ptr() if bias is not None else None, out.data_ptr(),
        m, n, k, xq.stride(0), wq.stride(0), out.stride(0),
        workspace.data_ptr(), workspace.numel(), flags, stream,
    )
    _lib.check(status, f"b200fp8_gemm_rowwise(M={m}, N={n}, K={k}, variant={variant})")
    return out


def fp8_gemm_rowwise_gather(
    xq: torch.Tensor,
    wq: torch.Tensor,
    x_scale: torch.Tensor,
    w_scale: torch.Tensor,
    y_copies: Sequence[int],
    ldy: int,
    bias: Optional[torch.Tensor] = None,
    variant: str = "auto",
    workspace: Optional[torch.Tensor] = None,
) -> None:
    """The GEMM with every tile of Y stored into several buffers at once (b200fp8_gemm_rowwise_gather): the fused
    form of GEMM + all-gather of a run sharded by rows.  y_copies are device addresses (valid in this process; the
    first one local, the others usually peer GPUs' memory mapped through dist.SharedRows) of where this call's M
    rows belong in each copy of the gathered matrix; ldy is their common row pitch in elements.  Asynchronous on the
    current stream; the ranks must synchronise with each other before anyone reads rows another rank wrote."""
    for t, name in ((xq, "xq"), (wq, "wq"), (x_scale, "x_scale"), (w_scale, "w_scale")):
        _require_cuda(t, name)
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1] or xq.stride(1) != 1 or wq.stride(1) != 1:
        raise ValueError("xq and wq must be [M, K] and [N, K] with K contiguous")
    m, k = xq.shape
    n = wq.shape[0]
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32 or x_scale.numel() != m or w_scale.numel() != n:
        raise ValueError("scales must be float32 with M and N elements")
    if bias is not None and (bias.dtype != torch.bfloat16 or bias.numel() != n or not bias.is_cuda):
        raise ValueError("bias must be a CUDA bfloat16 tensor with N elements")
    copies = [int(p) for p in y_copies]
    if not 1 <= len(copies) <= 8:
        raise ValueError("between 1 and 8 copies of Y")
    if workspace is None:
        workspace = get_workspace(xq.device, _lib.WORKSPACE_HEADER_BYTES)
    import ctypes

    arr = (ctypes.c_void_p * len(copies))(*copies)
    status = _lib.load().b200fp8_gemm_rowwise_gather(
        xq.data_ptr(), wq.data_ptr(), x_scale.contiguous().data_ptr(), w_scale.contiguous().data_ptr(),
        bias.data_ptr() if bias is not None else None, arr, len(copies), m, n, k, xq.stride(0), wq.stride(0), ldy,
        workspace.data_ptr(), workspace.numel(), _lib.VARIANTS[variant], torch.cuda.current_stream(xq.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_gemm_rowwise_gather(M={m}, N={n}, K={k}, copies={len(copies)})")


def fp8_row_quantize(x: torch.Tensor, recipe: str = "operator") -> Tuple[torch.Tensor, torch.Tensor]:
    """CUDA rowwise quantiser: (xq float8_e4m3fn [R, C], scale float32 [R]).

    recipe="operator" is the reference's `fp8_row_quantize` (operator.py:136-145) bit for bit, for
    bf16 / fp16 / fp32 x; recipe="fp32" is scale = max(rowabsmax, 1e-12) / 448 on fp32 x."""
    _require_cuda(x, "x")
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be [rows, cols] with cols contiguous")
    dtypes = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
    if x.dtype not in dtypes:
        raise ValueError(f"unsupported dtype {x.dtype}")
    recipes = {"operator": _lib.QUANT_OPERATOR, "fp32": _lib.QUANT_FP32}
    if recipe not in recipes:
        raise ValueError(f"unknown recipe {recipe!r}")
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    scale = torch.empty((rows,), dtype=torch.float32, device=x.device)
    status = _lib.load().b200fp8_row_quantize(
        x.data_ptr(), dtypes[x.dtype], recipes[recipe], rows, cols, x.stride(0), q.data_ptr(), q.stride(0),
        scale.data_ptr(), torch.cuda.current_stream(x.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_row_quantize({rows}x{cols}, {x.dtype}, {recipe})")
    return q.view(torch.float8_e4m3fn), scale


def fp8_block_quantize(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """CUDA 128x128 block quantiser, bit for bit the reference's `fp8_block_quantize`
    (tritonbench/operators/fp8_gemm_blockwise/operator.py:87-120): (xq float8_e4m3fn [M, K],
    scale float32 [ceil(M/128), ceil(K/128)] = 1 / multiplier)."""
    _require_cuda(x, "x")
    if x.dim() != 2 or x.stride(1) != 1:
        raise ValueError("x must be [rows, cols] with cols contiguous")
    dtypes = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}
    if x.dtype not in dtypes:
        raise ValueError(f"unsupported dtype {x.dtype}")
    rows, cols = x.shape
    q = torch.empty((rows, cols), dtype=torch.uint8, device=x.device)
    scale = torch.empty(((rows + 127) // 128, (cols + 127) // 128), dtype=torch.float32, device=x.device)
    status = _lib.load().b200fp8_block_quantize(
        x.data_ptr(), dtypes[x.dtype], rows, cols, x.stride(0), q.data_ptr(), q.stride(0), scale.data_ptr(),
        scale.stride(0), torch.cuda.current_stream(x.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_block_quantize({rows}x{cols}, {x.dtype})")
    return q.view(torch.float8_e4m3fn), scale


def _fused_row_quantize(producer: int, x1: torch.Tensor, x2: torch.Tensor, eps: float, round_bf16: bool, what: str):
    _require_cuda(x1, "x1")
    _require_cuda(x2, "x2")
    if x1.dtype != torch.bfloat16 or x2.dtype != torch.bfloat16:
        raise ValueError("inputs must be bfloat16")
    if x1.dim() != 2 or x1.stride(1) != 1:
        raise ValueError("x1 must be [rows, cols] with cols contiguous")
    rows, cols = x1.shape
    q = torch.empty((rows, cols), dtype=torch.uint8, device=x1.device)
    scale = torch.empty((rows,), dtype=torch.float32, device=x1.device)
    status = _lib.load().b200fp8_fused_row_quantize(
        producer, x1.data_ptr(), x2.data_ptr(), rows, cols, x1.stride(0), x2.stride(0) if x2.dim() == 2 else 0,
        float(eps), 1 if round_bf16 else 0, q.data_ptr(), q.stride(0), scale.data_ptr(),
        torch.cuda.current_stream(x1.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_fused_row_quantize({what}, {rows}x{cols})")
    return q.view(torch.float8_e4m3fn), scale


def rms_norm_fp8_rowwise_quant(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-5,
                               round_bf16: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm + rowwise e4m3 quantisation in one kernel, in the argument order of the call
    `rms_norm_fp8_rowwise_quant(x1, wd)` (tritonbench/operators/fp8_fused_quant_gemm_rowwise/operator.py:88):
    y = x * rsqrt(mean(x^2) + eps) * weight in fp32, then scale = max(rowabsmax, 1e-12) / 448.
    round_bf16=True rounds y to bf16 first (the unfused `rms_norm` then `quantize_fp8_row`, operator.py:98-103)."""
    if weight.dim() != 1 or weight.numel() != x.shape[1] or not weight.is_contiguous():
        raise ValueError("weight must be a contiguous vector with one element per column of x")
    return _fused_row_quantize(_lib.PRODUCER_RMS_NORM, x, weight, eps, round_bf16, "rms_norm")


def silu_mul_fp8_rowwise_quant(x1: torch.Tensor, x2: torch.Tensor, round_bf16: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """SiLU(x1) * x2 + rowwise e4m3 quantisation in one kernel (`silu_mul_fp8_rowwise_quant(x1, x2)`,
    tritonbench/operators/fp8_fused_quant_gemm_rowwise/operator.py:112); fp32 arithmetic;
    round_bf16=True rounds the product to bf16 first (`silu_mul` then `quantize_fp8_row`, operator.py:122-127)."""
    if x2.dim() != 2 or tuple(x2.shape) != tuple(x1.shape) or x2.stride(1) != 1:
        raise ValueError("x2 must have the shape of x1, cols contiguous")
    return _fused_row_quantize(_lib.PRODUCER_SILU_MUL, x1, x2, 0.0, round_bf16, "silu_mul")


def fp8_gemm_rowwise_grouped(
    xq: torch.Tensor, wq: torch.Tensor, m_sizes: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
    out: Optional[torch.Tensor] = None,
    variant: str = "auto",
    workspace: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Grouped GEMM in the argument order of the reference's
    `grouped_gemm_fp8_rowwise(group_A, group_B, m_sizes, a_scale, b_scale)`
    (tritonbench/operators/fp8_gemm_rowwise_grouped/operator.py:412-432): xq [M_total, K], wq [G*N, K] stacked,
    m_sizes int32 [G] on the device (never copied to the host), scales per row; returns bf16 [M_total, N].
    Pass `workspace` (256 zero bytes, see get_workspace) when the call is captured in a CUDA graph: the cached
    workspace is keyed by stream, and a capture stream would otherwise allocate a new one inside the capture."""
    for t, name in ((xq, "xq"), (wq, "wq"), (m_sizes, "m_sizes"), (x_scale, "x_scale"), (w_scale, "w_scale")):
        _require_cuda(t, name)
    if m_sizes.dtype != torch.int32 or m_sizes.dim() != 1 or not m_sizes.is_contiguous():
        raise ValueError("m_sizes must be a contiguous int32 vector")
    groups = m_sizes.numel()
    m_total, k = xq.shape
    if wq.shape[0] % groups != 0 or wq.shape[1] != k:
        raise ValueError("wq must be [G*N, K]")
    n = wq.shape[0] // groups
    if x_scale.numel() != m_total or w_scale.numel() != wq.shape[0]:
        raise ValueError("x_scale must have M_total elements and w_scale G*N elements")
    if out is None:
        out = torch.empty((m_total, n), dtype=torch.bfloat16, device=xq.device)
    if workspace is None:
        workspace = get_workspace(xq.device, _lib.WORKSPACE_HEADER_BYTES)
    status = _lib.load().b200fp8_gemm_rowwise_grouped(
        xq.data_ptr(), wq.data_ptr(), x_scale.contiguous().data_ptr(), w_scale.contiguous().data_ptr(), m_sizes.data_ptr(),
        groups, out.data_ptr(), m_total, n, k, xq.stride(0), wq.stride(0), out.stride(0),
        workspace.data_ptr(), workspace.numel(), _lib.VARIANTS[variant], torch.cuda.current_stream(xq.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_gemm_rowwise_grouped(M={m_total}, G={groups}, N={n}, K={k})")
    return out


def fp8_gemm_blockwise(xq: torch.Tensor, wq: torch.Tensor, x_scale: torch.Tensor, w_scale: torch.Tensor,
                       out: Optional[torch.Tensor] = None, tma_store: bool = True,
                       workspace: Optional[torch.Tensor] = None) -> torch.Tensor:
    """128x128 block-scaled GEMM in the argument order of the reference's `matmul_fp8_block(xq, wq, x_scale, w_scale)`
    (tritonbench/operators/fp8_gemm_blockwise/operator.py:139-149): x_scale [ceil(M/128), ceil(K/128)],
    w_scale [ceil(N/128), ceil(K/128)] float32 (the reciprocal multipliers); returns bf16 [M, N].
    `workspace`: as for fp8_gemm_rowwise_grouped."""
    for t, name in ((xq, "xq"), (wq, "wq"), (x_scale, "x_scale"), (w_scale, "w_scale")):
        _require_cuda(t, name)
    m, k = xq.shape
    n = wq.shape[0]
    kb = (k + 127) // 128
    if tuple(x_scale.shape) != ((m + 127) // 128, kb) or tuple(w_scale.shape) != ((n + 127) // 128, kb):
        raise ValueError("block scales must be [ceil(M/128), ceil(K/128)] and [ceil(N/128), ceil(K/128)]")
    if x_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise ValueError("scales must be float32")
    if x_scale.stride(1) != 1:
        x_scale = x_scale.contiguous()
    if w_scale.stride(1) != 1:
        w_scale = w_scale.contiguous()
    if out is None:
        out = torch.empty((m, n), dtype=torch.bfloat16, device=xq.device)
    if workspace is None:
        workspace = get_workspace(xq.device, _lib.WORKSPACE_HEADER_BYTES)
    status = _lib.load().b200fp8_gemm_blockwise(
        xq.data_ptr(), wq.data_ptr(), x_scale.data_ptr(), w_scale.data_ptr(), out.data_ptr(), m, n, k,
        xq.stride(0), wq.stride(0), out.stride(0), x_scale.stride(0), w_scale.stride(0),
        workspace.data_ptr(), workspace.numel(), 0 if tma_store else _lib.FLAG_NO_TMA_STORE,
        torch.cuda.current_stream(xq.device).cuda_stream,
    )
    _lib.check(status, f"b200fp8_gemm_blockwise(M={m}, N={n}, K={k})")
    return out


def fp8_gemm(a: torch.Tensor, b: torch.Tensor, scale_a=None, scale_b=None, out_dtype: torch.dtype = torch.float16,
             **kw) -> torch.Tensor:
    """The call of TritonBench's `fp8_gemm` operator, `torch._scaled_mm(a, b, scale_a, scale_b, out_dtype=...)`
    (tritonbench/operators/fp8_gemm/fp8_gemm.py:88-101): a [M, K] e4m3 row-major, b [K, N] e4m3 column-major
    (b.T contiguous), scales per tensor (scalars or None = 1.0) or per row / column ([M, 1] and [1, N])."""
    if b.dim() != 2 or b.stride(0) != 1:
        raise ValueError("b must be [K, N] with K contiguous (a transposed view of a row-major [N, K] tensor)")
    m, n = a.shape[0], b.shape[1]

    def vec(s, count):
        if s is None:
            return torch.ones(count, dtype=torch.float32, device=a.device)
        s = torch.as_tensor(s, dtype=torch.float32, device=a.device)
        return s.reshape(-1).expand(count).contiguous() if s.numel() == 1 else s.reshape(count).contiguous()

    return fp8_gemm_rowwise(a, b.t(), vec(scale_a, m), vec(scale_b, n), out_dtype=out_dtype, **kw)


_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16, torch.float32: _lib.DTYPE_FP32}


# A decode step makes these calls once per layer with kernels of a few microseconds: the checks below are written for
# their cost (get_device() is a tenth of comparing torch.device objects, the stream handle a thirtieth of a Stream object).
def _raw_stream_slow(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream_slow)


def _fresh_like(x: torch.Tensor) -> torch.Tensor:
    """An uninitialised tensor like x with its last dimension contiguous.  empty_like is the cheaper call, but of an
    expanded x it may make an expanded dimension the innermost one."""
    out = torch.empty_like(x)
    return out if out.stride(-1) == 1 else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _claim_out(out: torch.Tensor, like: torch.Tensor, name: str) -> None:
    """Checks a result that the caller gives, and tells autograd that it is written to: a backward pass that still needs what
    it held must not go on without it."""
    if out.shape != like.shape or out.dtype != like.dtype or out.get_device() != like.get_device() or out.stride(2) != 1:
        raise ValueError(f"{name} must have the input's shape, dtype and device, the last dimension contiguous")
    if any(st == 0 and n > 1 for st, n in zip(out.stride(), out.shape)):
        raise ValueError(f"{name} must not be expanded: several of its elements are one")
    if out is not like and out.data_ptr() == like.data_ptr() and any(
            a != b for a, b, n in zip(out.stride(), like.stride(), out.shape) if n > 1) and out.numel():
        raise ValueError(f"{name} must not lie where the input lies in another layout: elements would be overwritten unread")
    if out.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which these calls do not record for it")
    torch.autograd.graph.increment_version(out)


def _has_tangent(*tensors: Optional[torch.Tensor]) -> bool:
    return any(t is not None and _forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def _refuse_gradients(what: str, q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor) -> None:
    """The cache holds codes, so these calls have no gradient; a result that looks like a constant must not pass for one."""
    recorded = (k.requires_grad or v.requires_grad or (q is not None and q.requires_grad)) and torch.is_grad_enabled()
    if recorded or (_forward_ad._current_level >= 0 and _has_tangent(q, k, v)):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad(), or on detached tensors")


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, table, interleaved, transpose):
        ctx.save_for_backward(positions, table)
        ctx.save_for_forward(positions, table)
        ctx.form = (interleaved, transpose)
        return rotary(x, positions, table, interleaved, transpose)

    @staticmethod
    def backward(ctx, grad):
        positions, table = ctx.saved_tensors
        interleaved, transpose = ctx.form
        if grad.stride(2) != 1:
            grad = grad.contiguous()
        return rotary(grad, positions, table, interleaved, not transpose), None, None, None, None

    @staticmethod
    def jvp(ctx, x_tangent, *_):
        positions, table = ctx.saved_tensors
        interleaved, transpose = ctx.form
        if x_tangent.stride(2) != 1:
            x_tangent = x_tangent.contiguous()
        return rotary(x_tangent, positions, table, interleaved, transpose)


def rotary(x: torch.Tensor, positions: torch.Tensor, table: torch.Tensor, interleaved: bool = False,
           transpose: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary positions of x [tokens, heads, dim] (bf16, fp16 or fp32; any token and head stride, so a view of a fused
    projection's output will do): y_a = x_a cos - x_b sin, y_b = x_b cos + x_a sin for the pairs (i, i + rot/2) - or
    (2i, 2i + 1) if interleaved - of the first rot elements of a head, the others copied.  positions [tokens] int32 or
    int64; table float32 [max_positions, rot] from `rotary.rotary_table`; a position outside it gives NaN.
    fp32 arithmetic, one rounding.  out may be x, and must not overlap it otherwise.  transpose=True is the gradient with regard to x; a call on an x that
    requires one, or carries a forward tangent, is differentiable (with regard to x alone)."""
    device = x.get_device()
    if device < 0:
        _require_cuda(x, "x")
    if positions.get_device() != device or table.get_device() != device:
        raise ValueError("positions and table must be on x's device")
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"unsupported dtype {x.dtype}")
    if x.dim() != 3:
        raise ValueError("x must be [tokens, heads, dim]")
    tokens, heads, dim = x.shape
    x_token, x_head, one = x.stride()
    if one != 1 and dim > 1:
        raise ValueError("x must have dim contiguous")
    wide = positions.dtype is torch.int64
    if not wide and positions.dtype is not torch.int32 or positions.dim() != 1 or not positions.is_contiguous():
        raise ValueError("positions must be a contiguous int32 or int64 vector")
    if positions.numel() != tokens:
        raise ValueError("positions must have one entry per token")
    if table.dtype is not torch.float32 or table.dim() != 2 or not table.is_contiguous():
        raise ValueError("table must be a contiguous float32 [max_positions, rot]")
    max_pos, rot = table.shape
    if max_pos < 1 or not 2 <= rot <= dim or rot % 2:
        raise ValueError("the table needs a row, and an even width of at most dim")
    tangents = _forward_ad._current_level >= 0
    if (table.requires_grad and torch.is_grad_enabled()) or (tangents and _has_tangent(table)):
        raise ValueError("rotary has no gradient with regard to its table: pass table.detach()")
    if (x.requires_grad and torch.is_grad_enabled()) or (tangents and _has_tangent(x)):
        if out is not None:
            raise ValueError("out is not differentiable: leave it out, or call under torch.no_grad()")
        return _Rotary.apply(x, positions, table, interleaved, transpose)
    if out is None:
        out = _fresh_like(x)
    else:
        _claim_out(out, x, "out")
    if tokens == 0 or heads == 0:
        return out
    if device != torch.cuda.current_device():  # a launch on a stream of another device is an error
        with torch.cuda.device(device):
            return rotary(x, positions, table, interleaved, transpose, out)
    y_token, y_head, _ = out.stride()
    status = _lib.load().b200fp8_rotary(
        x.data_ptr(), dtype, out.data_ptr(), tokens, heads, dim, x_token, x_head, y_token, y_head, positions.data_ptr(), wide,
        table.data_ptr(), max_pos, rot, bool(interleaved), bool(transpose), _raw_stream(device))
    if status:
        _lib.check(status, f"b200fp8_rotary({tokens}x{heads}x{dim}, {x.dtype})")
    return out


def _elements_share_memory(t: torch.Tensor) -> bool:
    """Whether some elements of t are one (an expanded or overlapping view); also true of a few layouts that interleave
    their dimensions, which no cache has."""
    extent = 0  # offset of the last element of the dimensions so far
    for stride, n in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n > 1):
        if stride <= extent:
            return True
        extent += stride * (n - 1)
    return False


class Fp8KvCache:
    """A paged key/value cache in e4m3: k and v [num_pages, kv_heads, page_size, head_dim] float8_e4m3fn (any page, head
    and row strides that are multiples of 16 and below 2^31; head_dim contiguous), k_scale and v_scale [num_pages, kv_heads]
    float32; a value is code * scale, no scale is negative.  page_size 16, 32, 64 or 128; head_dim 64, 128 or 256.  The object
    describes the four tensors and keeps them alive; make one with `empty`, or around tensors of your own.  Its attributes
    cannot be replaced, and the tensors' memory must not be (`set_`, `.data`, `resize_`): make another cache instead.  Tensors that
    are expanded, overlap or are one (k and v) can be read, but not appended to."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "num_pages", "kv_heads", "page_size", "head_dim", "device", "descriptor", "read_only")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        for t, name in ((k, "k"), (v, "v"), (k_scale, "k_scale"), (v_scale, "v_scale")):
            _require_cuda(t, name)
            if t.device != k.device:
                raise ValueError("the cache's tensors must be on one device")
        if k.dim() != 4 or k.shape != v.shape or k.dtype != torch.float8_e4m3fn or v.dtype != torch.float8_e4m3fn:
            raise ValueError("k and v must be float8_e4m3fn [num_pages, kv_heads, page_size, head_dim]")
        pages, heads, size, dim = k.shape
        if heads < 1:
            raise ValueError("a cache needs at least one kv head")
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or tuple(s.shape) != (pages, heads):
                raise ValueError("k_scale and v_scale must be float32 [num_pages, kv_heads]")
        if size not in (16, 32, 64, 128) or dim not in (64, 128, 256):
            raise NotImplementedError(f"page_size {size}, head_dim {dim}: page_size must be 16, 32, 64 or 128, head_dim 64, 128 or 256")
        if k.stride(3) != 1 or v.stride(3) != 1:
            raise ValueError("head_dim must be contiguous in k and v")
        for t in (k, v):
            if t.data_ptr() % 16 or any(st % 16 for st, n in zip(t.stride()[:3], t.shape) if n > 1):
                raise NotImplementedError("rows of k and v must start on 16-byte boundaries")
        read_only = pages > 0 and (any(_elements_share_memory(t) for t in (k, v, k_scale, v_scale))
                                   or k.data_ptr() == v.data_ptr() or k_scale.data_ptr() == v_scale.data_ptr())
        descriptor = _lib.KV_CACHE.pack(
            k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *k.stride()[:3], *v.stride()[:3],
            *k_scale.stride(), *v_scale.stride(), pages, heads, size, dim)
        for name, value in zip(Fp8KvCache.__slots__, (k, v, k_scale, v_scale, pages, heads, size, dim, k.get_device(), descriptor, read_only)):
            object.__setattr__(self, name, value)

    def __setattr__(self, name, value):
        # the descriptor holds addresses: with another tensor in its place the kernels would go on using the old one's memory
        if name in Fp8KvCache.__slots__:
            raise AttributeError(f"an Fp8KvCache's {name} cannot be replaced: make another cache")
        object.__setattr__(self, name, value)

    def __delattr__(self, name):
        if name in Fp8KvCache.__slots__:
            raise AttributeError(f"an Fp8KvCache's {name} cannot be removed")
        object.__delattr__(self, name)

    def __copy__(self):
        return self

    def __reduce__(self):  # a deep or pickled copy describes its own tensors (codes as bytes: torch cannot load 8-bit floats)
        return _cache_of_bytes, (self.k.view(torch.uint8), self.v.view(torch.uint8), self.k_scale, self.v_scale)

    @classmethod
    def empty(cls, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> "Fp8KvCache":
        """A cache without tokens (codes and scales zero)."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.zeros(shape[:2], dtype=torch.float32, device=device) for _ in range(2))
        return cls(k, v, ks, vs)


def _cache_of_bytes(k, v, k_scale, v_scale) -> Fp8KvCache:
    return Fp8KvCache(k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), k_scale, v_scale)


def _pack_batch(tokens: int, cache: Fp8KvCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                cu_seqlens: Optional[torch.Tensor]) -> bytes:
    device = cache.device
    if block_table.get_device() != device or seq_lens.get_device() != device:
        raise ValueError("block_table and seq_lens must be on the cache's device")
    if seq_lens.dtype is not torch.int32 or seq_lens.dim() != 1 or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be a contiguous int32 vector")
    if block_table.dtype is not torch.int32 or block_table.dim() != 2:
        raise ValueError("block_table must be int32 [batch, pages]")
    batch, width = block_table.shape
    pitch, one = block_table.stride()
    if batch != seq_lens.shape[0]:
        raise ValueError("block_table and seq_lens must have one row and one entry per sequence")
    if one != 1 and width > 1:
        raise ValueError("block_table must have its pages contiguous")
    cu = 0
    if cu_seqlens is None:
        if tokens != batch:
            raise ValueError(f"{tokens} tokens for {batch} sequences: pass cu_seqlens unless every sequence has one")
    else:
        if cu_seqlens.dtype is not torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_contiguous() or cu_seqlens.shape[0] != batch + 1:
            raise ValueError("cu_seqlens must be a contiguous int32 vector with batch + 1 entries")
        if cu_seqlens.get_device() != device:
            raise ValueError("cu_seqlens must be on the cache's device")
        cu = cu_seqlens.data_ptr()
    return _lib.KV_BATCH.pack(block_table.data_ptr(), seq_lens.data_ptr(), cu, pitch, width, batch, tokens)


def fp8_kv_append(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor, cache: Fp8KvCache, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, table: Optional[torch.Tensor] = None,
                  interleaved: bool = False, q_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Rotary positions of q and k, then k and v quantised to e4m3 into the pages of their sequences, in one launch.
    Returns the rotated q (None if q is None).

    q [tokens, heads, head_dim], k and v [tokens, kv_heads, head_dim], bf16 or fp16, any token and head strides that are
    multiples of 8: views of the QKV projection's output will do.  The rows are the newest tokens of the batch's sequences
    behind one another, cu_seqlens [batch + 1] their bounds (None: one each).  seq_lens [batch] counts them, so the last
    row of sequence b has position seq_lens[b] - 1, and position j lies in page block_table[b, j // page_size].  All
    three are int32 on the device and never copied to the host.  table: `rotary.rotary_table` (its width a multiple of
    16), None for no rotation.

    One scale per page and kv head: the smallest power of two that takes the page's largest finite magnitude to at most
    448.  A page that already holds tokens keeps its scale, or is moved to a larger one.  Infinities and NaN are stored as
    NaN.  Rows whose position would be negative (seq_lens[b] = 0: a padded entry), positions behind the block table and
    pages outside the cache are skipped, their q is zero where the position is negative.  q_out (may be q, and must not
    overlap q, k and v otherwise) keeps its rows in front of cu_seqlens[0] and behind cu_seqlens[-1]; in a fresh result they
    are zero.  A page must not be appended to twice in one call (two sequences that share one, or a sequence that has it
    twice).  There is no gradient: q, k or v that
    require one are refused where gradients are recorded."""
    if not isinstance(cache, Fp8KvCache):
        raise ValueError("cache must be an Fp8KvCache")
    if cache.read_only:
        raise ValueError("the cache's tensors are expanded, overlap or are one: such a cache can be read, but not appended to")
    device, heads, dim = cache.device, cache.kv_heads, cache.head_dim
    dtype = k.dtype
    if k.get_device() != device or v.get_device() != device:
        raise ValueError("k and v must be on the cache's device")
    if k.dim() != 3 or k.shape[1] != heads or k.shape[2] != dim or v.shape != k.shape:
        raise ValueError(f"k and v must be [tokens, {heads}, {dim}]")
    if dtype is not torch.bfloat16 and dtype is not torch.float16 or v.dtype is not dtype:
        raise ValueError("k and v must be bfloat16 or float16, both the same")
    _refuse_gradients("fp8_kv_append", q, k, v)
    tokens = k.shape[0]
    k_token, k_head, k_one = k.stride()
    v_token, v_head, v_one = v.stride()
    if k_one != 1 or v_one != 1:
        raise ValueError("k and v must have head_dim contiguous")
    q_token = q_head = o_token = o_head = fill = 0
    q_ptr = o_ptr = table_ptr = None
    if q is not None:
        if q.get_device() != device or q.dim() != 3 or q.shape[0] != tokens or q.shape[2] != dim or q.dtype is not dtype:
            raise ValueError("q must be [tokens, heads, head_dim] with k's tokens, head_dim, dtype and device")
        heads = q.shape[1]
        if heads < 1 or heads % cache.kv_heads:
            raise ValueError(f"{heads} query heads cannot share {cache.kv_heads} kv heads")
        q_token, q_head, q_one = q.stride()
        if q_one != 1:
            raise ValueError("q must have head_dim contiguous")
        if q_out is None:
            q_out, fill = _fresh_like(q), 1
        else:
            _claim_out(q_out, q, "q_out")
        o_token, o_head, _ = q_out.stride()
        q_ptr, o_ptr = q.data_ptr(), q_out.data_ptr()
    elif q_out is not None:
        raise ValueError("q_out without q")
    max_pos = rot = 0
    if table is not None:
        if table.get_device() != device or table.dtype is not torch.float32 or table.dim() != 2 or not table.is_contiguous():
            raise ValueError("table must be a contiguous float32 [max_positions, rot] on the cache's device")
        max_pos, rot = table.shape
        if max_pos < 1 or not 2 <= rot <= dim or rot % 2:
            raise ValueError("the table needs a row, and an even width of at most head_dim")
        if table.requires_grad and torch.is_grad_enabled():
            raise ValueError("fp8_kv_append has no gradient with regard to its table: pass table.detach()")
        table_ptr = table.data_ptr()
    rows = _pack_batch(tokens, cache, block_table, seq_lens, cu_seqlens)
    args = (q_ptr, k.data_ptr(), v.data_ptr(), o_ptr, _DTYPES[dtype], heads, q_token, q_head, k_token, k_head, v_token, v_head,
            o_token, o_head, cache.descriptor, rows, table_ptr, max_pos, rot, bool(interleaved), fill, _raw_stream(device))
    if device == torch.cuda.current_device():
        status = _lib.load().b200fp8_kv_append(*args)
    else:
        with torch.cuda.device(device):
            status = _lib.load().b200fp8_kv_append(*args)
    if status:
        _lib.check(status, f"b200fp8_kv_append(tokens={tokens}, heads={heads}, kv_heads={cache.kv_heads}, dim={dim})")
    return q_out


def fp8_kv_attention(q: torch.Tensor, cache: Fp8KvCache, block_table: torch.Tensor, seq_lens: torch.Tensor,
                     cu_seqlens: Optional[torch.Tensor] = None, softmax_scale: Optional[float] = None,
                     out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Attention of the newest tokens of every sequence over the cache, each token over itself and all before it
    (a decode step, drafted tokens, a chunk of a prompt).  q [tokens, heads, head_dim] bf16 or fp16; heads / kv_heads
    neighbouring query heads share a kv head; block_table (any stride between its rows: sequences over the same pages may
    share one), seq_lens, cu_seqlens as for fp8_kv_append, which has stored the tokens' own k and v before.  softmax_scale:
    head_dim ** -0.5 by default.  Returns out in q's dtype (sums in fp32; the weights that multiply v are rounded to fp16),
    with return_lse also the natural logarithm of each softmax's denominator, float32 [tokens, heads], of weights in fp32.
    out may be q, and must not overlap it otherwise.

    Rows that see no token (position negative, or seq_lens[b] = 0) are zero with lse -inf.  Pages outside the cache
    (-1 for a page that has been dropped) and positions behind the block table count as not there.  Rows in front
    of cu_seqlens[0] and behind cu_seqlens[-1] keep what they hold in a given `out`; in a fresh one they are zero.  Built for
    up to a few dozen new tokens a sequence: the cache is read once per 16 query rows, with the work split over the context
    (a prompt of thousands of tokens works, at that rate).  The result does not depend on timing.  Small calls need no
    workspace, the others allocate theirs, so captured graphs and streams never share one.  There is no gradient: a q that
    requires one is refused where gradients are recorded."""
    if not isinstance(cache, Fp8KvCache):
        raise ValueError("cache must be an Fp8KvCache")
    device = cache.device
    dtype = q.dtype
    if q.get_device() != device:
        raise ValueError("q must be on the cache's device")
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        raise ValueError(f"q must be [tokens, heads, {cache.head_dim}]")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("q must be bfloat16 or float16")
    _refuse_gradients("fp8_kv_attention", None, q, q)
    tokens, heads, dim = q.shape
    if heads < 1 or heads % cache.kv_heads:
        raise ValueError(f"{heads} query heads cannot share {cache.kv_heads} kv heads")
    q_token, q_head, one = q.stride()
    if one != 1:
        raise ValueError("q must have head_dim contiguous")
    fill = 0
    if out is None:
        out, fill = _fresh_like(q), 1
    else:
        _claim_out(out, q, "out")
    o_token, o_head, _ = out.stride()
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    rows = _pack_batch(tokens, cache, block_table, seq_lens, cu_seqlens)
    if tokens:
        if device != torch.cuda.current_device():
            with torch.cuda.device(device):
                return fp8_kv_attention(q, cache, block_table, seq_lens, cu_seqlens, softmax_scale, None if fill else out, return_lse)
        lib = _lib.load()
        nbytes = lib.b200fp8_kv_attention_workspace_bytes(cache.descriptor, rows, heads)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None  # small calls need none
        status = lib.b200fp8_kv_attention(
            q.data_ptr(), out.data_ptr(), None if lse is None else lse.data_ptr(), _DTYPES[dtype], heads, q_token, q_head,
            o_token, o_head, cache.descriptor, rows, dim ** -0.5 if softmax_scale is None else softmax_scale, fill,
            None if ws is None else ws.data_ptr(), nbytes, _raw_stream(device))
        if status:
            _lib.check(status, f"b200fp8_kv_attention(tokens={tokens}, heads={heads}, kv_heads={cache.kv_heads}, dim={dim})")
    return (out, lse) if return_lse else out


def make_gemm_fn(xq, wq, x_scale, w_scale, bias=None, variant: str = "auto", reuse_out: bool = False,
                 overlap: bool = False, out_dtype: torch.dtype = torch.bfloat16,
                 split_config: Optional[Tuple[int, int]] = None) -> Callable:
    """Zero-argument closure in the shape the TritonBench harness wants from a backend
    (triton_op.py:765-785).  The workspace is allocated here, outside any timed or captured
    region; each call of the closure only enqueues the kernel."""
    m, k = xq.shape
    n = wq.shape[0]
    flags = _flags(variant, True)
    ws = get_workspace(xq.device, workspace_bytes(m, n, k, flags))
    out = torch.empty((m, n), dtype=out_dtype, device=xq.device) if reuse_out else None

    def fn():
        return fp8_gemm_rowwise(xq, wq, x_scale, w_scale, bias, out=out, variant=variant, workspace=ws, overlap=overlap,
                                out_dtype=out_dtype, split_config=split_config)

    return fn


def check_device_status(device: Optional[torch.device] = None) -> None:
    """Synchronise and raise if any kernel recorded a timed-out wait in a workspace."""
    torch.cuda.synchronize(device)
    lib = _lib.load()
    import ctypes

    for ws in list(_workspaces.values()):
        word = ctypes.c_uint32(0)
        status = lib.b200fp8_query_status(ws.data_ptr(), ctypes.byref(word))
        if status != _lib.OK:
            ws.zero_()
            _lib.check(status, f"device status word {word.value:#010x}")


class HostGemm:
    """Host-buffer GEMM: inputs and output are CPU tensors (pin them for full PCIe speed);
    every call copies in, runs the kernel, copies out and synchronises.

    set_weights(wq, w_scale, bias) uploads the weights once; calls that then pass wq=None send only X."""

    def __init__(self, m: int, n: int, k: int, variant: str = "auto", panels: Optional[Tuple[int, int]] = None):
        import ctypes

        self.shape = (m, n, k)
        self._ctx = ctypes.c_void_p()
        self._lib = _lib.load()
        _lib.check(
            self._lib.b200fp8_host_ctx_create(m, n, k, _flags(variant, True), ctypes.byref(self._ctx)),
            "b200fp8_host_ctx_create",
        )
        if panels is not None:
            _lib.check(self._lib.b200fp8_host_ctx_set_panels(self._ctx, panels[0], panels[1]), "b200fp8_host_ctx_set_panels")

    @staticmethod
    def _host(t, name):
        if t.is_cuda or not t.is_contiguous():
            raise ValueError(f"{name}: HostGemm takes contiguous CPU tensors")
        return t.data_ptr()

    def set_weights(self, wq, w_scale, bias=None) -> None:
        m, n, k = self.shape
        if wq is None:
            _lib.check(self._lib.b200fp8_host_ctx_set_weights(self._ctx, None, None, None), "b200fp8_host_ctx_set_weights")
            return
        if tuple(wq.shape) != (n, k) or w_scale.numel() != n or w_scale.dtype != torch.float32:
            raise ValueError("wq must be [N, K] and w_scale float32 [N]")
        _lib.check(
            self._lib.b200fp8_host_ctx_set_weights(
                self._ctx, self._host(wq, "wq"), self._host(w_scale, "w_scale"),
                self._host(bias, "bias") if bias is not None else None),
            "b200fp8_host_ctx_set_weights",
        )

    def __call__(self, xq, wq, x_scale, w_scale, bias=None, out=None) -> torch.Tensor:
        m, n, k = self.shape
        if tuple(xq.shape) != (m, k) or (wq is not None and tuple(wq.shape) != (n, k)):
            raise ValueError("shape differs from the context's")
        if x_scale.numel() != m or x_scale.dtype != torch.float32:
            raise ValueError("x_scale must be float32 [M]")
        if out is None:
            out = torch.empty((m, n), dtype=torch.bfloat16, pin_memory=True)
        elif tuple(out.shape) != (m, n) or out.dtype != torch.bfloat16:
            raise ValueError("out must be bfloat16 [M, N]")
        status = self._lib.b200fp8_gemm_rowwise_host(
            self._ctx, self._host(xq, "xq"), self._host(wq, "wq") if wq is not None else None,
            self._host(x_scale, "x_scale"), self._host(w_scale, "w_scale") if w_scale is not None else None,
            self._host(bias, "bias") if bias is not None else None, self._host(out, "out"),
        )
        _lib.check(status, "b200fp8_gemm_rowwise_host")
        return out

    def close(self) -> None:
        if self._ctx:
            self._lib.b200fp8_host_ctx_destroy(self._ctx)
            self._ctx = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
