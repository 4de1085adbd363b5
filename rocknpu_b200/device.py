"""Device-pointer entry points (include/rocknpu_b200.h) on torch CUDA tensors.

torch provides the device memory and the stream; the work is done by the
library's kernels.  Each function checks shapes and dtypes, queues the kernel
on the current torch stream (or the given one) and returns without waiting.
"""
from __future__ import annotations

import ctypes

import torch

from .capi import BLOCK_BYTES, GGML_BF16, GGML_F16, GGML_F32, F8Experts, MoeF8Args, lib

_TYPES = {torch.float32: GGML_F32, torch.float16: GGML_F16, torch.bfloat16: GGML_BF16}
F8_BLOCK = 128


def _stream(stream) -> int:
    if stream is None:
        stream = torch.cuda.current_stream()
    return stream.cuda_stream if hasattr(stream, "cuda_stream") else int(stream)


def _check(st: int, what: str) -> None:
    if st != 0:
        raise RuntimeError(f"{what} failed with status {st}")


def new_status(device=None) -> torch.Tensor:
    return torch.zeros(1, dtype=torch.int32, device=device or "cuda")


def prepare_w8(kind: int, blocks: torch.Tensor, k: int, n: int, status: torch.Tensor, stream=None):
    """K1: K-quant rows -> (int8 [n, k], f32 scales [n])."""
    assert blocks.is_cuda and blocks.dtype == torch.uint8 and blocks.is_contiguous()
    w = torch.empty((n, k), dtype=torch.int8, device=blocks.device)
    s = torch.empty(n, dtype=torch.float32, device=blocks.device)
    _check(lib().rocknpu_b200_prepare_w8(kind, blocks.data_ptr(), k, n, w.data_ptr(), s.data_ptr(),
                                         status.data_ptr(), _stream(stream)), "prepare_w8")
    return w, s


def quantize_rows(a: torch.Tensor, status: torch.Tensor, out: torch.Tensor | None = None,
                  scales: torch.Tensor | None = None, stream=None):
    """K2: f32 [m, k] -> (int8 [m, k], f32 scales [m])."""
    assert a.is_cuda and a.dtype == torch.float32 and a.is_contiguous() and a.dim() == 2
    m, k = a.shape
    out = torch.empty((m, k), dtype=torch.int8, device=a.device) if out is None else out
    scales = torch.empty(m, dtype=torch.float32, device=a.device) if scales is None else scales
    _check(lib().rocknpu_b200_quantize_rows(a.data_ptr(), m, k, out.data_ptr(), out.stride(0), scales.data_ptr(),
                                            status.data_ptr(), _stream(stream)), "quantize_rows")
    return out, scales


def workspace_bytes(m: int, n: int, k: int) -> int:
    return int(lib().rocknpu_b200_gemm_workspace_bytes(m, n, k))


def new_workspace(nbytes: int, device=None) -> torch.Tensor:
    """Zeroed split-K workspace (the GEMM keeps it zero between launches)."""
    return torch.zeros(max(nbytes, 1), dtype=torch.uint8, device=device or "cuda")


def gemm_w8a8(a8: torch.Tensor, a_scales: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor,
              status: torch.Tensor, out: torch.Tensor | None = None, acc: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, stream=None):
    """K3: (f32(acc) * a_s) * w_s with acc = a8 . w8^T exact int32."""
    m, k = a8.shape
    n = w8.shape[0]
    out = torch.empty((m, n), dtype=torch.float32, device=a8.device) if out is None else out
    ws_ptr = workspace.data_ptr() if workspace is not None else None
    ws_bytes = workspace.numel() if workspace is not None else 0
    _check(lib().rocknpu_b200_gemm_w8a8(a8.data_ptr(), a8.stride(0), a_scales.data_ptr(), w8.data_ptr(),
                                        w8.stride(0), w_scales.data_ptr(), out.data_ptr(), out.stride(0),
                                        acc.data_ptr() if acc is not None else None, m, k, n, ws_ptr, ws_bytes,
                                        status.data_ptr(), _stream(stream)), "gemm_w8a8")
    return out


def convert_f16(a: torch.Tensor, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """The FP16 executor's f32 -> f16 activation conversion (round to nearest even)."""
    assert a.is_cuda and a.dtype == torch.float32 and a.dim() == 2 and a.stride(1) == 1
    m, k = a.shape
    out = torch.empty((m, k), dtype=torch.float16, device=a.device) if out is None else out
    _check(lib().rocknpu_b200_convert_f16(a.data_ptr(), m, k, a.stride(0), out.data_ptr(), out.stride(0),
                                          _stream(stream)), "convert_f16")
    return out


def gemm_f16(a16: torch.Tensor, w16: torch.Tensor, status: torch.Tensor, out: torch.Tensor | None = None,
             stream=None):
    """K4: f16 [m, k] . f16 [n, k]^T accumulated in f32."""
    m, k = a16.shape
    n = w16.shape[0]
    out = torch.empty((m, n), dtype=torch.float32, device=a16.device) if out is None else out
    _check(lib().rocknpu_b200_gemm_f16(a16.data_ptr(), a16.stride(0), w16.data_ptr(), w16.stride(0), out.data_ptr(),
                                       out.stride(0), m, k, n, status.data_ptr(), _stream(stream)), "gemm_f16")
    return out


def gemv_w8a8(a8: torch.Tensor, a_scale: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor,
              out: torch.Tensor | None = None, stream=None):
    """K5: M=1 W8A8 GEMV."""
    n, k = w8.shape
    out = torch.empty(n, dtype=torch.float32, device=w8.device) if out is None else out
    _check(lib().rocknpu_b200_gemv_w8a8(a8.data_ptr(), a_scale.data_ptr(), w8.data_ptr(), w_scales.data_ptr(),
                                        out.data_ptr(), k, n, _stream(stream)), "gemv_w8a8")
    return out


def kq_layout(kind: int, blocks: torch.Tensor, k: int, n: int, stream=None) -> torch.Tensor:
    """Decode layout of a K-quant weight (device uint8 blocks, n rows of k)."""
    nbytes = int(lib().rocknpu_b200_kq_layout_bytes(kind, k, n))
    if nbytes == 0:
        raise ValueError(f"no decode layout for kind {kind}, k={k}")
    out = torch.empty(nbytes, dtype=torch.uint8, device=blocks.device)
    _check(lib().rocknpu_b200_kq_layout(kind, blocks.data_ptr(), k, n, out.data_ptr(), _stream(stream)), "kq_layout")
    return out


def gemv_kq(kind: int, layout: torch.Tensor, x: torch.Tensor, n: int, status: torch.Tensor,
            out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """K5b: y[n] = dequant(W) . x straight from the K-quant decode layout."""
    k = x.numel()
    out = torch.empty(n, dtype=torch.float32, device=x.device) if out is None else out
    _check(lib().rocknpu_b200_gemv_kq(kind, layout.data_ptr(), k, n, x.data_ptr(), out.data_ptr(),
                                      status.data_ptr(), _stream(stream)), "gemv_kq")
    return out


def matmul_w8a8(ctx, a: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor, out: torch.Tensor, stream=None):
    """K2 + K3 (K5 at m == 1) through a context's workspace.  On torch's
    default stream (handle 0, also what stream=None gives there) the work
    runs on the context's own stream: rocknpu_b200_context_check (or a device
    synchronisation) orders it before later reads of `out`."""
    m, k = a.shape
    n = w8.shape[0]
    _check(lib().rocknpu_b200_matmul_w8a8(ctx.handle, a.data_ptr(), w8.data_ptr(), w_scales.data_ptr(),
                                          out.data_ptr(), m, k, n, _stream(stream)), "matmul_w8a8")
    return out


# ---- e4m3 with a scale per block of 128 --------------------------------------
#
# e4m3 tensors are torch.float8_e4m3fn; scales are f32, per row and 128 columns
# for activations, per 128 x 128 block for weights.  These calls queue on the
# operands' own device (its current torch stream unless one is given).

def _f8_blocks(n: int) -> int:
    return (n + F8_BLOCK - 1) // F8_BLOCK


def _require(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _operands(first: torch.Tensor, *others) -> None:
    _require(first.is_cuda, "operands are CUDA tensors")
    for t in others:
        _require(t is None or t.device == first.device, "all operands are on one device")


def _status_word(status: torch.Tensor) -> None:
    _require(status.dtype == torch.int32 and status.numel() >= 1, "status is an int32 tensor (new_status)")


def _launch(name: str, device, stream, *args) -> None:
    """Call entry point `name` with `device` current; the stream goes last."""
    with torch.cuda.device(device):
        _check(getattr(lib(), f"rocknpu_b200_{name}")(*args, _stream(stream)), name)


def _f8_empty(*shape, device) -> torch.Tensor:
    """e4m3 tensor whose rows start at multiples of 16 bytes."""
    k16 = (shape[-1] + 15) // 16 * 16
    return torch.empty((*shape[:-1], k16), dtype=torch.float8_e4m3fn, device=device)[..., :shape[-1]]


def _f8_weight(w8: torch.Tensor, scales: torch.Tensor, what: str) -> None:
    n, k = w8.shape[-2:]
    _require(w8.dtype == torch.float8_e4m3fn and w8.stride(-1) == 1 and w8.stride(-2) >= k,
             f"{what} is an e4m3 tensor of whole rows")
    _require(scales.dtype == torch.float32 and scales.is_contiguous() and
             tuple(scales.shape) == (*w8.shape[:-2], _f8_blocks(n), _f8_blocks(k)),
             f"{what} scales are a contiguous f32 tensor, one per 128 x 128 block")


def quantize_rows_f8(a: torch.Tensor, status: torch.Tensor, out: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None, stream=None):
    """f32 / f16 / bf16 [m, k] -> (e4m3 [m, k], f32 scales [m, ceil(k / 128)])."""
    _operands(a, status, out, scales)
    _status_word(status)
    _require(a.dim() == 2 and a.dtype in _TYPES and a.stride(1) == 1, "a is an f32, f16 or bf16 matrix of whole rows")
    m, k = a.shape
    _require(m > 0 and k > 0, "a is not empty")
    out = _f8_empty(m, k, device=a.device) if out is None else out
    scales = torch.empty((m, _f8_blocks(k)), dtype=torch.float32, device=a.device) if scales is None else scales
    _require(out.dtype == torch.float8_e4m3fn and out.shape == a.shape and out.stride(1) == 1,
             "out is an e4m3 matrix of a's shape")
    _require(scales.dtype == torch.float32 and tuple(scales.shape) == (m, _f8_blocks(k)) and
             (scales.stride(1) == 1 or scales.shape[1] == 1), "scales are f32 [m, ceil(k / 128)]")
    _launch("quantize_rows_f8", a.device, stream, _TYPES[a.dtype], a.data_ptr(), m, k, _pitch(a), out.data_ptr(),
            _pitch(out), scales.data_ptr(), _pitch(scales), status.data_ptr())
    return out, scales


def _pitch(t: torch.Tensor) -> int:
    """Row pitch in elements; a single row's stride says nothing."""
    return t.stride(-2) if t.shape[-2] > 1 else max(t.shape[-1], t.stride(-2))


def prepare_f8(w: torch.Tensor, status: torch.Tensor, stream=None):
    """Dense weight(s) [n, k] or [experts, n, k] -> (e4m3 of the same shape,
    f32 scales [..., ceil(n / 128), ceil(k / 128)])."""
    _operands(w, status)
    _status_word(status)
    _require(w.dim() in (2, 3) and w.dtype in _TYPES and w.stride(-1) == 1 and w.numel() > 0,
             "w is an f32, f16 or bf16 matrix, or a stack of them, of whole rows")
    n, k = w.shape[-2:]
    count = w.shape[0] if w.dim() == 3 else 1
    ldw = _pitch(w)
    _require(count == 1 or w.stride(0) == n * ldw, "a stack of weights has no gaps between them")
    out = _f8_empty(*w.shape, device=w.device)
    scales = torch.empty((*w.shape[:-2], _f8_blocks(n), _f8_blocks(k)), dtype=torch.float32, device=w.device)
    _launch("prepare_f8", w.device, stream, _TYPES[w.dtype], w.data_ptr(), n, k, ldw, count, out.data_ptr(),
            (k + 15) // 16 * 16, scales.data_ptr(), status.data_ptr())
    return out, scales


def prepare_f8_q(kind: int, blocks: torch.Tensor, k: int, n: int, status: torch.Tensor, stream=None):
    """K-quant rows -> (e4m3 [n, k], f32 scales [ceil(n / 128), k / 128])."""
    _operands(blocks, status)
    _status_word(status)
    _require(blocks.dtype == torch.uint8 and blocks.is_contiguous(), "blocks are contiguous uint8")
    _require(kind in BLOCK_BYTES and k > 0 and n > 0 and k % 256 == 0 and
             blocks.numel() >= n * (k // 256) * BLOCK_BYTES[kind], "blocks hold n rows of k / 256 superblocks")
    out = torch.empty((n, k), dtype=torch.float8_e4m3fn, device=blocks.device)
    scales = torch.empty((_f8_blocks(n), _f8_blocks(k)), dtype=torch.float32, device=blocks.device)
    _launch("prepare_f8_q", blocks.device, stream, kind, blocks.data_ptr(), k, n, out.data_ptr(), k,
            scales.data_ptr(), status.data_ptr())
    return out, scales


def gemm_f8_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(lib().rocknpu_b200_gemm_f8_workspace_bytes(m, n, k))


def matmul_f8_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(lib().rocknpu_b200_matmul_f8_workspace_bytes(m, n, k))


def _f8_out(out, m: int, n: int, dtype, device) -> torch.Tensor:
    out = torch.empty((m, n), dtype=dtype, device=device) if out is None else out
    _require(out.dtype in _TYPES and tuple(out.shape) == (m, n) and (out.stride(1) == 1 or n == 1),
             f"out is an f32, f16 or bf16 matrix of shape {(m, n)}")
    return out


def gemm_f8(a8: torch.Tensor, a_scales: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor,
            status: torch.Tensor, out: torch.Tensor | None = None, out_dtype=torch.float32,
            workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Block-scaled e4m3 product a8 [m, k] . w8 [n, k]^T (quantize_rows_f8,
    prepare_f8).  Rows start at multiples of 16 bytes."""
    _operands(a8, a_scales, w8, w_scales, status, out, workspace)
    _status_word(status)
    _require(a8.dim() == 2 and a8.dtype == torch.float8_e4m3fn and a8.stride(1) == 1 and a8.numel() > 0,
             "a8 is an e4m3 matrix of whole rows")
    m, k = a8.shape
    _require(w8.dim() == 2 and w8.shape[1] == k and w8.numel() > 0, "w8 is [n, k]")
    _f8_weight(w8, w_scales, "w8")
    _require(a_scales.dtype == torch.float32 and tuple(a_scales.shape) == (m, _f8_blocks(k)) and
             (a_scales.stride(1) == 1 or a_scales.shape[1] == 1), "a_scales are f32 [m, ceil(k / 128)]")
    n = w8.shape[0]
    out = _f8_out(out, m, n, out_dtype, a8.device)
    _launch("gemm_f8", a8.device, stream, a8.data_ptr(), _pitch16(a8), a_scales.data_ptr(), _pitch(a_scales),
            w8.data_ptr(), _pitch16(w8), w_scales.data_ptr(), out.data_ptr(), _TYPES[out.dtype], _pitch(out), m, k, n,
            workspace.data_ptr() if workspace is not None else None,
            workspace.numel() * workspace.element_size() if workspace is not None else 0, status.data_ptr())
    return out


def _pitch16(t: torch.Tensor) -> int:
    """Row pitch of an e4m3 operand; a single row has none, and may end at k."""
    return t.stride(-2) if t.shape[-2] > 1 else (t.shape[-1] + 15) // 16 * 16


def matmul_f8(a: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor, status: torch.Tensor,
              workspace: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None, stream=None) -> torch.Tensor:
    """quantize_rows_f8 + gemm_f8: f32 / f16 / bf16 a [m, k] times a prepared
    weight; the result has a's type unless `out` or `out_dtype` says another.
    `workspace` (new_workspace of matmul_f8_workspace_bytes) is kept by the
    caller, one per stream on which calls may be in flight."""
    _operands(a, w8, w_scales, status, workspace, out)
    _status_word(status)
    _require(a.dim() == 2 and a.dtype in _TYPES and a.stride(1) == 1 and a.numel() > 0,
             "a is an f32, f16 or bf16 matrix of whole rows")
    m, k = a.shape
    _require(w8.dim() == 2 and w8.shape[1] == k and w8.numel() > 0, "w8 is [n, k]")
    _f8_weight(w8, w_scales, "w8")
    n = w8.shape[0]
    out = _f8_out(out, m, n, out_dtype or a.dtype, a.device)
    _launch("matmul_f8", a.device, stream, a.data_ptr(), _TYPES[a.dtype], _pitch(a), w8.data_ptr(), _pitch16(w8),
            w_scales.data_ptr(), out.data_ptr(), _TYPES[out.dtype], _pitch(out), m, k, n, workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), status.data_ptr())
    return out


def moe_f8_workspace_bytes(tokens: int, hidden: int, ffn: int, experts: int, top_k: int, dtype) -> int:
    """0 for a shape that moe_f8 does not take."""
    return int(lib().rocknpu_b200_moe_f8_workspace_bytes(tokens, hidden, ffn, experts, top_k, _TYPES[dtype]))


def _f8_experts(w8: torch.Tensor, scales: torch.Tensor, shape, what: str) -> F8Experts:
    _require(tuple(w8.shape) == shape, f"{what} is an e4m3 tensor of shape {shape}")
    _f8_weight(w8, scales, what)
    return F8Experts(w8.data_ptr(), _pitch16(w8), w8.stride(0), scales.data_ptr(), scales.stride(0))


def moe_f8(x: torch.Tensor, gate, up, down, status: torch.Tensor, workspace: torch.Tensor, *,
           router: torch.Tensor | None = None, top_k: int | None = None, renormalize: bool = True,
           ids: torch.Tensor | None = None, weights: torch.Tensor | None = None, out: torch.Tensor | None = None,
           stream=None):
    """A mixture-of-experts layer for up to 64 tokens x [t, hidden].

    gate, up and down are (e4m3, scales) pairs of stacked weights as
    prepare_f8 returns them, [e, ffn, hidden], [e, ffn, hidden] and
    [e, hidden, ffn].  With `router` [e, hidden] the layer picks top_k experts
    per token (softmax over the chosen ones, or over all with
    renormalize=False); without, int32 `ids` (negative: empty slot) and f32
    `weights` [t, top_k] say them.  Returns (out, ids, weights).
    `workspace`: new_workspace(moe_f8_workspace_bytes(...)), kept by the
    caller, one per stream on which calls may be in flight."""
    _operands(x, *gate, *up, *down, status, workspace, router, ids, weights, out)
    _status_word(status)
    _require(x.dim() == 2 and x.dtype in _TYPES and x.stride(1) == 1 and x.numel() > 0,
             "x is an f32, f16 or bf16 matrix of whole rows")
    t, h = x.shape
    _require(gate[0].dim() == 3, "gate is [experts, ffn, hidden]")
    e, f = gate[0].shape[:2]
    if router is not None:
        _require(top_k is not None and ids is None and weights is None, "a router goes with top_k, ids and weights without")
        _require(router.dtype in _TYPES and tuple(router.shape) == (e, h) and router.stride(1) == 1,
                 "router is an f32, f16 or bf16 matrix [experts, hidden]")
        ids = torch.empty((t, top_k), dtype=torch.int32, device=x.device)
        weights = torch.empty((t, top_k), dtype=torch.float32, device=x.device)
    else:
        _require(ids is not None and weights is not None, "without a router, ids and weights are given")
        top_k = ids.shape[1] if ids.dim() == 2 else 0
        _require(ids.dtype == torch.int32 and weights.dtype == torch.float32 and tuple(ids.shape) == (t, top_k) and
                 ids.shape == weights.shape and ids.is_contiguous() and weights.is_contiguous(),
                 "ids and weights are contiguous int32 and f32 [tokens, top_k]")
    out = _f8_out(out, t, h, x.dtype, x.device)
    _require(out.dtype == x.dtype, "out has x's type")
    args = MoeF8Args(t, h, f, e, top_k, _TYPES[x.dtype], x.data_ptr(), out.data_ptr(), _pitch(x), _pitch(out),
                     _f8_experts(*gate, (e, f, h), "gate"), _f8_experts(*up, (e, f, h), "up"),
                     _f8_experts(*down, (e, h, f), "down"), None if router is None else router.data_ptr(),
                     _TYPES[torch.float32 if router is None else router.dtype], 0 if router is None else _pitch(router),
                     1 if renormalize else 0, ids.data_ptr(), weights.data_ptr())
    _launch("moe_f8", x.device, stream, ctypes.byref(args), workspace.data_ptr(),
            workspace.numel() * workspace.element_size(), status.data_ptr())
    return out, ids, weights
