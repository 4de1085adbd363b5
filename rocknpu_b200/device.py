"""Device-pointer entry points (include/rocknpu_b200.h) on torch CUDA tensors.

torch provides the device memory and the stream; the work is done by the
library's kernels.  Each function checks shapes and dtypes, queues the kernel
on the current torch stream (or the given one) and returns without waiting.
"""
from __future__ import annotations

import struct

import torch

from .capi import BLOCK_BYTES, GGML_BF16, GGML_F16, GGML_F32, lib

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
# operands' own device (its current torch stream unless one is given).  A
# decode call's kernels take a few microseconds, so the checks are written to
# cost about as much: sizes and strides are read once, and messages are made
# only for an error.

def _f8_blocks(n: int) -> int:
    return (n + F8_BLOCK - 1) // F8_BLOCK


def _device_of(first: torch.Tensor, *others) -> int:
    dev = first.get_device()
    if dev < 0:
        raise ValueError("operands are CUDA tensors")
    for t in others:
        if t is not None and t.get_device() != dev:
            raise ValueError("all operands are on one device")
    return dev


_ENTRY = {}


def _launch(name: str, dev: int, *args) -> None:
    """Call entry point `name` on device `dev` and its current stream."""
    fn = _ENTRY.get(name)
    if fn is None:
        fn = _ENTRY[name] = getattr(lib(), "rocknpu_b200_" + name)
    handle = torch._C._cuda_getCurrentRawStream(dev)
    if torch._C._cuda_getDevice() == dev:
        st = fn(*args, handle)
    else:
        with torch.cuda.device(dev):
            st = fn(*args, handle)
    if st != 0:
        raise RuntimeError(f"{name} failed with status {st}")


def _on(stream, dev: int):
    """The given stream as the current one, so that what a call allocates
    belongs to it."""
    if not isinstance(stream, torch.cuda.Stream):
        handle = int(stream)
        stream = torch.cuda.ExternalStream(handle, device=dev) if handle else torch.cuda.default_stream(dev)
    if stream.device.index != dev:
        raise ValueError("the stream is on another device than the operands")
    return torch.cuda.stream(stream)


def _status_ptr(status: torch.Tensor) -> int:
    if status.dtype is not torch.int32 or status.numel() < 1:
        raise ValueError("status is an int32 tensor (new_status)")
    return status.data_ptr()


def _workspace(workspace: torch.Tensor):
    """(address, bytes); the bytes are the workspace's own, so no expanded or
    strided view."""
    if not workspace.is_contiguous():
        raise ValueError("workspace is contiguous (new_workspace)")
    return workspace.data_ptr(), workspace.nbytes


def _f8_empty(like: torch.Tensor, *shape) -> torch.Tensor:
    """e4m3 tensor on `like`'s device whose rows start at multiples of 16 bytes."""
    k = shape[-1]
    if k % 16 == 0:
        return like.new_empty(shape, dtype=torch.float8_e4m3fn)
    return like.new_empty((*shape[:-1], (k + 15) // 16 * 16), dtype=torch.float8_e4m3fn)[..., :k]


def _dense_rows(t: torch.Tensor, what: str):
    """(rows, columns, row pitch, type id) of a dense matrix of whole rows.  A
    single row's stride says nothing."""
    type_ = _TYPES.get(t.dtype)
    if type_ is None or t.dim() != 2 or t.numel() == 0:
        raise ValueError(f"{what} is an f32, f16 or bf16 matrix, not empty")
    (m, k), (ld, step) = t.shape, t.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{what} is a matrix of whole rows")
    return m, k, ld if m > 1 else max(k, ld), type_


def _f8_rows(t: torch.Tensor, what: str):
    """(rows, columns, row pitch) of an e4m3 operand; a single row may end at k."""
    if t.dtype is not torch.float8_e4m3fn or t.dim() != 2 or t.numel() == 0:
        raise ValueError(f"{what} is an e4m3 matrix, not empty")
    (m, k), (ld, step) = t.shape, t.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{what} is a matrix of whole rows")
    return m, k, ld if m > 1 else (k + 15) // 16 * 16


def _row_scales(s: torch.Tensor, m: int, k: int, what: str) -> int:
    """Row pitch of activation scales [m, ceil(k / 128)]."""
    kb = _f8_blocks(k)
    if s.dtype is not torch.float32 or s.shape != (m, kb):
        raise ValueError(f"{what} are f32 [m, ceil(k / 128)]")
    ld, step = s.stride()
    if step != 1 and kb > 1:
        raise ValueError(f"{what} are a matrix of whole rows")
    return ld if m > 1 else max(kb, ld)


def _weight_scales(s: torch.Tensor, shape, what: str) -> None:
    if s.dtype is not torch.float32 or s.shape != shape or not s.is_contiguous():
        raise ValueError(f"{what} scales are contiguous f32 {tuple(shape)}, one per 128 x 128 block")


def _dense_out(out, m: int, n: int, dtype, like: torch.Tensor):
    """(out, type id, row pitch), made when None."""
    if out is None:
        if dtype not in _TYPES:
            raise ValueError("results are f32, f16 or bf16")
        return like.new_empty((m, n), dtype=dtype), _TYPES[dtype], n
    rows, cols, ld, type_ = _dense_rows(out, "out")
    if rows != m or cols != n:
        raise ValueError(f"out has shape {(m, n)}")
    return out, type_, ld


def quantize_rows_f8(a: torch.Tensor, status: torch.Tensor, out: torch.Tensor | None = None,
                     scales: torch.Tensor | None = None, stream=None):
    """f32 / f16 / bf16 [m, k] -> (e4m3 [m, k], f32 scales [m, ceil(k / 128)])."""
    dev = _device_of(a, status, out, scales)
    if stream is not None:
        with _on(stream, dev):
            return quantize_rows_f8(a, status, out, scales)
    m, k, lda, type_ = _dense_rows(a, "a")
    if out is None:
        out = _f8_empty(a, m, k)
    if scales is None:
        scales = a.new_empty((m, _f8_blocks(k)), dtype=torch.float32)
    rows, cols, ld8 = _f8_rows(out, "out")
    if rows != m or cols != k:
        raise ValueError("out has a's shape")
    _launch("quantize_rows_f8", dev, type_, a.data_ptr(), m, k, lda, out.data_ptr(), ld8, scales.data_ptr(),
            _row_scales(scales, m, k, "scales"), _status_ptr(status))
    return out, scales


def prepare_f8(w: torch.Tensor, status: torch.Tensor, stream=None):
    """Dense weight(s) [n, k] or [experts, n, k] -> (e4m3 of the same shape,
    f32 scales [..., ceil(n / 128), ceil(k / 128)])."""
    dev = _device_of(w, status)
    if stream is not None:
        with _on(stream, dev):
            return prepare_f8(w, status)
    if w.dim() not in (2, 3):
        raise ValueError("w is a matrix or a stack of them")
    n, k, ldw, type_ = _dense_rows(w if w.dim() == 2 else w[0] if w.shape[0] else w.flatten(0, 1), "w")
    count = w.shape[0] if w.dim() == 3 else 1
    if count > 1 and w.stride(0) != n * ldw:
        raise ValueError("a stack of weights has no gaps between them")
    out = _f8_empty(w, *w.shape)
    scales = w.new_empty((*w.shape[:-2], _f8_blocks(n), _f8_blocks(k)), dtype=torch.float32)
    _launch("prepare_f8", dev, type_, w.data_ptr(), n, k, ldw, count, out.data_ptr(), (k + 15) // 16 * 16,
            scales.data_ptr(), _status_ptr(status))
    return out, scales


def prepare_f8_q(kind: int, blocks: torch.Tensor, k: int, n: int, status: torch.Tensor, stream=None):
    """K-quant rows -> (e4m3 [n, k], f32 scales [ceil(n / 128), k / 128])."""
    dev = _device_of(blocks, status)
    if stream is not None:
        with _on(stream, dev):
            return prepare_f8_q(kind, blocks, k, n, status)
    if blocks.dtype is not torch.uint8 or not blocks.is_contiguous():
        raise ValueError("blocks are contiguous uint8")
    if kind not in BLOCK_BYTES or k <= 0 or n <= 0 or k % 256 or blocks.numel() < n * (k // 256) * BLOCK_BYTES[kind]:
        raise ValueError("blocks hold n rows of k / 256 superblocks")
    out = blocks.new_empty((n, k), dtype=torch.float8_e4m3fn)
    scales = blocks.new_empty((_f8_blocks(n), _f8_blocks(k)), dtype=torch.float32)
    _launch("prepare_f8_q", dev, kind, blocks.data_ptr(), k, n, out.data_ptr(), k, scales.data_ptr(),
            _status_ptr(status))
    return out, scales


def gemm_f8_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(lib().rocknpu_b200_gemm_f8_workspace_bytes(m, n, k))


def matmul_f8_workspace_bytes(m: int, n: int, k: int) -> int:
    return int(lib().rocknpu_b200_matmul_f8_workspace_bytes(m, n, k))


def gemm_f8(a8: torch.Tensor, a_scales: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor,
            status: torch.Tensor, out: torch.Tensor | None = None, out_dtype=torch.float32,
            workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Block-scaled e4m3 product a8 [m, k] . w8 [n, k]^T (quantize_rows_f8,
    prepare_f8).  Rows start at multiples of 16 bytes."""
    dev = _device_of(a8, a_scales, w8, w_scales, status, out, workspace)
    if stream is not None:
        with _on(stream, dev):
            return gemm_f8(a8, a_scales, w8, w_scales, status, out, out_dtype, workspace)
    m, k, lda = _f8_rows(a8, "a8")
    n, kw, ldw = _f8_rows(w8, "w8")
    if kw != k:
        raise ValueError("w8 is [n, k]")
    _weight_scales(w_scales, (_f8_blocks(n), _f8_blocks(k)), "w8")
    out, out_type, ldo = _dense_out(out, m, n, out_dtype, a8)
    _launch("gemm_f8", dev, a8.data_ptr(), lda, a_scales.data_ptr(), _row_scales(a_scales, m, k, "a_scales"),
            w8.data_ptr(), ldw, w_scales.data_ptr(), out.data_ptr(), out_type, ldo, m, k, n,
            *((None, 0) if workspace is None else _workspace(workspace)), _status_ptr(status))
    return out


def matmul_f8(a: torch.Tensor, w8: torch.Tensor, w_scales: torch.Tensor, status: torch.Tensor,
              workspace: torch.Tensor, out: torch.Tensor | None = None, out_dtype=None, stream=None) -> torch.Tensor:
    """quantize_rows_f8 + gemm_f8: f32 / f16 / bf16 a [m, k] times a prepared
    weight; the result has a's type unless `out` or `out_dtype` says another
    (`out` is apart from `a`).
    `workspace` (new_workspace of matmul_f8_workspace_bytes) is kept by the
    caller, one per stream on which calls may be in flight."""
    dev = _device_of(a, w8, w_scales, status, workspace, out)
    if stream is not None:
        with _on(stream, dev):
            return matmul_f8(a, w8, w_scales, status, workspace, out, out_dtype)
    m, k, lda, type_ = _dense_rows(a, "a")
    n, kw, ldw = _f8_rows(w8, "w8")
    if kw != k:
        raise ValueError("w8 is [n, k]")
    _weight_scales(w_scales, (_f8_blocks(n), _f8_blocks(k)), "w8")
    out, out_type, ldo = _dense_out(out, m, n, out_dtype or a.dtype, a)
    _launch("matmul_f8", dev, a.data_ptr(), type_, lda, w8.data_ptr(), ldw, w_scales.data_ptr(),
            out.data_ptr(), out_type, ldo, m, k, n, *_workspace(workspace), _status_ptr(status))
    return out


def moe_f8_workspace_bytes(tokens: int, hidden: int, ffn: int, experts: int, top_k: int, dtype) -> int:
    """0 for a shape that moe_f8 does not take."""
    return int(lib().rocknpu_b200_moe_f8_workspace_bytes(tokens, hidden, ffn, experts, top_k, _TYPES[dtype]))


# The bytes of a rocknpu_b200_moe_f8_args (capi.MoeF8Args names its fields).
_MOE_ARGS = struct.Struct("@5N I PPNN PNNPN PNNPN PNNPN P I N i PP")


def _experts(weight, shape, what: str):
    """The fields of a rocknpu_b200_f8_experts."""
    w8, scales = weight
    if w8.dtype is not torch.float8_e4m3fn or w8.shape != shape:
        raise ValueError(f"{what} is an e4m3 tensor of shape {shape}")
    e, n, k = shape
    stride, ld, step = w8.stride()
    if step != 1 and k > 1:
        raise ValueError(f"{what} is a stack of matrices of whole rows")
    _weight_scales(scales, (e, _f8_blocks(n), _f8_blocks(k)), what)
    return w8.data_ptr(), ld if n > 1 else (k + 15) // 16 * 16, stride, scales.data_ptr(), scales.stride(0)


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
    dev = _device_of(x, *gate, *up, *down, status, workspace, router, ids, weights, out)
    if stream is not None:
        with _on(stream, dev):
            return moe_f8(x, gate, up, down, status, workspace, router=router, top_k=top_k, renormalize=renormalize,
                          ids=ids, weights=weights, out=out)
    t, h, ldx, type_ = _dense_rows(x, "x")
    if gate[0].dim() != 3:
        raise ValueError("gate is [experts, ffn, hidden]")
    e, f, _ = gate[0].shape
    if router is not None:
        if top_k is None or top_k < 1 or ids is not None or weights is not None:
            raise ValueError("a router goes with top_k, ids and weights without")
        rows, cols, ld_router, router_type = _dense_rows(router, "router")
        if rows != e or cols != h:
            raise ValueError("router is [experts, hidden]")
        ids = x.new_empty((t, top_k), dtype=torch.int32)
        weights = x.new_empty((t, top_k), dtype=torch.float32)
    else:
        ld_router = router_type = 0
        if ids is None or weights is None or ids.dim() != 2 or ids.shape[0] != t or ids.shape != weights.shape or \
                ids.dtype is not torch.int32 or weights.dtype is not torch.float32 or \
                not ids.is_contiguous() or not weights.is_contiguous():
            raise ValueError("without a router, ids and weights are contiguous int32 and f32 [tokens, top_k]")
        if top_k is not None and top_k != ids.shape[1]:
            raise ValueError("ids and weights are [tokens, top_k]")
        top_k = ids.shape[1]
    out, out_type, ldo = _dense_out(out, t, h, x.dtype, x)
    if out_type != type_:
        raise ValueError("out has x's type")
    args = _MOE_ARGS.pack(t, h, f, e, top_k, type_, x.data_ptr(), out.data_ptr(), ldx, ldo,
                          *_experts(gate, (e, f, h), "gate"), *_experts(up, (e, f, h), "up"),
                          *_experts(down, (e, h, f), "down"), 0 if router is None else router.data_ptr(), router_type,
                          ld_router, 1 if renormalize else 0, ids.data_ptr(), weights.data_ptr())
    _launch("moe_f8", dev, args, *_workspace(workspace), _status_ptr(status))
    return out, ids, weights
