"""Operators against a large vocabulary: one-table embedding lookup and the softmax cross entropy of a linear map
(csrc/embedding.hip, csrc/linear_xent.hip).  Exported by ``phc_gnn_amd.ops``.

Unlike the message-passing operators they take fp32, bf16 and fp16 tensors.  Sums, softmax statistics and losses are fp32 in
every case; gradients come in the type of their input, rounded once.  There is no CPU path."""
from __future__ import annotations

import contextlib
import ctypes as C
import os
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import lib as L

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def on_device(dev: torch.device):
    """Launches go to the tensors' device, whatever device is current."""
    return contextlib.nullcontext() if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _dtype_id(what: str, t: torch.Tensor) -> int:
    try:
        return L.DTYPE_IDS[t.dtype]
    except KeyError:
        raise L.PhcError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}") from None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A 2-D tensor the kernels can read in place: unit column stride, rows that do not overlap; anything else is copied."""
    if t.stride(1) == 1 and (t.stride(0) >= t.shape[1] or t.shape[0] == 1):
        return t
    return t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _int64(what: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise L.PhcError(f"{what}: int64 or int32 expected, got {t.dtype}")
    return t.to(torch.int64).contiguous()


def raw_stream(dev: torch.device) -> int:
    """The current stream of ``dev`` as a hipStream_t (``lib.stream_ptr`` without the Python stream object)."""
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _check_capture(who: str, *tensors: Optional[torch.Tensor]) -> None:
    """A leaf has ONE gradient node while any graph that ends in it lives, and autograd runs that node on the stream it was made on.  A
    backward captured on another stream would pull that stream into the capture, which ends the process when the capture ends: refused
    here, before anything is recorded."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves or not torch.is_grad_enabled() or not torch.cuda.is_current_stream_capturing():
        return
    for t in leaves:
        if _torch_ops().gradient_on_another_stream(t):
            raise L.PhcError(f"{who}: captured into a graph while an eager result of the same parameter, made on another stream, still holds its "
                             "autograd graph; detach or delete that result (or make it on the capture's stream) first")


_ops = None


def _torch_ops():
    """The operators of torch in ``phc_gnn_amd`` (csrc/torch_embedding.cpp), bound to the loaded engine."""
    global _ops
    if _ops is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libphc_torch.so")
        if not os.path.exists(path):
            raise L.PhcError(f"{path} not found: the operators of torch are not built (run `python -m phc_gnn_amd.build`)")
        lib = L.load()
        try:
            torch.ops.load_library(path)
            bind = C.CDLL(path).phc_torch_bind
        except (OSError, AttributeError) as exc:
            raise L.PhcError(f"cannot load {path}: {exc}; rebuild it") from exc
        bind.restype, bind.argtypes = None, [C.c_void_p] * 4
        bind(*(C.cast(f, C.c_void_p) for f in (lib.phc_embedding_fwd, lib.phc_embedding_bwd, lib.phc_embedding_bwd_ws_bytes, lib.phc_last_error)))
        _ops = torch.ops.phc_gnn_amd
    return _ops


# ---- embedding ------------------------------------------------------------------------------------------------------------------
def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``: ``weight`` [V, D], ``tokens`` int64 / int32 of any shape -> [*tokens.shape, D] in the weight's type.

    The gradient of ``weight`` is dense, ``scale`` times the sum of the rows' gradients per token in a fixed order (bitwise
    reproducible), zero in row ``padding_idx``.  A token outside [0, V) reads row 0, counts as 0 in the gradient and is reported by
    ``phc_gnn_amd.check_indices()``, like the encoders' feature values."""
    dev = L.require_device(tokens, weight)
    _dtype_id("embedding: weight", weight)
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise L.PhcError(f"embedding: weight [V, D] expected, got {tuple(weight.shape)}")
    _check_capture("embedding", weight)
    V = weight.shape[0]
    pad = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise L.PhcError(f"embedding: padding_idx {padding_idx} outside the {V} rows")
        pad = int(padding_idx) % V
    try:
        out = (_ops or _torch_ops()).embedding.default(_int64("embedding: tokens", tokens), weight, float(scale), pad)
    except RuntimeError as exc:
        if str(exc).startswith("phc_embedding_fwd"):
            raise L.PhcError(str(exc).splitlines()[0]) from None
        raise
    L.maybe_check_indices(dev)
    return out


# ---- softmax cross entropy of a linear map ----------------------------------------------------------------------------------------
def _xent_desc(x, w, bias, target, ignore_index, reduction, state, piece):
    d = L.LinearXentDesc()
    d.N, d.D = x.shape
    d.V = w.shape[0]
    d.ldx, d.ldw = _row_stride(x), _row_stride(w)
    d.ignore_index, d.piece = ignore_index, piece
    d.dtype, d.reduction = L.DTYPE_IDS[x.dtype], reduction
    d.x, d.W, d.bias, d.target = L.ptr(x), L.ptr(w), L.ptr(bias), L.ptr(target)
    d.state = L.ptr(state)
    return d


def _xent_workspace(lib, d, backward: int, dev) -> torch.Tensor:
    n = lib.phc_linear_xent_ws_bytes(C.byref(d), backward)
    if n == 0:
        raise L.PhcError(f"linear_cross_entropy: {lib.phc_last_error().decode()}")
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    d.ws, d.ws_bytes = ws.data_ptr(), n
    return ws


class _LinearCrossEntropyFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, target, ignore_index: int, reduction: int, piece: int):
        lib = L.load()
        dev = x.device
        N = x.shape[0]
        ctx.meta = (ignore_index, reduction, piece)
        if N == 0:
            ctx.save_for_backward(x, weight, bias)
            if reduction == 0:
                return torch.zeros(0, dtype=torch.float32, device=dev)
            return torch.full((), float("nan") if reduction == 2 else 0.0, dtype=torch.float32, device=dev)
        x_, w_ = _rows(x), _rows(weight)
        b_ = None if bias is None else bias.contiguous()
        loss = torch.empty((N,) if reduction == 0 else (), dtype=torch.float32, device=dev)
        state = torch.empty(lib.phc_linear_xent_state_bytes(N), dtype=torch.uint8, device=dev)
        d = _xent_desc(x_, w_, b_, target, ignore_index, reduction, state, piece)
        d.loss = L.ptr(loss)
        ws = _xent_workspace(lib, d, 0, dev)
        with on_device(dev):
            L.check(lib.phc_linear_xent_fwd(C.byref(d), raw_stream(dev)), "phc_linear_xent_fwd")
        del ws
        L.maybe_check_indices(dev)
        ctx.save_for_backward(x_, w_, b_, target, state)
        return loss

    @staticmethod
    def backward(ctx, dloss):
        return _xent_backward_once(ctx, dloss) if torch.is_grad_enabled() else _xent_backward(ctx, dloss)


def _xent_backward(ctx, dloss):
    lib = L.load()
    ignore_index, reduction, piece = ctx.meta
    need_x, need_w, need_b = ctx.needs_input_grad[:3]
    if len(ctx.saved_tensors) == 3:                          # no rows
        x, w, b = ctx.saved_tensors
        return (torch.zeros_like(x) if need_x else None, torch.zeros_like(w) if need_w else None,
                torch.zeros_like(b) if need_b else None, None, None, None, None)
    x, w, b, target, state = ctx.saved_tensors
    dev = x.device
    g = dloss.to(torch.float32).contiguous()
    dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if need_x else None
    dw = torch.empty(w.shape, dtype=w.dtype, device=dev) if need_w else None
    db = torch.empty(b.shape, dtype=b.dtype, device=dev) if need_b else None
    d = _xent_desc(x, w, b, target, ignore_index, reduction, state, piece)
    d.dloss, d.dx, d.dW, d.db = L.ptr(g), L.ptr(dx), L.ptr(dw), L.ptr(db)
    ws = _xent_workspace(lib, d, 1, dev)
    L.check(lib.phc_linear_xent_bwd(C.byref(d), raw_stream(dev)), "phc_linear_xent_bwd")       # (autograd has made dev the current device)
    del ws
    return dx, dw, db, None, None, None, None


_xent_backward_once = once_differentiable(_xent_backward)


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         ignore_index: int = -100, reduction: str = "mean", piece: int = 0) -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T + bias`` against ``target``, without the logits in memory.

    ``x`` [*, D] and ``weight`` [V, D] (and ``bias`` [V]) of one type (fp32, bf16, fp16), ``target`` [*] int64 / int32 -> fp32 loss: one
    value (``reduction`` "mean", "sum") or one for each row ("none").  Rows whose target is ``ignore_index`` have loss 0 and a zero
    gradient and stay out of the mean; the mean of no rows is NaN, as for an empty selection.  A bias of -inf takes a column out of the
    vocabulary.  A target outside [0, V) counts as 0 and is reported by ``phc_gnn_amd.check_indices()``.

    The backward computes the logits again, ``piece`` columns of the vocabulary at a time (0: as many as half a GiB of scratch holds; it
    grows with ``piece``).  fp32 inputs have to be finite; they are multiplied to the accuracy of fp32."""
    dev = L.require_device(x, weight, target, bias)
    _dtype_id("linear_cross_entropy: x", x)
    if weight.dim() != 2 or x.dim() < 1 or weight.shape[0] < 1 or weight.shape[1] < 1 or x.shape[-1] != weight.shape[1]:
        raise L.PhcError(f"linear_cross_entropy: x {tuple(x.shape)} does not fit weight {tuple(weight.shape)}")
    if weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise L.PhcError(f"linear_cross_entropy: x, weight and bias of one type expected, got {x.dtype}, {weight.dtype}"
                         + ("" if bias is None else f", {bias.dtype}"))
    if bias is not None and tuple(bias.shape) != (weight.shape[0],):
        raise L.PhcError(f"linear_cross_entropy: bias {tuple(bias.shape)} does not fit {weight.shape[0]} columns")
    if tuple(target.shape) != tuple(x.shape[:-1]):
        raise L.PhcError(f"linear_cross_entropy: target {tuple(target.shape)} does not fit x {tuple(x.shape)}")
    if reduction not in _REDUCTIONS:
        raise L.PhcError(f"linear_cross_entropy: unknown reduction '{reduction}' (known: {sorted(_REDUCTIONS)})")
    if piece < 0:
        raise L.PhcError(f"linear_cross_entropy: piece {piece}")
    _check_capture("linear_cross_entropy", x, weight, bias)
    t = _int64("linear_cross_entropy: target", target).reshape(-1)
    loss = _LinearCrossEntropyFn.apply(x.reshape(-1, x.shape[-1]), weight, bias, t, int(ignore_index), _REDUCTIONS[reduction], int(piece))
    return loss.reshape(target.shape) if reduction == "none" else loss
