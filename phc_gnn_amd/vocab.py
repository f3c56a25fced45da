"""Operators against a large vocabulary: one-table embedding lookup and the softmax cross entropy of a linear map
(csrc/embedding.hip, csrc/linear_xent.hip).  Exported by ``phc_gnn_amd.ops``.

Unlike the message-passing operators they take fp32, bf16 and fp16 tensors.  Sums, softmax statistics and losses are fp32 in
every case; gradients come in the type of their input.  There is no CPU path."""
from __future__ import annotations

import ctypes as C
import os
from typing import Optional

import torch

from . import lib as L

_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def _dtype_id(what: str, t: torch.Tensor) -> int:
    try:
        return L.DTYPE_IDS[t.dtype]
    except KeyError:
        raise L.PhcError(f"{what}: float32, bfloat16 or float16 expected, got {t.dtype}") from None


def _int64(what: str, t: torch.Tensor) -> torch.Tensor:
    if t.dtype not in (torch.int64, torch.int32):
        raise L.PhcError(f"{what}: int64 or int32 expected, got {t.dtype}")
    return t.to(torch.int64).contiguous()


def _check_capture(who: str, *tensors: Optional[torch.Tensor]) -> None:
    """A leaf has ONE gradient node while any graph that ends in it lives, and autograd runs that node on the stream it was made on.  A
    backward captured on another stream would pull that stream into the capture, which ends the process when the capture ends: refused
    here, before anything is recorded."""
    leaves = [t for t in tensors if t is not None and t.requires_grad and t.is_leaf]
    if not leaves or not torch.is_grad_enabled() or not torch.cuda.is_current_stream_capturing():
        return
    for t in leaves:
        if torch_ops().gradient_on_another_stream(t):
            raise L.PhcError(f"{who}: captured into a graph while an eager result of the same parameter, made on another stream, still holds its "
                             "autograd graph; detach or delete that result (or make it on the capture's stream) first")


# the order of phc_torch_bind
_BOUND = ("phc_embedding_fwd", "phc_embedding_bwd", "phc_embedding_bwd_ws_bytes", "phc_linear_xent_fwd", "phc_linear_xent_bwd",
          "phc_linear_xent_state_bytes", "phc_linear_xent_ws_bytes", "phc_grad_norm_ws_bytes", "phc_grad_norm_clip", "phc_last_error")
_ops = None


def torch_ops():
    """The operators of torch in ``phc_gnn_amd`` (csrc/torch_vocab.cpp), bound to the loaded engine."""
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
        bind.restype, bind.argtypes = None, [C.c_void_p * len(_BOUND)]
        bind((C.c_void_p * len(_BOUND))(*(C.cast(getattr(lib, f), C.c_void_p) for f in _BOUND)))
        _ops = torch.ops.phc_gnn_amd
    return _ops


def _call(name: str, dev: torch.device, *args) -> torch.Tensor:
    try:
        out = getattr(_ops or torch_ops(), name).default(*args)
    except RuntimeError as exc:
        if str(exc).startswith("phc_"):                            # (the engine's refusal; out of memory and the like stay what they are)
            raise L.PhcError(str(exc).splitlines()[0]) from None
        raise
    L.maybe_check_indices(dev)
    return out


# ---- embedding ------------------------------------------------------------------------------------------------------------------
def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0, padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[tokens]``: ``weight`` [V, D], ``tokens`` int64 / int32 of any shape -> [*tokens.shape, D] in the weight's type.

    The gradient of ``weight`` is dense, ``scale`` times the sum of the rows' gradients per token in a fixed order (fp32, rounded once;
    bitwise reproducible), zero in row ``padding_idx``.  A token outside [0, V) reads row 0, counts as 0 in the gradient and is reported by
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
    return _call("embedding", dev, _int64("embedding: tokens", tokens), weight, float(scale), pad)


# ---- softmax cross entropy of a linear map ----------------------------------------------------------------------------------------
def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, bias: Optional[torch.Tensor] = None,
                         ignore_index: int = -100, reduction: str = "mean", piece: int = 0) -> torch.Tensor:
    """Softmax cross entropy of the logits ``x @ weight.T + bias`` against ``target``, without the logits in memory.

    ``x`` [*, D] and ``weight`` [V, D] (and ``bias`` [V]) of one type (fp32, bf16, fp16), ``target`` [*] int64 / int32 -> fp32 loss: one
    value (``reduction`` "mean", "sum") or one for each row ("none").  Rows whose target is ``ignore_index`` have loss 0 and a zero
    gradient and stay out of the mean; the mean of no rows is NaN, as for an empty selection.  A bias of -inf takes a column out of the
    vocabulary.  A target outside [0, V) counts as 0 and is reported by ``phc_gnn_amd.check_indices()``.

    The backward computes the logits again, ``piece`` columns of the vocabulary at a time (0: as many as half a GiB of scratch holds, 2048 at
    least; it grows with ``piece``).  The forward takes as many as half a GiB holds, and ``piece`` at most where it has to lay W out anew (fp32 of
    more than 256 rows, rows that are not whole 16-byte pieces).  Beside a piece lie a copy of ``x`` and, in the backward, ``dx`` in fp32 if there
    are several pieces and up to 128 MiB for split products.

    fp32 inputs have to be finite; they are multiplied to the accuracy of fp32.  With 16-bit inputs the logits' gradients, over the largest
    upstream gradient, are rounded to that type before the products with ``weight`` and ``x`` (sums in fp32, results rounded); in fp16 rows whose
    upstream gradient is far below the largest one lose bits (what is below 2^-28 of it is rounded to multiples of 2^-38).  An infinite or NaN
    upstream gradient of one row stays in its row of ``dx``.  Second derivatives are refused."""
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
    return _call("linear_cross_entropy", dev, x, weight, bias, _int64("linear_cross_entropy: target", target), int(ignore_index),
                 _REDUCTIONS[reduction], int(piece))
