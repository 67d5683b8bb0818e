"""A mixture-of-experts layer for a few tokens (decode batches): router selection, gated FC1, FC2 and the weighted sum.

    ids, weights = moe_topk(logits, top_k)
    out[t] = sum_j weights[t, j] * W2[e] (silu(W1[e, :F] x[t]) * (W1[e, F:] x[t])),   e = ids[t, j]

The experts' weights are read once per batch and the routing stays on the device, as in ``grouped``: nothing is sorted or padded on
the host, and the three launches of ``moe_forward`` can be captured into a HIP graph.  Batches of more than 256 tokens and training
are ``grouped_linear``'s: there is no backward pass here, and a result of inputs that require a gradient raises when it is
differentiated.  The gate order is that of
``activation("swiglu", ...)``: activation half first.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _lib
from ._lib import api
from .grouped import GroupedTensor
from .tensor import DType, current_stream_ptr, refuse_gradient, te_dtype

__all__ = ["moe_topk", "moe_forward"]


def moe_topk(logits: torch.Tensor, top_k: int, renormalize: bool = True) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax over the last dim of ``logits`` [tokens, experts] (fp32 / bf16 / fp16, up to 1024 experts) and its ``top_k`` largest.

    Returns ``(ids int32 [tokens, top_k], weights fp32 [tokens, top_k])`` in falling order; equal logits go to the lowest index,
    NaN ranks last (and makes its token's weights NaN, except with ``renormalize`` where it is not chosen itself).  ``renormalize``
    divides a token's weights by their sum."""
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got {tuple(logits.shape)}")
    if logits.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if not logits.is_cuda:
        raise RuntimeError("the router runs on the GPU only (no CPU fallback in this library)")
    if logits.device.index != torch.cuda.current_device():
        with torch.cuda.device(logits.device):
            return moe_topk(logits, top_k, renormalize)
    logits = logits if logits.is_contiguous() else logits.contiguous()
    tokens, experts = logits.shape
    if not 1 <= top_k <= min(experts, 64):
        raise ValueError(f"top_k must be 1 to 64 and at most the number of experts ({experts}), got {top_k}")
    ids = torch.empty((tokens, top_k), dtype=torch.int32, device=logits.device)
    weights = torch.empty((tokens, top_k), dtype=torch.float32, device=logits.device)
    api.nvte_amd_moe_topk(logits.data_ptr(), ids.data_ptr(), weights.data_ptr(), tokens, experts, top_k, int(bool(renormalize)),
                          int(te_dtype(logits.dtype)), current_stream_ptr())
    if logits.requires_grad and torch.is_grad_enabled():
        weights, = refuse_gradient("moe_topk has no backward pass", weights)
    return ids, weights


def _expert_weight(name: str, w, scale_inv):
    """(tensor [experts, rows, cols], NVTE dtype, scale_inv or None) of a stacked tensor or a GroupedTensor."""
    if isinstance(w, GroupedTensor):
        if scale_inv is not None:
            raise ValueError(f"{name} is a GroupedTensor and carries its own scale_inv")
        if w.scaling_mode != _lib.NVTE_DELAYED_TENSOR_SCALING or w.rowwise_data is None:
            raise ValueError(f"{name} must hold row-wise data with per-tensor scaling")
        if w.first_dims is not None or w.last_dims is not None:
            raise ValueError(f"{name}'s members must all have one shape")
        rows, cols = w.logical_shape
        n = w.num_tensors
        dtype = w.fp8_dtype if w.fp8_dtype is not None else te_dtype(w.rowwise_data.dtype)
        return w.rowwise_data.view(n, rows // n, cols), dtype, w.scale_inv if w.fp8_dtype is not None else None
    if w.dim() != 3:
        raise ValueError(f"{name} must be [experts, rows, cols], got {tuple(w.shape)}")
    # raw bytes are E4M3 payloads, as everywhere in this package
    dtype = DType.kFloat8E4M3 if w.dtype == torch.uint8 else te_dtype(w.dtype)
    return w, dtype, scale_inv


def moe_forward(x: torch.Tensor, w_fc1: Union[torch.Tensor, GroupedTensor], w_fc2: Union[torch.Tensor, GroupedTensor],
                topk_ids: torch.Tensor, topk_weights: torch.Tensor, fc1_scale_inv: Optional[torch.Tensor] = None,
                fc2_scale_inv: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x [..., hidden] bf16 / fp16 with up to 256 tokens; w_fc1 [experts, 2 ffn, hidden], w_fc2 [experts, hidden, ffn] in x's dtype
    or FP8 E4M3 with ``scale_inv`` fp32 [experts] (or a ``GroupedTensor``, which carries its own); topk_ids int32 and
    topk_weights fp32 [tokens, top_k].  An id outside [0, experts) adds nothing; an id that a token names twice counts twice."""
    w1, t1, s1 = _expert_weight("w_fc1", w_fc1, fc1_scale_inv)
    w2, t2, s2 = _expert_weight("w_fc2", w_fc2, fc2_scale_inv)
    if x.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    experts, ffn2, hidden = w1.shape
    ffn = ffn2 // 2
    if x.dim() < 1 or x.shape[-1] != hidden:
        raise ValueError(f"x has shape {tuple(x.shape)}, but w_fc1 has {hidden} input features")
    if ffn2 % 2 or tuple(w2.shape) != (experts, hidden, ffn):
        raise ValueError(f"w_fc1 {tuple(w1.shape)} and w_fc2 {tuple(w2.shape)} are not [experts, 2 ffn, hidden] and "
                         "[experts, hidden, ffn]")
    if t1 != t2 or (t1 != DType.kFloat8E4M3 and t1 != te_dtype(x.dtype)):
        raise TypeError(f"weights must both be {x.dtype} or FP8 E4M3, got {t1.name} and {t2.name}")
    tokens = x.numel() // hidden if hidden else 0
    if topk_ids.dim() != 2 or topk_ids.shape != topk_weights.shape or topk_ids.shape[0] != tokens:
        raise ValueError(f"topk_ids {tuple(topk_ids.shape)} and topk_weights {tuple(topk_weights.shape)} must be [{tokens}, top_k]")
    if topk_ids.dtype != torch.int32 or topk_weights.dtype != torch.float32:
        raise TypeError(f"topk_ids must be int32 and topk_weights float32, got {topk_ids.dtype} and {topk_weights.dtype}")
    fp8 = t1 == DType.kFloat8E4M3
    for name, s in (("w_fc1", s1), ("w_fc2", s2)):
        if fp8 and (s is None or s.dtype != torch.float32 or s.numel() != experts):
            raise ValueError(f"{name} is FP8 and needs scale_inv, float32 [{experts}]")
        if not fp8 and s is not None:
            raise ValueError(f"{name} is not FP8 and takes no scale_inv")
    for name, t in (("x", x), ("w_fc1", w1), ("w_fc2", w2), ("topk_ids", topk_ids), ("topk_weights", topk_weights),
                    ("fc1_scale_inv", s1), ("fc2_scale_inv", s2)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}: this layer runs on the GPU only (no CPU fallback in this library)")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, but x is on {x.device}")
    if x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return moe_forward(x, w_fc1, w_fc2, topk_ids, topk_weights, fc1_scale_inv, fc2_scale_inv)
    if not (w1.is_contiguous() and w2.is_contiguous()):
        raise ValueError("expert weights must be contiguous")     # no silent copy of every expert
    dense = lambda t: t if t is None or t.is_contiguous() else t.contiguous()
    x2d, ids, weights, s1, s2 = dense(x), dense(topk_ids), dense(topk_weights), dense(s1), dense(s2)
    top_k = ids.shape[1]
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    size = api.nvte_amd_moe_forward_workspace_size(tokens, top_k, experts, hidden, ffn)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device)
    api.nvte_amd_moe_forward(x2d.data_ptr(), w1.data_ptr(), w2.data_ptr(), s1.data_ptr() if fp8 else 0,
                             s2.data_ptr() if fp8 else 0, ids.data_ptr(), weights.data_ptr(), out.data_ptr(), tokens, top_k,
                             experts, hidden, ffn, int(te_dtype(x.dtype)), int(t1), ws.data_ptr(), size, current_stream_ptr())
    if torch.is_grad_enabled() and (x.requires_grad or w1.requires_grad or w2.requires_grad or topk_weights.requires_grad):
        out, = refuse_gradient("moe_forward has no backward pass: train with GroupedLinear", out)
    return out
