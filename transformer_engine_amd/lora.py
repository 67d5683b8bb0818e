"""Low-rank adapters of many requests beside a shared projection.

Every token ``t`` names its adapter ``a = adapter_ids[t]`` (any value outside ``[0, num_adapters)``: none) and gets

    y[t]  = base[t]      + scaling[a] * B_a (A_a x[t])
    dx[t] = base_grad[t] + scaling[a] * A_a^T (B_a^T dy[t])
    dA_a  = sum_t scaling[a] (B_a^T dy[t]) x[t]^T        dB_a = sum_t dy[t] (scaling[a] A_a x[t])^T

with ``A [num_adapters, rank, in]`` and ``B [num_adapters, out, rank]``.  ``base`` is the shared projection's output, for
instance of ``linear.Linear``.  Tokens of one adapter need not be neighbours: a decode batch (one token per request), prompts
back to back and a training batch go through the same call.  ``lora_forward`` / ``lora_backward`` are the bare passes (as
``linear.linear_forward`` / ``linear_backward``), ``lora`` is differentiable, ``LoRALinear`` puts adapters beside a frozen FP8
``Linear``.

Everything is bf16 or fp16 (one dtype per call), rank vectors and sums are fp32, each result is rounded once.  Inputs may be
strided (they are copied then); workspaces come from the caller's stream, so every pass can be captured into a HIP graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from ._lib import api
from .linear import Linear, linear_backward, linear_forward
from .tensor import current_stream_ptr, refuse_gradient, te_dtype

__all__ = ["lora_forward", "lora_backward", "lora", "LoRALinear"]

_DTYPES = (torch.bfloat16, torch.float16)


class LoRASaved(NamedTuple):
    """What ``lora_backward`` needs of the forward pass."""
    x: torch.Tensor             # [tokens, in]
    a: torch.Tensor
    b: torch.Tensor
    adapter_ids: torch.Tensor   # [tokens]
    scaling: Optional[torch.Tensor]
    low: torch.Tensor           # fp32 partial sums of A x
    x_shape: Tuple[int, ...]


def _rows(name: str, t: torch.Tensor, like: torch.Tensor, shape) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, but expected {tuple(shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} has dtype {t.dtype}, but expected {like.dtype}")
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, but x is on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _check(x, a, b, adapter_ids, scaling):
    if x.dtype not in _DTYPES:
        raise TypeError(f"adapters take bfloat16 or float16 activations, got {x.dtype}")
    if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
        raise ValueError(f"expected a [num_adapters, rank, in] and b [num_adapters, out, rank], got {tuple(a.shape)} and "
                         f"{tuple(b.shape)}")
    if x.dim() < 1 or x.shape[-1] != a.shape[2]:
        raise ValueError(f"x has shape {tuple(x.shape)}, but a has {a.shape[2]} input features")
    if adapter_ids.dtype != torch.int32:
        raise TypeError(f"adapter_ids must be int32, got {adapter_ids.dtype}")
    if adapter_ids.shape != x.shape[:-1]:
        raise ValueError(f"adapter_ids has shape {tuple(adapter_ids.shape)}, but expected one id per token, {tuple(x.shape[:-1])}")
    for name, t in (("a", a), ("b", b)):
        if t.dtype != x.dtype:
            raise TypeError(f"{name} has dtype {t.dtype}, but x has {x.dtype}")
    if scaling is not None and (scaling.dtype != torch.float32 or scaling.shape != (a.shape[0],)):
        raise ValueError(f"scaling must be float32 [{a.shape[0]}], got {scaling.dtype} {tuple(scaling.shape)}")
    for name, t in (("x", x), ("a", a), ("b", b), ("adapter_ids", adapter_ids), ("scaling", scaling)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} is on {t.device}: adapters run on the GPU only (no CPU fallback in this library)")
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, but x is on {x.device}")


def _span(t: torch.Tensor):
    return t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()


def lora_forward(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor,
                 scaling: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None,
                 out: Optional[torch.Tensor] = None, needs_backward: bool = True):
    """Returns ``(y, saved)``, ``saved`` for ``lora_backward`` (None without ``needs_backward``).

    x [..., in], adapter_ids int32 [...], scaling fp32 [num_adapters] (default 1), base [..., out] (default 0).  ``out`` receives y
    and may be ``base`` itself; it must not overlap any other input."""
    _check(x, a, b, adapter_ids, scaling)
    if x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return lora_forward(x, a, b, adapter_ids, scaling, base, out, needs_backward)
    n, rank, k = a.shape
    o = b.shape[1]
    y_shape = x.shape[:-1] + (o,)
    x2d = x if x.is_contiguous() else x.contiguous()
    a, b = a if a.is_contiguous() else a.contiguous(), b if b.is_contiguous() else b.contiguous()
    ids = adapter_ids if adapter_ids.is_contiguous() else adapter_ids.contiguous()
    scaling = scaling if scaling is None or scaling.is_contiguous() else scaling.contiguous()
    if base is not None:
        base = _rows("base", base, x, y_shape)
    if out is None:
        out = torch.empty(y_shape, dtype=x.dtype, device=x.device)
    else:
        if out.shape != y_shape or out.dtype != x.dtype or out.device != x.device or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous {x.dtype} tensor of shape {tuple(y_shape)} on {x.device}")
        begin, end = _span(out)
        for name, t in (("x", x2d), ("a", a), ("b", b), ("adapter_ids", ids), ("scaling", scaling), ("base", base)):
            if t is None or (name == "base" and t.data_ptr() == begin):
                continue
            lo, hi = _span(t)
            if lo < end and begin < hi:
                raise ValueError(f"out overlaps {name}")
    tokens = ids.numel()
    low = torch.empty((api.nvte_amd_lora_num_slices(tokens, k), tokens, rank), dtype=torch.float32, device=x.device)
    size = api.nvte_amd_lora_forward_workspace_size(tokens, n)
    ws = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    api.nvte_amd_lora_forward(x2d.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(),
                              0 if scaling is None else scaling.data_ptr(), 0 if base is None else base.data_ptr(),
                              out.data_ptr(), low.data_ptr(), tokens, k, o, rank, n, int(te_dtype(x.dtype)),
                              ws.data_ptr() if size else 0, size, current_stream_ptr())
    saved = LoRASaved(x2d, a, b, ids, scaling, low, tuple(x.shape)) if needs_backward else None
    return out, saved


def lora_backward(dy: torch.Tensor, saved: LoRASaved, base_grad: Optional[torch.Tensor] = None,
                  grad_dtype: Optional[torch.dtype] = None, requires_dgrad: bool = True, requires_wgrad: bool = True):
    """Returns ``(dx, da, db)`` (None for what is not asked for).

    dy [..., out]; base_grad [..., in]: the gradient that the shared projection sends back, added to dx (default 0);
    grad_dtype: dtype of da and db, the adapters' own (default) or float32."""
    x, a, b, ids, scaling, low, x_shape = saved
    if x.device.index != torch.cuda.current_device():
        with torch.cuda.device(x.device):
            return lora_backward(dy, saved, base_grad, grad_dtype, requires_dgrad, requires_wgrad)
    n, rank, k = a.shape
    o = b.shape[1]
    dy = _rows("dy", dy, x, x_shape[:-1] + (o,))
    if base_grad is not None:
        base_grad = _rows("base_grad", base_grad, x, x_shape)
    gdt = grad_dtype or a.dtype
    if gdt not in (a.dtype, torch.float32):
        raise TypeError(f"grad_dtype must be {a.dtype} or torch.float32, got {gdt}")
    if not (requires_dgrad or requires_wgrad):
        return None, None, None
    tokens = ids.numel()
    dev = x.device
    dx = torch.empty(x_shape, dtype=x.dtype, device=dev) if requires_dgrad else None
    da = torch.empty(a.shape, dtype=gdt, device=dev) if requires_wgrad else None
    db = torch.empty(b.shape, dtype=gdt, device=dev) if requires_wgrad else None
    size = (api.nvte_amd_lora_backward_workspace_size(tokens, k, o, rank, n) if requires_wgrad
            else api.nvte_amd_lora_dgrad_workspace_size(tokens, o, rank, n))
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    ptr = lambda t: 0 if t is None else t.data_ptr()
    api.nvte_amd_lora_backward(x.data_ptr(), dy.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), ptr(scaling),
                               low.data_ptr(), ptr(base_grad), ptr(dx), ptr(da), ptr(db), tokens, k, o, rank, n,
                               int(te_dtype(x.dtype)), int(te_dtype(gdt)), ws.data_ptr(), size, current_stream_ptr())
    return dx, da, db


def _save(ctx, saved: LoRASaved):
    ctx.save_for_backward(saved.x, saved.a, saved.b, saved.adapter_ids, saved.scaling, saved.low)
    ctx.x_shape = saved.x_shape


def _load(ctx) -> LoRASaved:
    return LoRASaved(*ctx.saved_tensors, ctx.x_shape)


def _first_order(*grads):
    """What a backward pass returns: under ``create_graph`` gradients that raise when they are differentiated themselves."""
    return refuse_gradient("adapters have no second derivatives", *grads) if torch.is_grad_enabled() else grads


class _LoRAFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, adapter_ids, scaling, base):
        y, saved = lora_forward(x, a, b, adapter_ids, scaling, base)
        _save(ctx, saved)
        return y

    @staticmethod
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        dx, da, db = _first_order(*lora_backward(dy, _load(ctx), requires_dgrad=need[0], requires_wgrad=need[1] or need[2]))
        return dx, da, db, None, None, dy if need[5] else None


def lora(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, adapter_ids: torch.Tensor,
         scaling: Optional[torch.Tensor] = None, base: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``base + scaling * B (A x)``, differentiable once in x, a, b and base (``scaling`` is a constant)."""
    if scaling is not None and scaling.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("scaling is a constant of the adapters and gets no gradient: detach it")
    return _LoRAFn.apply(x, a, b, adapter_ids, scaling, base)


class _LoRALinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, adapter_ids, scaling, module):
        lin = module.linear
        base, (_, w8) = linear_forward(x, lin.weight, lin.bias, lin.fp8_state, is_first_microbatch=module._is_first_microbatch,
                                       needs_backward=module._needs_backward)
        # x's FP8 copy is the weight gradient's, which a frozen weight has not
        ctx.saved_q = (None, w8) if ctx.needs_input_grad[0] else None
        y, saved = lora_forward(x, a, b, adapter_ids, scaling, base=base, out=base)
        _save(ctx, saved)
        ctx.module = module
        return y

    @staticmethod
    def backward(ctx, dy):
        lin = ctx.module.linear
        need = ctx.needs_input_grad
        base_grad = None
        if need[0]:
            base_grad, _, _ = linear_backward(dy, ctx.saved_q, lin.fp8_state, requires_wgrad=False)
            base_grad = base_grad.reshape(ctx.x_shape)
            lin.fp8_state.update_bwd(lin.amax_group)
        dx, da, db = _first_order(*lora_backward(dy, _load(ctx), base_grad=base_grad, requires_dgrad=need[0],
                                                 requires_wgrad=need[1] or need[2]))
        return dx, da, db, None, None, None


class LoRALinear(torch.nn.Module):
    """A frozen FP8 ``Linear`` with trainable low-rank adapters beside it.

    ``lora_a`` [num_adapters, rank, in] starts random and ``lora_b`` [num_adapters, out, rank] at zero, so a new adapter changes
    nothing; ``scaling`` is ``alpha / rank`` for every adapter (``alpha`` defaults to the rank).  Without ``adapter_ids`` every token
    uses adapter 0.  A projection whose parameters require a gradient is refused: it would get none (``Linear`` and ``lora`` train
    both).  ``is_first_microbatch`` keeps the shared weight's FP8 copy over calls as ``Linear`` does."""

    def __init__(self, in_features: int, out_features: int, rank: int, num_adapters: int = 1, alpha: Optional[float] = None,
                 bias: bool = True, params_dtype: torch.dtype = torch.bfloat16, device="cuda", recipe=None):
        super().__init__()
        if params_dtype not in _DTYPES:
            raise TypeError(f"adapters take bfloat16 or float16 parameters, got {params_dtype}")
        if not 1 <= rank <= 128:
            raise ValueError(f"rank must be 1 to 128, got {rank}")
        self.linear = Linear(in_features, out_features, bias=bias, params_dtype=params_dtype, device=device, recipe=recipe)
        self.linear.requires_grad_(False)
        self.lora_a = torch.nn.Parameter(torch.empty(num_adapters, rank, in_features, dtype=params_dtype, device=device))
        torch.nn.init.normal_(self.lora_a, std=in_features ** -0.5)
        self.lora_b = torch.nn.Parameter(torch.zeros(num_adapters, out_features, rank, dtype=params_dtype, device=device))
        self.register_buffer("scaling", torch.full((num_adapters,), (rank if alpha is None else alpha) / rank,
                                                   dtype=torch.float32, device=device))

    def _apply(self, fn, *args, **kwargs):
        scaling = self.scaling
        super()._apply(fn, *args, **kwargs)
        if self.scaling.dtype != torch.float32:     # a cast of the parameters leaves the factor as it was
            self.scaling = scaling.to(self.scaling.device)
        return self

    def forward(self, x: torch.Tensor, adapter_ids: Optional[torch.Tensor] = None,
                is_first_microbatch: Optional[bool] = None) -> torch.Tensor:
        if adapter_ids is None:
            adapter_ids = torch.zeros(x.shape[:-1], dtype=torch.int32, device=x.device)
        _check(x, self.lora_a, self.lora_b, adapter_ids, self.scaling)
        if torch.is_grad_enabled() and any(p.requires_grad for p in self.linear.parameters()):
            raise RuntimeError("the projection of a LoRALinear is frozen, but its weight or bias requires a gradient: call "
                               "requires_grad_(False) on it, or use Linear and lora to train both")
        self._is_first_microbatch = is_first_microbatch
        self._needs_backward = torch.is_grad_enabled()
        y = _LoRALinearFn.apply(x, self.lora_a, self.lora_b, adapter_ids, self.scaling, self)
        self.linear.fp8_state.update_fwd(self.linear.amax_group)
        return y
