"""Layer norm over the last axis as an operator of its own, with gradients (swg_layer_norm_fwd / swg_layer_norm_bwd):

    y = (x - mean) / sqrt(var + eps) * weight + bias

for modules that train next to the denoiser: inside SwinGNN's own ops the norm is part of fused kernels.  ``x`` is
float32, bfloat16 or float16 with any leading shape and row stride; ``weight`` and ``bias`` (either may be None) are
float32 or of x's type, their gradients come in that type.  Means, variances and every sum are held in float32; the
gradients of weight and bias are reduced in a fixed order, so equal inputs give equal bits.
``LayerNorm`` is the module form: an ``nn.LayerNorm`` (same constructor, same ``state_dict``) whose forward runs here;
the networks take it as ``norm_layer``.
"""
import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib as L
from .engine import call_on, refuse_transforms

_TYPE = {torch.float32: L.SWG_F32, torch.bfloat16: L.SWG_BF16, torch.float16: L.SWG_F16}


def _rows(t, D):
    """t as [rows, D] with unit stride along D, without a copy where its strides allow it."""
    if D == 1:
        t = t.resolve_neg()  # the sign flag of z.conj().imag; wider rows of it have a stride of two, and their copy resolves it
    if t.dim() != 2:
        try:
            t = t.view(-1, D)
        except RuntimeError:
            t = t.reshape(-1, D)
    return t if D == 1 or t.stride(1) == 1 else t.contiguous()


def _like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, eps, keep):
    D = x.shape[-1]
    x2 = _rows(x, D)
    rows = x2.shape[0]
    y = _like(x)
    stat = mean = rstd = None
    if keep:
        stat = x2.new_empty((2, rows), dtype=torch.float32)  # mean, then 1 / sqrt(var + eps)
        mean = stat.data_ptr()
        rstd = mean + 4 * rows
    wt = weight if weight is not None else bias
    wtype = _TYPE[x.dtype if wt is None else wt.dtype]
    call_on(x.device, L.lib.swg_layer_norm_fwd, "swg_layer_norm_fwd", rows, D, x2.data_ptr(), x2.stride(0), _TYPE[x.dtype],
            _ptr(weight), _ptr(bias), wtype, eps, y.data_ptr(), D, mean, rstd)
    return y, x2, stat, wtype


_WS_FLOATS = {}  # (rows, D, type) -> size: plain numbers, asked for once


def _ws_floats(rows, D, xt):
    n = _WS_FLOATS.get((rows, D, xt))
    if n is None:
        if len(_WS_FLOATS) > 4096:
            _WS_FLOATS.clear()
        n = _WS_FLOATS[(rows, D, xt)] = L.lib.swg_layer_norm_bwd_workspace_bytes(rows, D, xt) // 4
    return n


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, x2, stat, ctx.wtype = _forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x2, weight, bias, stat)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, bias, stat = ctx.saved_tensors
        rows, D = x2.shape
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = _like(dy) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        dy = _rows(dy, D)
        xt = _TYPE[x2.dtype]
        nbytes, ws = 0, None
        if need_w or need_b:
            n = _ws_floats(rows, D, xt)
            nbytes, ws = 4 * n, stat.new_empty(n)
        mean = stat.data_ptr()
        call_on(x2.device, L.lib.swg_layer_norm_bwd, "swg_layer_norm_bwd", rows, D, x2.data_ptr(), x2.stride(0), dy.data_ptr(),
                dy.stride(0), xt, _ptr(weight), ctx.wtype, mean, mean + 4 * rows, _ptr(dx), D, _ptr(dw), _ptr(db), _ptr(ws),
                nbytes)
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """Layer norm of ``x`` over its last axis; differentiable once, in reverse mode (a forward-mode tangent, a trace and a
    second derivative are refused)."""
    refuse_transforms("layer_norm", (x, weight, bias))
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"layer_norm: a last axis to normalise is needed, got shape {tuple(x.shape)}")
    if x.dtype not in _TYPE:
        raise NotImplementedError(f"layer_norm: float32, bfloat16 or float16, got {x.dtype}")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        if t.shape != x.shape[-1:]:
            raise ValueError(f"layer_norm: {what} has shape {tuple(t.shape)}, the last axis {x.shape[-1]}")
        if t.dtype is not torch.float32 and t.dtype is not x.dtype:
            raise NotImplementedError(f"layer_norm: {what} in float32 or in x's {x.dtype}, got {t.dtype}")
        if t.device != x.device:
            raise RuntimeError(f"layer_norm: {what} is on {t.device}, x on {x.device}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise NotImplementedError("layer_norm: weight and bias of one type")
    if x.device.type != "cuda":
        raise RuntimeError("swingnn_amd runs on an MI355X only; there is no CPU fallback")
    if x.shape[-1] == 1:
        weight, bias = (t if t is None else t.resolve_neg() for t in (weight, bias))
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    return _forward(x, weight, bias, eps, False)[0]


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over one axis whose forward is ``layer_norm``.  Under autocast it does what ``nn.LayerNorm`` does
    there: half types are normalised and returned in float32 (``layer_norm`` itself takes what it is given)."""

    def __init__(self, *args, **kwargs):
        super().__init__(*args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise NotImplementedError("LayerNorm: one normalised axis")

    def forward(self, x):
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"LayerNorm: last axis {tuple(x.shape)[-1:]}, normalised shape {tuple(self.normalized_shape)}")
        weight, bias = self.weight, self.bias
        if torch.is_autocast_enabled("cuda"):
            x, weight, bias = (t.float() if t is not None and t.dtype in (torch.bfloat16, torch.float16) else t
                               for t in (x, weight, bias))
        return layer_norm(x, weight, bias, self.eps)
