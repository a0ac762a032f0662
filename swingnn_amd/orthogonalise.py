"""Newton-Schulz orthogonalisation of update matrices (swg_orthogonalise), the operator inside ``FusedMuonEMA``:

    X0 = G / (|G|_F + eps);   X <- a X + (b A + c A A) X  with  A = X X'   (a, b, c) = (3.4445, -4.7750, 2.0315)

It brings every singular value of G's normalised form towards 1 (into [0.68, 1.21] where it is not tiny) and keeps the
singular vectors: about U V' of G = U S V'.
"""
import torch

from . import _lib as L
from .engine import call_on, refuse_transforms

_TYPE = {torch.float32: L.SWG_F32, torch.bfloat16: L.SWG_BF16, torch.float16: L.SWG_F16}


def orthogonalise(g, steps=5, eps=1e-7, out_dtype=torch.bfloat16):
    """Orthogonalised matrices of ``g``: a tensor [rows, cols] or [batch, rows, cols], or a list of such tensors of any
    shapes (one type, one device), which go through the same launches.  float32, bfloat16 or float16 in; bfloat16 or
    float16 out: the products carry 11 bits, which leaves an error of 1e-3 ... 2e-3 of |O| beside the output's rounding (up
    to 3e-3 where all singular values are equal).  A zero matrix gives zero.  Not differentiable: a matrix that asks for a
    gradient in grad mode, one with a forward-mode tangent and a trace are refused.  The work is queued on the current
    stream and may be recorded into a graph."""
    single = isinstance(g, torch.Tensor)
    mats = [g] if single else list(g)
    refuse_transforms("orthogonalise", mats)
    if not 1 <= int(steps) <= 64:
        raise ValueError("orthogonalise: steps between 1 and 64")
    if not eps >= 0.0:
        raise ValueError("orthogonalise: eps >= 0")
    if out_dtype not in (torch.bfloat16, torch.float16):
        raise NotImplementedError(f"orthogonalise: bfloat16 or float16 out, got {out_dtype}")
    for t in mats:
        if t.dim() not in (2, 3):
            raise ValueError(f"orthogonalise: [rows, cols] or [batch, rows, cols], got shape {tuple(t.shape)}")
        if t.dtype not in _TYPE:
            raise NotImplementedError(f"orthogonalise: float32, bfloat16 or float16, got {t.dtype}")
        if t.dtype is not mats[0].dtype or t.device != mats[0].device:
            raise ValueError("orthogonalise: matrices of one type on one device")
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("orthogonalise has no gradient: call it under torch.no_grad() or on a detached matrix")
        if t.device.type != "cuda":
            raise RuntimeError("swingnn_amd runs on an MI355X only; there is no CPU fallback")
    if not mats:
        return []
    dev = mats[0].device
    outs, items, keep = [], (L.SwgOrthItem * len(mats))(), []
    for t, it in zip(mats, items):
        rows, cols = t.shape[-2:]
        t = t.detach().resolve_neg()  # z.conj().imag holds its sign as a flag, which a column keeps through what follows
        # a row of one element has no stride of its own
        if t.numel() and ((cols > 1 and t.stride(-1) != 1) or (rows > 1 and t.stride(-2) < cols)):
            t = t.contiguous()
        keep.append(t)
        out = torch.empty(t.shape, dtype=out_dtype, device=dev)
        outs.append(out)
        it.g, it.out = t.data_ptr(), out.data_ptr()
        it.ld_g, it.ld_out = (t.stride(-2) if rows > 1 else cols), cols
        it.bs_g, it.bs_out = (t.stride(0) if t.dim() == 3 else 0), rows * cols
        it.rows, it.cols, it.batch = rows, cols, (t.shape[0] if t.dim() == 3 else 1)
    nbytes = int(L.lib.swg_orthogonalise_workspace_bytes(len(mats), items))
    if nbytes == 0:
        raise L.SwgError("swg_orthogonalise_workspace_bytes: unsupported shapes")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    call_on(dev, L.lib.swg_orthogonalise, "swg_orthogonalise", len(mats), items, _TYPE[mats[0].dtype], _TYPE[out_dtype],
            int(steps), float(eps), ws.data_ptr(), nbytes)
    return outs[0] if single else outs
