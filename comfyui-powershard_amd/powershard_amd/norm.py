"""RMS norm whose rows go straight into quantized linears.

Between two blocks of a text decoder the residual stream is added to, normalized and, in front of W8A8 /
fp8 projections, quantized again by each of them.  RMSNorm does all three in one pass over the rows
(ops.add_rms_norm) when the linears that follow agree on what they multiply, and hands them the codes
(QuantLinear.forward_codes); in front of weight-only linears it returns the rows in their dtype.  The
reference runs its text encoders' norms as torch modules.
"""
import torch
from torch import nn

from . import ops
from .quant_linear import QuantizedRows, QuantLinear

__all__ = ["RMSNorm", "rows_for", "linear"]


def rows_for(linears):
    """("int8" or "fp8", ConvRot group) that all of the linears take, or None (16-bit rows)."""
    kinds = {x.input_codes() if isinstance(x, QuantLinear) else None for x in linears}
    return kinds.pop() if len(kinds) == 1 else None


def linear(module, rows, activation=None):
    """module(rows) for rows as RMSNorm returns them, the module's hooks included; activation as in
    QuantLinear.forward_act."""
    return module(rows) if activation is None else module.forward_act(rows, activation)


class RMSNorm(nn.Module):
    """y = h / sqrt(mean(h^2) + eps) * weight, h = x + residual, in fp32 on 16-bit rows."""

    def __init__(self, features, eps=1e-6, dtype=torch.bfloat16, device=None):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(features, dtype=dtype, device=device), requires_grad=False)
        self.eps = eps

    def forward(self, x, residual=None, linears=()):
        """(rows, h): rows for `linears` (QuantizedRows when rows_for names one kind of codes, else a tensor
        like x) and h = x + residual (x itself without a residual)."""
        kind = rows_for(linears) if linears else None
        flat = x.reshape(-1, x.shape[-1])
        res = None if residual is None else residual.reshape(flat.shape)
        codes, group = kind or (None, 0)
        out, scale, h = ops.add_rms_norm(flat, self.weight, self.eps, residual=res, codes=codes, rot_group=group)
        h = x if h is None else h.reshape(x.shape)
        if codes is None:
            return out.reshape(x.shape), h
        return QuantizedRows(out, scale, group, tuple(x.shape), x.dtype), h
