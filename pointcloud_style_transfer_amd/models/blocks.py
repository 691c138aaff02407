"""Pre-norm gated residual blocks on the MI355X kernels (csrc/rms_norm.hip, csrc/gated_linear.hip):

    s = x + delta                       the residual stream, delta the previous block's output
    n = RMSNorm(s)                      with the addition above in the same launch
    delta' = Linear(act(n Wg^T + bg) * (n Wu^T + bu))

Functions first (rms_norm, gated_linear with gradients; rms_norm_quant, quant_rows, gated_linear_quant for
serving in 8 bits), then the modules that hold their weights.  All may be captured into a HIP graph, a forward
with its backward together; as torch has it, no eager graph of the same leaves may be alive at a capture.
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .. import _hip
from . import _autograd as _ag


def _wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _no_grad_form(name, *tensors):
    if _wants_grad(*tensors):
        raise RuntimeError(f"{name}: no gradients flow through 8 bits; call it under torch.no_grad()")


def rms_norm(x, weight, residual=None, eps=1e-6):
    """Root-mean-square norm over the last dimension (at most 16384 wide) -> y like x, or with a
    residual (y, s), s = x + residual rounded to x's type and y its norm.  x float32, bfloat16 or
    float16; weight [D] of x's type or float32.  Differentiable in x, weight and residual."""
    if _wants_grad(x, weight, residual):
        return _ag.RMSNormFn.apply(x, weight, residual, float(eps))
    y, s, _ = _hip.rms_norm(x, weight, residual, float(eps))
    return y if residual is None else (y, s)


def rms_norm_quant(x, weight, residual=None, eps=1e-6):
    """rms_norm with an 8-bit output -> (q, scale) or (q, scale, s): q float8_e4m3fn like x, scale
    float32 [...] with y = q * scale; scale = max |y| / 448 of a row, 1 for a row of zeros."""
    _no_grad_form("rms_norm_quant", x, weight, residual)
    q, scale, s = _hip.rms_norm_quant(x, weight, residual, float(eps))
    return (q, scale) if residual is None else (q, scale, s)


def quant_rows(x):
    """x [..., D] -> (q float8_e4m3fn, scale float32 [...]), x = q * scale: what gated_linear_quant takes
    as weights."""
    _no_grad_form("quant_rows", x)
    return _hip.quant_rows(x)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, act="silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up), x [..., D], weights [F, D] -> [..., F], in one
    kernel.  Operands of one type (float32, bfloat16 or float16; under torch.autocast they are rounded
    to its type), biases of that type or float32; act "silu", "gelu" or "relu".  Differentiable; relu's gradient
    may fall on either side where the gate is within the rounding of its own sum (1e-6 of the terms) of zero."""
    if (x.dim() != 2 or torch.is_autocast_enabled("cuda") or _wants_grad(x, w_gate, w_up, b_gate, b_up)):
        return _ag.GatedLinearFn.apply(x, w_gate, w_up, b_gate, b_up, act)
    return _hip.gated_linear(x, w_gate, w_up, b_gate, b_up, act)


def gated_linear_quant(q, scale, w_gate, gate_scale, w_up, up_scale, b_gate=None, b_up=None, act="silu",
                       out_dtype=torch.bfloat16):
    """gated_linear on 8-bit operands: q float8_e4m3fn [..., D] with scale [...] (rms_norm_quant),
    weights float8_e4m3fn [F, D] with scales [F] (quant_rows), biases of out_dtype or float32 ->
    [..., F] in out_dtype (bfloat16 or float16: 8-bit products are not summed finely enough for float32)."""
    _no_grad_form("gated_linear_quant", scale, gate_scale, up_scale, b_gate, b_up)
    if q.dtype != torch.float8_e4m3fn:
        raise RuntimeError(f"gated_linear_quant: float8_e4m3fn operands, got {q.dtype}")
    h = _hip.gated_linear(q.reshape(-1, q.shape[-1]), w_gate, w_up, b_gate, b_up, act,
                          (scale, gate_scale, up_scale), out_dtype)
    return h.view(*q.shape[:-1], h.shape[-1])


class RMSNorm(nn.Module):
    """rms_norm with its weight."""

    def __init__(self, dim: int, eps: float = 1e-6):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x, residual=None):
        return rms_norm(x, self.weight, residual, self.eps)


class GatedLinear(nn.Module):
    """gated_linear with its weights."""

    def __init__(self, dim: int, hidden: int, act: str = "silu", bias: bool = True):
        super().__init__()
        if act not in _hip.ACTS:
            raise ValueError(f"act is one of {sorted(_hip.ACTS)}, got {act!r}")
        self.act = act
        self.gate = nn.Linear(dim, hidden, bias=bias)
        self.up = nn.Linear(dim, hidden, bias=bias)

    def forward(self, x):
        return gated_linear(x, self.gate.weight, self.up.weight, self.gate.bias, self.up.bias, self.act)


class GatedBlock(nn.Module):
    """A pre-norm gated residual block on (x, delta), delta the previous block's output:
    s = x + delta; forward -> (s, Dropout(Linear(GatedLinear(RMSNorm(s)))))."""

    def __init__(self, dim: int, hidden: int, act: str = "silu", dropout: float = 0.1):
        super().__init__()
        self.norm = RMSNorm(dim)
        self.ff = GatedLinear(dim, hidden, act)
        self.down = nn.Linear(hidden, dim)
        self.drop = nn.Dropout(dropout)

    def forward(self, x, delta=None):
        n, s = (self.norm(x), x) if delta is None else self.norm(x, delta)
        return s, self.drop(_ag.linear(self.ff(n), self.down))

    @torch.no_grad()
    def pack(self, eight: bool):
        """The weights as `infer` reads them: bfloat16, gate and up in 8 bits with their scales if `eight`."""
        ff = self.ff
        gate, up = ((quant_rows(w.detach()) if eight else (w.detach().to(torch.bfloat16),))
                    for w in (ff.gate.weight, ff.up.weight))
        return (self.norm.weight.detach().float(), (*gate, *up, ff.gate.bias.detach().float(), ff.up.bias.detach().float()),
                self.down.weight.detach().to(torch.bfloat16), self.down.bias.detach().float(), eight)

    @torch.no_grad()
    def infer(self, packed, x, delta=None):
        """forward without dropout and gradients on bfloat16 rows x, delta [M, dim]; packed: pack()."""
        w, ff, down, bias, eight = packed
        if eight:
            q, scale, *s = rms_norm_quant(x, w, delta, self.norm.eps)
            s = s[0] if s else x
            h = gated_linear_quant(q, scale, *ff, self.ff.act)
        else:
            n, s = (rms_norm(x, w, None, self.norm.eps), x) if delta is None else rms_norm(x, w, delta, self.norm.eps)
            h = _hip.gated_linear(n, *ff, self.ff.act)
        return s, _hip.gemm_ex(h, down, bias, epilogue=_hip.EP_BF16)
