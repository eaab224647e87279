"""Closer bounds than those of seq_cases for two of the norms' gradients.

Column sums: a lane adds its rows one after the other, the lane groups of a workgroup are joined, sixteen waves add the
workgroups' rows and are joined.  With at most 768 to 1 536 workgroups the longest chain of additions at the sizes used here is
    40 001 x 24 fp32: 2 rows a lane + 32 groups + 48 + 16 = 98,   9 001 x 600 bf16: 6 + 96 + 16 = 118,
    20 011 x 200 fp32: 7 + 4 + 48 + 16 = 75,
so CHAIN roundings of the magnitudes' sum, and not as many as there are rows.

The slope of a gate: p = rcp(1 + e), q = e p p, with e = exp(-z) off by at most 4 u (the hardware's 1 ulp is 2 u, the correction
of the exponent's product and its fma 1 u each), 1 + e by 1 u more, the reciprocal 2 u: p is off by 7 u of itself and q, with its
two products, by 4 + 14 + 2 = 20 u of itself; the SiLU's p + z q by one more rounding.  24 u of p + |z| q, relative to the value
also where the gate is all but open, plus the subnormals that the hardware replaces by 0."""
import torch

from tests import seq_cases as S

CHAIN = 160


def terms(x, y, weight, gate, scale, next_weight, activation, d_out, d_next, eps=1e-5):
    """The terms of d_next_weight and of d_weight (those of d_scale are weight / scale as large) in 64 bits, [rows, width]."""
    r = S.block_norm(x, y, weight, gate, scale, next_weight, activation, eps, d_out, d_next)
    X, Y, W = x.double(), y.double(), weight.double()
    inv = 1 / (Y.square().mean(1, keepdim=True) + eps).sqrt()
    f = torch.ones_like(X) if gate is None else {"none": gate.double(), "sigmoid": torch.sigmoid(gate.double()),
                                                 "silu": gate.double() * torch.sigmoid(gate.double())}[activation]
    out = X + scale.double() * f * Y * inv * W
    io = 1 / (out.square().mean(1, keepdim=True) + eps).sqrt()
    return d_next.double() * out * io, r["d_x"][0] * f * scale.double() * Y * inv, r


def column(reference, term, factor=1.0):
    """(value, bound) of a column sum from seq_cases' with the chain of additions in place of the rows."""
    value, bound = reference
    return value, bound - (term.shape[0] + 32 - CHAIN) * S.U * term.abs().sum(0) * factor


def gate_gradient(t, d_out, d_next, activation):
    """(value, bound) of d_gate, the slope's error relative to the slope."""
    wide = {k: (None if v is None else v.float()) for k, v in t.items()}
    r = S.block_norm(**wide, activation=activation, d_out=d_out.float(), d_next=d_next.float())
    z = t["gate"].double()
    p = torch.sigmoid(z)
    q = p * torch.sigmoid(-z)
    size = q if activation == "sigmoid" else p + z.abs() * q
    slope = q if activation == "sigmoid" else p + z * q
    y = t["y"].double()
    normed = y / (y.square().mean(1, keepdim=True) + 1e-5).sqrt() * t["weight"].double() * t["scale"].double()
    d, e_d = r["d_x"]
    value = d * normed * slope
    e = normed.abs() * (slope.abs() * e_d + d.abs() * (24 * S.U * size + 2.0 ** -126 * (1 + z.abs()))) + 32 * S.U * value.abs()
    return value, e + S.stored(value, t["gate"].dtype)
