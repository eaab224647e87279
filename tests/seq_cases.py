"""Plain 64-bit forms of the sequence operators with the error that the kernels' types allow, and the inputs the tests
share.

u = 2^-24 is half a step of fp32, half_step(t) that of a result's type.  Every bound is a sum of magnitudes times the
number of fp32 roundings that can have touched them, plus half a step of the stored result."""
import torch

U = 2.0 ** -24
GROUP = 64


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def stored(ref, dtype):
    """Half a step of a result of that size in its type (subnormal results: half of the smallest step)."""
    info = torch.finfo(dtype)
    return (ref.abs() * half_step(dtype)).clamp_min(info.smallest_normal * info.eps / 2)


def close(got, ref, bound, what):
    err = (got.double().cpu() - ref.cpu()).abs()
    bound = bound.cpu().expand_as(err)
    bad = ~(err <= bound)
    if bad.any():
        i = int(torch.where(bad, err / bound.clamp_min(1e-300), torch.zeros_like(err)).argmax())
        raise AssertionError("%s: %d of %d outside; worst at %d: got %r, is %r, allowed %.3g" % (
            what, int(bad.sum()), bad.numel(), i, float(got.reshape(-1)[i]), float(ref.reshape(-1)[i]),
            float(bound.reshape(-1)[i])))


# ---- recurrence -------------------------------------------------------------------------------------------------

def recurrence(gate, inp, state=None, reset=None, reverse=False, d_out=None, d_last=None):
    """name -> (value, bound) in float64 on the CPU.  A value is a sum of products; the magnitudes' sums run through the
    same recurrence.  A step rounds at most three times (the fma; where the time is split, also the product of the gates
    and the sum of the span), each time by u of the magnitudes' sum."""
    dt = inp.dtype
    g, b = gate.detach().double().cpu().expand(inp.shape), inp.detach().double().cpu()
    steps, n, d = b.shape
    keep = torch.ones(steps, n, 1, dtype=torch.bool) if reset is None else (reset.cpu() == 0)[:, :, None]
    keep = keep.expand(b.shape)
    zero = torch.zeros(n, d, dtype=torch.float64)
    h0 = zero if state is None else state.detach().double().cpu()
    order = list(range(steps))[::-1] if reverse else list(range(steps))
    out, err, before, err_before = (torch.zeros_like(b) for _ in range(4))
    h, m, e = h0, h0.abs(), zero
    for t in order:
        before[t], err_before[t] = h, e
        h = torch.where(keep[t], g[t] * h, zero) + b[t]
        m = torch.where(keep[t], g[t].abs() * m, zero) + b[t].abs()
        e = torch.where(keep[t], g[t].abs() * e, zero) + 3 * U * m
        out[t], err[t] = h, e
    r = {"out": (out, err + stored(out, dt)), "last": (h, e + stored(h, torch.float32))}
    if d_out is None and d_last is None:
        return r
    go = torch.zeros_like(b) if d_out is None else d_out.detach().double().cpu()
    c = zero if d_last is None else d_last.detach().double().cpu()
    mc, ec = c.abs(), zero
    d_inp, d_gate, e_inp, e_gate = (torch.zeros_like(b) for _ in range(4))
    for i in range(steps - 1, -1, -1):
        t = order[i]
        c, mc = c + go[t], mc + go[t].abs()
        ec = ec + 3 * U * mc
        d_inp[t], e_inp[t] = c, ec
        # `before` is read as stored: half a step of its type where it is an element of out, exact where it is state
        eh = err_before[t] + (stored(before[t], dt) if i else 0.0)
        dg = torch.where(keep[t], c * before[t], zero)
        d_gate[t] = dg
        e_gate[t] = torch.where(keep[t], ec * (before[t].abs() + eh) + c.abs() * eh + U * dg.abs(), zero)
        c = torch.where(keep[t], g[t] * c, zero)
        mc = torch.where(keep[t], g[t].abs() * mc, zero)
        ec = torch.where(keep[t], g[t].abs() * ec, zero)
    r.update(d_inp=(d_inp, e_inp + stored(d_inp, dt)), d_gate=(d_gate, e_gate + stored(d_gate, dt)),
             d_state=(c, ec + stored(c, torch.float32)))
    return r


# ---- norms --------------------------------------------------------------------------------------------------------

def through8(x):
    """What the 8-bit codes of x [R, D] stand for, from the definition in fp32 steps."""
    r, d = x.shape
    groups = -(-d // GROUP) if d else 0
    p = torch.zeros(r, groups * GROUP)
    p[:, :d] = x.detach().float().cpu()
    p = p.reshape(r, groups, GROUP)
    top = p.abs().amax(-1, keepdim=True)
    full = torch.full_like(top, 127.0)
    tiny, bad = top < 2.0 ** -120, ~torch.isfinite(top)
    inverse = torch.where(tiny | bad, torch.zeros_like(top), full / top)
    scale = torch.where(tiny, torch.zeros_like(top), top / full)
    scale = torch.where(bad, torch.full_like(top, float("nan")), scale)
    code = torch.where(inverse == 0, torch.zeros_like(p), torch.round(p * inverse))
    return (code * scale).reshape(r, -1)[:, :d], code.reshape(r, -1)[:, :d], scale.reshape(r, groups)


def block_norm(x, y=None, weight=None, gate=None, scale=None, next_weight=None, activation="silu", eps=1e-5, d_out=None,
               d_next=None, checkpoint=False):
    """name -> (value, bound) in float64 on the CPU.

    Roundings, as counts c of u relative to the magnitudes' sums: a row's sum of squares takes at most 7 serial additions
    in a lane, 6 over a wave's lanes and 16 over the waves, which the inverse root halves: with its own rounding, the
    quotient and the gate's exponential (about 4) no factor of a term is off by more than 32 u.  A second sum over the row
    (the gradient's) adds as many again: 64 u.  Column sums add at most `rows` further terms one after the other.
    The sigmoid is a hardware reciprocal, 0 in place of a subnormal result: off by less than 2^-126, and z times that."""
    dt = x.dtype
    c1, c2 = 32 * U, 96 * U

    def f64(t):
        return None if t is None else t.detach().double().cpu()

    X, Y, W, Z, S, W2 = f64(x), f64(y), f64(weight), f64(gate), f64(scale), f64(next_weight)
    rows, width = X.shape
    one = torch.ones(width, dtype=torch.float64)
    S = one if S is None else S

    def act(z):
        if z is None:
            return torch.ones_like(X), torch.zeros_like(X)
        p = torch.sigmoid(z)
        return {"none": (z, torch.ones_like(z)), "sigmoid": (p, p * torch.sigmoid(-z)),
                "silu": (z * p, p + z * p * torch.sigmoid(-z))}[activation]

    def inv(v):
        return 1 / (v.square().mean(1, keepdim=True) + eps).sqrt()

    def flushed(z):
        return 0.0 if z is None or activation == "none" else 2.0 ** -126 * (1 + z.abs())

    r = {}
    out, bound = X, torch.zeros_like(X)
    if Y is not None:
        iy = inv(Y)
        f, _ = act(Z)
        branch = S * f * Y * iy * W
        out = X + branch
        bound = c1 * branch.abs() + (S * Y * iy * W).abs() * flushed(Z) + U * out.abs()
        r["out"] = (out, bound + stored(out, dt))
    if W2 is not None:
        io = inv(out)
        nxt = out * io * W2
        # an error of out reaches next directly and through the row's inverse root
        rel = (bound * out.abs()).mean(1, keepdim=True) * io * io
        e = io * W2.abs() * bound + nxt.abs() * (rel + c1)
        r["next"] = (nxt, e + stored(nxt, dt))
    if d_out is None and d_next is None:
        return r
    if checkpoint:
        if Y is None:
            X = through8(x)[0].double()
            out = X
        else:
            Y = through8(y)[0].double()
            Z = None if gate is None else through8(gate)[0].double()
    zero = torch.zeros_like(X)
    GO, GN = (zero if t is None else f64(t) for t in (d_out, d_next))
    f, slope = act(Z)
    if Y is not None:
        unit = Y * iy
        branch = S * f * unit * W
        out = X + branch
        bound = c1 * branch.abs() + (S * unit * W).abs() * flushed(Z) + U * out.abs()
    e_d = torch.zeros_like(X)
    d = GO
    if W2 is not None:
        u2 = out * io
        e_u2 = io * bound + c1 * u2.abs()
        t = GN * W2
        dot = (t * u2).mean(1, keepdim=True)
        e_dot = (t.abs() * e_u2).mean(1, keepdim=True) + c1 * (t * u2).abs().mean(1, keepdim=True)
        d = GO + io * (t - u2 * dot)
        e_d = io * (e_u2 * dot.abs() + u2.abs() * e_dot) + c2 * (io * (t.abs() + (u2 * dot).abs()) + GO.abs())
        terms = GN * u2
        r["d_next_weight"] = _column(terms, GN.abs() * e_u2, rows)
    r["d_x"] = (d, e_d + stored(d, dt))
    if Y is None:
        return r
    normed = unit * W
    dg = d * S * normed * slope
    # the slope is p + z p (1 - p): 1 - p is off by u, not by u of itself
    e_slope = (4 * U * (1 + (Z.abs() if Z is not None else 0.0))) if gate is not None and activation != "none" else 0.0
    e_slope = e_slope + flushed(Z)
    e_dg = (S * normed).abs() * (slope.abs() * e_d + d.abs() * e_slope) + c1 * dg.abs()
    r["d_gate"] = (dg, e_dg + stored(dg, dt))
    r["d_scale"] = _column(d * f * normed, (f * normed).abs() * e_d + c1 * (d * f * normed).abs() +
                           (d * normed).abs() * flushed(Z), rows)
    top = d * S * f
    e_top = (S * f).abs() * e_d + c1 * top.abs() + (d * S).abs() * flushed(Z)
    r["d_weight"] = _column(top * unit, unit.abs() * e_top + c1 * (top * unit).abs(), rows)
    t, e_t = top * W, e_top * W.abs()
    dot = (t * unit).mean(1, keepdim=True)
    e_dot = (e_t * unit.abs()).mean(1, keepdim=True) + c1 * (t * unit).abs().mean(1, keepdim=True)
    dy = iy * (t - unit * dot)
    e_dy = iy * (e_t + unit.abs() * e_dot) + c2 * iy * (t.abs() + (unit * dot).abs())
    r["d_y"] = (dy, e_dy + stored(dy, dt))
    return r


def _column(terms, e, rows):
    ref = terms.sum(0)
    return ref, e.sum(0) + (rows + 32) * U * terms.abs().sum(0) + stored(ref, torch.float32)
