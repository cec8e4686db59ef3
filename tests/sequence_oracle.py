"""The sequence operators in 64 bits, from their formulas, token by token and
differentiated by autograd, and the magnitudes that bound a kernel's error.

``magnitude=True`` computes the same sums over the absolute values of their
terms: a result that a kernel forms in f32 along paths of relative error at most
k differs from the exact one by at most k times that magnitude.
"""
import torch

F64 = torch.float64


def lengths_to_ptr(lens, lead=0):
    ptr = [lead]
    for n in lens:
        ptr.append(ptr[-1] + n)
    return ptr


class _Fixed(torch.autograd.Function):
    """``value`` whose derivative by ``leaf`` is ``slope``."""

    @staticmethod
    def forward(ctx, leaf, value, slope):
        ctx.save_for_backward(slope)
        return value.clone()

    @staticmethod
    def backward(ctx, g):
        (slope,) = ctx.saved_tensors
        return g * slope, None, None


def scan(x, dt, a, b, c, d, z, dt_bias, softplus, lens, start, magnitude=False):
    """(y [tokens, channels], final [seqs, channels, states]); every argument f64,
    b and c [tokens, groups, states], start [seqs, channels, states] or None."""
    ch, ns = a.shape
    per = ch // b.shape[1]
    u = dt if dt_bias is None else dt + dt_bias
    s = torch.nn.functional.softplus(u, threshold=60) if softplus else u
    if magnitude:
        x, b, c = x.abs(), b.abs(), c.abs()
        d = None if d is None else d.abs()
        start = None if start is None else start.abs()
        s = s if softplus else _Fixed.apply(s, s.abs().detach(), torch.ones_like(s))
    ys, finals, at = [], [], 0
    for i, n in enumerate(lens):
        h = torch.zeros(ch, ns, dtype=F64) if start is None else start[i]
        for t in range(at, at + n):
            arg = s[t][:, None] * a
            if magnitude:  # the derivative by s and a in absolute value
                mag = s[t][:, None] * a.abs()
                e = _Fixed.apply(mag, torch.exp(arg).detach(), torch.exp(arg).detach())
            else:
                e = torch.exp(arg)
            h = e * h + (s[t] * x[t])[:, None] * b[t].repeat_interleave(per, 0)
            o = (h * c[t].repeat_interleave(per, 0)).sum(1)
            ys.append(o if d is None else o + d * x[t])
        finals.append(h)
        at += n
    y = torch.stack(ys) if ys else torch.zeros(0, ch, dtype=F64) + 0 * x[:0]
    if z is not None and len(ys):
        sig = torch.sigmoid(z[:at])
        gate = z[:at] * sig
        if magnitude:
            gate = _Fixed.apply(z[:at], gate.abs().detach(), (sig * (1 + z[:at].abs())).detach())
        y = y * gate
    return y, (torch.stack(finals) if finals else torch.zeros(0, ch, ns, dtype=F64))


def scan_bound(dt, a, dt_bias, softplus, lens, tokens, channels, backward=False):
    """The relative error of a path through the scan in f32: at most the longest
    sequence's exponentials (each 2^-22 of its own, and its argument's roundings
    and the step's error, together below 2^-21 of the argument), once forwards
    and for gradients once backwards, and the roundings of the sums it enters."""
    u = dt if dt_bias is None else dt + dt_bias
    s = torch.nn.functional.softplus(u, threshold=60) if softplus else u.abs()
    most = float((s.max(0).values[:, None] * a.abs()).max()) if s.numel() else 0.0
    steps = max(lens, default=0) * (2 if backward else 1)
    return steps * (2.0 ** -22 + most * 2.0 ** -21) + (64 + (tokens + channels if backward else 0)) * 2.0 ** -24


def conv(x, w, bias, silu, lens, start, magnitude=False):
    """(y, final [seqs, width - 1, channels])."""
    ch, width = w.shape
    if magnitude:
        x, w = x.abs(), w.abs()
        bias = None if bias is None else bias.abs()
        start = None if start is None else start.abs()
    ys, finals, at = [], [], 0
    for i, n in enumerate(lens):
        begin = torch.zeros(width - 1, ch, dtype=F64) if start is None else start[i]
        line = torch.cat([begin, x[at:at + n]])
        u = sum(line[k:k + n] * w[:, k] for k in range(width))
        ys.append(u if bias is None else u + bias)
        finals.append(line[n:])
        at += n
    u = torch.cat(ys) if ys else x[:0]
    if silu:
        if magnitude:  # |u sigmoid(u)| <= |u|; slope below 1.1, and its change below 0.5 per change of u
            y = _Fixed.apply(u, 1.1 * u.detach(), 1.1 + 0.5 * u.detach())
        else:
            y = u * torch.sigmoid(u)
    else:
        y = u
    return y, (torch.stack(finals) if finals else torch.zeros(0, width - 1, ch, dtype=F64))


def norm(x, w, bias, eps):
    mean = x.mean(1)
    off = x - mean[:, None]
    rstd = (off.square().mean(1) + eps) ** -0.5
    y = off * rstd[:, None]
    y = y if w is None else y * w
    return (y if bias is None else y + bias), mean, rstd


def half_step(dtype):
    """The relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


def check(got, want, magnitude, k, what=""):
    """|got - want| <= k * magnitude + half a step of got's type (a subnormal's step at least)."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    g = got.detach().cpu().to(F64)
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    room = k * magnitude.abs() + half_step(got.dtype) * (want.abs() + k * magnitude.abs()) + tiny
    bad = ~((g - want).abs() <= room)
    if bad.any():
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: got {g.reshape(-1)[i]:.9g} want "
                             f"{want.reshape(-1)[i]:.9g} room {room.reshape(-1)[i]:.3g}")
