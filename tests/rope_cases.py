"""The norms and the rotation of queries and keys in 64 bits (angles in the host's extended
precision), with what each output may be off by.

Bounds, in units u = 2^-24 of an f32 operation. A head's sum of squares adds positive terms over
chains of at most 16 additions: 17 u relative, half of it in the root; with the mean, eps, the root
itself (4 u), x r and the weight (3 u) y is off by at most 20 u. The angle's fractional turn is
rounded to f32 (half a turn at most: 2 pi 2^-25 rad, 3.2 u), sine and cosine of it by at most 4 u, and
up to positions of 2^31 the 64-bit product is off by 8 u more; each product and the sum by 1 u. So a
rotated output is within (20 + 16 + 2) u (|a| + |b|) of its pair, held to 48 u; then it is rounded
once, by at most half a step of its type.

The gradient of x is r (g - h mean(g h)) with h = x r and g a rotated, weighted gradient: each g is
off by at most 24 u of its pair's (|z1| + |z2|) |w|, h by 20 u, the mean's chain adds 17 u: held to 96 u
of r (G + |h| mean(G |h|)), G = (|z1| + |z2|) |w|. A weight's gradient sums terms off by 48 u over a
chain of at most 96 + heads ceil(tokens / 1024) additions (the kernels' workgroups are 1024 at least
where there are as many tokens, each adding its own tokens' heads)."""
import numpy as np
import torch

U = 2.0 ** -24


def half_step(dtype, x):
    """What rounding once to ``dtype`` is off by: half a step of the value, or of the smallest normal."""
    i = torch.finfo(dtype)
    return x.abs() * (i.eps / 2) + i.tiny * i.eps / 2


def turns(freq, positions, n, d, interleaved):
    """cos and sin [tokens, 1, D] with 1 and 0 behind the rotated elements, each element's partner and
    the sign of the sine in it."""
    p = np.asarray(positions, dtype=np.longdouble)[:, None] * freq.double().numpy().astype(np.longdouble)
    c = torch.ones(len(positions), 1, d, dtype=torch.float64)
    s = torch.zeros(len(positions), 1, d, dtype=torch.float64)
    partner, j = torch.arange(d), torch.arange(n)
    a, b = (2 * j, 2 * j + 1) if interleaved else (j, j + n)
    cos, sin = (torch.from_numpy(f(p).astype(np.float64)) for f in (np.cos, np.sin))
    c[:, 0, a], c[:, 0, b], s[:, 0, a], s[:, 0, b] = cos, cos, -sin, sin
    partner[a], partner[b] = b, a
    return c, s, partner


def _weight(w, d, unit):
    return torch.ones(d, dtype=torch.float64) if w is None else w.double() + (1.0 if unit else 0.0)


def forward(x, w, unit, eps, turn):
    """x [tokens, heads, D]: the output and its bound before rounding."""
    c, s, partner = turn
    x = x.double()
    y = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * _weight(w, x.shape[-1], unit)
    rotated = (partner != torch.arange(x.shape[-1])).double()
    return y * c + y[..., partner] * s, 48 * U * (y.abs() + y[..., partner].abs() * rotated)


def backward(x, w, unit, eps, turn, z):
    """(dx, its bound, dw, its bound) before rounding."""
    c, s, partner = turn
    x, z, wt = x.double(), z.double(), _weight(w, x.shape[-1], unit)
    rotated = (partner != torch.arange(x.shape[-1])).double()
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    h = x * r
    u = z * c - z[..., partner] * s
    big = z.abs() + z[..., partner].abs() * rotated
    g, gbig = u * wt, big * wt.abs()
    dx = r * (g - h * (g * h).mean(-1, keepdim=True))
    dxb = 96 * U * r * (gbig + h.abs() * (gbig * h.abs()).mean(-1, keepdim=True))
    chain = 96 + x.shape[1] * -(-x.shape[0] // 1024)
    return dx, dxb, (u * h).sum((0, 1)), (48 + chain) * U * (big * h.abs()).sum((0, 1))


def held(name, got, want, bound):
    """``got`` within ``bound`` and one rounding of ``want``."""
    got = got.detach().cpu()
    off = (got.double() - want).abs()
    most = bound + half_step(got.dtype, want.abs() + bound)
    worst = float((off / most.clamp(min=1e-300)).max()) if off.numel() else 0.0
    print(f"{name}: {worst:.3f} of the bound", flush=True)
    assert not torch.isnan(off).any(), name
    assert worst <= 1.0, (name, worst)
