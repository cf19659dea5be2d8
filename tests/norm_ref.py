"""Normed rotation and its gradients in 64 bits from the definitions, for tests, with bounds.

u = 2^-24, e = finfo.eps / 2 half a step of the type.  A row's sum of D squares is off by D u of itself, its root by half of
that and two steps: r, and with it n = x r w, by (D / 2 + 8) u.  The rotation adds 8 u (tests of rotary) of |n_a| + |n_b|
and its three products and sums.  Together (D / 2 + 24) u of the pair's sum, and e of the result.
The gradient g = R^T dy is off by 8 u of |dy_a| + |dy_b| = G, the mean of D products by D u more: dx by (2 D + 64) u of
r (G |w| + |n| mean(G |w n|)), a weight's gradient, a sum over N rows, by (N + D + 64) u of sum G |x r|."""
import torch

U = 2.0 ** -24


def _turn(x, positions, inv_freq, sections, pos_scale, rope_scale, inverse):
    """(rotated, pair sums) of x (T, H, D)."""
    half = len(inv_freq)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)])
    scale = float(torch.tensor(pos_scale, dtype=torch.float32))
    angle = positions.double()[axis].t() * scale * inv_freq.double()                 # (T, half)
    rope = float(torch.tensor(rope_scale, dtype=torch.float32))
    c, s = torch.cos(angle)[:, None] * rope, torch.sin(angle)[:, None] * rope * (-1 if inverse else 1)
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    out = torch.cat([a * c - b * s, b * c + a * s, rest], dim=-1)
    size = (a.abs() + b.abs()) * abs(rope)
    return out, torch.cat([size, size, rest.abs()], dim=-1)


def forward(x, weight, positions, inv_freq, sections, eps, pos_scale=1.0, rope_scale=1.0):
    """(y, bound) of x (T, H, D) on the host."""
    e, D = torch.finfo(x.dtype).eps / 2, x.shape[-1]
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    x = x.double().cpu()
    w = 1.0 if weight is None else weight.double().cpu()
    n = x / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32))) * w
    y, size = _turn(n, positions.cpu(), inv_freq.cpu(), sections, pos_scale, rope_scale, False)
    return y, (D / 2 + 24) * U * size + e * y.abs() * 1.01 + tiny


def gradients(dy, x, weight, positions, inv_freq, sections, eps, pos_scale=1.0, rope_scale=1.0):
    """((dx, bound), (dweight, bound)) on the host."""
    e, D = torch.finfo(x.dtype).eps / 2, x.shape[-1]
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    x, dy = x.double().cpu(), dy.double().cpu()
    w = torch.ones(D, dtype=torch.float64) if weight is None else weight.double().cpu()
    r = 1 / torch.sqrt(x.square().mean(dim=-1, keepdim=True) + float(torch.tensor(eps, dtype=torch.float32)))
    n = x * r
    g, size = _turn(dy, positions.cpu(), inv_freq.cpu(), sections, pos_scale, rope_scale, True)
    dx = r * (g * w - n * (g * w * n).mean(dim=-1, keepdim=True))
    reach = r * (size * w.abs() + n.abs() * (size * (w * n).abs()).mean(dim=-1, keepdim=True))
    dw = (g * n).sum(dim=(0, 1))
    rows = x.shape[0] * x.shape[1]
    ew = e if weight is None else torch.finfo(weight.dtype).eps / 2
    return ((dx, (2 * D + 64) * U * reach + e * dx.abs() * 1.01 + tiny),
            (dw, (rows + D + 64) * U * (size * n.abs()).sum(dim=(0, 1)) + ew * dw.abs() * 1.01 + tiny))
