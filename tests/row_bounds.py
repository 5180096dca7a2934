"""Plain 64-bit LayerNorm / embedding and error bounds for the kernels' float32 arithmetic, used by the row operators' tests.

u = 2^-24 is the largest relative error of one float32 operation. A sum whose additions are at most K deep is off by at most
K u times the sum of the magnitudes. The kernels add at most 48 + D / 256 deep along a row (a thread's own values, then a
tree over the threads), and over R rows never deeper than R, nor deeper than 48 + R / 64 + 1300 (a thread's rows, the
warps, then the parts one after another). Rounding a result to type t adds half a step: finfo(t).eps / 2 relative, or half
of the smallest subnormal number.
"""
import torch

U = 2.0 ** -24


def half_step(y, kind):
    f = torch.finfo(kind)
    return torch.clamp(y.abs() * (f.eps / 2), min=f.tiny * f.eps / 2)


def layernorm64(x, w, b, eps):
    """Result, mean, rstd of the rows of a matrix, and the largest errors allowed for each (before the final rounding)."""
    x = x.double()
    d = x.shape[1]
    k = 48 + d / 256
    m = x.mean(1, keepdim=True)
    var = ((x - m) ** 2).mean(1, keepdim=True)
    r = 1 / torch.sqrt(var + eps)
    h = (x - m) * r
    w = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if b is None else b.double()
    y = h * w + b
    # the mean: the sum and the division
    dm = U * ((k + 2) * x.abs().mean(1, keepdim=True))
    # rstd: half of the variance's relative error (sum, squares, differences, product, epsilon) and that of a wrong mean, then a
    # square root and a division; epsilon itself is rounded to float32
    dr = r * (U * ((k + 7) / 2 + 3) + 0.5 * (dm * r) ** 2)
    dy = U * (h * w).abs() * 4 + (h * w).abs() * dr / r + dm * r * w.abs() + U * y.abs()
    return (y, m[:, 0], r[:, 0]), (dy, dm[:, 0] + U * m[:, 0].abs(), dr[:, 0])


def layernorm_backward64(g, x, m, r, w):
    """dx, dw, db from float32 statistics taken as they are, and the largest errors allowed (before the final rounding)."""
    g, x, m, r = g.double(), x.double(), m.double().reshape(-1, 1), r.double().reshape(-1, 1)
    rows, d = x.shape
    k = 48 + d / 256
    kr = min(rows, 48 + rows / 64 + 1300)
    h = (x - m) * r
    gw = g if w is None else g * w.double()
    c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    dx = r * (gw - c1 - h * c2)
    dc1 = U * (k + 4) * gw.abs().mean(1, keepdim=True)
    dc2 = U * (k + 8) * (gw * h).abs().mean(1, keepdim=True)
    ex = r * (U * (6 * gw.abs() + 6 * c1.abs() + 8 * (h * c2).abs()) + dc1 + h.abs() * dc2)
    dw, db = (g * h).sum(0), g.sum(0)
    ew = U * (kr + 4) * (g * h).abs().sum(0)
    eb = U * (kr + 2) * g.abs().sum(0)
    return (dx, dw, db), (ex, ew, eb)


def check(got, want, bound, what=""):
    """|got - want| <= bound + half a step of got's type (of the values the bound allows), everywhere."""
    kind = got.dtype
    err = (got.double() - want).abs()
    limit = bound + half_step(want.abs() + bound, kind)
    bad = ~(err <= limit)
    if bool(bad.any()):
        i = int((err / limit).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst at {i}: got {got.flatten()[i].item()}, "
                             f"want {want.flatten()[i].item()}, allowed {limit.flatten()[i].item()}")
