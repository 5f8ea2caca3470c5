"""The 8-bit activation checkpoint format and its operators in float64, element by element from
their definitions (csrc/act8.h states them): what tests/test_act8_host.py and
tests/test_gpu_act8.py compare with."""
import torch

U = 2.0 ** -24                              # half a step of f32
STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def two_to(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def pack(x):
    """-> (q int8 [rows, P], scale uint8 [rows, P / 32])."""
    rows, C = x.shape
    P = -(-C // 32) * 32
    v = torch.zeros(rows, P, dtype=torch.float64, device=x.device)
    v[:, :C] = x.double()
    v = v.view(rows, P // 32, 32)
    bad = ~(v.abs() <= 127 * 2.0 ** 121).all(-1)
    a = torch.where(bad, torch.zeros((), dtype=torch.float64, device=x.device), v.abs().amax(-1))
    e = torch.full(a.shape, -126, dtype=torch.int64, device=x.device)
    for step in (128, 64, 32, 16, 8, 4, 2, 1):           # the smallest e with a <= 127 * 2^e
        e = torch.where(a > 127 * two_to(e + step - 1), e + step, e)
    q = torch.round(v / two_to(e).unsqueeze(-1))
    q = torch.where(bad.unsqueeze(-1), torch.zeros_like(q), q)
    scale = torch.where(bad, torch.full_like(e, 255), e + 127)
    return q.to(torch.int8).view(rows, P), scale.to(torch.uint8)


def values(q, scale, C):
    rows = q.shape[0]
    s = torch.where(scale == 255, torch.full(scale.shape, float("nan"), dtype=torch.float64, device=q.device),
                    two_to(scale.long() - 127))
    return (q.double().view(rows, -1, 32) * s.unsqueeze(-1)).view(rows, -1)[:, :C]


def stand_for(x):
    return values(*pack(x), x.shape[1])


def tail(a):
    return 0.5 * torch.special.erfc(a / 2.0 ** 0.5)


def phi(a):
    return torch.exp(-a * a / 2) / (2 * torch.pi) ** 0.5


def gelu(x, gy):
    """-> y, gx and how far the kernels may be off.  The kernels take the normal tail as Q(a) =
    M(a) phi(a): M within 3.4e-7 (f32) / 9e-6 (bf16) plus a dozen roundings, phi with the
    hardware's 2^x (2 steps) of an argument that two roundings put a^2 2^-24 off; then the
    result's own rounding."""
    fit = 3.4e-7 if x.dtype == torch.float32 else 9e-6
    v, h, g = x.double(), stand_for(x), gy.double()
    y = torch.where(v < 0, v * tail(-v), v * (1 - tail(v)))
    a = v.abs()
    tol_y = a * tail(a) * (fit + 20 * U + a * a * U) + 2 * U * a + STEP[x.dtype] * y.abs()
    slope = torch.where(h < 0, tail(-h), 1 - tail(h)) + h * phi(h)
    a = h.abs()
    tol_s = (tail(a) * fit + (a * phi(a) + tail(a)) * (20 * U + a * a * U)) + 2 * U
    return y, g * slope, tol_y, g.abs() * tol_s + (STEP[x.dtype] + U) * (g * slope).abs()


def layer_norm(x, w, b, gy, eps, gs=None):
    """-> y, gx, gw, gb and how far each may be off: a row's sums are trees and chains of at most
    64 additions of f32, so a mean is off by at most 64 U of the mean magnitude and the rest
    follows; sums over rows are chains of at most (rows / workgroups + 64) additions, counted as
    128 for the sizes tested; then the result's own rounding."""
    n, step = 64 * U, STEP[x.dtype]
    v, w64, b64, g = x.double(), w.double(), b.double(), gy.double()
    mu = v.mean(1, keepdim=True)
    var = ((v - mu) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    xh = (v - mu) * rs
    d_mu = n * v.abs().mean(1, keepdim=True) + U * v.abs().amax(1, keepdim=True)
    d_rs = 2 * n + rs * rs * d_mu ** 2                       # relative
    y = xh * w64 + b64
    tol_y = w64.abs() * (rs * (d_mu + 2 * U * v.abs()) + xh.abs() * (d_rs + 4 * U)) + 2 * U * b64.abs() + step * y.abs()
    h = stand_for(x)
    xh = (h - mu) * rs
    d_xh = rs * (d_mu + 2 * U * h.abs()) + xh.abs() * (d_rs + 4 * U)
    gn = g * w64
    c1, c2 = gn.mean(1, keepdim=True), (gn * xh).mean(1, keepdim=True)
    gx = rs * (gn - c1 - xh * c2)
    d_c1 = n * gn.abs().mean(1, keepdim=True)
    d_c2 = n * (gn * xh).abs().mean(1, keepdim=True) + (gn.abs() * d_xh).mean(1, keepdim=True)
    tol_gx = rs * (4 * U * gn.abs() + d_c1 + xh.abs() * d_c2 + d_xh * c2.abs() + 4 * U * (xh * c2).abs())
    tol_gx = tol_gx + (d_rs + 4 * U) * gx.abs()
    if gs is not None:
        gx = gx + gs.double()
    gw, gb = (g * xh).sum(0), g.sum(0)
    tol_gw = (g.abs() * d_xh).sum(0) + 128 * U * (g * xh).abs().sum(0) + step * gw.abs()
    tol_gb = 128 * U * g.abs().sum(0) + step * gb.abs()
    return (y, gx, gw, gb), (tol_y, tol_gx + (step + U) * gx.abs(), tol_gw, tol_gb)


def wgrad(gy, q, scale, C, out_dtype):
    """-> dw, db and how far they may be off: exact products, every one added once in f32 (the
    matrix units may cut where they add: a whole step), then the result's own rounding."""
    g, h = gy.double(), values(q, scale, C)
    T = g.shape[0]
    dw, db = g.t().contiguous() @ h, g.sum(0)
    mag = g.abs().t().contiguous() @ h.abs()
    n = 2 * U * (T + 64)
    return dw, db, n * mag + STEP[out_dtype] * dw.abs(), n * g.abs().sum(0) + STEP[out_dtype] * db.abs()


def within(got, want, tol, what=""):
    """got is as far from want as tol allows, and not a number exactly where want is not."""
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    nan = torch.isnan(want)
    assert bool((torch.isnan(got) == nan).all()), f"{what}: NaNs in other places"
    tol = tol.expand_as(want)
    bad = ~nan & ~((got - want).abs() <= tol) & (got != want)
    if bool(bad.any()):
        i = int(torch.nonzero(bad.reshape(-1))[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; at {i} got {got.reshape(-1)[i].item()}, "
                             f"want {want.reshape(-1)[i].item()} +- {tol.reshape(-1)[i].item()}")
