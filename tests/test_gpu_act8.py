"""GPU tests of the 8-bit activation checkpoints (csrc/act8.hip, act8_norm.hip, act8_wgrad.hip)
against their definitions in float64 (tests/_act8ref.py, which also derives the tolerances)."""
import pytest
import torch
import torch.nn.functional as F

import _act8ref as ref

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _ops():
    from visionseg import ops
    return ops


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _act(rows, C, dtype, seed, zeros=True):
    g = _gen(seed)
    size = torch.exp(torch.randn(C, generator=g, device=DEV))
    x = torch.randn(rows, C, generator=g, device=DEV) * size + 0.5 * size
    if zeros and rows > 2:
        x[rows // 2] = 0
    return x.to(dtype)


def _grad(rows, C, dtype, seed):
    return (1e-2 * torch.randn(rows, C, generator=_gen(seed), device=DEV)).to(dtype)


def _on_grid(rows, C, dtype, seed):
    """Values that their own checkpoint holds exactly."""
    return ref.stand_for(_act(rows, C, dtype, seed)).to(dtype)


SIZES = [(1, 1), (1, 32), (3, 7), (2, 31), (5, 33), (64, 64), (100, 96), (33, 100), (257, 200), (4, 1003), (1000, 256),
         (3, 8192)]


# ------------------------------------------------------------------------------- pack / unpack
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", SIZES + [(3, 20011)])
def test_pack_is_exact(rows, C, dtype):
    ops = _ops()
    x = _act(rows, C, dtype, rows + C)
    q, s = ops.act8_pack(x)
    rq, rs = ref.pack(x)
    assert q.dtype == torch.int8 and s.dtype == torch.uint8
    assert torch.equal(q, rq) and torch.equal(s, rs)
    for out in (F32, BF16):
        assert torch.equal(ops.act8_unpack(q, s, C, out).double(), ref.values(rq, rs, C))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack_special_values(dtype):
    ops = _ops()
    x = _act(16, 70, F32, 5)
    top = 127 * 2.0 ** 121
    x[0] = 0
    x[1] = 127 * 2.0 ** -3                                  # exactly 127 steps
    x[2] = torch.nextafter(torch.tensor(127 * 2.0 ** -3), torch.tensor(1e9)).item()
    x[3] *= 1e-42                                           # denormals
    x[4] = top
    x[5, 3] = float("inf")
    x[6, 40] = float("nan")
    x[7, 69] = -float("inf")
    x[8] = torch.nextafter(torch.tensor(top), torch.tensor(float("inf"))).item()
    x[9] = -torch.finfo(F32).max
    x[10] = torch.arange(70, device=DEV) + 0.5              # ties
    x[11] = -x[10]
    x[12, :32] = 1e-45
    x = x.to(dtype)
    q, s = ops.act8_pack(x)
    rq, rs = ref.pack(x)
    assert torch.equal(q, rq) and torch.equal(s, rs)
    v = ops.act8_unpack(q, s, 70, dtype)
    want = ref.values(rq, rs, 70)
    assert torch.equal(torch.isnan(v), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(v.double()), torch.nan_to_num(want))
    # a NaN whose payload fills the low bits
    n = torch.full((1, 40), 0x7F800001, dtype=torch.int32, device=DEV).view(F32)
    q, s = ops.act8_pack(n)
    assert not bool(q.any()) and bool((s == 255).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_pack_strides_and_shapes(dtype):
    ops = _ops()
    wide = _act(50, 3 * 45 + 1, dtype, 9)
    for x in (wide[:, 45:90], wide[:, 1:46], wide[::2, 3:35], wide[:1, :33].expand(7, 33), wide.t(), wide[3:3],
              wide[:, :0]):
        q, s = ops.act8_pack(x)
        rq, rs = ref.pack(x.contiguous())
        assert torch.equal(q, rq) and torch.equal(s, rs)
    x = _act(2 * 3 * 5, 40, dtype, 10).view(2, 3, 5, 40)
    q, s = ops.act8_pack(x)
    assert q.shape == (2, 3, 5, 64) and s.shape == (2, 3, 5, 2)
    v = ops.act8_unpack(q, s, 40, dtype)
    assert torch.equal(v.view(30, 40).double(), ref.stand_for(x.view(30, 40)))
    q, s = ops.act8_pack(x[0, 0, 0])                        # one dimension
    assert torch.equal(q, ops.act8_pack(x)[0][0, 0, 0])
    # a permuted checkpoint is read as the rows it is
    q, s = ops.act8_pack(x)
    v2 = ops.act8_unpack(q.transpose(0, 2), s.transpose(0, 2), 40, dtype)
    assert torch.equal(v2, v.transpose(0, 2))


def test_pack_neighbours_stay():
    """q and scale of a view's rows are written, nothing around them."""
    from visionseg import _lib as L
    x = _act(5, 40, F32, 3)
    q = torch.full((7, 64), 99, dtype=torch.int8, device=DEV)
    s = torch.full((7, 2), 99, dtype=torch.uint8, device=DEV)
    L.check(L.lib().vs_act8_pack(0, L.ptr(x), 40, L.ptr(q[1:]), L.ptr(s[1:]), 5, 40, L.stream(x)), "pack")
    rq, rs = ref.pack(x)
    assert torch.equal(q[1:6], rq) and torch.equal(s[1:6], rs)
    assert bool((q[[0, 6]] == 99).all()) and bool((s[[0, 6]] == 99).all())
    y = torch.full((7, 40), 99.0, device=DEV)
    L.check(L.lib().vs_act8_unpack(0, L.ptr(q[1:]), L.ptr(s[1:]), L.ptr(y[1:]), 5, 40, L.stream(x)), "unpack")
    assert torch.equal(y[1:6].double(), ref.values(rq, rs, 40)) and bool((y[[0, 6]] == 99).all())


# ------------------------------------------------------------------------------- GELU
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", SIZES)
def test_gelu(rows, C, dtype):
    ops = _ops()
    x, gy = _act(rows, C, dtype, rows * C), _grad(rows, C, dtype, 1)
    x = x.requires_grad_()
    y = ops.gelu_act8(x)
    (gx,) = torch.autograd.grad(y, x, gy)
    ry, rgx, ty, tgx = ref.gelu(x.detach(), gy)
    ref.within(y.detach(), ry, ty, "y")
    ref.within(gx, rgx, tgx, "gx")
    with torch.no_grad():
        assert torch.equal(ops.gelu_act8(x), y)
    # the activation again, in the backward's pass
    from visionseg import _lib as L
    q, s = ops.act8_pack(x.detach())
    g2, y2 = L.tops().act8_gelu_bwd(gy, q, s, True)
    assert torch.equal(g2, gx)
    h = ref.stand_for(x.detach()).to(dtype)
    hy, _, th, _ = ref.gelu(h, gy)
    ref.within(y2, hy, th, "recomputed y")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gelu_over_the_range(dtype):
    """Every magnitude from 2^-30 to beyond the density's last number, both signs, and the ends."""
    ops = _ops()
    a = torch.cat([torch.logspace(-9, 1.3, 6000, device=DEV), torch.linspace(0, 45, 6000, device=DEV)])
    x = torch.cat([a, -a]).view(-1, 1).to(dtype)             # a block of one feature: 7 bits and more
    gy = torch.ones_like(x)
    xg = x.clone().requires_grad_()
    y = ops.gelu_act8(xg)
    (gx,) = torch.autograd.grad(y, xg, gy)
    ry, rgx, ty, tgx = ref.gelu(x, gy)
    ref.within(y.detach(), ry, ty, "y")
    ref.within(gx, rgx, tgx, "gx")
    ends = torch.tensor([[float("inf")], [-float("inf")], [float("nan")], [0.0], [-0.0], [3e38], [-3e38]], device=DEV,
                        dtype=dtype).requires_grad_()
    y = ops.gelu_act8(ends)
    (gx,) = torch.autograd.grad(y, ends, torch.ones_like(ends))
    y = y.detach().flatten().tolist()
    assert y[0] == float("inf") and y[1] == 0 and y[2] != y[2] and y[3] == 0 and y[4] == 0 and y[5] > 2.9e38
    assert y[6] == 0
    gx = gx.flatten().tolist()
    # at 0 the slope is 1 - M(0) phi(0): _act8ref.gelu's bound at a = 0, and the rounding
    near = 0.5 * ((3.4e-7 if dtype == F32 else 9e-6) + 20 * ref.U) + 2 * ref.U + ref.STEP[dtype] * 0.5
    assert all(v != v for v in gx[:3]) and abs(gx[3] - 0.5) <= near and abs(gx[4] - 0.5) <= near
    assert gx[5] == 1 and gx[6] == 0


def test_gelu_gradient_against_differences():
    ops = _ops()
    x = _on_grid(40, 70, F32, 8)
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ops.gelu_act8(xg).sum(), xg)
    d = 1e-6                                                 # f64: error ~ d^2 / 6 |gelu'''| + 1e-16 / d
    v = x.double()
    diff = (F.gelu(v + d) - F.gelu(v - d)) / (2 * d)
    assert float((gx.double() - diff).abs().max()) < 2e-6


# ------------------------------------------------------------------------------- LayerNorm
NORM = [(1, 1), (1, 32), (3, 7), (5, 33), (100, 96), (257, 192), (33, 100), (64, 64), (77, 128), (500, 384), (9, 1003),
        (12, 768), (7, 1536), (6, 2048), (5, 2056), (3, 4099), (2, 8192), (4099, 24)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,C", NORM)
def test_layer_norm(rows, C, dtype, residual):
    ops = _ops()
    x, gy = _act(rows, C, dtype, rows * C + 1), _grad(rows, C, dtype, 2)
    g = _gen(3)
    w = (1 + 0.3 * torch.randn(C, generator=g, device=DEV)).to(dtype).requires_grad_()
    b = (0.3 * torch.randn(C, generator=g, device=DEV)).to(dtype).requires_grad_()
    xg = x.clone().requires_grad_()
    gs = None
    if residual:
        r = _act(rows, C, dtype, 4).requires_grad_()
        gs = _grad(rows, C, dtype, 5)
        s, y = ops.add_layer_norm_act8(xg, r, w, b)
        want_s = (x.float() + r.detach().float()).to(dtype)
        assert torch.equal(s.detach(), want_s)
        gx, gr, gw, gb = torch.autograd.grad((s, y), (xg, r, w, b), (gs, gy))
        assert torch.equal(gx, gr)
        base = want_s
    else:
        y = ops.layer_norm_act8(xg, w, b)
        gx, gw, gb = torch.autograd.grad(y, (xg, w, b), gy)
        base = x
    want, tol = ref.layer_norm(base, w.detach(), b.detach(), gy, 1e-5, gs)
    for name, got, a, t in zip(("y", "gx", "gw", "gb"), (y.detach(), gx, gw, gb), want, tol):
        ref.within(got, a, t, name)
    again = torch.autograd.grad(ops.layer_norm_act8(xg, w, b), (w, b), gy) if not residual else None
    assert again is None or (torch.equal(again[0], gw) and torch.equal(again[1], gb))       # deterministic


def test_layer_norm_gradient_against_differences():
    ops = _ops()
    x = _on_grid(6, 70, F32, 11)
    w = torch.linspace(0.5, 1.5, 70, device=DEV)
    b = torch.linspace(-1, 1, 70, device=DEV)
    gy = _grad(6, 70, F32, 12) * 100
    xg = x.clone().requires_grad_()
    (gx,) = torch.autograd.grad(ops.layer_norm_act8(xg, w, b), xg, gy)
    d = 1e-6

    def loss(v):
        return (F.layer_norm(v, (70,), w.double(), b.double()) * gy.double()).sum(1)

    for c in range(0, 70, 9):
        e = torch.zeros(70, dtype=torch.float64, device=DEV)
        e[c] = d
        diff = (loss(x.double() + e) - loss(x.double() - e)) / (2 * d)
        # the row of zeros has rstd = 316: the third derivative's term is rstd^3 d^2
        assert bool(((gx[:, c].double() - diff).abs() <= 1e-4 * (1 + gx.double().abs().amax(1))).all())


def test_layer_norm_partial_gradients():
    """Any of the four gradients alone, an output that is not used, no gradient at all."""
    ops = _ops()
    x, r = _act(20, 40, F32, 1), _act(20, 40, F32, 2)
    w, b = torch.rand(40, device=DEV) + 0.5, torch.rand(40, device=DEV)
    gy, gs = _grad(20, 40, F32, 3), _grad(20, 40, F32, 4)
    full = [t.clone().requires_grad_() for t in (x, r, w, b)]
    s, y = ops.add_layer_norm_act8(*full)
    want = torch.autograd.grad((s, y), full, (gs, gy))
    for k in range(4):
        ts = [t.clone() for t in (x, r, w, b)]
        ts[k].requires_grad_()
        s1, y1 = ops.add_layer_norm_act8(*ts)
        assert torch.equal(s1, s) and torch.equal(y1, y)
        outs, gos = ((s1, y1), (gs, gy)) if k < 2 else ((y1,), (gy,))
        assert torch.equal(torch.autograd.grad(outs, ts[k], gos)[0], want[k])
    s, y = ops.add_layer_norm_act8(*full)
    gx, gr, gw, gb = torch.autograd.grad(s, full, gs)        # y unused
    assert torch.equal(gx, gs) and torch.equal(gr, gs) and not bool(gw.any()) and not bool(gb.any())
    s, y = ops.add_layer_norm_act8(*full)
    gx = torch.autograd.grad(y, full[0], gy)[0]              # s unused
    want_gx, tol = ref.layer_norm(s.detach(), w, b, gy, 1e-5)
    ref.within(gx, want_gx[1], tol[1], "gx")
    with torch.no_grad():
        s2, y2 = ops.add_layer_norm_act8(*full)
    assert torch.equal(s2, s) and torch.equal(y2, y) and not y2.requires_grad
    # the same tensor as both summands
    t = x.clone().requires_grad_()
    s, y = ops.add_layer_norm_act8(t, t, w, b)
    g2 = torch.autograd.grad((s, y), t, (gs, gy))[0]
    want2, tol2 = ref.layer_norm(2 * x, w, b, gy, 1e-5, gs)
    ref.within(g2, 2 * want2[1], 2 * tol2[1], "gx of both")


def test_layer_norm_non_finite_row():
    """A NaN or an infinity stays in its row (and reaches the sums over rows)."""
    ops = _ops()
    x = _act(9, 64, F32, 21)
    x[2, 5], x[4, 60] = float("inf"), float("nan")
    w, b = torch.ones(64, device=DEV), torch.zeros(64, device=DEV)
    xg = x.clone().requires_grad_()
    y = ops.layer_norm_act8(xg, w, b)
    (gx,) = torch.autograd.grad(y, xg, _grad(9, 64, F32, 22))
    bad = torch.tensor([r in (2, 4) for r in range(9)], device=DEV)
    assert bool(torch.isnan(y[bad]).any(1).all()) and bool(torch.isfinite(y[~bad]).all())
    assert bool(torch.isnan(gx[bad]).all()) and bool(torch.isfinite(gx[~bad]).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_layer_norm_window_rows(dtype):
    """y in the Swin window layout, gradients from there: the plain form's rows, permuted."""
    ops = _ops()
    B, H, W, C, ws, shift = 2, 9, 10, 96, 7, 3
    wr = ops.window_rows(B, H, W, ws, shift, torch.device(DEV, 0))
    x = _act(B * H * W, C, dtype, 31).requires_grad_()
    r = _act(B * H * W, C, dtype, 32).requires_grad_()
    w = torch.rand(C, device=DEV).to(dtype).requires_grad_()
    b = torch.rand(C, device=DEV).to(dtype).requires_grad_()
    s, y = ops.add_layer_norm_act8(x, r, w, b, 1e-5, wrows=wr)
    s0, y0 = ops.add_layer_norm_act8(x, r, w, b, 1e-5)
    assert y.shape == (wr.total, C) and torch.equal(s, s0)
    assert torch.equal(y[wr.rows.long()], y0) and not bool(y[wr.pad].any())
    gw_ = _grad(wr.total, C, dtype, 33)
    gs = _grad(B * H * W, C, dtype, 34)
    a = torch.autograd.grad((s, y), (x, r, w, b), (gs, gw_))
    c = torch.autograd.grad((s0, y0), (x, r, w, b), (gs, gw_[wr.rows.long()]))
    assert all(torch.equal(p, q) for p, q in zip(a, c))


def test_layer_norm_row_map_outside():
    """A row map that points outside: nothing is written, zeros are read."""
    from visionseg import _lib as L
    t = L.tops()
    x = _act(6, 40, F32, 41)
    w, b = torch.ones(40, device=DEV), torch.zeros(40, device=DEV)
    rows = torch.tensor([2, -1, 0, 4, 1 << 30, 3], dtype=torch.int32, device=DEV)
    s, y, q, sc, mean, rstd = t.act8_layer_norm_fwd(x, None, w, b, 1e-5, rows, 5, True)
    y0 = t.act8_layer_norm_fwd(x, None, w, b, 1e-5)[1]
    assert y.shape == (5, 40) and torch.equal(y[[2, 0, 4, 3]], y0[[0, 2, 3, 5]])
    gy = _grad(5, 40, F32, 42)
    gx, gw, gb = t.act8_layer_norm_bwd(gy, None, q, sc, w, mean, rstd, rows)
    full = torch.zeros(6, 40, device=DEV)
    full[[0, 2, 3, 5]] = gy[[2, 0, 4, 3]]
    gx0, gw0, gb0 = t.act8_layer_norm_bwd(full, None, q, sc, w, mean, rstd)
    assert torch.equal(gx, gx0) and torch.equal(gw, gw0) and torch.equal(gb, gb0)


def test_norm_and_gelu_without_rows():
    ops = _ops()
    w, b = (torch.ones(40, device=DEV).requires_grad_() for _ in range(2))
    x = torch.empty(0, 40, device=DEV).requires_grad_()
    y = ops.layer_norm_act8(x, w, b)
    gx, gw, gb = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == gx.shape == (0, 40) and not bool(gw.any()) and not bool(gb.any())
    assert torch.autograd.grad(ops.gelu_act8(x).sum(), x)[0].shape == (0, 40)


# ------------------------------------------------------------------------------- weight gradient
WGRAD = [(1, 1, 1), (1, 32, 32), (3, 7, 5), (63, 64, 128), (64, 128, 128), (65, 129, 127), (400, 256, 256),
         (1000, 96, 288), (777, 100, 33), (513, 33, 513), (5000, 64, 40), (20000, 130, 70), (300, 1003, 299)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,N", WGRAD)
def test_wgrad(T, K, N, dtype):
    ops = _ops()
    x, gy = _act(T, K, dtype, T + K), _grad(T, N, dtype, N)
    q, s = ops.act8_pack(x)
    for out in (F32, BF16):
        dw, db = ops.act8_wgrad(gy, q, s, K, out, bias=True)
        assert dw.dtype == db.dtype == out
        rw, rb, tw, tb = ref.wgrad(gy, q, s, K, out)
        ref.within(dw, rw, tw, "dw")
        ref.within(db, rb, tb, "db")
        assert torch.equal(ops.act8_wgrad(gy, q, s, K, out), dw)       # deterministic, no bias


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wgrad_strides(dtype):
    ops = _ops()
    T, K, N = 300, 70, 45
    q, s = ops.act8_pack(_act(T, K, dtype, 1))
    wide = _grad(T, 3 * N + 2, dtype, 2)
    for gy in (wide[:, N:2 * N], wide[:, 1:1 + N], wide[:, ::3][:, :N], wide[:1, :N].expand(T, N),
               wide[:, :N].reshape(3, 100, N)):
        shape = (*gy.shape[:-1], -1)
        dw, db = ops.act8_wgrad(gy, q.view(shape), s.view(shape), K, F32, bias=True)
        rw, rb, tw, tb = ref.wgrad(gy.reshape(T, N), q, s, K, F32)
        ref.within(dw, rw, tw, "dw")
        ref.within(db, rb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_wgrad_special_values(dtype):
    """NaN and infinities go where the products take them, and nowhere else."""
    ops = _ops()
    T, K, N = 200, 64, 48
    x, gy = _act(T, K, dtype, 3), _grad(T, N, dtype, 4)
    x[7, 40] = float("inf")                                  # the block of columns 32..63
    gy[9, 5], gy[10, 6], gy[11, 7] = float("inf"), float("nan"), -float("inf")
    x[9] = x[11] = 1
    q, s = ops.act8_pack(x)
    dw, db = ops.act8_wgrad(gy, q, s, K, F32, bias=True)
    assert bool(torch.isnan(dw[:, 32:]).all())
    d = dw[:, :32]
    assert bool((d[5] == float("inf")).all()) and bool(torch.isnan(d[6]).all()) and bool((d[7] == -float("inf")).all())
    ok = [n for n in range(N) if n not in (5, 6, 7)]
    assert bool(torch.isfinite(d[ok]).all())
    assert db[5] == float("inf") and bool(torch.isnan(db[6])) and db[7] == -float("inf")
    assert bool(torch.isfinite(db[ok]).all())
    if dtype == F32:                                         # a NaN whose payload fills the low bits
        gy = _grad(T, N, dtype, 4)
        gy.view(torch.int32)[3, 2] = 0x7F800001
        dw = ops.act8_wgrad(gy, *ops.act8_pack(torch.ones(T, K, device=DEV)), K, F32)
        assert bool(torch.isnan(dw[2]).all()) and bool(torch.isfinite(dw[3:]).all())
        # the whole range of f32: parts that bf16 rounds away or flushes would show
        gy = torch.full((1, 3), 1.0 + 2.0 ** -23, device=DEV)
        gy[0, 1], gy[0, 2] = 3.4e38, 1.1754944e-38 * (1 + 2.0 ** -20)
        dw = ops.act8_wgrad(gy, *ops.act8_pack(torch.ones(1, 32, device=DEV)), 32, F32)
        assert bool((dw[:2] == gy[0, :2, None]).all())
        assert bool(((dw[2] - gy[0, 2]).abs() <= 2.0 ** -126 * 2.0 ** -7).all())


def test_wgrad_without_tokens_or_outputs():
    ops = _ops()
    q, s = ops.act8_pack(torch.empty(0, 40, device=DEV))
    dw, db = ops.act8_wgrad(torch.empty(0, 24, device=DEV), q, s, 40, F32, bias=True)
    assert dw.shape == (24, 40) and not bool(dw.any()) and not bool(db.any())
    q, s = ops.act8_pack(torch.ones(4, 40, device=DEV))
    dw, db = ops.act8_wgrad(torch.empty(4, 0, device=DEV), q, s, 40, F32, bias=True)
    assert dw.shape == (0, 40) and db.shape == (0,)


# ------------------------------------------------------------------------------- refusals
def test_refusals():
    ops = _ops()
    from visionseg import _lib as L
    x = torch.ones(8, 40, device=DEV)
    w = torch.ones(40, device=DEV)
    q, s = ops.act8_pack(x)
    bad = [
        (lambda: ops.act8_pack(x.half()), "float32 or bfloat16"),
        (lambda: ops.act8_pack(x[0, 0]), "dimension"),
        (lambda: ops.act8_unpack(q, s, 20, F32), "not a checkpoint"),
        (lambda: ops.act8_unpack(q, s, 65, F32), "not a checkpoint"),
        (lambda: ops.act8_unpack(q[:4], s, 40, F32), "not a checkpoint"),
        (lambda: ops.act8_unpack(q, s.to(torch.int8), 40, F32), "uint8"),
        (lambda: ops.act8_unpack(q, s, 40, torch.float16), "float32 or bfloat16"),
        (lambda: ops.act8_wgrad(x[:4], q, s, 40, F32), "rows"),
        (lambda: ops.act8_wgrad(x, q, s, 0, F32), "feature"),
        (lambda: ops.act8_wgrad(x, q, s, 40, torch.float64), "float32 or bfloat16"),
        (lambda: ops.gelu_act8(x.double()), "float32 or bfloat16"),
        (lambda: ops.layer_norm_act8(x, w.bfloat16(), w), "dtype"),
        (lambda: ops.layer_norm_act8(x, w[:39], w), "weight and bias"),
        (lambda: ops.layer_norm_act8(torch.ones(2, 8200, device=DEV), torch.ones(8200, device=DEV),
                                     torch.ones(8200, device=DEV)), "8192"),
        (lambda: ops.add_layer_norm_act8(x, x[:4], w, w), "shaped"),
        (lambda: ops.add_layer_norm_act8(x, x.bfloat16(), w, w), "shaped"),
        (lambda: L.tops().act8_gelu_bwd(x[:4], q, s), "rows"),
        (lambda: L.tops().act8_layer_norm_bwd(x[:4], None, q, s, w, torch.ones(8, device=DEV),
                                              torch.ones(8, device=DEV)), "rows"),
        (lambda: L.tops().act8_layer_norm_bwd(x, x[:4], q, s, w, torch.ones(8, device=DEV),
                                              torch.ones(8, device=DEV)), "grad_s"),
        (lambda: L.tops().act8_layer_norm_bwd(x, None, q, s, w, torch.ones(7, device=DEV),
                                              torch.ones(8, device=DEV)), "mean"),
    ]
    for call, msg in bad:
        with pytest.raises(RuntimeError, match=msg):
            call()
    with pytest.raises(RuntimeError, match="HIP device|devices"):
        ops.act8_unpack(q, s.cpu(), 40, F32)
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(ops.gelu_act8(xg).sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                                   # once differentiable


# ------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,bias", [(F32, True), (BF16, True), (F32, False)])
def test_linear_and_mlp(dtype, bias):
    """linear_act8 and mlp_act8 on an input that its checkpoint holds exactly."""
    from visionseg.linear import linear_act8, mlp_act8
    g = _gen(1)
    C, Hd, T = 96, 200, 640
    x = _on_grid(T, C, dtype, 2).view(2, T // 2, C)
    w1, w2 = ((0.1 * torch.randn(*s, generator=g, device=DEV)).to(dtype) for s in ((Hd, C), (C, Hd)))
    b1, b2 = ((torch.randn(n, generator=g, device=DEV)).to(dtype) if bias else None for n in (Hd, C))
    gy = _grad(T, Hd, dtype, 4).view(2, T // 2, Hd)

    def grads(fn, ts, gout):
        ts = [t.detach().clone().requires_grad_() if t is not None else None for t in ts]
        y = fn(*ts)
        return y, torch.autograd.grad(y, [t for t in ts if t is not None], gout)

    y, gr = grads(linear_act8, (x, w1, b1), gy)
    y0, gr0 = grads(F.linear, [t.double() if t is not None else None for t in (x, w1, b1)], gy.double())
    # a chain of n <= 640 additions of f32: each is off by U of a partial sum of k terms, in the root
    # mean square U sqrt(k), all of them U n / sqrt(2) terms against a sum of sqrt(n): U sqrt(n / 2)
    tol = 4 * ref.STEP[dtype] + 2 * ref.U * (T / 2) ** 0.5
    y, y0 = y.detach(), y0.detach()
    for a, c in zip((y, *gr), (y0, *gr0)):
        assert float((a.double() - c).norm() / c.norm()) < tol

    # the MLP's backward from its formulas at the pre-activation's checkpoint
    gy = _grad(T, C, dtype, 5).view(2, T // 2, C)
    args = (x, w1, b1, w2, b2)
    y, gr = grads(mlp_act8, args, gy)
    pre = F.linear(x, w1, b1).view(T, Hd)                    # the library call that the MLP makes
    h, x64, g64 = ref.stand_for(pre), x.double().view(T, C), gy.double().view(T, C)
    gh = (g64 @ w2.double()) * (1 - ref.tail(h) + h * ref.phi(h))
    want = [gh @ w1.double(), gh.t() @ x64, gh.sum(0), g64.t() @ (h * (1 - ref.tail(h))), g64.sum(0)]
    want = [v for v, t in zip(want, args) if t is not None]
    p64 = pre.double()
    y0 = (p64 * (1 - ref.tail(p64))) @ w2.double().t() + (b2.double() if bias else 0)
    tol = 8 * ref.STEP[dtype] + 4 * ref.U * (T / 2) ** 0.5   # up to four roundings to the type on the way
    for a, c in zip((y.detach(), *gr), (y0, *want)):
        assert float((a.double().view(c.shape) - c).norm() / c.norm()) < tol
    # a frozen part
    for k in range(5):
        if args[k] is None:
            continue
        ts = [t.detach().clone() if t is not None else None for t in args]
        ts[k].requires_grad_()
        (gk,) = torch.autograd.grad(mlp_act8(*ts), ts[k], gy)
        i = [j for j in range(5) if args[j] is not None].index(k)
        assert float((gk.double() - gr[i].double()).norm() / gr[i].double().norm()) < tol


def _block(act8, dtype, seed=0):
    from visionseg.model import M2FConfig, SwinBackbone
    torch.manual_seed(seed)
    cfg = M2FConfig(embed_dim=96, depths=(2, 2), num_heads=(3, 6), window_size=7, act8=act8)
    return SwinBackbone(cfg).to(DEV, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_swin_backbone(dtype):
    """The Swin backbone under M2FConfig.act8: the same features, gradients within what 8 bits
    cost, less memory."""
    px = torch.randn(1, 3, 224, 256, generator=_gen(1), device=DEV).to(dtype)
    out = {}
    for act8 in (False, True):
        net = _block(act8, dtype)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        feats = net(px)
        kept = torch.cuda.memory_allocated() - base
        gos = [_grad(f.numel(), 1, dtype, i).view(f.shape) for i, f in enumerate(feats)]
        grads = torch.autograd.grad(feats, list(net.parameters()), gos)
        out[act8] = ([f.detach() for f in feats], grads, kept)
    for a, c in zip(out[True][0], out[False][0]):
        assert float((a.double() - c.double()).norm() / c.double().norm()) < (1e-5 if dtype == F32 else 2e-2)
    for a, c in zip(out[True][1], out[False][1]):
        assert float((a.double() - c.double()).norm()) <= 0.05 * float(c.double().norm()) + 1e-12
    assert out[True][2] < 0.75 * out[False][2], (out[True][2], out[False][2])


def test_trainer():
    """Training steps of the whole model under M2FConfig.act8, replayed as HIP graphs and eager: the
    same losses and weights, to the noise of the float atomics elsewhere in the model (the bounds of
    tests/test_gpu_graphs.py)."""
    import copy
    from test_gpu_graphs import _compare, _run
    from visionseg.criterion import SetCriterion
    from visionseg.data import synthetic_batch
    from visionseg.model import M2FConfig, Mask2Former
    from visionseg.train import Trainer
    dev = torch.device(DEV, 0)
    cfg = M2FConfig.preset("swin_t", num_queries=20, act8=True)
    model = Mask2Former(cfg).init_weights(seed=0)
    batch = synthetic_batch(2, 256, seed=1, device=dev)
    ta = Trainer(copy.deepcopy(model), SetCriterion(cfg), device=dev)
    tb = Trainer(copy.deepcopy(model), SetCriterion(cfg), device=dev, graphs=True, graph_warmup=2)
    la, lb = _run(ta, [batch] * 6), _run(tb, [batch] * 6)
    assert tb.captures == 1
    _compare(ta, tb, la, lb)


def test_predictor_and_checkpoints():
    """Without gradients the act8 model keeps nothing and predicts what it does in training; its
    state dict is the plain model's."""
    from visionseg.model import M2FConfig, Mask2Former
    kw = dict(embed_dim=32, depths=(2, 2, 2, 2), num_heads=(1, 2, 4, 8), feature_size=64, mask_feature_size=64,
              hidden_dim=64, enc_ffn=128, dec_ffn=128, dec_heads=2, enc_layers=2, dec_layers=4, num_queries=10)
    torch.manual_seed(4)
    plain, packed = Mask2Former(M2FConfig(**kw)), Mask2Former(M2FConfig(act8=True, **kw))
    packed.load_state_dict(plain.state_dict())
    plain, packed = plain.to(DEV), packed.to(DEV)
    im = torch.randn(1, 3, 128, 160, generator=_gen(1), device=DEV)
    with torch.no_grad():
        a, b = plain.backbone(im), packed.backbone(im)
        kept = packed.backbone(im)
    for x, y, z in zip(a, b, kept):
        assert torch.equal(y, z)
        assert float((x - y).norm() / x.norm()) < 1e-5
    with torch.enable_grad():
        for y, z in zip(b, packed.backbone(im)):
            # (the Linears of training and inference may be different GEMMs)
            assert float((y - z.detach()).norm() / y.norm()) < 1e-5


def test_inference_mode_and_one_dimension():
    ops = _ops()
    x = _act(5, 40, F32, 1)
    w, b = torch.rand(40, device=DEV).requires_grad_(), torch.rand(40, device=DEV).requires_grad_()
    want = ops.layer_norm_act8(x, w, b).detach(), ops.gelu_act8(x)
    with torch.inference_mode():
        assert torch.equal(ops.layer_norm_act8(x, w, b), want[0]) and torch.equal(ops.gelu_act8(x), want[1])
        assert torch.equal(ops.add_layer_norm_act8(x, x, w, b)[0], 2 * x)
    # one row without a dimension for it: the same as a matrix of one row
    assert torch.equal(ops.gelu_act8(x[1]), want[1][1]) and torch.equal(ops.layer_norm_act8(x[1], w, b), want[0][1])
    q, s = ops.act8_pack(x[1])
    assert torch.equal(ops.act8_unpack(q, s, 40, F32), ops.act8_unpack(*ops.act8_pack(x), 40, F32)[1])
    gy = _grad(5, 24, F32, 2)
    assert torch.equal(ops.act8_wgrad(gy[1], q, s, 40, F32), ops.act8_wgrad(gy[1:2], q[None], s[None], 40, F32))


def test_whole_gradients_by_expansion():
    """The gradient that sum() sends back is one number without strides."""
    ops = _ops()
    x = _act(6, 40, F32, 1).requires_grad_()
    w, b = torch.rand(40, device=DEV).requires_grad_(), torch.rand(40, device=DEV).requires_grad_()
    for f, ts in ((lambda: ops.gelu_act8(x), (x,)), (lambda: ops.layer_norm_act8(x, w, b), (x, w, b))):
        a = torch.autograd.grad(f().sum(), ts)
        y = f()
        c = torch.autograd.grad(y, ts, torch.ones_like(y))
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    q, s = ops.act8_pack(x.detach())
    one = torch.ones((), device=DEV).expand(6, 24)
    dw, db = ops.act8_wgrad(one, q, s, 40, F32, bias=True)
    dw0, db0 = ops.act8_wgrad(one.contiguous(), q, s, 40, F32, bias=True)
    assert torch.equal(dw, dw0) and torch.equal(db, db0)


def test_two_streams_at_once():
    ops = _ops()
    sets = [(_act(20000, 256, BF16, k), _grad(20000, 256, BF16, 10 + k)) for k in range(2)]
    want = [ops.act8_wgrad(gy, *ops.act8_pack(x), 256, F32, bias=True) for x, gy in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, (x, gy) in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(ops.act8_wgrad(gy, *ops.act8_pack(x), 256, F32, bias=True))
        torch.cuda.synchronize()
        for (a, b), (c, d) in zip(got, want):
            assert torch.equal(a, c) and torch.equal(b, d)


def test_on_another_stream():
    ops = _ops()
    side = torch.cuda.Stream()
    x, gy = _act(3000, 200, BF16, 1), _grad(3000, 96, BF16, 2)
    want = ops.act8_wgrad(gy, *ops.act8_pack(x), 200, F32)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.act8_wgrad(gy, *ops.act8_pack(x), 200, F32)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_captured_and_replayed():
    """Forward and backward of the set captured twice, the two graphs replayed in turn with eager
    work between: every replay gives the eager result for the inputs it finds."""
    ops = _ops()
    from visionseg import linear
    C, N, T = 96, 130, 700
    w = torch.rand(C, device=DEV).bfloat16().requires_grad_()
    b = torch.rand(C, device=DEV).bfloat16().requires_grad_()
    wl = torch.randn(N, C, generator=_gen(2), device=DEV).bfloat16().requires_grad_()
    bl = torch.rand(N, device=DEV).bfloat16().requires_grad_()

    def step(x, gy):
        y = ops.gelu_act8(linear.linear_act8(ops.layer_norm_act8(x, w, b), wl, bl))
        return (y.detach(), *torch.autograd.grad(y, (x, w, b, wl, bl), gy))

    def data(seed):
        return _act(T, C, BF16, seed), _grad(T, N, BF16, seed + 50)

    graphs = []
    for k in range(2):
        x, gy = data(k)
        x = x.requires_grad_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(x, gy)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(x, gy)
        graphs.append((g, x, gy, out))
    for turn in range(3):
        for k, (g, x, gy, out) in enumerate(graphs):
            nx, ngy = data(10 * turn + k)
            with torch.no_grad():
                x.copy_(nx)
            gy.copy_(ngy)
            g.replay()
            torch.cuda.synchronize()
            want = step(nx.requires_grad_(), ngy)
            assert all(torch.equal(a, c) for a, c in zip(out, want)), (turn, k)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two devices")
def test_on_another_device():
    ops = _ops()
    x = _act(100, 70, F32, 1)
    q, s = ops.act8_pack(x.to("cuda:1"))
    assert q.device.index == 1 and torch.equal(q.to(DEV), ops.act8_pack(x)[0])


def test_rows_beyond_32_bits():
    """More than 2^32 elements: the last rows are packed and read back like the first."""
    ops = _ops()
    rows, C = (1 << 32) // 1000 + 7, 1000
    x = torch.zeros(rows, C, device=DEV, dtype=BF16)
    some = _act(5, C, BF16, 3)
    at = [0, 1, (1 << 31) // C, rows - 2, rows - 1]
    x[at] = some
    q, s = ops.act8_pack(x)
    rq, rs = ref.pack(some)
    assert torch.equal(q[at], rq) and torch.equal(s[at], rs)
    x.zero_()
    v = ops.act8_unpack(q, s, C, BF16)
    assert torch.equal(v[at].double(), ref.values(rq, rs, C))
    del x, v
    gy = torch.zeros(rows, 8, device=DEV, dtype=BF16)
    gs = _grad(5, 8, BF16, 4)
    gy[at] = gs
    dw = ops.act8_wgrad(gy, q, s, C, F32)
    rw, _, tw, _ = ref.wgrad(gs, rq, rs, C, F32)
    ref.within(dw, rw, tw, "dw")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,N,pitch,first", [
    (1, 40, 9, 9, 1), (130, 40, 9, 9, 1), (130, 40, 9, 11, 2), (1000, 300, 517, 517, 0), (1000, 300, 517, 519, 1),
    (1000, 300, 518, 519, 3), (6000, 515, 515, 515, 0), (6000, 515, 514, 514, 1), (9000, 1030, 1031, 1031, 1)])
def test_wgrad_row_starts(T, K, N, pitch, first, dtype):
    """Rows that begin anywhere; the gradient's last value is its storage's last, and what lies in
    front of a row and behind it is NaN."""
    ops = _ops()
    q, s = ops.act8_pack(_act(T, K, dtype, 5))
    flat = torch.full((first + (T - 1) * pitch + N,), float("nan"), device=DEV, dtype=dtype)
    gy = flat.as_strided((T, N), (pitch, 1), first)
    gy.copy_(_grad(T, N, dtype, 6))
    dw, db = ops.act8_wgrad(gy, q, s, K, F32, bias=True)
    rw, rb, tw, tb = ref.wgrad(gy.contiguous(), q, s, K, F32)
    ref.within(dw, rw, tw, "dw")
    ref.within(db, rb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N", [40, 257])
def test_wgrad_rows_far_apart(N, dtype):
    """64 rows that span more than 2^31 bytes: addressed row by row."""
    ops = _ops()
    T, K, pitch = 70, 100, 1 << 24
    q, s = ops.act8_pack(_act(T, K, dtype, 7))
    flat = torch.empty((T - 1) * pitch + N, device=DEV, dtype=dtype)
    gy = flat.as_strided((T, N), (pitch, 1))
    gy.copy_(_grad(T, N, dtype, 8))
    dw, db = ops.act8_wgrad(gy, q, s, K, F32, bias=True)
    rw, rb, tw, tb = ref.wgrad(gy.contiguous(), q, s, K, F32)
    ref.within(dw, rw, tw, "dw")
    ref.within(db, rb, tb, "db")


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,N", [(100000, 20, 18), (200000, 96, 95), (200000, 96, 96), (16384, 384, 1536),
                                   (40001, 1030, 1030), (40001, 1029, 1031)])
def test_wgrad_tiles(T, K, N, dtype):
    """Sizes from the smallest output tile with hundreds of splits to the largest one."""
    ops = _ops()
    x, gy = _act(T, K, dtype, 9), _grad(T, N, dtype, 10)
    q, s = ops.act8_pack(x)
    del x
    dw, db = ops.act8_wgrad(gy, q, s, K, F32, bias=True)
    rw, rb, tw, tb = ref.wgrad(gy, q, s, K, F32)
    ref.within(dw, rw, tw, "dw")
    ref.within(db, rb, tb, "db")
    assert torch.equal(ops.act8_wgrad(gy, q, s, K, F32), dw)
