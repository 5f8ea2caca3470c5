"""GPU tests of the weight gradient from 8-bit checkpoints, to the last bit, on every output tile of
csrc/act8_wgrad.hip with and without splits of the tokens and in every way it reads a gradient."""
import pytest
import torch

import _act8exact as ex

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16

# T, K, N.  An odd N: bf16 rows that begin inside a dword
BF16_SIZES = [
    (65, 129, 127), (400, 256, 256), (5000, 64, 40), (100000, 20, 18), (100000, 20, 19),       # 64 x 64
    (130, 1030, 2048), (130, 1030, 2047), (4000, 4100, 96), (200000, 96, 96), (200000, 96, 95),  # 128 x 128
    (200, 4100, 1030), (200, 4100, 1031), (4000, 4100, 130), (4000, 4100, 131), (16384, 96, 2047),  # 256 x 128
    (200, 4100, 2048), (200, 4100, 2047), (4001, 4100, 516), (4001, 4100, 515)]                 # 256 x 256
F32_SIZES = [
    (65, 130, 130), (1000, 96, 96), (10007, 203, 299), (150000, 20, 18),                   # 64 x 64
    (130, 1030, 2047), (4000, 96, 2047), (2000, 4100, 96),                                      # 128 x 128
    (200, 1030, 4100), (4000, 130, 2047), (9000, 2048, 96)]                                     # 128 x 256


def _check(gy, q, scale, dw, db, K):
    from visionseg import ops
    for out in (F32, BF16):
        gw, gb = ops.act8_wgrad(gy, q, scale, K, out, bias=True)
        ex.same(gw, dw, "dw")
        ex.same(gb, db, "db")
        ex.same(ops.act8_wgrad(gy, q, scale, K, out), dw, "dw without db")


@pytest.mark.parametrize("T,K,N,dtype", [(*s, BF16) for s in BF16_SIZES] + [(*s, F32) for s in F32_SIZES])
def test_whole_numbers(T, K, N, dtype):
    _check(*ex.whole(T, N, K, dtype, T + K + N, DEV), K)


@pytest.mark.parametrize("T,K,N", F32_SIZES)
def test_three_parts(T, K, N):
    _check(*ex.parts(T, N, K, T + K + N, DEV), K)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("T,K,N,pitch,first", [
    (200, 4100, 2047, 2049, 1), (200, 4100, 2048, 2051, 3), (130, 1030, 2047, 2048, 1), (4000, 130, 2047, 2047, 1),
    (400, 256, 256, 263, 5)])
def test_row_starts(T, K, N, pitch, first, dtype):
    """Rows that begin anywhere in a wider buffer of NaN."""
    for gy, q, scale, dw, db in (ex.whole(T, N, K, dtype, 1, DEV),) + ((ex.parts(T, N, K, 2, DEV),) if dtype == F32 else ()):
        flat = torch.full((first + (T - 1) * pitch + N,), float("nan"), device=DEV, dtype=dtype)
        rows = flat.as_strided((T, N), (pitch, 1), first)
        rows.copy_(gy)
        _check(rows, q, scale, dw, db, K)


@pytest.mark.parametrize("T,K,N", [(70, 100, 40), (70, 1030, 2047), (70, 4100, 1030)])
def test_rows_far_apart(T, K, N):
    """64 rows that span more than 2^31 bytes, on each kind of tile."""
    pitch = 1 << 24
    gy, q, scale, dw, db = ex.whole(T, N, K, BF16, 3, DEV)
    rows = torch.empty((T - 1) * pitch + N, device=DEV, dtype=BF16).as_strided((T, N), (pitch, 1))
    rows.copy_(gy)
    _check(rows, q, scale, dw, db, K)
    del rows
    gy, q, scale, dw, db = ex.parts(T, N, K, 4, DEV)
    rows = torch.empty((T - 1) * pitch + N, device=DEV).as_strided((T, N), (pitch, 1))
    rows.copy_(gy)
    _check(rows, q, scale, dw, db, K)


def test_three_parts_down_to_denormals():
    """A gradient of 2^-110 or more is the sum of its parts; below, bf16's last bit, 2^-133, is where they
    are cut (towards zero: off by less than that, times |h|)."""
    from visionseg import ops
    g = torch.Generator(device=DEV).manual_seed(1)
    for he in (0, 20, -10):
        q, scale = ops.act8_pack(torch.full((1, 32), 2.0 ** he, device=DEV))
        for e in (-149, -140, -134, -133, -130, -127, -126, -120, -118, -112, -111, -110, -109, -104, -103, -96):
            v = (torch.randint(1 << 23, 1 << 24, (1, 515), generator=g, device=DEV) | 1).double() * 2.0 ** (e - 23)
            gy = v.float()                                   # (rounded below 2^-126)
            dw = ops.act8_wgrad(gy, q, scale, 32, F32).double()
            want = (gy.double() * 2.0 ** he).view(-1, 1).expand_as(dw)
            if e >= -110:
                assert torch.equal(dw, want), (he, e)
            else:
                # (and the result's own rounding where it is a denormal)
                assert bool(((dw - want).abs() < 2.0 ** (he - 133) + (2.0 ** -150 if he < 0 else 0)).all()), (he, e)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_checkpoint_error_bound(dtype):
    """At most 1 / 127 of the block's largest magnitude, or 2^-127."""
    from visionseg import ops
    g = torch.Generator(device=DEV).manual_seed(2)
    x = torch.randn(4000, 64, generator=g, device=DEV, dtype=torch.float64)
    x = (x * 2.0 ** torch.linspace(-148, 125, 4000, device=DEV, dtype=torch.float64).view(-1, 1)).to(dtype)
    v = ops.act8_unpack(*ops.act8_pack(x), 64, F32).double()
    a = x.double().view(4000, 2, 32).abs().amax(-1, keepdim=True)
    off = (v - x.double()).view(4000, 2, 32).abs()
    held = (a <= 127 * 2.0 ** 121).expand_as(off)            # above: NaN
    assert bool((off <= torch.clamp(a / 127, min=2.0 ** -127))[held].all())
    assert bool(torch.isnan(off[~held]).all())


def test_gelu_f32_in_the_norm():
    """f32 GELU and its gradient against float64, in the norm.  One rounding is off by U = 2^-24 at most and
    0.41 U in the root mean square over significands.  With h ~ N(0, 1): gx = gy (1 + d), d ~ -0.35 =
    (a - M) phi.  M: two roundings and the fit's 0.22 U; a - M: one; phi: 0.6 U of the exponential, 0.41 U
    of its factor, 0.3 U of its argument; d: one; each of them times 0.35; 1 + d and the product with gy: one
    each, of 0.75.  The root of the squares is 0.6 U of 0.75, 0.8 U: 0.9 U allowed.  y = max(x, 0) - a M phi:
    x M phi is 0.25 of y in the mean, the last rounding whole: 0.45 U, 0.5 U allowed."""
    from visionseg import ops
    U = 2.0 ** -24
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(20000, 64, generator=g, device=DEV) * torch.exp(0.6 * torch.randn(64, generator=g, device=DEV))
    gy = torch.randn(20000, 64, generator=g, device=DEV)
    x = ops.act8_unpack(*ops.act8_pack(x), 64, F32).requires_grad_()          # its own checkpoint
    y = ops.gelu_act8(x)
    (gx,) = torch.autograd.grad(y, x, gy)
    v = x.detach().double()
    cdf = 0.5 * torch.special.erfc(-v / 2.0 ** 0.5)
    want_y, want_gx = v * cdf, gy.double() * (cdf + v * torch.exp(-v * v / 2) / (2 * torch.pi) ** 0.5)
    assert float((y.detach().double() - want_y).norm() / want_y.norm()) <= 0.5 * U
    assert float((gx.double() - want_gx).norm() / want_gx.norm()) <= 0.9 * U


def test_norm_and_gelu_beyond_32_bits():
    """Tensors of more than 2^32 elements: rows there come out as they do in a tensor of their own."""
    from visionseg import ops
    C = 1000
    rows = (1 << 32) // C + 9
    at = torch.tensor([0, 1, (1 << 31) // C, (1 << 31) // C + 1, rows - 2, rows - 1], device=DEV)
    g = torch.Generator(device=DEV).manual_seed(4)
    some, grad = (torch.randn(6, C, generator=g, device=DEV).to(BF16) for _ in range(2))
    w, b = (torch.rand(C, generator=g, device=DEV).to(BF16).requires_grad_() for _ in range(2))
    few = some.clone().requires_grad_()
    want = ops.layer_norm_act8(few, w, b), ops.gelu_act8(few)
    want_gx = torch.autograd.grad(want[0], few, grad)[0], torch.autograd.grad(want[1], few, grad)[0]
    x = torch.zeros(rows, C, device=DEV, dtype=BF16)
    x[at] = some
    x.requires_grad_()
    gy = torch.zeros(rows, C, device=DEV, dtype=BF16)
    gy[at] = grad
    for k, op in enumerate((lambda: ops.layer_norm_act8(x, w, b), lambda: ops.gelu_act8(x))):
        y = op()
        assert torch.equal(y.detach()[at], want[k].detach())
        gx = torch.autograd.grad(y, x, gy)[0]
        assert torch.equal(gx[at], want_gx[k])
        del y, gx
    # a width without remainder (the kernels' flat form)
    n = (1 << 32) // 1024 + 5
    z = torch.zeros(n, 1024, device=DEV, dtype=BF16)
    tail = torch.randn(3, 1024, generator=g, device=DEV).to(BF16)
    z[-3:] = tail
    assert torch.equal(ops.gelu_act8(z)[-3:], ops.gelu_act8(tail))


def test_weight_gradient_of_more_than_32_bits():
    """dW of more than 2^32 values."""
    from visionseg import ops
    T, N, K = 3, 66001, 66004
    g = torch.Generator(device=DEV).manual_seed(5)
    gy = torch.randint(-1, 2, (T, N), generator=g, device=DEV, dtype=torch.int8).to(BF16)
    x = torch.randint(-15, 16, (T, K), generator=g, device=DEV, dtype=torch.int8).to(BF16)
    q, scale = ops.act8_pack(x)
    h = ops.act8_unpack(q, scale, K, F32).double()
    dw, db = ops.act8_wgrad(gy, q, scale, K, BF16, bias=True)
    ex.same(db, gy.double().sum(0), "db")
    for r in (0, 1, (1 << 31) // K, (1 << 32) // K - 1, (1 << 32) // K, N - 1):
        ex.same(dw[r], (gy[:, r].double()[:, None] * h).sum(0), f"row {r}")
    cols = torch.tensor([0, 31, 32, K // 2, K - 1], device=DEV)
    ex.same(dw[:, cols], gy.double().t().contiguous() @ h[:, cols].contiguous(), "columns")
