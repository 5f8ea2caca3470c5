"""Operands of the weight gradient whose sums float32 holds exactly, in any order and association,
so that a result is right to the last bit or wrong: a bound that grows with the tokens cannot hide
a chunk that was left out or a part of a float32 gradient that was dropped.

whole()  every gradient -1, 0 or 1, every q in -15..15, every step 1/2, 1 or 2: a sum over T tokens is
         a whole number of halves of at most 60 T < 2^24.
parts()  float32: one token a column of the gradient, its value a full 24-bit significand (odd, so that
         none of its three bf16 parts is zero but by chance), q = +-1 and steps of 1/4..4: a product is
         the gradient moved by a power of two, and the parts add up to it without rounding.

Both -> gy [T, N], q int8 [T, P], scale uint8 [T, P / 32], dw float64 [N, K], db float64 [N]."""
import torch


def _values(q, scale, K):
    step = ((scale.long() - 127 + 1023) << 52).view(torch.float64)
    return (q.double().view(q.shape[0], -1, 32) * step.unsqueeze(-1)).view(q.shape[0], -1)[:, :K].contiguous()


def product(gy, q, scale, K):
    g = gy.double()
    return g.t().contiguous() @ _values(q, scale, K), g.sum(0)


def _checkpoint(T, K, g, device, lo, hi, steps):
    P = -(-K // 32) * 32
    q = torch.randint(lo, hi + 1, (T, P), generator=g, device=device, dtype=torch.int8)
    q[:, K:] = 0
    return q, torch.randint(127 - steps, 128 + steps, (T, P // 32), generator=g, device=device, dtype=torch.uint8)


def whole(T, N, K, dtype, seed, device):
    assert 60 * T < 1 << 24
    g = torch.Generator(device=device).manual_seed(seed)
    gy = torch.randint(-1, 2, (T, N), generator=g, device=device, dtype=torch.int8).to(dtype)
    q, scale = _checkpoint(T, K, g, device, -15, 15, 1)
    return (gy, q, scale, *product(gy, q, scale, K))


def parts(T, N, K, seed, device):
    g = torch.Generator(device=device).manual_seed(seed)
    at = torch.randint(0, T, (N,), generator=g, device=device)
    ends = [t for t in (0, T - 1, 31, 32, 63, 64) if t < T][:N]
    at[:len(ends)] = torch.tensor(ends, device=device)
    v = (torch.randint(1 << 23, 1 << 24, (N,), generator=g, device=device) | 1).float()
    v = torch.ldexp(v, torch.randint(-60, -20, (N,), generator=g, device=device))
    v = torch.where(torch.rand(N, generator=g, device=device) < 0.5, v, -v)
    gy = torch.zeros(T, N, device=device)
    gy[at, torch.arange(N, device=device)] = v
    q, scale = _checkpoint(T, K, g, device, 0, 1, 2)
    q[:, :K] = 2 * q[:, :K] - 1
    return (gy, q, scale, *product(gy, q, scale, K))


def same(got, want, what):
    """got (float32 or bfloat16) is want (float64, exact in float32), rounded once."""
    exact = want.float()
    assert torch.equal(exact.double(), want), what
    assert torch.equal(got, exact.to(got.dtype)), f"{what}: {int((got != exact.to(got.dtype)).sum())} of {got.numel()}"
