"""GPU tests of how the 8-bit activation checkpoints behave under autograd: repeated backward
passes, forward mode, empty sizes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
F32, BF16 = torch.float32, torch.bfloat16


def _rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


@pytest.mark.parametrize("dtype,T", [(F32, 300), (BF16, 300), (BF16, 5000)])
def test_a_second_backward_over_a_retained_graph(dtype, T):
    """Every op's gradients come out the same twice (5000 tokens: the input gradients on the token
    GEMM, whose transposed weights the first pass has already used up)."""
    from visionseg import ops
    from visionseg.linear import linear_act8, mlp_act8
    C, H = 96, 384
    x, r = _rand((T, C), dtype, 1), _rand((T, C), dtype, 2)
    w, b = _rand((C,), dtype, 3), _rand((C,), dtype, 4)
    w1, b1, w2, b2 = _rand((H, C), dtype, 5, 0.1), _rand((H,), dtype, 6), _rand((C, H), dtype, 7, 0.1), _rand((C,), dtype, 8)
    for fn, ts in ((lambda *a: ops.gelu_act8(*a), (x,)), (lambda *a: ops.layer_norm_act8(*a), (x, w, b)),
                   (lambda *a: ops.add_layer_norm_act8(*a)[1], (x, r, w, b)), (linear_act8, (x, w1, b1)),
                   (mlp_act8, (x, w1, b1, w2, b2))):
        ts = [t.clone().requires_grad_() for t in ts]
        y = fn(*ts)
        gy = _rand(y.shape, dtype, 9)
        first = torch.autograd.grad(y, ts, gy, retain_graph=True)
        again = torch.autograd.grad(y, ts, gy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))
