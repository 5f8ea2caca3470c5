"""The Linears of the 8-bit activation checkpoints without a GPU: their autograd Functions on CPU
tensors, with plain torch in the place of the kernels (the reference of the GPU tests)."""
import pytest
import torch

import _act8ref as ref
from visionseg import linear, ops


@pytest.fixture
def plain_kernels(monkeypatch):
    def gelu_bwd(gy, q, scale, recompute):
        h = ref.values(q, scale, gy.shape[-1])
        slope = 1 - ref.tail(h) + h * ref.phi(h)
        return (gy.double() * slope).to(gy.dtype), (h * (1 - ref.tail(h))).to(gy.dtype) if recompute else None

    def wgrad(gy, q, scale, features, out_dtype, bias=False):
        dw = (gy.double().t() @ ref.values(q, scale, features)).to(out_dtype)
        return (dw, gy.double().sum(0).to(out_dtype)) if bias else dw

    monkeypatch.setattr(ops, "act8_pack", lambda x: ref.pack(x))
    monkeypatch.setattr(ops, "act8_wgrad", wgrad)
    monkeypatch.setattr(ops, "_act8", lambda: {
        "act8_gelu_fwd": lambda x, keep: (torch.nn.functional.gelu(x), *ref.pack(x)),
        "act8_gelu_bwd": gelu_bwd})


def _leaves(*shapes):
    g = torch.Generator().manual_seed(3)
    return [torch.randn(*s, generator=g, requires_grad=True) for s in shapes]


def test_a_second_backward_over_a_retained_graph(plain_kernels):
    x, w1, b1, w2, b2 = _leaves((2, 5, 40), (24, 40), (24,), (40, 24), (40,))
    for fn, ts, n in ((linear._LinearAct8Fn, (x, w1, b1), 24), (linear._MlpAct8Fn, (x, w1, b1, w2, b2), 40)):
        y = fn.apply(*ts)
        gy = torch.randn(2, 5, n, generator=torch.Generator().manual_seed(4))
        first = torch.autograd.grad(y, ts, gy, retain_graph=True)
        again = torch.autograd.grad(y, ts, gy)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_a_tangent_is_refused():
    """Forward mode, with and without a reverse-mode gradient as well: refused before the device is
    looked at."""
    import torch.autograd.forward_ad as fwd
    from visionseg import _lib as L
    t = L.tops()
    x, r, w, b = torch.randn(3, 40), torch.randn(3, 40), torch.ones(40), torch.zeros(40)
    for grad in (False, True):
        with fwd.dual_level():
            def dual(v):
                return fwd.make_dual(v.clone().requires_grad_(grad), torch.ones_like(v))
            for call in (lambda: t.gelu_act8(dual(x)), lambda: t.layer_norm_act8(dual(x), w, b, 1e-5),
                         lambda: t.layer_norm_act8(x, dual(w), b, 1e-5), lambda: t.layer_norm_act8(x, w, dual(b), 1e-5),
                         lambda: t.add_layer_norm_act8(dual(x), r, w, b, 1e-5),
                         lambda: t.add_layer_norm_act8(x, dual(r), w, b, 1e-5)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()


@pytest.mark.parametrize("rows,C", [(1 << 27, 256), ((1 << 27) - 7, 250), (1 << 32, 1), (33, 1 << 30), ((1 << 30) + 1, 32)])
def test_tensors_beyond_one_launch_are_refused(rows, C):
    """2^32 threads or more: refused before any HIP call, by name."""
    import ctypes
    from visionseg import _lib as L
    lib, p = L.lib(), ctypes.c_void_p(16)
    for rc in (lib.vs_act8_pack(1, p, C, p, p, rows, C, None), lib.vs_act8_unpack(1, p, p, p, rows, C, None),
               lib.vs_act8_gelu_forward(1, p, p, p, p, rows, C, None),
               lib.vs_act8_gelu_backward(1, p, p, p, p, p, rows, C, None)):
        assert rc == -1 and b"too large" in lib.vs_last_error()
