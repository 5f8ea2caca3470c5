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


def test_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    from visionseg import _lib as L, ops
    from visionseg.linear import linear_act8, mlp_act8
    t = L.tops()
    x, r, w, b = _rand((6, 40), F32, 1), _rand((6, 40), F32, 2), _rand((40,), F32, 3), _rand((40,), F32, 4)
    wl = _rand((24, 40), F32, 5).requires_grad_()
    wb = _rand((40, 24), F32, 6)
    q, s = ops.act8_pack(x)
    mean, rstd = _rand((6,), F32, 7), _rand((6,), F32, 8)
    for grad in (False, True):
        with fwd.dual_level():
            def dual(v):
                return fwd.make_dual(v.detach().clone().requires_grad_(grad), torch.ones_like(v))
            for call in (lambda: ops.gelu_act8(dual(x)), lambda: ops.layer_norm_act8(dual(x), w, b),
                         lambda: ops.layer_norm_act8(x, dual(w), b), lambda: ops.layer_norm_act8(x, w, dual(b)),
                         lambda: ops.add_layer_norm_act8(dual(x), r, w, b),
                         lambda: ops.add_layer_norm_act8(x, dual(r), w, b),
                         lambda: ops.act8_wgrad(dual(x), q, s, 40, F32), lambda: t.act8_gelu_bwd(dual(x), q, s),
                         lambda: t.act8_layer_norm_bwd(dual(x), None, q, s, w, mean, rstd),
                         lambda: t.act8_layer_norm_bwd(x, dual(r), q, s, w, mean, rstd),
                         lambda: linear_act8(dual(x), wl), lambda: mlp_act8(dual(x), wl, None, wb, None)):
                with pytest.raises(RuntimeError, match="forward-mode|forward mode|jvp"):
                    call()
    # a tangent of the gradient that arrives
    y = ops.gelu_act8(x.clone().requires_grad_())
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        y.backward(fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_linears_of_no_inputs_or_outputs(dtype):
    """What F.linear gives, gradients too."""
    import torch.nn.functional as F
    from visionseg.linear import linear_act8, mlp_act8

    def plain_mlp(x, w1, b1, w2, b2):
        return F.linear(F.gelu(F.linear(x, w1, b1)), w2, b2)

    def compare(fn, plain, shapes):
        ts = [_rand(s, dtype, k).requires_grad_() for k, s in enumerate(shapes)]
        got, want = fn(*ts), plain(*ts)
        assert got.shape == want.shape and torch.equal(got, want)
        for a, b in zip(torch.autograd.grad(got.sum(), ts, allow_unused=True),
                        torch.autograd.grad(want.sum(), ts, allow_unused=True)):
            assert (a is None) == (b is None) and (a is None or (a.shape == b.shape and torch.equal(a, b)))

    for T, K, N in ((0, 40, 24), (5, 0, 24), (5, 40, 0), (0, 0, 3), (0, 3, 0)):
        compare(linear_act8, F.linear, ((T, K), (N, K), (N,)))
    for T, C, H, O in ((0, 40, 24, 8), (5, 0, 24, 8), (5, 40, 0, 8), (5, 40, 24, 0)):
        compare(mlp_act8, plain_mlp, ((T, C), (H, C), (H,), (O, H), (O,)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_kernel_timer_books_what_is_moved(dtype):
    """bench's kernel table: every op's forward and backward is timed, with its algorithmic bytes."""
    from visionseg import ops
    from visionseg.linear import mlp_act8
    from visionseg.profiling import KernelTimer
    T, C, N, e = 70, 40, 24, dtype.itemsize
    n, ck = T * C, T * (64 + 2)
    x, r = _rand((T, C), dtype, 1).requires_grad_(), _rand((T, C), dtype, 2).requires_grad_()
    w, b = _rand((C,), dtype, 3).requires_grad_(), _rand((C,), dtype, 4)
    gy = _rand((T, N), dtype, 5)
    w1, w2 = _rand((N, C), dtype, 6).requires_grad_(), _rand((C, N), dtype, 7).requires_grad_()
    with KernelTimer() as t:
        q, s = ops.act8_pack(x.detach())
        ops.act8_unpack(q, s, C, dtype)
        ops.act8_wgrad(gy, q, s, C, F32, bias=True)
        ops.gelu_act8(x).sum().backward()
        ops.layer_norm_act8(x, w, b).sum().backward()
        ops.add_layer_norm_act8(x, r, w, b)[1].sum().backward()
    with KernelTimer() as m:
        mlp_act8(x, w1, None, w2, None).sum().backward()
    with torch.no_grad(), KernelTimer() as f:
        ops.gelu_act8(x)
    ops.gelu_act8(x).sum().backward()                        # no timer: nothing is booked
    torch.cuda.synchronize()
    want = {"act8_pack": n * e + ck, "act8_unpack": n * e + ck, "act8_wgrad": T * N * e + ck + N * C * 4,
            "gelu_act8": 2 * n * e + ck, "gelu_act8_bwd": 2 * n * e + ck,
            "layer_norm_act8": 2 * n * e + ck, "layer_norm_act8_bwd": 2 * n * e + ck,
            "add_layer_norm_act8": 4 * n * e + ck, "add_layer_norm_act8_bwd": 3 * n * e + ck}
    got = t.summary()
    assert {k: v["bytes"] for k, v in got.items()} == want
    assert all(v["launches"] == 1 and v["total_ms"] > 0 for v in got.values())
    assert got["act8_wgrad"]["flops"] == 2 * T * N * C
    hk = T * (32 + 1)
    got = m.summary()
    assert got["act8_gelu_fwd"]["bytes"] == 2 * T * N * e + hk and got["act8_gelu_bwd"]["bytes"] == 3 * T * N * e + hk
    assert {k: v["bytes"] for k, v in f.summary().items()} == {"gelu_act8": 2 * n * e}


def test_backbone_under_autocast():
    """M2FConfig.act8 under autocast: the norms are the plain ones, the qkv projections and MLPs keep
    8 bits (test_gpu_act8.test_swin_backbone has the bounds of the types without it)."""
    from visionseg.model import M2FConfig, SwinBackbone
    px = _rand((1, 3, 224, 256), F32, 1)
    out = {}
    for act8 in (False, True):
        torch.manual_seed(0)
        net = SwinBackbone(M2FConfig(embed_dim=96, depths=(2, 2), num_heads=(3, 6), window_size=7, act8=act8)).to(DEV)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        with torch.autocast("cuda", torch.bfloat16):
            feats = net(px)
        kept = torch.cuda.memory_allocated() - base
        grads = torch.autograd.grad(feats, list(net.parameters()), [_rand(f.shape, f.dtype, i) for i, f in enumerate(feats)])
        out[act8] = (feats, grads, kept)
    for a, c in zip(out[True][0], out[False][0]):
        assert a.dtype == c.dtype
        a, c = a.detach().double(), c.detach().double()
        assert float((a - c).norm() / c.norm()) < 2e-2
    for a, c in zip(out[True][1], out[False][1]):
        assert a.dtype == c.dtype == F32
        assert float((a.double() - c.double()).norm()) <= 0.05 * float(c.double().norm()) + 1e-12
    assert out[True][2] < out[False][2]


@pytest.mark.parametrize("T", [50, 5000])
def test_parameters_that_do_not_belong(T):
    """A bias of another size or device, a weight of another device: what F.linear says to them (at
    5000 tokens the token GEMM would read the bias itself)."""
    import torch.nn.functional as F
    from visionseg import ops
    from visionseg.linear import linear_act8, linear_tokens, mlp_act8
    x, w, b = _rand((T, 96), BF16, 1), _rand((288, 96), BF16, 2).requires_grad_(), _rand((288,), BF16, 3)
    w2, b2 = _rand((96, 288), BF16, 4), _rand((96,), BF16, 5)
    for wrong in (b[:7], b.cpu(), b.view(1, 288)[:, :5]):
        with pytest.raises(RuntimeError):
            F.linear(x, w, wrong)
        for call in (lambda: linear_act8(x, w, wrong), lambda: mlp_act8(x, w, wrong, w2, b2),
                     lambda: linear_tokens(x, w, wrong)):
            with pytest.raises((RuntimeError, ValueError)):
                call()
        with pytest.raises((RuntimeError, ValueError)):
            ops.token_gemm(x, w.detach(), wrong)
    with pytest.raises(RuntimeError):
        linear_act8(x, w.detach().cpu().requires_grad_(), b)
    one = b[:1]                                              # one value for every output, as F.linear takes it
    assert torch.equal(linear_act8(x, w, one), F.linear(x, w, one))


@pytest.mark.parametrize("T", [300, 5000])
@pytest.mark.parametrize("how", ["recomputed", "offloaded"])
def test_saved_tensors_elsewhere(how, T):
    """A block under torch's own activation checkpointing or offloading: the same results."""
    from torch.utils.checkpoint import checkpoint
    from visionseg import ops
    from visionseg.linear import linear_act8, mlp_act8
    C, H = 96, 384
    ts = [_rand(s, BF16, k, 1.0 if k < 2 else 0.1).requires_grad_() for k, s in enumerate(
        ((T, C), (T, C), (C,), (C,), (C, C), (C,), (H, C), (H,), (C, H), (C,)))]

    def block(x, r, w, b, wq, bq, w1, b1, w2, b2):
        s, y = ops.add_layer_norm_act8(x, r, w, b)
        y = ops.gelu_act8(linear_act8(y, wq, bq))
        return s + mlp_act8(ops.layer_norm_act8(y, w, b), w1, b1, w2, b2)

    gy = _rand((T, C), BF16, 20)
    want = block(*ts)
    grads = torch.autograd.grad(want, ts, gy)
    if how == "recomputed":
        got = checkpoint(block, *ts, use_reentrant=False)
        again = torch.autograd.grad(got, ts, gy)
    else:
        with torch.autograd.graph.save_on_cpu():
            got = block(*ts)
        again = torch.autograd.grad(got, ts, gy)
    assert torch.equal(got, want) and all(torch.equal(a, b) for a, b in zip(again, grads))
