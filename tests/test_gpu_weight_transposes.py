"""GPU tests of the token Linears' batched weight transposes (linear._WT) where forwards and backwards
of several streams and captures are open at once."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16 = torch.bfloat16
T, C, H = 5000, 96, 288                    # sizes whose input gradients run on the token GEMM


def _rand(shape, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(BF16)


def _kinds():
    from visionseg.linear import linear_act8, linear_tokens, mlp_act8
    one = ((T, C), (H, C), (H,))
    return {"linear_tokens": (linear_tokens, one), "linear_act8": (linear_act8, one),
            "mlp_act8": (mlp_act8, one + ((C, H), (C,)))}


def _leaves(shapes, seed):
    return [_rand(s, seed + k, 1.0 if k == 0 else 0.1).requires_grad_() for k, s in enumerate(shapes)]


def _grads(y, ts, seed):
    return torch.autograd.grad(y, ts, _rand(y.shape, seed))


def test_capture_ids():
    from visionseg import _lib as L
    lib = L.lib()
    side = torch.cuda.Stream()

    def here():
        return lib.vs_stream_capture_id(torch.cuda.current_stream().cuda_stream)

    ids = []
    x = torch.zeros(4, device=DEV)
    assert here() == 0 and lib.vs_stream_capture_id(side.cuda_stream) == 0
    for _ in range(2):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            a = here()
            x.add_(1)
            ids += [a, here()]
        assert here() == 0 and lib.vs_stream_capture_id(side.cuda_stream) == 0
    assert ids[0] == ids[1] != 0 and ids[2] == ids[3] != 0 and ids[0] != ids[2]


@pytest.mark.parametrize("kind", ["linear_tokens", "linear_act8", "mlp_act8"])
def test_two_streams_open_at_once(kind):
    """Forwards on two streams, then both backwards: the first backward leaves the other stream's
    weights to that stream."""
    from visionseg import linear
    fn, shapes = _kinds()[kind]
    sets = [_leaves(shapes, 10 * k) for k in range(2)]
    want = [_grads(fn(*ts), ts, 7) for ts in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        ys, got = [], []
        for s, ts in zip(streams, sets):
            with torch.cuda.stream(s):
                ys.append(fn(*ts))
        open_before = len(linear._WT.pending)
        for s, ts, y in zip(streams, sets, ys):
            with torch.cuda.stream(s):
                got.append(_grads(y, ts, 7))
            assert len(linear._WT.pending) < open_before
            open_before = len(linear._WT.pending)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("same_stream", [False, True])
@pytest.mark.parametrize("kind", ["linear_tokens", "linear_act8", "mlp_act8"])
def test_an_open_eager_forward_beside_a_capture(kind, same_stream):
    """An eager forward waits for its backward while a step on other tensors is captured; the captured
    launch is not run then, and at replays must not touch what the eager one has freed."""
    fn, shapes = _kinds()[kind]
    eager, caught = _leaves(shapes, 0), _leaves(shapes, 20)
    want_eager = _grads(fn(*eager), eager, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = _grads(fn(*caught), caught, 8)                # (warms up the capture stream too)
        if same_stream:
            y = fn(*eager)
    if not same_stream:
        y = fn(*eager)
    torch.cuda.synchronize()
    gy = _rand(y.shape, 8)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        yc = fn(*caught)
        got = torch.autograd.grad(yc, caught, gy)
    back = _grads(y, eager, 7)                               # (on the stream of its forward)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(back, want_eager))
    del y, back
    for _ in range(3):
        fresh = [torch.full_like(t, 3.0) for t in eager]     # memory that the eager step has given back
        for t in got:
            t.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        assert all(bool((t == 3.0).all()) for t in fresh)
