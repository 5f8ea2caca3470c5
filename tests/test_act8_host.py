"""8-bit activation checkpoints without a GPU: the reference of the GPU tests against the format's
definition, the C entry points' refusals (made before any HIP call), the Python ops' refusals and
the configuration switch."""
import ctypes

import pytest
import torch

import _act8ref as ref
from visionseg import _lib as L

P16 = ctypes.c_void_p(16)
NULL = ctypes.c_void_p(0)


def test_reference_matches_the_definition():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(40, 70, generator=g) * torch.exp(4 * torch.randn(40, 1, generator=g))
    x[0] = 0
    x[1] = 127 * 2.0 ** -3                           # exactly 127 steps
    x[2] = torch.nextafter(torch.tensor(127 * 2.0 ** -3), torch.tensor(1e9)).item()
    x[3] *= 1e-42
    x[4] = 127 * 2.0 ** 121
    x[7] = torch.nextafter(torch.tensor(127 * 2.0 ** 121), torch.tensor(float("inf"))).item()
    x[5, 3], x[6, 40] = float("inf"), float("nan")
    q, s = ref.pack(x)
    for r in range(40):
        for b in range(3):
            blk = x[r, 32 * b:32 * b + 32].double()
            if not bool((blk.abs() <= 127 * 2.0 ** 121).all()):
                assert s[r, b] == 255 and not bool(q[r, 32 * b:32 * b + 32].any())
                continue
            a, e = float(blk.abs().max()), int(s[r, b]) - 127
            assert a <= 127 * 2.0 ** e and (e == -126 or a > 127 * 2.0 ** (e - 1))
            want = [round(float(v) / 2.0 ** e) for v in blk]          # ties to even
            assert q[r, 32 * b:32 * b + len(want)].tolist() == want
    assert not bool(q[:, 70:].any())
    v = ref.values(q, s, 70)
    fin = (x.abs() <= 127 * 2.0 ** 121).all(1)
    assert float((v - x.double())[fin].abs().max() / 3.4e38) <= 1 / 127
    assert bool((v[fin].to(torch.bfloat16).double() == v[fin]).all())     # exact in bf16


def test_c_entry_points_refuse():
    lib = L.lib()

    def refused(rc, msg):
        assert rc == -1, rc
        assert msg in lib.vs_last_error(), lib.vs_last_error()

    refused(lib.vs_act8_pack(2, P16, 8, P16, P16, 4, 8, None), b"dtype")
    refused(lib.vs_act8_pack(0, P16, 8, P16, P16, -1, 8, None), b"rows")
    refused(lib.vs_act8_pack(0, P16, 8, P16, P16, 4, -8, None), b"features")
    refused(lib.vs_act8_pack(0, P16, -8, P16, P16, 4, 8, None), b"stride")
    refused(lib.vs_act8_pack(0, NULL, 8, P16, P16, 4, 8, None), b"null")
    refused(lib.vs_act8_pack(0, P16, 8, ctypes.c_void_p(20), P16, 4, 8, None), b"aligned")
    refused(lib.vs_act8_pack(0, P16, 1 << 30, P16, P16, 1 << 30, 1 << 30, None), b"too large")
    refused(lib.vs_act8_unpack(1, P16, NULL, P16, 4, 8, None), b"null")
    refused(lib.vs_act8_unpack(7, P16, P16, P16, 4, 8, None), b"dtype")
    refused(lib.vs_act8_gelu_forward(1, P16, P16, P16, NULL, 4, 8, None), b"both or neither")
    refused(lib.vs_act8_gelu_backward(1, NULL, P16, P16, P16, P16, 4, 8, None), b"null")
    refused(lib.vs_act8_layer_norm_forward(1, P16, P16, P16, P16, NULL, P16, P16, P16, P16, P16, 4, 8, 1e-5, None, 0,
                                           None), b"both or neither")
    refused(lib.vs_act8_layer_norm_forward(1, P16, None, P16, P16, None, P16, P16, P16, P16, P16, 4, 8193, 1e-5, None,
                                           0, None), b"8192")
    refused(lib.vs_act8_layer_norm_forward(1, P16, None, P16, P16, None, P16, P16, P16, P16, P16, 4, 0, 1e-5, None,
                                           0, None), b"features")
    refused(lib.vs_act8_layer_norm_backward(1, P16, None, P16, P16, P16, P16, P16, P16, P16, P16, NULL, 4, 8, None, 0,
                                            None), b"null")
    refused(lib.vs_act8_wgrad(1, 3, P16, 8, P16, P16, P16, P16, P16, 4, 8, 8, None), b"dtypes")
    refused(lib.vs_act8_wgrad(1, 1, P16, 8, P16, P16, P16, P16, P16, -4, 8, 8, None), b"sizes")
    refused(lib.vs_act8_wgrad(1, 1, P16, 8, P16, P16, P16, P16, P16, 4, 8, 0, None), b"K > 0")
    refused(lib.vs_act8_wgrad(1, 1, P16, 8, ctypes.c_void_p(24), P16, P16, P16, P16, 4, 8, 8, None), b"aligned")
    refused(lib.vs_act8_wgrad(1, 1, NULL, 8, P16, P16, P16, P16, P16, 4, 8, 8, None), b"null")
    need = lib.vs_act8_wgrad_workspace_bytes(1, 65536, 64, 64)
    assert need > 0
    refused(lib.vs_act8_wgrad(1, 1, P16, 64, P16, P16, P16, P16, NULL, 65536, 64, 64, None), b"workspace")
    # nothing to do: no pointer is looked at
    assert lib.vs_act8_pack(0, NULL, 0, NULL, NULL, 0, 8, None) == 0
    assert lib.vs_act8_unpack(0, NULL, NULL, NULL, 8, 0, None) == 0
    assert lib.vs_act8_gelu_forward(0, NULL, NULL, NULL, NULL, 0, 8, None) == 0
    assert lib.vs_act8_layer_norm_backward_workspace_bytes(0, 64) > 0
    assert lib.vs_act8_layer_norm_backward_workspace_bytes(4, 0) == 0
    assert lib.vs_act8_wgrad_workspace_bytes(1, -1, 8, 8) == 0


def test_ops_refuse_cpu_tensors():
    from visionseg import ops
    x, w = torch.zeros(4, 32), torch.zeros(32)
    q, s = torch.zeros(4, 32, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8)
    for call in (lambda: ops.act8_pack(x), lambda: ops.act8_unpack(q, s, 32, torch.float32),
                 lambda: ops.act8_wgrad(x, q, s, 32, torch.float32), lambda: ops.gelu_act8(x),
                 lambda: ops.layer_norm_act8(x, w, w), lambda: ops.add_layer_norm_act8(x, x, w, w)):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


def test_linear_act8_on_the_cpu_is_the_plain_composition():
    from visionseg.linear import linear_act8, mlp_act8
    import torch.nn.functional as F
    g = torch.Generator().manual_seed(1)
    x, w1, w2 = (torch.randn(*s, generator=g, requires_grad=True) for s in ((5, 8), (16, 8), (8, 16)))
    b1 = torch.randn(16, generator=g)
    assert torch.equal(linear_act8(x, w1, b1), F.linear(x, w1, b1))
    assert torch.equal(mlp_act8(x, w1, b1, w2, None), F.linear(F.gelu(F.linear(x, w1, b1)), w2))


def test_config_switch():
    from visionseg.model import M2FConfig, SwinBackbone
    cfg = M2FConfig.preset("swin_t", act8=True)
    assert M2FConfig.from_dict(cfg.to_dict()).act8
    assert all(blk.act8 and blk.mlp.act8 for st in SwinBackbone(cfg).stages for blk in st.blocks)
    assert not any(blk.act8 or blk.mlp.act8 for st in SwinBackbone(M2FConfig()).stages for blk in st.blocks)
    with pytest.raises(ValueError, match="act8"):
        SwinBackbone(M2FConfig.preset("swin_t", act8=True, linear_fp8=True))


def test_wgrad_refuses_gradients_off_their_alignment():
    lib = L.lib()
    for dtype, address in ((0, 18), (1, 17)):                 # f32 on 2 B, bf16 on 1 B
        rc = lib.vs_act8_wgrad(dtype, 1, ctypes.c_void_p(address), 8, P16, P16, P16, P16, P16, 4, 8, 8, None)
        assert rc == -1 and b"aligned to its elements" in lib.vs_last_error()
