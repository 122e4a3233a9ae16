"""8-bit dense layers (ops/int8.py, FullyConnectedLayer.quantize_int8_) on CPU: definition, refusals, the serving rule of the layer; argument checks of the C entry point."""
import copy
import ctypes

import pytest
import torch

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import amax, int8
from stylegan_v_amd.training.layers import FullyConnectedLayer, MappingNetwork, normalize_2nd_moment


def _rows(m, k, seed):
    return torch.randint(-128, 128, [m, k], generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def test_definition():
    a, b = _rows(3, 21, 1), _rows(5, 21, 2)
    sa, sb, bias = torch.rand(3) + 0.5, torch.rand(5) + 0.5, torch.randn(5)
    want = (a.long() @ b.long().t()).double() * sa.double()[:, None] * sb.double() + bias.double()
    assert torch.equal(int8.matmul(a, sa, b, sb, bias=bias, act='linear'), want.float())
    got = int8.matmul(a, sa, b, sb, bias=bias, act='lrelu', act_gain=2.0)
    assert torch.allclose(got.double(), 2 * torch.maximum(want, want * 0.2), rtol=1e-6)
    got = int8.matmul(a.view(1, 3, 21), sa.view(1, 3), b, sb, dtype=torch.bfloat16)
    assert got.shape == (1, 3, 5) and got.dtype == torch.bfloat16
    assert int8.matmul(a[:0], sa[:0], b, sb).shape == (0, 5) and int8.matmul(a, sa, b[:0], sb[:0]).shape == (3, 0)


def test_refusals():
    a, b, sa, sb = _rows(3, 8, 1), _rows(5, 8, 2), torch.ones(3), torch.ones(5)
    bad = [(a.float(), sa, b, sb, {}), (a, sa, b.float(), sb, {}), (a, torch.ones(4), b, sb, {}), (a, sa.double(), b, sb, {}), (a, sa, b, torch.ones(3), {}), (a, sa, b[:, :7], sb, {}),
           (a, sa, b.view(1, 5, 8), sb.view(1, 5), {}), (a, sa, b, sb, dict(dtype=torch.float64)), (a, sa, b, sb, dict(act='relu')), (a, sa, b, sb, dict(bias=torch.ones(4))),
           (a, sa, b, sb, dict(bias=torch.ones(5, dtype=torch.float16))), (a[:, :0], sa, b[:, :0], sb, {}), (a, sa, b, sb.clone().requires_grad_(True), {})]
    for x, s, w, ws, kw in bad:
        with pytest.raises(RuntimeError):
            int8.matmul(x, s, w, ws, **kw)
    long = torch.zeros([1, int8.max_inner + 1], dtype=torch.int8)
    with pytest.raises(RuntimeError, match='131071'):
        int8.matmul(long, torch.ones(1), long, torch.ones(1))
    for q, s, kw in ((a.float(), sa, {}), (a, sb, {}), (a, sa, dict(dtype=torch.float64))):
        with pytest.raises(RuntimeError):
            int8.dequantize_rows(q, s, **kw)


def test_layer_serves_in_8_bits_without_gradients_only():
    torch.manual_seed(0)
    layer = FullyConnectedLayer(24, 10, activation='lrelu', lr_multiplier=0.01, bias_init=1)
    keys = set(layer.state_dict())
    x = torch.randn([6, 24])
    with torch.no_grad():
        want = layer(x)
        assert layer.quantize_int8_() is layer and set(layer.state_dict()) == keys
        got = layer(x)
    # q of either operand is off by at most half a step: |dy| <= gain * sum_k (|dx w| + |x dw| + |dx dw|), dx <= sx / 2, dw <= sw / 2
    w = layer.weight.detach() * layer.weight_gain
    sx, sw = x.abs().amax(dim=1) / 127, w.abs().amax(dim=1) / 127
    bound = 2 ** 0.5 * (sx[:, None] / 2 * w.abs().sum(dim=1) + x.abs().sum(dim=1, keepdim=True) * sw / 2 + 24 * sx[:, None] * sw / 4)
    assert (got - want).abs().le(bound + 1e-6).all() and not torch.equal(got, want)
    assert torch.equal(layer(x), want) and layer(x).requires_grad                       # gradients enabled: the fp32 layer
    with torch.no_grad():
        assert torch.allclose(layer(x, gain=3.0), got * 3.0, rtol=1e-6)
        assert layer(x.view(2, 3, 24)).shape == (2, 3, 10)
        twin = copy.deepcopy(layer)                       # a copy has parameters of its own
        with pytest.raises(RuntimeError, match='quantise it again'):
            twin(x)
        assert torch.equal(twin.quantize_int8_()(x), got)
        volume = torch.randn([2, 24, 24])                 # the input norm runs over dimension 1, with three dimensions too
        assert torch.equal(layer(volume, normalize_input=True), layer(normalize_2nd_moment(volume)))
        layer.weight.add_(0.1)
        with pytest.raises(RuntimeError, match='quantise it again'):
            layer(x)
        layer.quantize_int8_()(x)
        layer.quantize_int8_()
        amax.graph_replayed()                             # a replayed graph may have written the parameters behind their version counters
        with pytest.raises(RuntimeError, match='quantise it again'):
            layer(x)
        layer.quantize_int8_()
        layer.weight.data = layer.weight.data * 2         # (a new tensor behind the parameter leaves its version as it was)
        with pytest.raises(RuntimeError, match='quantise it again'):
            layer(x)
        layer.quantize_int8_().half().float()             # (... and so does a round trip through another type)
        with pytest.raises(RuntimeError, match='quantise it again'):
            layer(x)
        old = copy.deepcopy(layer)
        old.__dict__.pop('_int8', None)                   # a layer from before it had an 8-bit form
        assert old(x).shape == (6, 10)
        assert layer.quantize_int8_().bfloat16()._int8 is not None
        with pytest.raises(RuntimeError, match='quantise it again'):
            layer(x)
    with pytest.raises(RuntimeError, match='tanh'):
        FullyConnectedLayer(4, 4, activation='tanh').quantize_int8_()


def test_mapping_network_in_8_bits():
    torch.manual_seed(1)
    net = MappingNetwork(z_dim=32, c_dim=3, w_dim=32, num_ws=4, num_layers=2).eval()
    z, c = torch.randn([16, 32]), torch.randn([16, 3])
    with torch.no_grad():
        want = net(z, c)
        got = net.quantize_int8_()(z, c)
    assert got.shape == want.shape
    # three layers, each with two operands off by up to half a step of 1/127 of a row's maximum: ~ 3 * sqrt(2) * (max / rms ~ 3) * 1/127/sqrt(12) = 3 % of the result's size
    assert (got - want).norm() / want.norm() < 0.06


def test_training_goes_on_beside_a_served_average():
    """The averaged generator served in 8 bits inside a training process: the steps run, and the average refuses to serve numbers of an older state."""
    from stylegan_v_amd.training import config as cfgs, train_step
    g_kwargs, d_kwargs = cfgs.small_test_model_kwargs(res=32)
    cfg = cfgs.Config(r1_gamma=1.0, lr=0.0025, betas=(0.0, 0.99), ema_kimg=1.0, ema_rampup=0.05, G_reg_interval=4, D_reg_interval=16, pl_weight=0.0)
    ts = train_step.TrainStep(g_kwargs, d_kwargs, cfg, device='cpu', batch_gpu=2)
    z, c, keys = torch.randn([2, 32]), torch.zeros([2, 0]), set(ts.G_ema.state_dict())
    with torch.no_grad():
        ts.G_ema.mapping.quantize_int8_()(z, c)
    ts.step()
    assert set(ts.G_ema.state_dict()) == keys
    with torch.no_grad():
        with pytest.raises(RuntimeError, match='quantise it again'):
            ts.G_ema.mapping(z, c)
        ts.G_ema.mapping.quantize_int8_()(z, c)


def test_argument_checks_of_the_c_entry_without_gpu():
    lib = custom_ops.get_native()
    F32 = custom_ops.SGV_F32
    buf = (ctypes.c_float * 256)()
    addr = (ctypes.addressof(buf) + 15) // 16 * 16
    p = custom_ops.Int8GemmParams()
    assert lib.sgv_int8_gemm(p, F32, None) == -1
    p.m, p.n, p.k = 1, 1, 131072
    assert lib.sgv_int8_gemm(p, F32, None) == -2
    p.k, p.act = 32, 2
    assert lib.sgv_int8_gemm(p, F32, None) == -1 and b'act' in lib.sgv_last_error()
    p.act = 1
    assert lib.sgv_int8_gemm(p, F32, None) == -1 and b'NULL' in lib.sgv_last_error()
    p.a, p.b, p.a_scale, p.b_scale, p.c, p.lda, p.ldb, p.ldc = addr, addr + 1, addr, addr, addr, 32, 32, 1
    assert lib.sgv_int8_gemm(p, F32, None) == -1 and b'16 bytes' in lib.sgv_last_error()
    p.b, p.lda = addr, 24
    assert lib.sgv_int8_gemm(p, F32, None) == -1
    p.lda, p.ldc = 32, 0
    assert lib.sgv_int8_gemm(p, F32, None) == -1 and b'overlap' in lib.sgv_last_error()
    p.ldc, p.lda = 1, 1 << 23
    assert lib.sgv_int8_gemm(p, F32, None) == -2 and b'apart' in lib.sgv_last_error()
    p.lda = 32
    assert lib.sgv_int8_gemm(p, custom_ops.SGV_F64, None) == -3
    p.m = 0
    assert lib.sgv_int8_gemm(p, F32, None) == 0
    assert ctypes.sizeof(custom_ops.Int8GemmParams) == 96
