"""Row norm and 8-bit product on the GPU while torch records a graph of operations (torch.jit.trace, make_fx): a launch does not show in such a graph.

`rms_norm` leaves its formula there; the 8-bit operators and the layers that serve with them refuse."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn
from stylegan_v_amd.training.layers import FullyConnectedLayer, MappingNetwork

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def _recorders():
    return (lambda f, *x: torch.jit.trace(f, x, check_trace=False), lambda f, *x: make_fx(f)(*x))


@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
@pytest.mark.parametrize('grad', [False, True])
@pytest.mark.parametrize('recorder', [0, 1])
def test_a_recorded_norm_computes(recorder, grad):
    w, r = _rand(40, seed=2), _rand(6, 40, seed=3)
    w.requires_grad_(grad)
    x, other = _rand(6, 40, seed=1), _rand(6, 40, seed=4)
    with torch.set_grad_enabled(grad):
        graph = _recorders()[recorder](lambda a, b: rn.rms_norm(a, b, r, 1e-6), x, w)        # (an input: a trace holds no constant that requires gradients)
        want = rn.rms_norm(other, w, r, 1e-6)
        for _ in range(2):
            got = graph(other, w)
            assert torch.equal(got[1], want[1])
            assert ((got[0] - want[0]).abs() <= 100 * U * want[0].abs()).all()       # two forms of the same fp32 value: 44 U each
        one = _recorders()[recorder](lambda a: rn.rms_norm(a), x)(other)
    assert (one - rn.rms_norm(other)).abs().max() <= 100 * U * one.abs().max()


@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
@pytest.mark.parametrize('recorder', [0, 1])
def test_8_bit_operators_are_not_recorded(recorder):
    x, q, s = _rand(4, 64, seed=1), torch.ones([5, 64], dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    a, sa = torch.ones([4, 64], dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    layer, net = FullyConnectedLayer(64, 8).to(DEV), MappingNetwork(z_dim=64, c_dim=0, w_dim=64, num_ws=2, num_layers=2).to(DEV).eval()
    with torch.no_grad():
        layer.quantize_int8_()
        net.quantize_int8_()
        served = layer(x)
        for call in (lambda t: rn.rms_norm_int8(t)[1], lambda t: int8.quantize_rows(t)[1], lambda t: int8.dequantize_rows(a, sa + t[:, 0]), lambda t: int8.matmul(a, sa + t[:, 0], q, s),
                     lambda t: int8.dense(t, q, s), lambda t: layer(t), lambda t: net(t, t[:, :0])):
            with pytest.raises(RuntimeError, match='trace'):
                _recorders()[recorder](call, x)
        assert torch.equal(layer(x), served)           # and serves on
