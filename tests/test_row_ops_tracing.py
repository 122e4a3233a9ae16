"""The torch side of the row operators while torch records a graph of operations: it tells so, whatever the tensors' device.  (On the CPU the operators themselves are torch operations.)"""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn


class _Passing(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def test_the_torch_side_tells_that_a_graph_is_recorded():
    ops = custom_ops.get_row_ops()
    x, q, s = torch.ones([2, 16]), torch.ones([2, 16], dtype=torch.int8), torch.ones(2)
    for call in (lambda t: ops.rms_norm(t, None, None, 1e-8), lambda t: ops.rms_norm_int8(t, None, None, 1e-8, True), lambda t: ops.dequantize_rows(q, t[:, 0], 0),
                 lambda t: ops.matmul(q, t[:, 0], q, s, None, 1, 0.0, 1.0, 0), lambda t: ops.dense(t, q, s, None, 1, 0.0, 1.0, False, 1e-8)):
        with pytest.raises(ops.Watched, match='trace'):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(ops.Watched, match='trace'):
            make_fx(call)(x)
        with _Passing(), pytest.raises(ops.Refused) as plain:         # a mode that records nothing
            call(x)
        assert not isinstance(plain.value, ops.Watched)


@pytest.mark.filterwarnings('ignore::torch.jit.TracerWarning')
def test_traces_on_the_cpu():
    x, other, w = torch.randn([4, 16]), torch.randn([4, 16]), torch.randn(16)
    q, s = int8.quantize_rows(torch.randn([8, 16]))
    for call in (lambda t: rn.rms_norm(t, w), lambda t: int8.dense(t, q, s, act='lrelu')):
        assert torch.equal(torch.jit.trace(call, (x,), check_trace=False)(other), call(other))
