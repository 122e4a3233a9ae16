"""Row norm and its 8-bit output (ops/rms_norm.py) on CPU: the definition, its gradient against differences, refusals; and the argument checks of the C entry points."""
import ctypes

import pytest
import torch

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn


def _rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def test_definition_and_gradient_by_differences():
    x, r, w = _rand(3, 7, seed=1).requires_grad_(True), _rand(3, 7, seed=2).requires_grad_(True), _rand(7, seed=3).requires_grad_(True)
    y, h = rn.rms_norm(x, w, r, eps=0.1)
    assert torch.equal(h, x + r)
    assert torch.allclose(y, (x + r) / ((x + r).square().mean(dim=1, keepdim=True) + 0.1).sqrt() * w, rtol=1e-12)
    assert torch.autograd.gradcheck(lambda *a: rn.rms_norm(*a, eps=0.1), (x, w, r))
    assert torch.autograd.gradcheck(lambda a: rn.rms_norm(a), (x,))


def test_the_torch_side_is_built_and_takes_no_cpu_tensors():
    ops = custom_ops.get_row_ops()
    x, q = torch.zeros([2, 16]), torch.zeros([2, 16], dtype=torch.int8)
    for call in (lambda: ops.rms_norm(x, None, None, 1e-8), lambda: ops.rms_norm_int8(x, None, None, 1e-8, True), lambda: ops.dequantize_rows(q, x[:, 0], 0),
                 lambda: ops.matmul(q, x[:, 0], q, x[:, 0], None, 1, 0.0, 1.0, 0), lambda: ops.dense(x, q, x[:, 0], None, 1, 0.0, 1.0, False, 1e-8)):
        with pytest.raises(ops.Refused):
            call()
    assert issubclass(ops.Refused, RuntimeError)


def test_int8_output_on_cpu():
    x = torch.tensor([[1.0, -2.0, 0.5, 0.25], [0.0, 0.0, 0.0, 0.0], [1.0, float('nan'), 0.0, 0.0], [1.0, float('inf'), 0.0, 0.0], [254.0, 1.0, 3.0, -5.0]])
    q, s = int8.quantize_rows(x)
    assert q.tolist()[0] == [64, -127, 32, 16] and q.tolist()[1] == [0, 0, 0, 0] and q.tolist()[2] == [0, 0, 0, 0] and q.tolist()[3] == [0, 0, 0, 0]
    assert q.tolist()[4] == [127, 0, 2, -2]             # 0.5, 1.5, -2.5: halves go to the even neighbour
    assert s[0] == torch.tensor(2.0 / 127) and s[1] == 0 and s[2].isnan() and s[3].isnan()
    x = _rand(6, 40, seed=5, dtype=torch.float32)
    r, w = _rand(6, 40, seed=6, dtype=torch.float32), _rand(40, seed=7, dtype=torch.float32)
    q, s, h = rn.rms_norm_int8(x, w, r)
    y, h2 = rn.rms_norm(x, w, r)
    assert torch.equal(h, h2) and q.dtype == torch.int8 and s.shape == (6,)
    back = int8.dequantize_rows(q, s)
    assert (back - y).abs().amax(dim=1).le(s * 0.5001).all()             # half a step


@pytest.mark.parametrize('shape', [(0, 8), (2, 0, 8), (8,), (2, 3, 8)])
def test_shapes(shape):
    x = _rand(*shape, dtype=torch.float32)
    y, h = rn.rms_norm(x, residual=x)
    q, s = rn.rms_norm_int8(x)
    assert y.shape == h.shape == q.shape == x.shape and s.shape == x.shape[:-1]


def test_refusals():
    x = torch.zeros([2, 8])
    for bad in (torch.zeros([2, 0]), torch.zeros([]), torch.zeros([2, 8], dtype=torch.int32), torch.zeros([2, 8], dtype=torch.complex64)):
        with pytest.raises(RuntimeError):
            rn.rms_norm(bad)
    for w in (torch.zeros([7]), torch.zeros([1, 8]), torch.zeros([8], dtype=torch.float16)):
        with pytest.raises(RuntimeError, match='weight'):
            rn.rms_norm(x, weight=w)
    for r in (torch.zeros([8]), torch.zeros([2, 8], dtype=torch.float16)):
        with pytest.raises(RuntimeError, match='residual'):
            rn.rms_norm(x, residual=r)
    for eps in (-1e-3, float('nan')):
        with pytest.raises(RuntimeError, match='eps'):
            rn.rms_norm(x, eps=eps)
    xg = torch.zeros([2, 8], requires_grad=True)
    with pytest.raises(RuntimeError, match='no gradient'):
        rn.rms_norm_int8(xg)
    with pytest.raises(RuntimeError, match='no gradient'):
        int8.quantize_rows(xg)
    with torch.no_grad():
        rn.rms_norm_int8(xg)
        int8.quantize_rows(xg)


def test_argument_checks_of_the_c_entries_without_gpu():
    lib = custom_ops.get_native()
    F32 = custom_ops.SGV_F32
    buf = (ctypes.c_float * 256)()
    addr = (ctypes.addressof(buf) + 15) // 16 * 16
    p = custom_ops.RmsNormParams()
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'cols' in lib.sgv_last_error()
    p.rows, p.cols, p.normalize = 1, 8, 1
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'NULL' in lib.sgv_last_error()
    p.x = p.y = p.q = p.q_scale = addr
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'one output' in lib.sgv_last_error()
    p.y, p.q_stride = None, 8
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'16' in lib.sgv_last_error()
    p.q, p.q_stride = addr + 4, 16
    assert lib.sgv_rms_norm(p, F32, None) == -1
    p.q, p.residual = addr, addr
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'residual' in lib.sgv_last_error()
    p.residual, p.eps = None, -1.0
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'eps' in lib.sgv_last_error()
    p.eps = 0.0
    assert lib.sgv_rms_norm(p, custom_ops.SGV_F64, None) == -3
    p.cols = 1 << 26
    assert lib.sgv_rms_norm(p, F32, None) == -2
    p.rows, p.cols = 0, 8
    assert lib.sgv_rms_norm(p, F32, None) == 0                          # nothing to do
    q, p.y, p.normalize = p.q, addr, 0
    p.q, p.rows = None, 1
    assert lib.sgv_rms_norm(p, F32, None) == -1 and b'8-bit' in lib.sgv_last_error()
    b = custom_ops.RmsNormBackwardParams()
    assert lib.sgv_rms_norm_backward(b, F32, None) == -1
    b.rows, b.cols, b.dy, b.h, b.inv_rms, b.dweight = 4, 8, addr, addr, addr, addr
    assert lib.sgv_rms_norm_backward(b, F32, None) == -1 and b'no weight' in lib.sgv_last_error()
    b.weight = addr
    assert lib.sgv_rms_norm_backward(b, F32, None) == -1 and b'workspace' in lib.sgv_last_error()
    assert lib.sgv_rms_norm_backward_workspace_bytes(4, 8, F32) == 32 and lib.sgv_rms_norm_backward_workspace_bytes(4, 8, custom_ops.SGV_F64) == 0
    assert lib.sgv_dequantize_rows(None, 8, None, None, 1, 8, F32, None) == -1
    assert lib.sgv_dequantize_rows(addr, 8, addr, addr, 1, 8, custom_ops.SGV_F64, None) == -3
    assert ctypes.sizeof(custom_ops.RmsNormParams) == 112 and ctypes.sizeof(custom_ops.RmsNormBackwardParams) == 112
