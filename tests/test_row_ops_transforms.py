"""Row norm and 8-bit operators on the CPU under derivatives of forward mode and function transforms: the norm follows them, the 8-bit operators have no gradient."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn


def _rand(*shape, seed=0, dtype=torch.float64):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype)


def test_forward_mode_of_the_norm():
    x, w, r = _rand(3, 7, seed=1), _rand(7, seed=2), _rand(3, 7, seed=3)
    tx, tw, tr = _rand(3, 7, seed=4), _rand(7, seed=5), _rand(3, 7, seed=6)
    (y, h), (ty, th) = torch.func.jvp(lambda *a: rn.rms_norm(*a, eps=0.1), (x, w, r), (tx, tw, tr))
    e = 1e-6
    up, down = [rn.rms_norm(x + s * e * tx, w + s * e * tw, r + s * e * tr, eps=0.1)[0] for s in (1, -1)]
    assert torch.allclose(ty, (up - down) / (2 * e), rtol=1e-7, atol=1e-8) and torch.allclose(th, tx + tr, rtol=1e-14)      # (differences: error e^2 + 1e-16 / e)
    assert torch.allclose(torch.func.vmap(lambda a: rn.rms_norm(a, w, eps=0.1))(x), rn.rms_norm(x, w, eps=0.1), rtol=1e-14)


def test_8_bit_operators_refuse_tangents():
    x, q, s = _rand(4, 16, dtype=torch.float32), torch.ones([4, 16], dtype=torch.int8), torch.ones(4)
    with fwd.dual_level(), torch.no_grad():
        d, ds = fwd.make_dual(x, x), fwd.make_dual(s, s)
        for call in (lambda: rn.rms_norm_int8(d), lambda: rn.rms_norm_int8(x, None, d), lambda: int8.quantize_rows(d), lambda: int8.dequantize_rows(q, ds), lambda: int8.matmul(q, ds, q, s),
                     lambda: int8.matmul(q, s, q, ds), lambda: int8.matmul(q, s, q, s, bias=ds), lambda: int8.dense(d, q, s), lambda: int8.dense(x, q, ds)):
            with pytest.raises(RuntimeError, match='no gradient'):
                call()
        int8.dense(d.detach(), q, s)


def test_the_torch_side_tells_what_follows_a_tensor():
    ops = custom_ops.get_row_ops()
    x, q, s = torch.ones([2, 16]), torch.ones([2, 16], dtype=torch.int8), torch.ones(2)
    assert issubclass(ops.Watched, ops.Refused)
    calls = (lambda t: ops.rms_norm(t, None, None, 1e-8), lambda t: ops.rms_norm(x, t[0], None, 1e-8), lambda t: ops.rms_norm(x, None, t, 1e-8), lambda t: ops.rms_norm_int8(t, None, None, 1e-8, True),
             lambda t: ops.dequantize_rows(q, t[:, 0], 0), lambda t: ops.matmul(q, t[:, 0], q, s, None, 1, 0.0, 1.0, 0), lambda t: ops.matmul(q, s, q, t[:, 0], None, 1, 0.0, 1.0, 0),
             lambda t: ops.matmul(q, s, q, s, t[:, 0], 1, 0.0, 1.0, 0), lambda t: ops.dense(t, q, s, None, 1, 0.0, 1.0, False, 1e-8))
    for call in calls:
        with fwd.dual_level(), pytest.raises(ops.Watched, match='no gradient'):
            call(fwd.make_dual(x, x))
        with pytest.raises(ops.Watched, match='transform'):
            torch.func.vmap(call)(torch.stack([x, x]))
        with pytest.raises(ops.Refused) as plain:          # (and a plain CPU tensor is refused for being one)
            call(x)
        assert not isinstance(plain.value, ops.Watched)
