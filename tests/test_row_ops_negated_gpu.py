"""Row operators on the GPU with views whose elements are stored with the other sign (torch's negative bit): the values count, not what lies in memory."""
import pytest
import torch

from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def test_negated_views():
    """A view whose elements are stored with the other sign (the imaginary part of a conjugate): one column, so that no copy is made for the strides' sake."""
    z = torch.complex(_rand(6, 1, seed=1), _rand(6, 1, seed=2))
    v = z.conj().imag
    assert v.is_neg()
    plain = v.resolve_neg().clone()
    w = torch.complex(_rand(1, seed=3), _rand(1, seed=4)).conj().imag
    assert torch.equal(rn.rms_norm(v, eps=1.0), rn.rms_norm(plain, eps=1.0))
    assert torch.equal(rn.rms_norm(plain, w, eps=1.0), rn.rms_norm(plain, w.resolve_neg(), eps=1.0))
    assert torch.equal(rn.rms_norm(plain, residual=v, eps=1.0)[1], plain + plain)
    assert torch.equal(int8.quantize_rows(v)[0], int8.quantize_rows(plain)[0])
    wide, scales = torch.ones([6, 4], dtype=torch.int8, device=DEV), v[:, 0]
    assert torch.equal(int8.dequantize_rows(wide, scales), int8.dequantize_rows(wide, plain[:, 0]))
    assert torch.equal(int8.matmul(wide, scales, wide, scales, bias=scales), int8.matmul(wide, plain[:, 0], wide, plain[:, 0], bias=plain[:, 0]))
    neg = torch._neg_view(_rand(5, 64, seed=5))
    assert neg.is_neg() and torch.equal(rn.rms_norm(neg), rn.rms_norm(neg.resolve_neg()))
    assert torch.equal(int8.dense(neg, wide.new_ones([3, 64]), torch.ones(3, device=DEV)), int8.dense(neg.resolve_neg(), wide.new_ones([3, 64]), torch.ones(3, device=DEV)))
    x = _rand(5, 64, seed=6).requires_grad_(True)
    r = _rand(5, 64, seed=7)
    y, h = rn.rms_norm(x, residual=r)
    (got,) = torch.autograd.grad([y, h], [x], [neg, neg], retain_graph=True)
    (want,) = torch.autograd.grad([y, h], [x], [neg.resolve_neg()] * 2, retain_graph=True)
    assert torch.equal(got, want)
    xn = torch._neg_view(x)
    (got,) = torch.autograd.grad(rn.rms_norm(xn), [x], r)
    (want,) = torch.autograd.grad(rn.rms_norm(-x), [x], r)
    assert torch.equal(got, want)
