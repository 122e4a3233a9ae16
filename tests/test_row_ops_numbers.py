"""Row norm on the CPU at the ends of fp32's range: the same values as the kernel's, in both directions."""
import pytest
import torch

from stylegan_v_amd.torch_utils.ops import rms_norm as rn


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('scale,eps', [(1e30, 1e-8), (3e38, 0.0), (1e20, 1e-8), (1e-25, 0.0), (1e-37, 0.0)])
def test_rows_out_of_range(scale, eps, dtype):
    g = torch.Generator().manual_seed(0)
    x = (torch.rand([3, 40], generator=g, dtype=torch.float64) * scale).to(dtype)
    w, dy = torch.rand([40], generator=g).to(dtype), torch.rand([3, 40], generator=g).to(dtype)
    h = x.double().requires_grad_(True)
    w64 = w.double().requires_grad_(True)
    want = h * (h.square().mean(dim=1, keepdim=True) + eps).rsqrt() * w64
    wx, ww = torch.autograd.grad(want, (h, w64), dy.double())
    x.requires_grad_(True)
    w.requires_grad_(True)
    y = rn.rms_norm(x, w, eps=eps)
    gx, gw = torch.autograd.grad(y, (x, w), dy)
    step = torch.finfo(dtype).eps
    # y and the sum over three rows in fp32: a few roundings, and one to the type; dx: a difference of terms no larger than inv * max(dy w), which a subnormal result rounds to 1e-40
    assert ((y.double() - want).abs() <= (4 * 2.0 ** -24 + step / 2 * 1.001) * want).all()
    assert ((gw.double() - ww).abs() <= (8 * 2.0 ** -24 + step) * ww).all()
    inv = (x.detach().double().square().mean(dim=1, keepdim=True) + eps).rsqrt()
    size = inv * (dy.double() * w.detach().double()).abs().amax(dim=1, keepdim=True) * (1 + 40 ** 0.5)
    fine = size < torch.finfo(dtype).max                      # (1e-37: the gradient is 1e37 and fits)
    assert fine.all() and ((gx.double() - wx).abs() <= (8 * 2.0 ** -24 + step) * size + 1e-40).all()
    q, s = rn.rms_norm_int8(x.detach(), w.detach(), eps=eps)
    assert (q * s[:, None] - want.detach()).abs().amax(dim=1).le(s * 0.51).all()
