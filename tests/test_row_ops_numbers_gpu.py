"""Row norm on the GPU at the ends of fp32's range: the forms of a value that are not a launch of the kernel alone."""
import pytest
import torch

from stylegan_v_amd.torch_utils.ops import rms_norm as rn

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
EPS = 1e-6


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def _formula(x, w, r, eps):
    h = x + r
    return h * (h.square().mean(dim=-1, keepdim=True) + eps).rsqrt() * w, h


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('scale', [1e30, 1e20, 1.0, 1e-25])
def test_second_derivative_of_rows_out_of_range(dtype, scale):
    """The gradient under create_graph is the first-order kernel's, and its own gradient the formula's, whatever the rows' size."""
    eps = 0.0
    ins = [(_rand(4, 50, seed=1) * scale).to(dtype), _rand(50, seed=2, dtype=dtype), (_rand(4, 50, seed=3) * scale).to(dtype)]
    dy = _rand(4, 50, seed=4, dtype=dtype)
    a = [t.clone().requires_grad_(True) for t in ins]
    first = torch.autograd.grad(rn.rms_norm(*a, eps=eps)[0], a, dy)
    b = [t.clone().requires_grad_(True) for t in ins]
    under = torch.autograd.grad(rn.rms_norm(*b, eps=eps)[0], b, dy, create_graph=True)
    # both forms are within 200 U of the exact gradient's terms, whose size is at most a few times the largest of a row's; and each is rounded once to the type
    for got, want in zip(under, first):
        assert torch.isfinite(got).all() and want.any()
        assert (got.double() - want.double()).abs().max() <= (2000 * U + 2 * torch.finfo(dtype).eps) * want.double().abs().max()
    v = _rand(50, seed=5, dtype=dtype)
    (second,) = torch.autograd.grad(under[1], b[0], v)
    # the same in 64 bits, on the stream as it was rounded
    h64 = (ins[0].double() + ins[2].double()).to(dtype).double().requires_grad_(True)
    w64 = ins[1].double().requires_grad_(True)
    y64, _ = _formula(h64, w64, torch.zeros_like(h64), eps)
    (gw,) = torch.autograd.grad(y64, w64, dy.double(), create_graph=True)
    (want,) = torch.autograd.grad(gw, h64, v.double())
    assert torch.isfinite(second).all()
    top = torch.finfo(dtype).smallest_normal           # (1e30: the second derivative is 1e-30 and below)
    assert (second.double() - want).abs().max() <= (2000 * U + 4 * torch.finfo(dtype).eps) * want.abs().max() + top


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('cols', [40, 4096, 16384, 20000])
def test_scale_near_the_end_of_the_range(dtype, cols):
    """max |y| beyond fp32's end, a 127th of it inside: the scale is a number, whatever |h w| is."""
    x = torch.zeros([3, cols], device=DEV)
    x[0, 1], x[1, 2], x[2, 3] = 0.5, 1e-3, 1e6
    x = x.to(dtype)
    w = torch.full([cols], 1.0 / cols ** 0.5, device=DEV, dtype=torch.float64).mul(2e39).clamp(max=3e38).to(dtype)
    q, s = rn.rms_norm_int8(x, w, eps=0.0)
    want = (w.double().max() * cols ** 0.5 / 127).item()            # y = sqrt(cols) w at the only element of a row
    assert want < 3.4e38 and ((s.double() - want).abs() <= 60 * U * want).all(), (s.tolist(), want)
    assert torch.equal(q.double(), 127.0 * (x != 0))


@pytest.mark.parametrize('cols', [(1 << 25) + 40, (1 << 26) - 16, (1 << 26) - 15, (1 << 26) - 1])
def test_weight_gradient_of_the_longest_rows(cols):
    """Up to the longest rows there are, 2^26 - 1: a thread of a launch for each 64th of a column would be 2^32 of them, one more than a launch may have."""
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip('needs 20 GB of device memory')
    g = torch.Generator(device=DEV).manual_seed(cols)
    x, dy = [torch.empty([2, cols], dtype=torch.float16, device=DEV).normal_(generator=g) for _ in range(2)]
    w = torch.ones([cols], dtype=torch.float16, device=DEV).requires_grad_(True)
    (dw,) = torch.autograd.grad(rn.rms_norm(x, w, eps=EPS), [w], dy)
    inv = (x.double().square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    for part in (slice(0, 1 << 20), slice(1 << 25, (1 << 25) + (1 << 20)), slice(cols - (1 << 20), cols)):
        t = dy[:, part].double() * x[:, part].double() * inv
        want, size = t.sum(dim=0), t.abs().sum(dim=0)
        # 1 / rms within 44 U, three roundings of each product, one of the sum; half a step of fp16
        assert ((dw[part].double() - want).abs() <= 48 * U * size + 2.0 ** -11 * want.abs() * 1.0001 + 2.0 ** -24).all()
