"""Row norm and 8-bit product on the GPU under what sees torch's operations only, not a launch: derivatives of forward mode, function transforms, tracers.

`rms_norm` takes its formula in torch operations there; the 8-bit operators, which have no gradient, refuse."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
EPS = 1e-6


def _rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64).to(dtype).to(DEV)


def _pushed(x, w, r, tx, tw, tr):
    """(dy, dh, the sizes of dy's terms) in 64 bits: dy = inv (dh - xh mean(xh dh)) w + xh dw."""
    def f64(t):
        return torch.zeros(1, dtype=torch.float64, device=DEV) if t is None else t.double()
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    h, dh = h.double(), (f64(tx) + f64(tr)).expand(h.shape)
    weight = torch.ones(h.shape[-1], dtype=torch.float64, device=DEV) if w is None else w.double()
    inv = (h.square().mean(dim=-1, keepdim=True) + EPS).rsqrt()
    xh = h * inv
    dy = inv * (dh - xh * (xh * dh).mean(dim=-1, keepdim=True)) * weight + xh * f64(tw)
    size = inv * (dh.abs() + xh.abs() * (xh * dh).abs().mean(dim=-1, keepdim=True)) * weight.abs() + (xh * f64(tw)).abs()
    return dy, dh, size


def _near(got, want, size, dtype, rounded, units=20):
    # at most `units` roundings of fp32 in the terms, `rounded` ones to the rows' type, half a step of the result
    info = torch.finfo(dtype)
    tol = (units * U + rounded * info.eps / 2) * size + info.eps / 2 * want.abs() * 1.0001 + (1 + rounded) * info.smallest_normal * info.eps
    assert got.dtype == dtype and got.shape == want.shape
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f'{(err / tol).max().item():.3g} of the tolerance'


@pytest.mark.parametrize('dtype', [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize('which', ['x', 'w', 'r', 'xwr'])
@pytest.mark.parametrize('requires_grad', [False, True])
def test_forward_mode(dtype, which, requires_grad):
    ins = dict(x=_rand(5, 100, seed=1, dtype=dtype), w=_rand(100, seed=2, dtype=dtype), r=_rand(5, 100, seed=3, dtype=dtype))
    tangents = {k: _rand(*ins[k].shape, seed=4 + i, dtype=dtype) for i, k in enumerate('xwr') if k in which}
    dy, dh, size = _pushed(ins['x'], ins['w'], ins['r'], *[tangents.get(k) for k in 'xwr'])
    if requires_grad:
        ins = {k: t.requires_grad_(True) for k, t in ins.items()}
    with fwd.dual_level():
        dual = {k: fwd.make_dual(t, tangents[k]) if k in which else t for k, t in ins.items()}
        y, h = rn.rms_norm(dual['x'], dual['w'], dual['r'], EPS)
        ty, th = fwd.unpack_dual(y).tangent, fwd.unpack_dual(h).tangent
        assert ty is not None and (th is not None) == (which != 'w')
        _near(ty, dy, size, dtype, 2)                  # the tangent of h and that of the sum in front of it are tensors of the type too
        if th is not None:
            _near(th, dh, dh.abs(), dtype, 0)
        plain = rn.rms_norm(ins['x'].detach(), ins['w'].detach(), ins['r'].detach(), EPS)
        _near(fwd.unpack_dual(y).primal, plain[0].double(), plain[0].double().abs(), dtype, 2, 44 + 20)      # (the kernel's 44, the formula's)
        assert torch.equal(fwd.unpack_dual(h).primal, plain[1])
    before = custom_ops.launch_count()
    rn.rms_norm(ins['x'], ins['w'], ins['r'], EPS)      # the level is left: the kernel again
    assert custom_ops.launch_count() - before == 1


def test_forward_mode_over_a_gradient():
    """The gradient's own tangent, by a dual gradient of the output: linear in it."""
    x, w, r = [t.requires_grad_(True) for t in (_rand(4, 60, seed=1), _rand(60, seed=2), _rand(4, 60, seed=3))]
    dy, dh, ty, th = _rand(4, 60, seed=4), _rand(4, 60, seed=5), _rand(4, 60, seed=6), _rand(4, 60, seed=7)
    y, h = rn.rms_norm(x, w, r, EPS)
    want = torch.autograd.grad([y, h], [x, w, r], [ty, th], retain_graph=True)
    with fwd.dual_level():
        found = torch.autograd.grad([y, h], [x, w, r], [fwd.make_dual(dy, ty), fwd.make_dual(dh, th)], retain_graph=True)
        for got, ref in zip(found, want):
            t = fwd.unpack_dual(got).tangent
            assert t is not None and (t - ref).norm() <= 200 * U * ref.norm()
    (gx,) = torch.autograd.grad(h, [x], dh, retain_graph=True)          # (the stream alone)
    assert torch.equal(gx, dh)


def test_function_transforms():
    x, w = _rand(6, 40, seed=1), _rand(40, seed=2)
    tx = _rand(6, 40, seed=3)
    plain = rn.rms_norm(x, w, eps=EPS)
    ye = plain.double()
    _near(torch.func.vmap(lambda a: rn.rms_norm(a, w, eps=EPS))(x), ye, ye.abs(), torch.float32, 2, 44 + 20)
    y, t = torch.func.jvp(lambda a: rn.rms_norm(a, w, eps=EPS), (x,), (tx,))
    dy, _, size = _pushed(x, w, None, tx, None, None)
    _near(y, ye, ye.abs(), torch.float32, 2, 44 + 20)
    _near(t, dy, size, torch.float32, 0)
    xg = x.clone().requires_grad_(True)
    (want,) = torch.autograd.grad(rn.rms_norm(xg, w, eps=EPS), [xg], tx)
    _, pull = torch.func.vjp(lambda a: rn.rms_norm(a, w, eps=EPS), x)
    assert (pull(tx)[0] - want).norm() <= 200 * U * want.norm()
    # a batch of gradients at once: a transform that only the backward pass sees
    yg = rn.rms_norm(xg, w, eps=EPS)
    many = torch.stack([tx, 2 * tx, _rand(6, 40, seed=5)])
    (batched,) = torch.autograd.grad(yg, [xg], many, is_grads_batched=True, retain_graph=True)
    for i in range(3):
        (one,) = torch.autograd.grad(yg, [xg], many[i], retain_graph=True)
        assert (batched[i] - one).norm() <= 200 * U * one.norm()


def test_8_bit_operators_refuse_what_they_cannot_follow():
    x, q, s = _rand(4, 64, seed=1), torch.ones([5, 64], dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)
    a, sa = torch.ones([4, 64], dtype=torch.int8, device=DEV), torch.ones(4, device=DEV)
    bias, w = torch.ones(5, device=DEV), torch.ones(64, device=DEV)

    def dual(t):
        return fwd.make_dual(t, torch.ones_like(t))
    with fwd.dual_level():
        for call in (lambda: rn.rms_norm_int8(dual(x)), lambda: rn.rms_norm_int8(x, dual(w)), lambda: rn.rms_norm_int8(x, None, dual(x)), lambda: int8.quantize_rows(dual(x)),
                     lambda: int8.dequantize_rows(a, dual(sa)), lambda: int8.matmul(a, dual(sa), q, s), lambda: int8.matmul(a, sa, q, dual(s)),
                     lambda: int8.matmul(a, sa, q, s, bias=dual(bias)), lambda: int8.dense(dual(x), q, s), lambda: int8.dense(x, q, dual(s)), lambda: int8.dense(x, q, s, bias=dual(bias))):
            with pytest.raises(RuntimeError, match='no gradient'):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match='no gradient'):       # (a tangent goes through no_grad)
                call()
        assert torch.equal(int8.dense(dual(x).detach(), q, s), int8.dense(x, q, s))
    for call in (rn.rms_norm_int8, int8.quantize_rows, lambda t: int8.dense(t, q, s), lambda t: int8.dequantize_rows(a[0], t.sum()), lambda t: int8.matmul(a[0], t.sum(), q, s)):
        with pytest.raises(RuntimeError, match='transform'):
            torch.func.vmap(call)(x)
