"""Row norm kernels (csrc/rms_norm.hip through ops/rms_norm.py) against the definition in 64 bits: forward, gradient, 8-bit output, at the lengths where the kernel changes,
with rows that hold nothing, infinities, NaN and values at the ends of their type.

Tolerances count roundings, U = 2^-24 for fp32 and eps/2 of the output's type.  inv: a sum of squares over at most 64 terms per thread and 12 tree levels, relative error
76 U, half of that in the root, 3 U for the division and the root: 41 U.  y = h * inv * w: 44 U.  dx: three terms of at most 41 + 76 + 44 + 5 < 200 U of their size."""
import pytest
import torch

from stylegan_v_amd.torch_utils import custom_ops
from stylegan_v_amd.torch_utils.ops import int8, rms_norm as rn

pytestmark = pytest.mark.gpu
DEV = 'cuda'
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# both sides of every border of the dispatch: one thread, 8, 16, 32 lanes, one wave x 1, 2, 4 vectors, a workgroup x 2, 4, 8, the walking kernel; whole vectors and not
LENGTHS = [1, 3, 4, 7, 8, 15, 16, 31, 32, 33, 64, 65, 120, 128, 129, 255, 256, 257, 511, 512, 513, 1024, 1025, 1111, 2048, 2049, 2900, 4096, 4100, 5121, 8192, 8193, 9000, 13313, 16384, 16385, 40001]


def _rand(*shape, seed=0, dtype=torch.float32, scale=1.0):
    return (torch.randn(list(shape), generator=torch.Generator().manual_seed(seed), dtype=torch.float64) * scale).to(dtype).to(DEV)


def _half(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps        # the spacing of the smallest values


def _check(got, want, size, units, what):
    """|got - want| <= units * U * size + half a step of got's type."""
    tol = units * U * size + _half(got.dtype) * want.abs() * 1.0001 + _tiny(got.dtype)
    err = (got.double() - want).abs()
    assert (err <= tol).all(), f'{what}: {(err / tol).max().item():.3g} of the tolerance'


def _exact(x, w, r, eps):
    h = x if r is None else (x.double() + r.double()).to(x.dtype)
    hd = h.double()
    inv = (hd.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    return h, hd, inv, (hd * inv if w is None else hd * inv * w.double())


def _exact8(h, w, inv):
    u = h.double() if w is None else h.double() * w.double()
    top = u.abs().amax(dim=-1, keepdim=True)
    q = torch.where(top > 0, torch.round(u * 127.0 / top), torch.zeros_like(u))
    return q, (top * inv / 127.0).squeeze(-1)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cols', LENGTHS)
def test_forward_gradient_and_8_bits(cols, dtype):
    rows, eps = 6, 1e-6
    for residual, weight in ((False, None), (True, dtype), (True, torch.float32), (False, dtype)):
        x = _rand(rows, cols, seed=cols, dtype=dtype)
        r = _rand(rows, cols, seed=cols + 1, dtype=dtype, scale=3) if residual else None
        w = _rand(cols, seed=cols + 2, dtype=weight) if weight else None
        x[2] = 0
        if r is not None:
            r[2] = 0                     # a row of padding
        leaves = [t.requires_grad_(True) for t in (x, w, r) if t is not None]
        dy, dh = _rand(rows, cols, seed=cols + 3, dtype=dtype), _rand(rows, cols, seed=cols + 4, dtype=dtype)
        before = custom_ops.launch_count()
        out = rn.rms_norm(x, w, r, eps)
        assert custom_ops.launch_count() - before == 1
        y, h = out if residual else (out, x)
        grads = torch.autograd.grad([y, h] if residual else [y], leaves, [dy, dh] if residual else [dy])
        assert custom_ops.launch_count() - before == 2
        he, hd, inv, ye = _exact(x.detach(), w.detach() if w is not None else None, r.detach() if residual else None, eps)
        assert torch.equal(h.detach(), he)
        _check(y.detach(), ye, ye.abs(), 44, 'y')
        g = dy.double() * (w.detach().double() if w is not None else 1.0)
        xh = hd * inv
        along = (g * xh).abs().mean(dim=1, keepdim=True)
        dx = inv * (g - xh * (g * xh).mean(dim=1, keepdim=True)) + (dh.double() if residual else 0.0)
        size = inv * (g.abs() + xh.abs() * along) + (dh.double().abs() if residual else 0.0)
        _check(grads[0], dx, size, 200, 'dx')
        if residual:
            assert torch.equal(grads[0], grads[-1])
        if w is not None:
            assert grads[1].dtype == w.dtype
            _check(grads[1], (dy.double() * xh).sum(dim=0), (dy.double() * xh).abs().sum(dim=0), 44 + rows, 'dw')
        with torch.no_grad():
            got = rn.rms_norm_int8(x, w, r, eps)
        qe, se = _exact8(he, w.detach() if w is not None else None, inv)
        assert torch.equal(got[0].double(), qe), f'{(got[0].double() != qe).sum().item()} of {qe.numel()} values differ'
        _check(got[1], se, se, 46, 'scale')
        if residual:
            assert torch.equal(got[2], he)
        q, s = int8.quantize_rows(x.detach())
        qe, se = _exact8(x.detach(), None, torch.ones_like(inv))
        assert torch.equal(q.double(), qe)
        _check(s, se, se, 2, 'scale of quantize_rows')
        back = int8.dequantize_rows(q, s, dtype=dtype)
        _check(back, q.double() * s.double().unsqueeze(1), (q.double() * s.double().unsqueeze(1)).abs(), 1, 'dequantize_rows')
        assert q.data_ptr() % 16 == 0 and q.stride(0) % 16 == 0
        if cols % 16:                    # the storage behind the last column is written, with zeros
            wide = q.as_strided([rows, q.stride(0)], [q.stride(0), 1])
            assert not wide[:, cols:].any()


@pytest.mark.parametrize('rows', [1, 2, 5, 511, 2047, 2049, 5000])
@pytest.mark.parametrize('cols', [3, 24, 57, 120, 200, 520, 2900])
def test_many_rows_weight_gradient(rows, cols):
    x, w, dy = _rand(rows, cols, seed=rows), _rand(cols, seed=1), _rand(rows, cols, seed=rows + 2)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(rn.rms_norm(x, w), (x, w), dy)
    _, hd, inv, _ = _exact(x.detach(), None, None, 1e-8)
    t = dy.double() * hd * inv
    # a thread adds at most rows / 256 + 4 rows (one workgroup takes every 256th), then 6 levels of a wave, 4 waves, 1024 / 64 partial sums and 6 levels
    _check(dw, t.sum(dim=0), t.abs().sum(dim=0), 44 + rows / 256 + 4 + 6 + 4 + 16 + 6, 'dw')
    again = torch.autograd.grad(rn.rms_norm(x, w), (x, w), dy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)          # a fixed order: the same bits


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('cols', [40, 5000, 20000])
def test_rows_with_nan_infinities_and_extremes(dtype, cols):
    top = torch.finfo(dtype).max
    x = _rand(8, cols, seed=9, dtype=dtype)
    x[0, 3] = float('nan')
    x[1, 5] = float('inf')
    x[2, 7] = -float('inf')
    x[3] = -top                                    # masks of the type's lowest value
    x[4] = top
    x[5, :] = 0
    x[5, 1] = torch.finfo(dtype).smallest_normal
    x[6, 0] = -top
    _, hd, inv, ye = _exact(x, None, None, 1e-8)
    y = rn.rms_norm(x)
    fin = torch.isfinite(ye)
    assert torch.equal(torch.isfinite(y), fin)
    _check(torch.where(fin, y, torch.zeros_like(y)), torch.where(fin, ye, torch.zeros_like(ye)), torch.where(fin, ye, torch.zeros_like(ye)).abs(), 60, 'y')
    q, s = rn.rms_norm_int8(x)
    assert s[:3].isnan().all() and not q[:3].any()
    qe, se = _exact8(x[3:], None, inv[3:])
    assert torch.equal(q[3:].double(), qe)
    _check(s[3:], se, se, 60, 'scale')
    q, s = int8.quantize_rows(x)
    assert s[:3].isnan().all() and not q[:3].any()
    assert torch.equal(q[3:].double(), qe)
    # a weight that takes the products beyond fp32, and one that takes them below it
    if dtype != torch.float16:
        for scale in (1e30, 1e-30):
            w = (_rand(cols, seed=3, dtype=torch.float64) * scale).to(dtype)
            xs = _rand(3, cols, seed=4, dtype=dtype, scale=scale)
            q, s = rn.rms_norm_int8(xs, w, eps=0.0)
            qe, se = _exact8(xs, w, xs.double().square().mean(dim=1, keepdim=True).rsqrt())
            assert torch.equal(q.double(), qe)
            _check(s, se, se, 60, 'scale')
    if dtype == torch.float32:                     # squares far below fp32's range under an eps that does not cover them
        xs = _rand(3, cols, seed=4, scale=1e-25)
        ye = xs.double() * xs.double().square().mean(dim=1, keepdim=True).rsqrt()
        _check(rn.rms_norm(xs, eps=0.0), ye, ye.abs(), 60, 'y')


def test_border_values_are_decided_exactly():
    """Values on and next to the border between two steps: k + 1/2 steps of a maximum that makes them representable, and their neighbours in fp32."""
    for top in (127.0, 254.0, 3.0, 2.0 ** -20 * 127, 1.0):
        k = torch.arange(-126, 127, dtype=torch.float64) + 0.5
        mid = (k * top / 127.0).float()
        row = torch.cat([torch.tensor([top]), mid, torch.nextafter(mid, torch.tensor(float('inf'))), torch.nextafter(mid, torch.tensor(-float('inf')))]).to(DEV)[None]
        for w in (None, torch.full([row.shape[1]], 3.0, device=DEV), _rand(row.shape[1], seed=2).abs() + 0.5):
            q, _ = rn.rms_norm_int8(row, w)
            assert torch.equal(q.double(), _exact8(row, w, torch.ones(1, 1, device=DEV, dtype=torch.float64))[0])
    bits = torch.randint(-128, 129, [64, 1000], generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)      # whole numbers: many exact halves
    bits[:, 0] = 254
    q, _ = int8.quantize_rows(bits)
    assert torch.equal(q.double(), _exact8(bits, None, torch.ones(64, 1, device=DEV, dtype=torch.float64))[0])


@pytest.mark.parametrize('dtype', TYPES)
def test_strides_and_alignments(dtype):
    base = _rand(9, 700, seed=1, dtype=dtype)
    views = [base[:, 3:520], base[:, 1:513], base[::2], base[2:3], base.t()[5:70], base[:1].expand(5, 700), base[:, ::3], base.view(3, 3, 700)[:, 1:, :512], base[4], base[:, 7:8]]
    for v in views:
        w = _rand(v.shape[-1] + 1, seed=2, dtype=dtype)[1:]
        for r in (None, v.clone(), v.flip(0)):
            h, hd, inv, ye = _exact(v, w, r, 1e-8)
            out = rn.rms_norm(v, w, r)
            y = out if r is None else out[0]
            assert y.shape == v.shape
            _check(y, ye, ye.abs(), 44, 'y')
            q, s = rn.rms_norm_int8(v, w, r)[:2]
            qe, _ = _exact8(h, w, inv)
            assert q.shape == v.shape and s.shape == v.shape[:-1] and torch.equal(q.double(), qe)
        x = v.detach().clone().requires_grad_(True)
        y = rn.rms_norm(x, w)
        (dx,) = torch.autograd.grad(y.sum(), x)                             # dy with strides of zero
        x64 = v.detach().double().requires_grad_(True)
        (want,) = torch.autograd.grad(rn.rms_norm_ref(x64, w.double()).sum(), x64)
        _, hd, inv, _ = _exact(v, w, None, 1e-8)
        g, xh = w.double().expand(v.shape), hd * inv
        _check(dx, want, inv * (g.abs() + xh.abs() * (g * xh).abs().mean(dim=-1, keepdim=True)), 200, 'dx')
    y3, h3 = rn.rms_norm(base.view(3, 3, 700), residual=base.view(3, 3, 700))
    assert y3.shape == h3.shape == (3, 3, 700)


def test_gradients_of_some_inputs_only_and_of_one_output_only():
    x, r, w = _rand(5, 100, seed=1), _rand(5, 100, seed=2), _rand(100, seed=3)
    dy = _rand(5, 100, seed=4)
    full = [t.clone().requires_grad_(True) for t in (x, w, r)]
    y, h = rn.rms_norm(full[0], full[1], full[2])
    want = torch.autograd.grad(y, full, dy, retain_graph=True)
    only_h = torch.autograd.grad(h, [full[0], full[2]], dy, retain_graph=True)
    assert torch.equal(only_h[0], dy) and torch.equal(only_h[1], dy)
    assert torch.autograd.grad(h, [full[1]], dy, allow_unused=True)[0] is None
    for k in range(3):
        ins = [t.clone().requires_grad_(i == k) for i, t in enumerate((x, w, r))]
        (got,) = torch.autograd.grad(rn.rms_norm(ins[0], ins[1], ins[2])[0], [ins[k]], dy)
        assert torch.equal(got, want[k])
    same = x.clone().requires_grad_(True)                                   # one tensor as both
    y, h = rn.rms_norm(same, None, same)
    (g,) = torch.autograd.grad(y, same, dy)
    t = x.clone().requires_grad_(True)
    (one,) = torch.autograd.grad(rn.rms_norm(t + t), t, dy)
    assert torch.allclose(g, one, rtol=1e-5, atol=1e-5)


def test_second_derivative():
    x, w, r = [t.requires_grad_(True) for t in (_rand(4, 50, seed=1), _rand(50, seed=2), _rand(4, 50, seed=3))]

    def penalty(fn, *ins):
        y, h = fn(*ins)
        (gx,) = torch.autograd.grad((y * y * y).sum() + (h * h).sum(), ins[0], create_graph=True)
        return torch.autograd.grad(gx.square().sum() + y.sum(), ins)
    got = penalty(lambda *a: rn.rms_norm(*a, eps=1e-3), x, w, r)
    want = penalty(lambda *a: rn.rms_norm_ref(*a, eps=1e-3), *[t.detach().double().requires_grad_(True) for t in (x, w, r)])
    for a, b in zip(got, want):
        assert (a.double() - b).norm() / b.norm() < 1e-5        # 50-term fp32 sums, differentiated twice: ~100 U = 6e-6


def test_gradient_against_differences():
    x, w, dy, v = _rand(3, 600, seed=1, dtype=torch.float64), _rand(600, seed=2, dtype=torch.float64), _rand(3, 600, seed=3, dtype=torch.float64), _rand(3, 600, seed=4, dtype=torch.float64)
    f = lambda t: (rn.rms_norm_ref(t, w) * dy).sum().item()     # noqa: E731
    slope = (f(x + 1e-5 * v) - f(x - 1e-5 * v)) / 2e-5          # error of the difference: 1e-10 of the third derivative
    xf = x.float().requires_grad_(True)
    (dx,) = torch.autograd.grad(rn.rms_norm(xf, w.float()), xf, dy.float())
    assert abs((dx.double() * v).sum().item() - slope) < 200 * U * (dx.double() * v).abs().sum().item() * 2


def test_refusals_on_the_gpu():
    x = _rand(2, 8)
    with pytest.raises(RuntimeError, match='dtype'):
        rn.rms_norm(x.double())
    with pytest.raises(RuntimeError, match='device'):
        rn.rms_norm(x, residual=x.cpu())
    with pytest.raises(RuntimeError, match='weight'):
        rn.rms_norm(x, weight=torch.ones(8))
    assert rn.rms_norm(x[:0]).shape == (0, 8) and rn.rms_norm_int8(x[:0])[0].shape == (0, 8)
    e, w = x[:0].clone().requires_grad_(True), torch.ones(8, device=DEV, requires_grad=True)
    de, dw = torch.autograd.grad(rn.rms_norm(e, w).sum(), (e, w))
    assert de.shape == (0, 8) and not dw.any()


def test_empty_batches_and_lost_inputs():
    for shape in ((0, 24), (2, 0, 24), (0, 3, 24)):
        x = torch.empty(shape, device=DEV, requires_grad=True)
        y, h = rn.rms_norm(x, None, torch.empty(shape, device=DEV))
        assert y.shape == h.shape == shape
        (dx,) = torch.autograd.grad([y, h], [x], [torch.empty(shape, device=DEV)] * 2)
        assert dx.shape == shape
        with torch.no_grad():
            q, s = rn.rms_norm_int8(x)
            assert q.shape == shape and s.shape == shape[:-1] and int8.dequantize_rows(q, s).shape == shape
            assert int8.matmul(q, s, torch.ones([5, 24], dtype=torch.int8, device=DEV), torch.ones(5, device=DEV)).shape == shape[:-1] + (5,)
            assert int8.dense(x, torch.ones([5, 24], dtype=torch.int8, device=DEV), torch.ones(5, device=DEV), normalize=True).shape == shape[:-1] + (5,)
    x, w = _rand(4, 24).requires_grad_(True), torch.ones(24, device=DEV, requires_grad=True)
    y, h = rn.rms_norm(x, w, x)
    h.add_(1)                                       # the gradient needs the stream as it was
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.sum().backward()


def test_two_threads_on_two_streams():
    import threading
    sets = [(_rand(700, 1111).requires_grad_(True), _rand(1111).requires_grad_(True), _rand(700, 1111)) for _ in range(2)]

    def once(x, w, dy):
        y = rn.rms_norm(x, w)
        with torch.no_grad():
            q, s = rn.rms_norm_int8(x, w)
            p = int8.matmul(q, s, q, s)
        return torch.autograd.grad(y, (x, w), dy) + (y.detach(), q, s, p)

    want = [once(*s) for s in sets]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got = once(*sets[i])
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_streams_and_graph_replays():
    x, r, w, dy = _rand(300, 1000, seed=1), _rand(300, 1000, seed=2), _rand(1000, seed=3), _rand(300, 1000, seed=4)
    ins = [t.clone().requires_grad_(True) for t in (x, w, r)]

    def step():
        y, h = rn.rms_norm(*ins)
        grads = torch.autograd.grad([y, h], ins, [dy, dy])
        with torch.no_grad():
            q, s = rn.rms_norm_int8(ins[0], ins[1])
            back = int8.dequantize_rows(q, s)
        return [y.detach(), h.detach(), *grads, q, s, back]
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):                                   # two captured graphs of the same call, each with a workspace of its own
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for seed in range(3):
        with torch.no_grad():
            ins[0].copy_(_rand(300, 1000, seed=10 + seed))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = step()
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_more_than_2_31_elements():
    rows, cols = 65600, 32768 + 8
    free = torch.cuda.mem_get_info()[0]
    if free < 40 << 30:
        pytest.skip('needs 40 GB of device memory')
    x = torch.empty([rows, cols], dtype=torch.bfloat16, device=DEV)
    x.normal_(generator=torch.Generator(device=DEV).manual_seed(0))
    pick = torch.tensor([0, 1, rows // 2, rows - 2, rows - 1], device=DEV)
    y, h = rn.rms_norm(x, residual=x)
    he, _, inv, ye = _exact(x[pick], None, x[pick], 1e-8)
    assert torch.equal(h[pick], he)
    _check(y[pick], ye, ye.abs(), 44, 'y')
    del y, h
    q, s = int8.quantize_rows(x)
    qe, _ = _exact8(x[pick], None, torch.ones_like(inv))
    assert torch.equal(q[pick].double(), qe)
    back = int8.dequantize_rows(q, s, dtype=torch.bfloat16)
    assert torch.equal(back[pick], (q[pick].float() * s[pick].unsqueeze(1)).to(torch.bfloat16))
    del back, q
    xg = x.requires_grad_(True)
    (dx,) = torch.autograd.grad(rn.rms_norm(xg), xg, x.detach())
    hd = x.detach()[pick].double()
    inv = (hd.square().mean(dim=1, keepdim=True) + 1e-8).rsqrt()
    xh = hd * inv
    want = inv * (hd - xh * (hd * xh).mean(dim=1, keepdim=True))
    _check(dx[pick], want, inv * (hd.abs() + xh.abs() * (hd * xh).abs().mean(dim=1, keepdim=True)), 200, 'dx')
