"""Root-mean-square norm of rows with a learned weight, the addition of a residual stream, and an output in the rows' type or in 8 bits (csrc/rms_norm.hip).

``rms_norm(x, weight, residual, eps)`` is ``normalize_2nd_moment`` of the mapping network (src/training/layers.py:16-18) over the last dimension as an operator with
a gradient of its own:

    h = x + residual                      (rounded to x's type: h is the residual stream that goes on, and the norm sees what goes on)
    y = h * rsqrt(mean(h^2) + eps) * weight

One launch forward and one backward (two with a weight, whose gradient is a sum over all rows; its order is fixed, so equal inputs give equal bits).  A gradient that is
itself differentiated (``create_graph``) takes the same formula as a composition of torch ops.

``rms_norm_int8`` gives y in 8 bits with one scale per row -- the left operand of ``ops.int8.matmul`` -- in the same single pass: y is never written in its own type.
It serves inference and has no gradient.

Statistics are fp32 whatever the rows' type (fp32, fp16, bf16).  CPU tensors take the plain torch formulation.
"""
import torch

from .. import custom_ops

_forward = custom_ops.PackedEntry('sgv_rms_norm', custom_ops.RmsNormParams)
_backward = custom_ops.PackedEntry('sgv_rms_norm_backward', custom_ops.RmsNormBackwardParams)
_DTYPE_CODES = {torch.float32: custom_ops.SGV_F32, torch.float16: custom_ops.SGV_F16, torch.bfloat16: custom_ops.SGV_BF16}


def check_no_grad(what, *tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError(f'{what} serves inference and has no gradient: call it under torch.no_grad() or with detached tensors')


def _check(what, x, weight, residual, eps):
    if not isinstance(x, torch.Tensor) or x.ndim < 1 or x.shape[-1] < 1:
        raise RuntimeError(f'{what}: x must be a tensor of rows (at least one dimension, the last one not empty)')
    dtype = x.dtype
    if dtype not in _DTYPE_CODES and not (dtype == torch.float64 and not x.is_cuda):
        raise RuntimeError(f'{what}: unsupported dtype {dtype}')
    if not eps >= 0:
        raise RuntimeError(f'{what}: eps must be >= 0')
    if weight is not None:
        if weight.ndim != 1 or weight.shape[0] != x.shape[-1]:
            raise RuntimeError(f'{what}: weight must have one element per column')
        if (weight.dtype != dtype and weight.dtype != torch.float32) or weight.device != x.device:
            raise RuntimeError(f'{what}: weight must have the type of x or fp32, on the device of x')
    if residual is not None and (residual.shape != x.shape or residual.dtype != dtype or residual.device != x.device):
        raise RuntimeError(f'{what}: residual must have the same shape, dtype, and device as x')


def row_view(t):
    """t as [rows, columns] with unit stride along a row: a view where t allows one, else a copy."""
    if t.is_contiguous():
        return t if t.ndim == 2 else t.view(-1, t.shape[-1])
    cols = t.shape[-1]
    if t.ndim != 2:
        t = t.reshape(-1, cols)
    if cols > 1 and t.stride(1) != 1:
        t = t.contiguous()
    return t


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _stride(t):
    return 0 if t is None else t.stride(0)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def launch_forward(x, weight, residual, eps, int8, normalize=True, want_inv=False):
    """(y or q, h or None, inv_rms or None, scale or None), all as rows; x and residual: ``row_view``s on a GPU, weight dense."""
    rows, cols = x.shape
    h = None if residual is None else x.new_empty((rows, cols))
    inv = x.new_empty(rows, dtype=torch.float32) if want_inv else None
    if int8:      # rows on 16 bytes, zeros behind the last column: what the 8-bit product reads
        pitch = (cols + 15) // 16 * 16
        y, scale = x.new_empty((rows, pitch), dtype=torch.int8), x.new_empty(rows, dtype=torch.float32)
    else:
        pitch = cols
        y, scale = x.new_empty((rows, cols)), None
    if rows:
        out = y.data_ptr()
        _forward(x, _DTYPE_CODES[x.dtype], x.data_ptr(), _ptr(residual), _ptr(weight), 0 if int8 else out, _ptr(h), _ptr(inv), out if int8 else 0, _ptr(scale), rows, _stride(x),
                 _stride(residual), pitch, cols, weight is not None and weight.dtype == torch.float32, normalize, eps)
    return (y[:, :cols] if pitch != cols else y), h, inv, scale


def _launch_backward(dy, h, dh, weight, inv, need_dx, need_dw):
    rows, cols = h.shape
    dx = h.new_empty((rows, cols)) if need_dx else None
    dw = torch.empty_like(weight) if need_dw else None
    if rows == 0:
        return dx, (dw.zero_() if need_dw else None)
    code = _DTYPE_CODES[h.dtype]
    size = custom_ops.get_native().sgv_rms_norm_backward_workspace_bytes(rows, cols, code) if need_dw else 0
    work = inv.new_empty(size // 4) if need_dw else None
    _backward(h, code, dy.data_ptr(), h.data_ptr(), _ptr(dh), _ptr(weight), inv.data_ptr(), _ptr(dx), _ptr(dw), _ptr(work), size, rows, _stride(dy), _stride(h), _stride(dh), cols,
              weight is not None and weight.dtype == torch.float32)
    return dx, dw


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def rms_norm_ref(x, weight=None, residual=None, eps=1e-8):
    """The definition, in torch ops."""
    h = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
    y = _wide(h) * (_wide(h).square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    if weight is not None:
        y = y * _wide(weight)
    y = y.to(x.dtype)
    return y if residual is None else (y, h)


def _gradient_ref(dy, h, dh, weight, eps):
    """(dx, dweight) in torch ops: what the backward kernel computes, differentiable once more."""
    hf = h.float()
    inv = (hf.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    dx = dw = None
    if dy is not None:
        xh, g = hf * inv, dy.float()
        if weight is not None:
            dw = (g * xh).sum(dim=0).to(weight.dtype)
            g = g * weight.float()
        dx = inv * (g - xh * (g * xh).mean(dim=-1, keepdim=True))
    if dh is not None:
        dx = dh.float() if dx is None else dx + dh.float()
    return (dx.to(h.dtype) if dx is not None else None), dw


class _RmsNormFn(torch.autograd.Function):
    """Rows in, rows out: y, or (y, h) with a residual."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, h, inv, _ = launch_forward(x, _dense(weight), residual, eps, int8=False, want_inv=True)
        ctx.eps, ctx.inv = eps, inv
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x if residual is None else h, weight)
        return y if residual is None else (y, h)

    @staticmethod
    def backward(ctx, dy, dh=None):
        h, weight = ctx.saved_tensors
        need_x, need_w, need_r, _ = ctx.needs_input_grad
        need_w = need_w and dy is not None
        if torch.is_grad_enabled():
            dx, dw = _gradient_ref(dy, h, dh, weight, ctx.eps)
        elif dy is None:
            dx, dw = dh, None
        else:
            if dy.stride(1) != 1 and dy.shape[1] != 1:
                dy = dy.contiguous()
            if dh is not None and dh.stride(1) != 1 and dh.shape[1] != 1:
                dh = dh.contiguous()
            dx, dw = _launch_backward(dy, h, dh, _dense(weight), ctx.inv, need_x or need_r, need_w)
        return (dx if need_x else None), (dw if need_w else None), (dx if need_r else None), None


def rms_norm(x, weight=None, residual=None, eps=1e-8):
    """x [..., K], weight [K] (x's type or fp32) or None, residual like x or None -> y like x; with a residual (y, h), h = x + residual."""
    _check('rms_norm', x, weight, residual, eps)
    if not x.is_cuda:
        return rms_norm_ref(x, weight, residual, eps)
    rows, res = row_view(x), None if residual is None else row_view(residual)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (residual is not None and residual.requires_grad)):
        out = _RmsNormFn.apply(rows, weight, res, eps)
    else:
        out = launch_forward(rows, _dense(weight), res, eps, int8=False)
        out = out[0] if residual is None else out[:2]
    if x.ndim == 2:
        return out
    return out.view(x.shape) if residual is None else (out[0].view(x.shape), out[1].view(x.shape))


def quantize_ref(u, factor):
    """(q, scale) of rows u in fp64: q = 127 u / max|u| to nearest even, scale = max|u| * factor / 127; a row with a NaN or an infinity: NaN and zeros."""
    top = u.abs().amax(dim=-1, keepdim=True)
    fine = torch.isfinite(top) & (top > 0)
    q = torch.where(fine, torch.round(u * 127.0 / torch.where(fine, top, torch.ones_like(top))), torch.zeros_like(u))
    scale = torch.where(torch.isfinite(top), top * factor / 127.0, torch.full_like(top, float('nan')))
    return q.to(torch.int8), scale.squeeze(-1).float()


def rms_norm_int8(x, weight=None, residual=None, eps=1e-8):
    """``rms_norm`` with y in 8 bits: (q [..., K] int8, scale [...] fp32), with a residual (q, scale, h).  y stands for q * scale: scale = max|y| / 127 of each row and
    q = y / scale rounded to nearest even (of the exact quotient).  A row of zeros has scale 0; a row with a NaN or an infinity in y has scale NaN and q = 0.
    The rows of q start on 16 bytes (q is a view of wider storage where K is no multiple of 16), as ``ops.int8.matmul`` wants them."""
    _check('rms_norm_int8', x, weight, residual, eps)
    check_no_grad('rms_norm_int8', x, weight, residual)
    if not x.is_cuda:
        h = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
        u = h.double()
        factor = (u.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
        q, scale = quantize_ref(u if weight is None else u * weight.double(), factor)
        return (q, scale) if residual is None else (q, scale, h)
    q, h, _, scale = launch_forward(row_view(x), _dense(weight), None if residual is None else row_view(residual), eps, int8=True)
    if x.ndim != 2:
        q, scale = q.unflatten(0, x.shape[:-1]) if x.ndim > 2 else q[0], scale.view(x.shape[:-1])
        h = h.view(x.shape) if h is not None else None
    return (q, scale) if residual is None else (q, scale, h)
