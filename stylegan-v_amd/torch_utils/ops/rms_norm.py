"""Root-mean-square norm of rows with a learned weight, the addition of a residual stream, and an output in the rows' type or in 8 bits (csrc/rms_norm.hip).

``rms_norm(x, weight, residual, eps)`` is ``normalize_2nd_moment`` of the mapping network (src/training/layers.py:16-18) over the last dimension as an operator with
a gradient of its own:

    h = x + residual                      (rounded to x's type: h is the residual stream that goes on, and the norm sees what goes on)
    y = h * rsqrt(mean(h^2) + eps) * weight

One launch forward and one backward (two with a weight, whose gradient is a sum over all rows; its order is fixed, so equal inputs give equal bits).  A gradient that is
itself differentiated (``create_graph``) takes the same formula as a composition of torch ops, and so do both directions under derivatives of forward mode, function
transforms (``torch.func``) and while a graph of torch's operations is recorded (``torch.jit.trace``, ``make_fx``).

``rms_norm_int8`` gives y in 8 bits with one scale per row -- the left operand of ``ops.int8.matmul`` -- in the same single pass: y is never written in its own type.
It serves inference and has no gradient.

Statistics are fp32 whatever the rows' type (fp32, fp16, bf16), fp64 for rows whose squares leave fp32's range; eps and 1 / rms are fp32 numbers.  CPU tensors take the plain
torch formulation.
"""
import torch
import torch.autograd.forward_ad as _fwd

from .. import custom_ops

_DTYPE_CODES = {torch.float32: custom_ops.SGV_F32, torch.float16: custom_ops.SGV_F16, torch.bfloat16: custom_ops.SGV_BF16}


def check_no_grad(what, *tensors):
    for t in tensors:
        if t is None:
            continue
        if torch.is_grad_enabled() and t.requires_grad:
            raise RuntimeError(f'{what} serves inference and has no gradient: call it under torch.no_grad() or with detached tensors')
        if _fwd.unpack_dual(t).tangent is not None:
            raise RuntimeError(f'{what} serves inference and has no gradient, of forward mode neither: call it with detached tensors')


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


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def rms_norm_ref(x, weight=None, residual=None, eps=1e-8):
    """The definition, in torch ops.  The norm is fp64: squares of what fp32 and bf16 hold leave fp32's range."""
    h = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
    hd = h.double()
    y = hd * (hd.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    y = y if x.dtype == torch.float64 else y.float()
    if weight is not None:
        y = y * _wide(weight)
    y = y.to(x.dtype)
    return y if residual is None else (y, h)


def rms_norm(x, weight=None, residual=None, eps=1e-8):
    """x [..., K], weight [K] (x's type or fp32) or None, residual like x or None -> y like x; with a residual (y, h), h = x + residual."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        ops = custom_ops.get_row_ops()
        try:
            out = ops.rms_norm(x, weight, residual, eps)
        except ops.Watched:
            _check('rms_norm', x, weight, residual, eps)
            return rms_norm_ref(x, weight, residual, eps)
        except (ops.Refused, TypeError):
            _check('rms_norm', x, weight, residual, eps)
            raise
        return out[0] if residual is None else out
    _check('rms_norm', x, weight, residual, eps)
    return rms_norm_ref(x, weight, residual, eps)


def quantize_ref(u, factor):
    """(q, scale) of rows u in fp64: q = 127 u / max|u| to nearest even, scale = max|u| * factor / 127; a row with a NaN or an infinity: NaN and zeros."""
    top = u.abs().amax(dim=-1, keepdim=True)
    fine = torch.isfinite(top) & (top > 0)
    q = torch.where(fine, torch.round(u * 127.0 / torch.where(fine, top, torch.ones_like(top))), torch.zeros_like(u))
    scale = torch.where(torch.isfinite(top), top * factor / 127.0, torch.full_like(top, float('nan')))
    return q.to(torch.int8), scale.squeeze(-1).float()


def rms_norm_int8(x, weight=None, residual=None, eps=1e-8):
    """``rms_norm`` with y in 8 bits: (q [..., K] int8, scale [...] fp32), with a residual (q, scale, h).  y stands for q * scale: scale = max|y| / 127 of each row and
    q = y / scale rounded to nearest even (of the exact quotient).  A row of zeros has scale 0 (NaN under eps = 0, as its y); a row with a NaN or an infinity in y has scale NaN and q = 0.
    The rows of q start on 16 bytes (q is a view of wider storage where K is no multiple of 16), as ``ops.int8.matmul`` wants them."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        out = launch_int8('rms_norm_int8', x, weight, residual, eps, True)
        return out[:2] if residual is None else out
    _check('rms_norm_int8', x, weight, residual, eps)
    check_no_grad('rms_norm_int8', x, weight, residual)
    h = x if residual is None else (_wide(x) + _wide(residual)).to(x.dtype)
    u = h.double()
    factor = (u.square().mean(dim=-1, keepdim=True) + eps).rsqrt()
    q, scale = quantize_ref(u if weight is None else u * weight.double(), factor)
    return (q, scale) if residual is None else (q, scale, h)


def launch_int8(what, x, weight, residual, eps, normalize):
    """(q, scale, h or None) of a GPU tensor."""
    ops = custom_ops.get_row_ops()
    try:
        return ops.rms_norm_int8(x, weight, residual, eps, normalize)
    except ops.Watched as seen:
        raise RuntimeError(f'{what} {seen}') from None
    except (ops.Refused, TypeError):
        _check(what, x, weight, residual, eps)
        check_no_grad(what, x, weight, residual)
        raise
