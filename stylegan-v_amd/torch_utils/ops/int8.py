"""Dense layers in 8-bit integers (csrc/int8_gemm.hip, csrc/rms_norm.hip): rows quantised with one scale each, and their matrix product.

    quantize_rows(x)                          -> q int8, scale = max|x| / 127 per row
    matmul(a, a_scale, b, b_scale, ...)       -> act((a b^T) * a_scale * b_scale + bias) * act_gain
    dense(x, weight, weight_scale, ...)       -> FullyConnectedLayer.forward (src/training/layers.py:108-138) with 8-bit operands

A weight is quantised once (``quantize_rows(weight)``: one scale per output channel), activations at every call (one scale per token).  The sums are exact 32-bit integers,
so a result depends neither on how the product is split nor on the other rows of a batch; scales, bias and activation are applied in fp32, rounded once to the output's type.
All of it serves inference and has no gradient.  CPU tensors take the plain torch formulation.  On the GPU a call is a launch that torch's tracers and function transforms
would not see: it refuses them.
"""
import torch

from .. import custom_ops
from . import bias_act as _ba
from . import rms_norm as _rn

max_inner = 131071     # 128 * 128 * K has to fit in a signed 32-bit sum
_acts = {name: (spec.cuda_idx, spec.def_alpha, spec.def_gain) for name, spec in _ba.activation_funcs.items() if name in ('linear', 'lrelu')}


def quantize_rows(x):
    """x [..., K] -> (q [..., K] int8, scale [...] fp32): x stands for q * scale, q = x / scale to nearest even; zero and non-finite rows as in ``rms_norm_int8``.
    The rows of q start on 16 bytes, as ``matmul`` wants them."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        return _rn.launch_int8('quantize_rows', x, None, None, 0.0, False)[:2]
    _rn._check('quantize_rows', x, None, None, 0.0)
    _rn.check_no_grad('quantize_rows', x)
    return _rn.quantize_ref(x.double(), 1.0)


def dequantize_rows(q, scale, dtype=torch.float32):
    """q [..., K] int8, scale [...] fp32 -> q * scale in ``dtype``, dense."""
    if isinstance(q, torch.Tensor) and q.is_cuda:
        ops = custom_ops.get_row_ops()
        try:
            return ops.dequantize_rows(q, scale, _rn._DTYPE_CODES[dtype])
        except ops.Watched as seen:
            raise RuntimeError(f'dequantize_rows {seen}') from None
        except (ops.Refused, TypeError, KeyError):
            _check_dequantize(q, scale, dtype)
            raise
    _check_dequantize(q, scale, dtype)
    return (q.float() * scale.unsqueeze(-1)).to(dtype)


def _check_rows(what, name, q, scale):
    if not isinstance(q, torch.Tensor) or q.dtype != torch.int8 or q.ndim < 1 or q.shape[-1] < 1:
        raise RuntimeError(f'{what}: {name} must be int8 rows (at least one dimension, the last one not empty)')
    if scale.dtype != torch.float32 or scale.shape != q.shape[:-1] or scale.device != q.device:
        raise RuntimeError(f'{what}: the scales of {name} must be fp32, one per row, on its device')


def _check_dequantize(q, scale, dtype):
    _check_rows('dequantize_rows', 'q', q, scale)
    if dtype not in _rn._DTYPE_CODES:
        raise RuntimeError(f'dequantize_rows: unsupported dtype {dtype}')
    _rn.check_no_grad('dequantize_rows', scale)


def _check_layer(what, cols, device, b, b_scale, bias, dtype, act):
    _check_rows(what, 'b', b, b_scale)
    if b.ndim != 2 or b.shape[1] != cols or b.device != device:
        raise RuntimeError(f'{what}: b must be [N, K] with the K of a, on the device of a')
    if cols > max_inner:
        raise RuntimeError(f'{what}: K is at most {max_inner} (a sum of 128 * 128 * K has to fit in 32 bits)')
    if dtype not in _rn._DTYPE_CODES:
        raise RuntimeError(f'{what}: unsupported dtype {dtype}')
    if act not in _acts:
        raise RuntimeError(f'{what}: unsupported activation {act}')
    if bias is not None and (bias.ndim != 1 or bias.shape[0] != b.shape[0] or bias.dtype != torch.float32 or bias.device != device):
        raise RuntimeError(f'{what}: bias must be fp32, one element per row of b, on the device of a')


def _check_matmul(a, a_scale, b, b_scale, bias, dtype, act):
    _check_rows('matmul', 'a', a, a_scale)
    _check_layer('matmul', a.shape[-1], a.device, b, b_scale, bias, dtype, act)
    _rn.check_no_grad('matmul', a_scale, b_scale, bias)


def _matmul_ref(a, a_scale, b, b_scale, bias, act, gain, dtype):
    v = torch.matmul(a.double(), b.double().t()) * a_scale.double().unsqueeze(-1) * b_scale.double()     # (whole numbers below 2^53: exact)
    if bias is not None:
        v = v + bias.double()
    if act == 'lrelu':
        v = torch.where(v > 0, v, v * _ba.activation_funcs[act].def_alpha)
    return (v * gain).to(dtype)


def matmul(a, a_scale, b, b_scale, bias=None, act='linear', act_gain=None, dtype=torch.float32):
    """a [..., K] int8 with a_scale [...], b [N, K] int8 with b_scale [N], bias [N] or None -> [..., N] in ``dtype`` (fp32, fp16, bf16).
    ``act``: 'linear' or 'lrelu'; ``act_gain``: its gain (default: the activation's own, sqrt(2) for lrelu).  Rows of a and b that start on 16 bytes and can be read up to
    the next multiple of 16 columns are taken as they are, others are copied first."""
    if isinstance(a, torch.Tensor) and a.is_cuda:
        ops = custom_ops.get_row_ops()
        try:
            kind, alpha, gain = _acts[act]
            return ops.matmul(a, a_scale, b, b_scale, bias, kind, alpha, gain if act_gain is None else act_gain, _rn._DTYPE_CODES[dtype])
        except ops.Watched as seen:
            raise RuntimeError(f'matmul {seen}') from None
        except (ops.Refused, TypeError, KeyError):
            _check_matmul(a, a_scale, b, b_scale, bias, dtype, act)
            raise
    _check_matmul(a, a_scale, b, b_scale, bias, dtype, act)
    return _matmul_ref(a, a_scale, b, b_scale, bias, act, _acts[act][2] if act_gain is None else act_gain, dtype)


def dense(x, weight, weight_scale, bias=None, act='linear', act_gain=None, normalize=False, eps=1e-8):
    """x [..., K] fp32 / fp16 / bf16, weight [N, K] int8 with weight_scale [N] (``quantize_rows`` of the layer's weight), bias [N] fp32 -> [..., N] in x's type.
    ``normalize``: the rows of x through ``rms_norm`` (no weight) first, in the same pass that quantises them."""
    if isinstance(x, torch.Tensor) and x.is_cuda:
        ops = custom_ops.get_row_ops()
        try:
            kind, alpha, gain = _acts[act]
            return ops.dense(x, weight, weight_scale, bias, kind, alpha, gain if act_gain is None else act_gain, normalize, eps)
        except ops.Watched as seen:
            raise RuntimeError(f'dense {seen}') from None
        except (ops.Refused, TypeError, KeyError):
            _rn._check('dense', x, None, None, eps)
            _check_layer('dense', x.shape[-1], x.device, weight, weight_scale, bias, x.dtype, act)
            _rn.check_no_grad('dense', x, weight_scale, bias)
            raise
    q, scale = _rn.rms_norm_int8(x, eps=eps) if normalize else quantize_rows(x)
    return matmul(q, scale, weight, weight_scale, bias=bias, act=act, act_gain=act_gain, dtype=x.dtype)
