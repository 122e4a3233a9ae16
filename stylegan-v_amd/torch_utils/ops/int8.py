"""Dense layers in 8-bit integers (csrc/int8_gemm.hip, csrc/rms_norm.hip): rows quantised with one scale each, and their matrix product.

    quantize_rows(x)                          -> q int8, scale = max|x| / 127 per row
    matmul(a, a_scale, b, b_scale, ...)       -> act((a b^T) * a_scale * b_scale + bias) * act_gain
    dense(x, weight, weight_scale, ...)       -> FullyConnectedLayer.forward (src/training/layers.py:108-138) with 8-bit operands

A weight is quantised once (``quantize_rows(weight)``: one scale per output channel), activations at every call (one scale per token).  The sums are exact 32-bit integers,
so a result depends neither on how the product is split nor on the other rows of a batch; scales, bias and activation are applied in fp32, rounded once to the output's type.
All of it serves inference and has no gradient.  CPU tensors take the plain torch formulation.
"""
import torch

from .. import custom_ops
from . import bias_act as _ba
from . import rms_norm as _rn

_gemm = custom_ops.PackedEntry('sgv_int8_gemm', custom_ops.Int8GemmParams)
max_inner = 131071     # 128 * 128 * K has to fit in a signed 32-bit sum
max_stride = 1 << 23   # bytes between two rows that the product takes as they are


def quantize_rows(x):
    """x [..., K] -> (q [..., K] int8, scale [...] fp32): x stands for q * scale, q = x / scale to nearest even; zero and non-finite rows as in ``rms_norm_int8``.
    The rows of q start on 16 bytes, as ``matmul`` wants them."""
    _rn._check('quantize_rows', x, None, None, 0.0)
    _rn.check_no_grad('quantize_rows', x)
    if not x.is_cuda:
        return _rn.quantize_ref(x.double(), 1.0)
    q, _, _, scale = _rn.launch_forward(_rn.row_view(x), None, None, 0.0, int8=True, normalize=False)
    if x.ndim != 2:
        q, scale = q.unflatten(0, x.shape[:-1]) if x.ndim > 2 else q[0], scale.view(x.shape[:-1])
    return q, scale


def dequantize_rows(q, scale, dtype=torch.float32):
    """q [..., K] int8, scale [...] fp32 -> q * scale in ``dtype``, dense."""
    _check_rows('dequantize_rows', 'q', q, scale)
    if dtype not in _rn._DTYPE_CODES:
        raise RuntimeError(f'dequantize_rows: unsupported dtype {dtype}')
    _rn.check_no_grad('dequantize_rows', scale)
    if not q.is_cuda:
        return (q.float() * scale.unsqueeze(-1)).to(dtype)
    out = q.new_empty(q.shape, dtype=dtype)
    rows = _rn.row_view(q)
    if rows.shape[0]:
        scale = _rn._dense(scale)
        lib = custom_ops.get_native()
        with custom_ops.device_guard(q):
            custom_ops.check(lib.sgv_dequantize_rows(rows.data_ptr(), rows.stride(0), scale.data_ptr(), out.data_ptr(), rows.shape[0], rows.shape[1], _rn._DTYPE_CODES[dtype],
                                                     custom_ops.raw_stream(q)), lib)
    return out


def _check_rows(what, name, q, scale):
    if not isinstance(q, torch.Tensor) or q.dtype != torch.int8 or q.ndim < 1 or q.shape[-1] < 1:
        raise RuntimeError(f'{what}: {name} must be int8 rows (at least one dimension, the last one not empty)')
    if scale.dtype != torch.float32 or scale.shape != q.shape[:-1] or scale.device != q.device:
        raise RuntimeError(f'{what}: the scales of {name} must be fp32, one per row, on its device')


def _product_rows(q):
    """(tensor to keep, rows, row stride in bytes): the rows of q starting on 16 bytes and readable up to the next multiple of 16 columns -- q itself where it is so (what
    ``quantize_rows`` and ``rms_norm_int8`` return, and any dense K % 16 == 0 tensor), else a copy."""
    q = _rn.row_view(q)
    rows, cols = q.shape
    pitch = (cols + 15) // 16 * 16
    stride = q.stride(0) if rows > 1 else pitch
    if stride % 16 == 0 and stride < max_stride and q.data_ptr() % 16 == 0 and (cols == pitch or q.storage_offset() + (rows - 1) * stride + pitch <= q.untyped_storage().nbytes()):
        return q, rows, stride
    out = q.new_empty((rows, pitch))
    out[:, :cols].copy_(q)          # (what lies behind the last column is ignored)
    return out, rows, pitch


def _matmul_ref(a, a_scale, b, b_scale, bias, act, gain, dtype):
    v = torch.matmul(a.double(), b.double().t()) * a_scale.double().unsqueeze(-1) * b_scale.double()     # (whole numbers below 2^53: exact)
    if bias is not None:
        v = v + bias.double()
    if act == 'lrelu':
        v = torch.where(v > 0, v, v * _ba.activation_funcs[act].def_alpha)
    return (v * gain).to(dtype)


def _check_layer(what, cols, device, b, b_scale, bias, dtype, act):
    _check_rows(what, 'b', b, b_scale)
    if b.ndim != 2 or b.shape[1] != cols or b.device != device:
        raise RuntimeError(f'{what}: b must be [N, K] with the K of a, on the device of a')
    if cols > max_inner:
        raise RuntimeError(f'{what}: K is at most {max_inner} (a sum of 128 * 128 * K has to fit in 32 bits)')
    if dtype not in _rn._DTYPE_CODES:
        raise RuntimeError(f'{what}: unsupported dtype {dtype}')
    if act not in ('linear', 'lrelu'):
        raise RuntimeError(f'{what}: unsupported activation {act}')
    if bias is not None and (bias.ndim != 1 or bias.shape[0] != b.shape[0] or bias.dtype != torch.float32 or bias.device != device):
        raise RuntimeError(f'{what}: bias must be fp32, one element per row of b, on the device of a')


def _launch(a, m, lda, a_scale, b, b_scale, bias, act, act_gain, out):
    """out = the product of the rows of a (dense scales) with the rows of b."""
    n, cols = b.shape
    br, _, ldb = _product_rows(b)
    sb, bc = _rn._dense(b_scale), _rn._dense(bias)
    spec = _ba.activation_funcs[act]
    _gemm(out, _rn._DTYPE_CODES[out.dtype], a.data_ptr(), br.data_ptr(), a_scale.data_ptr(), sb.data_ptr(), _rn._ptr(bc), out.data_ptr(), lda, ldb, n, m, n, cols, spec.cuda_idx,
          spec.def_alpha, spec.def_gain if act_gain is None else act_gain)
    return out


def matmul(a, a_scale, b, b_scale, bias=None, act='linear', act_gain=None, dtype=torch.float32):
    """a [..., K] int8 with a_scale [...], b [N, K] int8 with b_scale [N], bias [N] or None -> [..., N] in ``dtype`` (fp32, fp16, bf16).
    ``act``: 'linear' or 'lrelu'; ``act_gain``: its gain (default: the activation's own, sqrt(2) for lrelu)."""
    _check_rows('matmul', 'a', a, a_scale)
    _check_layer('matmul', a.shape[-1], a.device, b, b_scale, bias, dtype, act)
    _rn.check_no_grad('matmul', a_scale, b_scale, bias)
    if not a.is_cuda:
        return _matmul_ref(a, a_scale, b, b_scale, bias, act, _ba.activation_funcs[act].def_gain if act_gain is None else act_gain, dtype)
    out = a.new_empty(a.shape[:-1] + b.shape[:1], dtype=dtype)
    if out.numel():
        rows, m, lda = _product_rows(a)
        _launch(rows, m, lda, _rn._dense(a_scale), b, b_scale, bias, act, act_gain, out)
    return out


def dense(x, weight, weight_scale, bias=None, act='linear', act_gain=None, normalize=False, eps=1e-8):
    """x [..., K] fp32 / fp16 / bf16, weight [N, K] int8 with weight_scale [N] (``quantize_rows`` of the layer's weight), bias [N] fp32 -> [..., N] in x's type.
    ``normalize``: the rows of x through ``rms_norm`` (no weight) first, in the same pass that quantises them."""
    if not x.is_cuda:
        q, scale = _rn.rms_norm_int8(x, eps=eps) if normalize else quantize_rows(x)
        return matmul(q, scale, weight, weight_scale, bias=bias, act=act, act_gain=act_gain, dtype=x.dtype)
    _rn._check('dense', x, None, None, eps)
    _check_layer('dense', x.shape[-1], x.device, weight, weight_scale, bias, x.dtype, act)
    _rn.check_no_grad('dense', x, weight_scale, bias)
    out = x.new_empty(x.shape[:-1] + weight.shape[:1])
    if out.numel():
        q, _, _, scale = _rn.launch_forward(_rn.row_view(x), None, None, eps, int8=True, normalize=normalize)
        _launch(q, q.shape[0], q.stride(0), scale, weight, weight_scale, bias, act, act_gain, out)
    return out
