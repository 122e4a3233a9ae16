"""Cases of the row norm and the 8-bit integer product: the calls that are timed, and their plain forms.

`run` with ``own = False`` computes an operator from elementary torch operations; with ``own = True`` it makes the calls a user makes of
``stylegan_v_amd.torch_utils.ops.rms_norm`` and ``stylegan_v_amd.torch_utils.ops.int8``.

Kinds of cases (a case is a dict of plain values):

``norm``     training: y = rms_norm(x + residual, weight), with the gradients of x (which is the residual's too) and of the weight
``norm8``    serving: the same norm with an 8-bit output and one scale per row, returned as the values it stands for, beside the residual stream
``product``  8-bit integers [rows, inner] x [cols, inner]^T with one scale per row of either, bias, activation
``dense``    the operators together, as the mapping network of the generator is served in 8 bits: norm -> product -> quantise -> product ...
"""
import math

import torch

own = False

EPS = 1e-8                                   # of the framework's normalize_2nd_moment
TYPES = {'float32': torch.float32, 'float16': torch.float16, 'bfloat16': torch.bfloat16}
SIZE = {'float32': 4, 'float16': 2, 'bfloat16': 2}


def listed():
    return [
        # the latents of one batch of 32 videos at the mapping network's input, in training: a few microseconds of work, bound by the launches
        dict(name='norm_mapping_input', kind='norm', rows=32, cols=512, type='float32', weight=False, residual=False),
        # odd everything: rows that are no multiple of a vector load, a padded batch (its last rows are zeros)
        dict(name='norm_odd_rows', kind='norm', rows=2049, cols=1111, type='float16', weight=True, residual=True),
        # a training batch of token rows in the usual 16-bit type
        dict(name='norm_training_batch', kind='norm', rows=16384, cols=4096, type='bfloat16', weight=True, residual=True),
        # one token of a served model: latency
        dict(name='norm8_one_token', kind='norm8', rows=1, cols=4096, type='bfloat16', weight=True, residual=True),
        # odd sizes in 32 bits, no residual
        dict(name='norm8_odd_rows', kind='norm8', rows=300, cols=1111, type='float32', weight=True, residual=False),
        # a long prompt: the largest stream that is normed and quantised
        dict(name='norm8_prompt', kind='norm8', rows=8192, cols=8192, type='bfloat16', weight=True, residual=True),
        # one token through a large layer: the weight is read once, nothing else counts
        dict(name='product_one_token', kind='product', rows=1, cols=8192, inner=8192, type='bfloat16', bias=False, act='linear'),
        # the dense layer of the discriminator's epilogue (512 channels x 4 x 4 -> 512) on a batch of 32: few rows, a long sum
        dict(name='product_epilogue_head', kind='product', rows=32, cols=512, inner=8192, type='float32', bias=True, act='lrelu'),
        # ten thousand latents through one mapping layer (the estimate of the mean w), rows not a multiple of a tile
        dict(name='product_mapping_layer', kind='product', rows=10007, cols=512, inner=512, type='float32', bias=True, act='lrelu'),
        # nothing divides anything
        dict(name='product_odd', kind='product', rows=777, cols=1001, inner=1030, type='float16', bias=True, act='linear'),
        # a long prompt through a large square layer: the matrix pipe's rate
        dict(name='product_prompt', kind='product', rows=8192, cols=8192, inner=8192, type='bfloat16', bias=False, act='linear'),
        # the two mapping layers served in 8 bits, for a batch of 1024 latents
        dict(name='dense_mapping_network', kind='dense', rows=1024, width=512, layers=2, type='bfloat16'),
    ]


def _spread(rng, lo, hi):
    """A whole number spread over its logarithm; every other one is rounded to a multiple of 64 where it is large enough."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if v >= 96 and rng.random() < 0.5:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choice(['norm', 'norm8', 'product', 'product', 'dense'])
    kind_type = rng.choice(sorted(TYPES))
    if kind in ('norm', 'norm8'):
        cols = _spread(rng, 8, 16384)
        rows = _spread(rng, 1, max(2, min(32768, 16384 * 2048 // cols)))
        return dict(kind=kind, rows=rows, cols=cols, type=kind_type, weight=rng.random() < 0.8, residual=rng.random() < 0.6)
    if kind == 'product':
        return dict(kind=kind, rows=_spread(rng, 1, 8192), cols=_spread(rng, 8, 8192), inner=_spread(rng, 16, 8192), type=kind_type, bias=rng.random() < 0.5,
                    act=rng.choice(['linear', 'lrelu']))
    return dict(kind='dense', rows=_spread(rng, 1, 8192), width=_spread(rng, 32, 1024), layers=rng.choice([1, 2, 3]), type=rng.choice(['bfloat16', 'float16']))


def _int8_rows(rows, inner, g, device):
    """Rows of whole numbers as a quantiser leaves them (bell-shaped, clipped to +-127), in storage whose rows start on 16 bytes."""
    pitch = (inner + 15) // 16 * 16
    v = torch.randn([rows, pitch], generator=g, device=device).mul_(127.0 / 4.0).round_().clamp_(-127, 127).to(torch.int8)
    v[:, inner:] = 0
    return v[:, :inner]


def prepare(case, seed):
    device = 'cuda' if torch.cuda.is_available() else 'cpu'
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(*size, scale=1.0, shift=0.0):
        return torch.randn(list(size), generator=g, device=device).mul_(scale).add_(shift)

    s = dict(case=case)
    kind = case['kind']
    if kind in ('norm', 'norm8'):
        t, rows, cols = TYPES[case['type']], case['rows'], case['cols']
        wide = torch.exp(normal(cols, scale=0.5))                       # some channels are several times larger than others
        s['x'] = (normal(rows, cols) * wide).to(t)
        if case['residual']:
            s['residual'] = (normal(rows, cols, scale=2.0) * wide).to(t)
        if case['weight']:
            s['weight'] = normal(cols, scale=0.2, shift=1.0).to(t)
        if rows >= 64:                                                  # the padding of a batch: rows of zeros
            for name in ('x', 'residual'):
                if name in s:
                    s[name][rows - rows // 50:] = 0
        if kind == 'norm':
            s['dy'] = normal(rows, cols).to(t)
            if case['residual']:
                s['dh'] = normal(rows, cols).to(t)
            if own:                                                     # leaves of an autograd graph, as a training program holds them
                for name in ('x', 'residual', 'weight'):
                    if name in s:
                        s[name].requires_grad_(True)
    elif kind == 'product':
        rows, cols, inner = case['rows'], case['cols'], case['inner']
        s['a'], s['b'] = _int8_rows(rows, inner, g, device), _int8_rows(cols, inner, g, device)
        s['a_scale'] = torch.rand([rows], generator=g, device=device).mul_(0.02).add_(0.01)
        s['b_scale'] = torch.rand([cols], generator=g, device=device).add_(0.5).mul_(0.03 / math.sqrt(inner))
        if case['bias']:
            s['bias'] = normal(cols, scale=0.1)
    else:
        width = case['width']
        s['x'] = normal(case['rows'], width).to(TYPES[case['type']])
        s['stack'] = [(_int8_rows(width, width, g, device), torch.rand([width], generator=g, device=device).add_(0.5).mul_(0.03 / math.sqrt(width)), normal(width, scale=0.1))
                      for _ in range(case['layers'])]
    return s


# ---------------------------------------------------------------------------------------------------------------------------------------
# the plain forms

def _activate(v, act):
    return torch.where(v > 0, v, v * 0.2) * math.sqrt(2) if act == 'lrelu' else v


def _plain_stream(x, residual):
    """x + residual, rounded to the tensors' type: the residual stream, which is a tensor of that type, and what the norm sees."""
    return x if residual is None else (x.float() + residual.float()).to(x.dtype)


def _plain_inverse(h):
    return torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS)


def _plain_quantise(u, peak):
    """(whole numbers, scale) of rows u with the largest magnitude `peak` of what they stand for.  In 64 bits: a value halfway between two whole numbers has to be seen as one."""
    u = u.double()
    top = u.abs().amax(dim=1, keepdim=True)
    q = torch.where(top > 0, torch.round(u * 127.0 / top), torch.zeros_like(u))
    return q.float(), (peak / 127.0).float()


def _plain_norm8(x, weight, residual):
    h = _plain_stream(x, residual)
    u = h.double() if weight is None else h.double() * weight.double()
    y = u.float() * _plain_inverse(h.float())
    q, scale = _plain_quantise(u, y.abs().amax(dim=1, keepdim=True))
    return h, q, scale


def _plain_product(a, a_scale, b, b_scale, bias, act, t):
    v = (a.float() @ b.float().t()) * a_scale[:, None] * b_scale[None, :]
    if bias is not None:
        v = v + bias[None, :]
    return _activate(v, act).to(t)


def _plain_norm(s):
    x, weight, residual, dy = s['x'], s.get('weight'), s.get('residual'), s['dy']
    h = _plain_stream(x, residual)
    hf, gf = h.float(), dy.float()
    inverse = _plain_inverse(hf)
    xh = hf * inverse
    y = xh if weight is None else xh * weight.float()
    out = dict(y=y.to(x.dtype))
    if weight is not None:
        out['dweight'] = (gf * xh).sum(dim=0).to(weight.dtype)
        gf = gf * weight.float()
    dx = inverse * (gf - xh * (gf * xh).mean(dim=1, keepdim=True))
    if residual is not None:
        dx = dx + s['dh'].float()
        out['h'] = h
    out['dx'] = dx.to(x.dtype)
    return out


def _run_plain(s):
    case = s['case']
    kind = case['kind']
    if kind == 'norm':
        return _plain_norm(s)
    if kind == 'norm8':
        h, q, scale = _plain_norm8(s['x'], s.get('weight'), s.get('residual'))
        out = dict(values=q * scale)
        if 'residual' in s:
            out['h'] = h
        return out
    if kind == 'product':
        return _plain_product(s['a'], s['a_scale'], s['b'], s['b_scale'], s.get('bias'), case['act'], TYPES[case['type']])
    x, t = s['x'], TYPES[case['type']]
    for i, (b, b_scale, bias) in enumerate(s['stack']):
        if i == 0:
            _, q, scale = _plain_norm8(x, None, None)
        else:
            q, scale = _plain_quantise(x, x.float().abs().amax(dim=1, keepdim=True))
        x = _plain_product(q, scale[:, 0], b, b_scale, bias, 'lrelu', t)
    return x


# ---------------------------------------------------------------------------------------------------------------------------------------
# the framework's calls

def _run_own(s):
    from stylegan_v_amd.torch_utils.ops import int8, rms_norm
    case = s['case']
    kind = case['kind']
    if kind == 'norm':
        x, weight, residual = s['x'], s.get('weight'), s.get('residual')
        if residual is None:
            y = rms_norm.rms_norm(x, weight=weight, eps=EPS)
            outs, grads, out = [y], [s['dy']], dict(y=y.detach())
        else:
            y, h = rms_norm.rms_norm(x, weight=weight, residual=residual, eps=EPS)
            outs, grads, out = [y, h], [s['dy'], s['dh']], dict(y=y.detach(), h=h.detach())
        leaves = [t for t in (x, residual, weight) if t is not None]
        found = torch.autograd.grad(outs, leaves, grads)
        out['dx'] = found[0]
        if weight is not None:
            out['dweight'] = found[-1]
        return out
    if kind == 'norm8':
        got = rms_norm.rms_norm_int8(s['x'], weight=s.get('weight'), residual=s.get('residual'), eps=EPS)
        out = dict(values=int8.dequantize_rows(got[0], got[1], dtype=torch.float32))
        if 'residual' in s:
            out['h'] = got[2]
        return out
    if kind == 'product':
        return int8.matmul(s['a'], s['a_scale'], s['b'], s['b_scale'], bias=s.get('bias'), act=case['act'], dtype=TYPES[case['type']])
    x = s['x']
    for i, (b, b_scale, bias) in enumerate(s['stack']):
        x = int8.dense(x, b, b_scale, bias=bias, act='lrelu', normalize=(i == 0))
    return x


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------------------------------------------

def work(case):
    kind = case['kind']
    if kind in ('norm', 'norm8'):
        n, t = case['rows'] * case['cols'], SIZE[case['type']]
        streams = 2 if case['residual'] else 1                                  # x, residual
        w = case['cols'] * t if case['weight'] else 0
        if kind == 'norm':
            moved = n * t * (streams + 1 + 1 + 1) + (2 * n * t if case['residual'] else 0) + 2 * w      # x (residual) dy -> y dx; dh -> h; weight and its gradient
            return dict(bytes=moved, flops=12 * n)
        return dict(bytes=n * (t * streams + 4 + (t if case['residual'] else 0)) + w, flops=8 * n)       # ... -> values, h
    if kind == 'product':
        m, n, k = case['rows'], case['cols'], case['inner']
        return dict(bytes=m * k + n * k + m * n * SIZE[case['type']] + 4 * (m + n + (n if case['bias'] else 0)), flops=2 * m * n * k)
    m, n, depth = case['rows'], case['width'], case['layers']
    return dict(bytes=2 * m * n * SIZE[case['type']] + depth * (n * n + 8 * n), flops=2 * m * n * n * depth)


def exact(case, seed):
    """From the definitions, in 64 bits.  (The residual stream, the layers' outputs and the whole numbers are what they are defined as: tensors of the case's type, 8-bit values.)"""
    s = prepare(case, seed)
    t = TYPES[case['type']]
    f64 = torch.float64

    def wide(name):
        v = s.get(name)
        return None if v is None else v.detach().to(f64)

    def eight(u, factor):
        """Rows u: values of the 8-bit grid whose last step is the row's largest magnitude, times `factor` (one per row)."""
        step = u.abs().max(dim=1).values / 127
        whole = torch.zeros_like(u)
        some = step > 0
        biggest = u[some].abs().max(dim=1).values
        whole[some] = ((u[some] * 127) / biggest.unsqueeze(1)).round()
        return whole * (step * factor).unsqueeze(1)

    if case['kind'] in ('norm', 'norm8'):
        stream = wide('x')
        if case['residual']:
            stream = (stream + wide('residual')).to(t).to(f64)
        gamma = wide('weight') if case['weight'] else torch.ones(case['cols'], dtype=f64, device=stream.device)
        power = torch.linalg.vector_norm(stream, dim=1) ** 2 / case['cols'] + EPS
        if case['kind'] == 'norm8':
            out = dict(values=eight(stream * gamma, power ** -0.5))
        else:
            dy = wide('dy')
            out = dict(y=stream / power.sqrt().unsqueeze(1) * gamma)
            # dL/dh_j = dy_j w_j / sigma - h_j (sum_k dy_k w_k h_k) / (K sigma^3)
            along = torch.sum(dy * gamma * stream, dim=1) / (case['cols'] * power ** 1.5)
            dx = dy * gamma / power.sqrt().unsqueeze(1) - stream * along.unsqueeze(1)
            out['dx'] = dx + wide('dh') if case['residual'] else dx
            if case['weight']:
                out['dweight'] = torch.sum(dy * stream / power.sqrt().unsqueeze(1), dim=0)
        if case['residual']:
            out['h'] = stream
        return out

    def layer(left, right, right_scale, bias, act):
        v = torch.matmul(left, (right.to(f64) * right_scale.to(f64).unsqueeze(1)).t().contiguous())
        if bias is not None:
            v = v + bias.to(f64)
        return torch.maximum(v, v / 5) * math.sqrt(2.0) if act == 'lrelu' else v

    if case['kind'] == 'product':
        return layer(wide('a') * wide('a_scale').unsqueeze(1), s['b'], s['b_scale'], s.get('bias'), case['act'])
    x = wide('x')
    for i, (b, b_scale, bias) in enumerate(s['stack']):
        x = eight(x, (x.pow(2).mean(dim=1) + EPS).rsqrt() if i == 0 else torch.ones_like(x[:, 0]))
        x = layer(x, b, b_scale, bias, 'lrelu')
        if i + 1 < case['layers']:
            x = x.to(t).to(f64)
    return x
