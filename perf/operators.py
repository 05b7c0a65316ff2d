"""The 8-bit decoder operators as a user calls them, with plain forms in elementary torch operations.

The operators turn the projections around the packed attention to 8 bits. Numbers are
held as e4m3 with fp32 scales: activations with one scale per row and group of 128
columns, weights with one per block of 128 x 128.

    quantize   q, s = e4m3 rows of x
    norm       x + y, then RMSNorm and its weight, as e4m3 rows
    linear     C = A W^T of e4m3 rows and e4m3 weight blocks, in bf16 or fp32
    gate_up    silu(A G^T) * (A U^T) as e4m3 rows: the input of the down projection

A scale is max(amax of its group, 2^-100) / 448, and q = e4m3(x * 448 / amax): 448 is
the largest e4m3 value, and the floor keeps the quotients of a group of zeros finite.
"""
import functools
import math
import sys
from pathlib import Path

import torch

own = False

GROUP = 128
E4M3_MAX = 448.0
FLOOR = 2.0 ** -100
EPS = 1e-5
# no case computes or writes more than these (the largest listed products)
MOST_MACS = 4096 ** 3
MOST_OUT = 4096 * 5120


def listed():
    return [
        # the attention output of one 64-token frame, before the output projection
        dict(name='quantize frame', op='quantize', rows=64, width=960),
        # a long prompt's activations, MLP width: bandwidth
        dict(name='quantize prompt', op='quantize', rows=8191, width=2560),
        # the norm between two blocks of a decode step: latency
        dict(name='norm decode', op='norm', rows=1, width=960, residual=True),
        # the same for eight requests' 64-token frames stepped together
        dict(name='norm frames', op='norm', rows=512, width=960, residual=True),
        # a prompt at a generic large width, the first layer's form (no residual yet)
        dict(name='norm prompt', op='norm', rows=4097, width=4096, residual=False),
        # the joined QKV projection of one token
        dict(name='linear decode qkv', op='linear', rows=1, out=1600, width=960, dtype='bfloat16'),
        # the down projection of one 64-token frame
        dict(name='linear frame down', op='linear', rows=64, out=960, width=2560, dtype='bfloat16'),
        # fp32 logits over the vocabulary for a scored candidate (24 tokens and the one before)
        dict(name='linear logits', op='linear', rows=25, out=49280, width=960, dtype='float32'),
        # odd sizes: the last column group, tile and weight block are partial
        dict(name='linear ragged', op='linear', rows=333, out=1001, width=1040, dtype='bfloat16'),
        # a generic square product: the tensor cores' rate
        dict(name='linear square', op='linear', rows=4096, out=4096, width=4096, dtype='bfloat16'),
        # the MLP's joined gate / up of a scored candidate
        dict(name='gate_up candidate', op='gate_up', rows=25, out=2560, width=960),
        # the same for 64 frames of 64 tokens
        dict(name='gate_up frames', op='gate_up', rows=4096, out=2560, width=960),
    ]


def _log(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm."""
    return min(high, max(low, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(('quantize', 'norm', 'linear', 'linear', 'gate_up'))
    rows = _log(rng, 1, 8192)
    width = 16 * _log(rng, 1, 512)  # 16 to 8192: rows of q begin 16 bytes apart
    if op in ('quantize', 'norm'):
        rows = min(rows, 8191 * 2560 // width)
        case = dict(op=op, rows=rows, width=width)
        if op == 'norm':
            case['residual'] = rng.random() < 0.75
        return case
    out = _log(rng, 1, 49280) if op == 'linear' else 16 * _log(rng, 1, 512)
    macs = MOST_MACS if op == 'linear' else MOST_MACS // 2
    rows = max(1, min(rows, MOST_OUT // out, macs // (out * width)))
    case = dict(op=op, rows=rows, out=out, width=width)
    if op == 'linear':
        case['dtype'] = 'float32' if rng.random() < 0.25 else 'bfloat16'
    return case


# -- inputs -----------------------------------------------------------------------

def _activations(rows, width, gen):
    """Hidden states: normal, with a spread of channel sizes and a few large channels."""
    size = torch.exp(0.5 * torch.randn(width, generator=gen, device='cuda'))
    large = torch.rand(width, generator=gen, device='cuda') < 0.01
    return torch.randn(rows, width, generator=gen, device='cuda') * torch.where(large, 12.0 * size, size)


def _as_rows(x):
    """e4m3 rows with a scale per row and group of 128 columns, of a 32-bit x [rows, width]."""
    rows, width = x.shape
    groups = -(-width // GROUP)
    x = torch.nn.functional.pad(x, (0, groups * GROUP - width)).view(rows, groups, GROUP)
    amax = x.abs().amax(-1).clamp_min(FLOOR)
    q = (x * (E4M3_MAX / amax)[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.reshape(rows, groups * GROUP)[:, :width]
    return q.contiguous().to(torch.float8_e4m3fn), amax / E4M3_MAX


def _as_blocks(w):
    """e4m3 weights with a scale per 128 x 128 block, of a 32-bit w [out, width]."""
    out, width = w.shape
    a, b = -(-out // GROUP), -(-width // GROUP)
    w = torch.nn.functional.pad(w, (0, b * GROUP - width, 0, a * GROUP - out)).view(a, GROUP, b, GROUP)
    amax = w.abs().amax((1, 3)).clamp_min(FLOOR)
    q = (w * (E4M3_MAX / amax)[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    q = q.reshape(a * GROUP, b * GROUP)[:out, :width]
    return q.contiguous().to(torch.float8_e4m3fn), amax / E4M3_MAX


def _weights(out, width, gen):
    return _as_blocks(torch.randn(out, width, generator=gen, device='cuda') * width ** -0.5)


def prepare(case, seed):
    gen = torch.Generator(device='cuda').manual_seed(seed)
    op, rows, width = case['op'], case['rows'], case['width']
    x = _activations(rows, width, gen)
    if op == 'quantize':
        return dict(op=op, x=x.bfloat16())
    if op == 'norm':
        y = torch.randn(rows, width, generator=gen, device='cuda').bfloat16() if case['residual'] else None
        weight = (1 + 0.2 * torch.randn(width, generator=gen, device='cuda')).bfloat16()
        return dict(op=op, x=x.bfloat16(), y=y, weight=weight)
    state = dict(op=op, a=_as_rows(x))
    if op == 'linear':
        return dict(state, w=_weights(case['out'], width, gen), dtype=getattr(torch, case['dtype']))
    return dict(state, gate=_weights(case['out'], width, gen), up=_weights(case['out'], width, gen))


# -- one pass ---------------------------------------------------------------------

def _rows_values(a):
    """The 32-bit values that e4m3 rows stand for."""
    q, scale = a
    return q.float() * scale.repeat_interleave(GROUP, 1)[:, :q.shape[1]]


def _blocks_values(w):
    """The 32-bit values that e4m3 weight blocks stand for."""
    q, scale = w
    scale = scale.repeat_interleave(GROUP, 0)[:q.shape[0]].repeat_interleave(GROUP, 1)
    return q.float() * scale[:, :q.shape[1]]


def _plain(state):
    op = state['op']
    if op == 'quantize':
        return _as_rows(state['x'].float())
    if op == 'norm':
        # the residual stream itself is bf16: what the next block adds to is what is normed
        x = state['x'] if state['y'] is None else (state['x'].float() + state['y'].float()).bfloat16()
        v = x.float()
        h = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * state['weight'].float()
        q, scale = _as_rows(h)
        return (q, scale) if state['y'] is None else (x, q, scale)
    a = _rows_values(state['a'])
    if op == 'linear':
        return (a @ _blocks_values(state['w']).T).to(state['dtype'])
    g, u = a @ _blocks_values(state['gate']).T, a @ _blocks_values(state['up']).T
    return _as_rows(g / (1 + torch.exp(-g)) * u)


@functools.cache
def _ops():
    """The framework's operators, imported once as a user's program does."""
    package = str(Path(__file__).resolve().parent.parent / 'dynamic-kv-cache_b200')
    if package not in sys.path:
        sys.path.insert(0, package)
    from src import gpu_ops
    return gpu_ops


def run(state):
    if not own:
        return _plain(state)
    ops, op = _ops(), state['op']
    if op == 'quantize':
        return ops.fp8_quantize(state['x'])
    if op == 'norm':
        x, a = ops.add_rms_fp8(state['x'], state['y'], state['weight'], EPS)
        return a if state['y'] is None else (x, *a)
    if op == 'linear':
        return ops.fp8_linear(state['a'], state['w'], state['dtype'])
    return ops.fp8_gate_up(state['a'], state['gate'], state['up'])


# -- what a pass cannot do without ------------------------------------------------

def work(case):
    op, m, k = case['op'], case['rows'], case['width']
    groups = -(-k // GROUP)
    rows8 = m * k + 4 * m * groups  # e4m3 rows and their scales
    if op == 'quantize':
        return {'bytes': 2 * m * k + rows8, 'flops': 3 * m * k}
    if op == 'norm':
        added = 4 * m * k if case['residual'] else 0  # the other summand, and the sum
        return {'bytes': 2 * m * k + added + 2 * k + rows8, 'flops': 7 * m * k}
    n = case['out']
    blocks8 = n * k + 4 * -(-n // GROUP) * groups
    if op == 'linear':
        return {'bytes': rows8 + blocks8 + m * n * (4 if case['dtype'] == 'float32' else 2), 'flops': 2 * m * n * k}
    return {'bytes': rows8 + 2 * blocks8 + m * n + 4 * m * -(-n // GROUP), 'flops': 4 * m * n * k}


# -- the definitions in 64 bits ---------------------------------------------------
# An output held in 8 bits is given before its rounding to e4m3, as the others are
# given before theirs to bf16 or fp32.

def _exact_rows(x):
    columns = torch.arange(x.shape[1], device=x.device) // GROUP
    scale = torch.full((x.shape[0], int(columns[-1]) + 1), FLOOR, dtype=torch.float64, device=x.device)
    scale = scale.scatter_reduce(1, columns.expand_as(x), x.abs(), 'amax') / E4M3_MAX
    return x / scale[:, columns], scale


def _exact_product(a, w):
    (qa, sa), (qw, sw) = ([t.double() for t in pair] for pair in (a, w))
    out = torch.arange(qw.shape[0], device=qw.device) // GROUP
    total = torch.zeros(qa.shape[0], qw.shape[0], dtype=torch.float64, device=qa.device)
    for group in range(sa.shape[1]):  # each group's product has one scale per row and one per block
        columns = slice(group * GROUP, (group + 1) * GROUP)
        total += torch.einsum('mk,nk->mn', qa[:, columns], qw[:, columns]) * sa[:, group, None] * sw[out, group]
    return total


def exact(case, seed):
    state = prepare(case, seed)
    op = case['op']
    if op == 'quantize':
        return _exact_rows(state['x'].double())
    if op == 'norm':
        x = state['x'].double()
        if case['residual']:
            total = x + state['y'].double()
            x = total.bfloat16().double()  # the residual stream is bf16 by definition
        rms = (x.square().sum(-1, keepdim=True) / case['width'] + EPS).sqrt()
        q, scale = _exact_rows(x / rms * state['weight'].double())
        return (total, q, scale) if case['residual'] else (q, scale)
    if op == 'linear':
        return _exact_product(state['a'], state['w'])
    g, u = _exact_product(state['a'], state['gate']), _exact_product(state['a'], state['up'])
    return _exact_rows(torch.special.expit(g) * g * u)
