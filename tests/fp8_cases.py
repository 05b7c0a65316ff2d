"""64-bit forms of the 8-bit decoder operators and the tolerances their tests share.

Rounding: to e4m3 at most half a step, 2^-4 of a value of at least 2^-6 and 2^-10 below
(the step of the smallest binades is 2^-9); to the other types finfo.eps / 2 (bf16 2^-8,
fp32 2^-24). Sums: n products added in fp32 in any order are off by
at most n * 2^-23 of the sum of their magnitudes (2^-24 per rounding, twice that where an
adder truncates)."""
import torch

GROUP, TOP, FLOOR = 128, 448.0, 2.0 ** -100


def groups(width):
    return -(-width // GROUP)


def row_values(a):
    """The 64-bit values of e4m3 rows (q [..., k], scale [..., groups])."""
    q, s = a
    return q.double() * s.double().repeat_interleave(GROUP, -1)[..., :q.shape[-1]]


def block_values(w):
    q, s = w
    s = s.double().repeat_interleave(GROUP, 0)[:q.shape[0]].repeat_interleave(GROUP, 1)
    return q.double() * s[:, :q.shape[1]]


def row_scales(h):
    """The scale [..., groups] of each column group of 64-bit rows h."""
    pad = torch.nn.functional.pad(h, (0, groups(h.shape[-1]) * GROUP - h.shape[-1]))
    amax = pad.unflatten(-1, (-1, GROUP)).abs().amax(-1)
    return amax.clamp_min(FLOOR) / TOP


def _quotients(amax):
    """448 / amax and amax / 448, one IEEE division each (torch makes a product with a rounded
    reciprocal of a division by or of a number)."""
    top = torch.full_like(amax, TOP)
    return top / amax, amax / top


def torch_rows(x):
    """fp32 rows as e4m3 rows, every step one IEEE fp32 operation."""
    s = row_scales(x.double())
    amax = (s * TOP).float()
    inverse, scale = _quotients(amax)
    inverse = inverse.repeat_interleave(GROUP, -1)[..., :x.shape[-1]]
    return (x.float() * inverse).to(torch.float8_e4m3fn), scale


def torch_blocks(w):
    n, k = w.shape
    pad = torch.nn.functional.pad(w.float(), (0, groups(k) * GROUP - k, 0, groups(n) * GROUP - n))
    amax = pad.view(groups(n), GROUP, groups(k), GROUP).abs().amax((1, 3)).clamp_min(FLOOR)
    inverse, scale = _quotients(amax)
    inverse = inverse.repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]
    return (w.float() * inverse).to(torch.float8_e4m3fn), scale


def check_rows(actual, h, off):
    """e4m3 rows `actual` against the 64-bit values h they stand for, which the kernel's
    fp32 arithmetic may have missed by `off` (elementwise) before the one rounding."""
    q, s = actual
    exact = row_scales(h)
    reach = torch.nn.functional.pad(off, (0, groups(h.shape[-1]) * GROUP - h.shape[-1])).unflatten(-1, (-1, GROUP))
    # the largest magnitude may be off by its own error; amax / 448 is one more fp32 rounding
    assert ((s.double() - exact).abs() <= reach.amax(-1) / TOP + exact * 2 ** -23).all()
    # one step of the quotient's rounding, three fp32 roundings (448 / amax, the product, the scale)
    scale = s.double().repeat_interleave(GROUP, -1)[..., :h.shape[-1]]
    half = torch.maximum(h.abs() / scale, torch.tensor(2.0 ** -6, device=h.device).double()) * 2 ** -4
    bound = scale * half * (1 + 2 ** -20) + off * (1 + 2 ** -3) + h.abs() * 2 ** -22
    miss = (q.double() * scale - h).abs() - bound
    assert (miss <= 0).all(), float(miss.max())


def check_product(actual, a, w):
    """A linear layer's output against the 64-bit product of the values a and w stand for."""
    av, wv = row_values(a).flatten(0, -2), block_values(w)
    exact, mass = av @ wv.T, av.abs() @ wv.abs().T
    got = actual.double().flatten(0, -2)
    step = torch.finfo(actual.dtype).eps / 2
    bound = exact.abs() * step * (1 + 2 ** -10) + mass * (av.shape[1] + 8) * 2 ** -23
    miss = (got - exact).abs() - bound
    assert (miss <= 0).all(), float(miss.max())
    # the errors of n roundings do not line up over a whole matrix: sqrt(n) of them, in the 2-norm
    n = av.shape[1] + 8
    assert (got - exact).norm() <= exact.norm() * step + mass.norm() * n ** 0.5 * 2 ** -23


def check_gate_up(actual, a, gate, up):
    av, gv, uv = row_values(a).flatten(0, -2), block_values(gate), block_values(up)
    g, u = av @ gv.T, av @ uv.T
    n = (av.shape[1] + 8) * 2 ** -23
    dg, du = (av.abs() @ gv.abs().T) * n, (av.abs() @ uv.abs().T) * n
    h = g * torch.sigmoid(g) * u
    # |silu'| <= 1.1, |silu(g)| <= |g|; exp, the quotient and the product round a few times more
    off = 1.1 * dg * (u.abs() + du) + (g.abs() + dg) * du + h.abs() * 2 ** -20 + 2.0 ** -120
    check_rows(tuple(t.flatten(0, -2) for t in actual), h, off)
