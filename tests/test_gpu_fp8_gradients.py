"""The 8-bit operators have no derivative: every tensor operand that autograd would have to follow,
backward or forward, is refused, and the same operands are taken where it does not."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD

import fp8_cases as F
from src import gpu_ops as G

pytestmark = pytest.mark.gpu

M, N, K = 5, 144, 256


def _operands():
    gen = torch.Generator().manual_seed(0)
    a = F.torch_rows(torch.randn(M, K, generator=gen).cuda())
    w, u = (F.torch_blocks(torch.randn(N, K, generator=gen).bfloat16().cuda()) for _ in range(2))
    x, y = (torch.randn(M, K, generator=gen).bfloat16().cuda() for _ in range(2))
    weight = torch.ones(K, device='cuda').bfloat16()
    flat = lambda *groups: [t for g in groups for t in (g if isinstance(g, tuple) else (g,))]
    return {
        'quantize': (flat(x), lambda x: G.fp8_quantize(x)),
        'quantize_weight': (flat(x), lambda x: G.fp8_quantize_weight(x)),
        'norm': (flat(x, y, weight), lambda x, y, w: G.add_rms_fp8(x, y, w, 1e-5)),
        'linear': (flat(a, w), lambda q, s, w, ws: G.fp8_linear((q, s), (w, ws))),
        'gate_up': (flat(a, w, u), lambda q, s, g, gs, u, us: G.fp8_gate_up((q, s), (g, gs), (u, us))),
    }


CASES = [(op, i) for op, n in (('quantize', 1), ('quantize_weight', 1), ('norm', 3), ('linear', 4), ('gate_up', 6))
         for i in range(n)]


@pytest.mark.parametrize('op,i', CASES)
def test_an_operand_that_requires_a_gradient(cuda, op, i):
    operands, call = _operands()[op]
    operands[i] = operands[i].detach().clone().requires_grad_()
    with pytest.raises(ValueError, match='backward'):
        call(*operands)
    with torch.no_grad():
        call(*operands)
    call(*(t.detach() for t in operands))


@pytest.mark.parametrize('op,i', CASES)
def test_an_operand_with_a_tangent(cuda, op, i):
    operands, call = _operands()[op]
    primal = operands[i]
    tangent = torch.ones_like(primal, dtype=torch.float32).to(primal.dtype)
    with fwAD.dual_level():
        operands[i] = fwAD.make_dual(primal, tangent)
        with pytest.raises(ValueError, match='tangent'):
            call(*operands)
        with torch.no_grad(), pytest.raises(ValueError, match='tangent'):  # no_grad leaves tangents on
            call(*operands)
        with torch.inference_mode():
            call(*operands)
