"""GPU checks of the 8-bit products in the kernels, stage counts and splits that the plan chooses at
few tokens (test_fp8_plans_host.py: these lists and test_gpu_fp8_ops.py's reach every one of them)."""
import pytest
import torch

import fp8_cases as F
from src import gpu_ops as G

pytestmark = pytest.mark.gpu

# 16, 32 and 64 tokens a tile; three stages (more blocks than SMs) and four; one block a tile and several
LINEAR = [(1, 49280, 144), (9, 30001, 400), (25, 49280, 960), (31, 30002, 144), (17, 5121, 8192), (27, 8193, 4112), (20, 961, 8192),
          (64, 30001, 1040), (50, 2561, 8192)]
GATE_UP = [(129, 4096, 128), (128, 2560, 960), (256, 2560, 960), (33, 16384, 144), (200, 1600, 2048), (700, 5120, 272),
           (300, 960, 8192), (40, 5120, 4112), (20, 960, 8192), (129, 976, 8208)]


def _rows(gen, m, k):
    return F.torch_rows((torch.randn(m, k, generator=gen) * torch.exp(torch.randn(k, generator=gen))).cuda())


def _blocks(gen, n, k):
    return F.torch_blocks((torch.randn(n, k, generator=gen) * k ** -0.5).bfloat16().cuda())


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k', LINEAR)
def test_linear(cuda, m, n, k, dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    a, w = _rows(gen, m, k), _blocks(gen, n, k)
    out = G.fp8_linear(a, w, dtype)
    F.check_product(out, a, w)
    assert torch.equal(G.fp8_linear(a, w, dtype), out)


@pytest.mark.parametrize('m,n,k', GATE_UP)
def test_gate_up(cuda, m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    a, gate, up = _rows(gen, m, k), _blocks(gen, n, k), _blocks(gen, n, k)
    out = G.fp8_gate_up(a, gate, up)
    F.check_gate_up(out, a, gate, up)
    again = G.fp8_gate_up(a, gate, up)
    assert torch.equal(again.q.view(torch.uint8), out.q.view(torch.uint8)) and torch.equal(again.scale, out.scale)


@pytest.mark.parametrize('m,n,k', GATE_UP)
def test_a_row_of_nan_keeps_to_itself(cuda, m, n, k):
    gen = torch.Generator().manual_seed(m)
    (q, s), gate, up = _rows(gen, m, k), _blocks(gen, n, k), _blocks(gen, n, k)
    ref = G.fp8_gate_up((q, s), gate, up)
    s[m // 2, -1] = float('nan')
    out = G.fp8_gate_up((q, s), gate, up)
    keep = torch.arange(m, device='cuda') != m // 2
    assert torch.isnan(out.scale[m // 2]).all() and torch.isnan(out.q[m // 2].float()).all()
    assert torch.equal(out.q[keep].view(torch.uint8), ref.q[keep].view(torch.uint8))
    assert torch.equal(out.scale[keep], ref.scale[keep])
