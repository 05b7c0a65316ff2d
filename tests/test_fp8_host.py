"""CPU checks of the 8-bit operators: what their entry points refuse on the host, before any
launch, and the 64-bit forms the GPU tests compare against."""
import pytest
import torch

import fp8_cases as F
from src import gpu_kernels as K
from src import gpu_ops as G

P = 0x10000  # fake but 16-byte aligned: every call below ends in host validation


def _refused(fn, base, over, text):
    args = dict(base)
    args.update(over)
    assert getattr(K.LIB, fn)(*args.values()) == K.DKV_EINVAL
    assert text in K.LIB.dkv_last_error().decode()


@pytest.mark.parametrize('over,text', [
    (dict(width=24), 'multiple of 16'), (dict(width=0), 'multiple of 16'), (dict(width=16400), 'multiple of 16'),
    (dict(rows=-1), 'negative'), (dict(x=None), 'null'), (dict(q=None), 'null'), (dict(scale=None), 'null'),
    (dict(x=P + 8), 'aligned'), (dict(q=P + 4), 'aligned'), (dict(scale=P + 2), 'aligned'), (dict(xs=952), 'strides'),
    (dict(xs=964), 'strides'), (dict(rows=1 << 31), 'too many rows'),
])
def test_quantize_refuses(over, text):
    _refused('dkv_fp8_quantize', dict(x=P, q=P, scale=P, rows=4, width=960, xs=960, stream=None), over, text)


@pytest.mark.parametrize('over,text', [
    (dict(k=40), 'multiple of 16'), (dict(n=0), 'rows'), (dict(n=(1 << 24) + 1), 'rows'), (dict(w=None), 'null'),
    (dict(w=P + 2), 'aligned'), (dict(ws=944), 'strides'),
])
def test_quantize_weight_refuses(over, text):
    _refused('dkv_fp8_quantize_weight', dict(w=P, q=P, scale=P, n=160, k=960, ws=960, stream=None), over, text)


@pytest.mark.parametrize('over,text', [
    (dict(width=1000), 'multiple of 16'), (dict(rows=-2), 'negative'), (dict(eps=-1e-5), 'eps'),
    (dict(eps=float('nan')), 'eps'), (dict(x_out=None), 'null'), (dict(weight=None), 'null'), (dict(y=P + 8), 'aligned'),
    (dict(ys=952), 'strides'), (dict(os=961), 'strides'), (dict(rows=1 << 31), 'too many'),
])
def test_norm_refuses(over, text):
    _refused('dkv_add_rms_norm_fp8', dict(x=P, y=P, x_out=P, q=P, scale=P, weight=P, rows=4, width=960, xs=960, ys=960,
                                          os=960, eps=1e-5, stream=None), over, text)


@pytest.mark.parametrize('over,text', [
    (dict(k=1000), 'multiple of 16'), (dict(bits=8), 'bf16 (16) or fp32 (32)'), (dict(m=-1), 'rows'),
    (dict(m=(1 << 21) + 1), 'rows'), (dict(n=0), 'weight rows'), (dict(a=None), 'null'), (dict(ws_=None), 'null'),
    (dict(out=P + 4), 'aligned'), (dict(as_=952), 'strides'), (dict(ws=968), 'strides'),
])
def test_linear_refuses(over, text):
    _refused('dkv_fp8_linear', dict(a=P, sa=P, w=P, ws_=P, out=P, bits=16, m=5, n=7, k=960, as_=960, ws=960, stream=None),
             over, text)


@pytest.mark.parametrize('over,text', [
    (dict(k=8), 'multiple of 16'), (dict(n=24), 'multiple of 16'), (dict(n=16400), 'multiple of 16'),
    (dict(m=-1), 'rows'), (dict(up=None), 'null'), (dict(scale=None), 'null'), (dict(q=P + 1), 'aligned'),
    (dict(us=944), 'strides'), (dict(gs=970), 'strides'),
])
def test_gate_up_refuses(over, text):
    _refused('dkv_fp8_gate_up', dict(a=P, sa=P, gate=P, sg=P, up=P, su=P, q=P, scale=P, m=5, n=160, k=960, as_=960,
                                     gs=960, us=960, stream=None), over, text)


def test_no_rows_is_no_launch():
    assert K.LIB.dkv_fp8_quantize(None, None, None, 0, 960, 960, None) == K.DKV_OK
    assert K.LIB.dkv_add_rms_norm_fp8(None, None, None, None, None, None, 0, 960, 960, 0, 0, 1e-5, None) == K.DKV_OK
    assert K.LIB.dkv_fp8_linear(None, None, None, None, None, 16, 0, 7, 960, 960, 960, None) == K.DKV_OK
    assert K.LIB.dkv_fp8_gate_up(None, None, None, None, None, None, None, None, 0, 160, 960, 960, 960, 960,
                                 None) == K.DKV_OK


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(2, 1)
    w = (torch.zeros(16, 64).to(torch.float8_e4m3fn), torch.ones(1, 1))
    for call in (lambda: G.fp8_quantize(x), lambda: G.fp8_quantize_weight(x),
                 lambda: G.add_rms_fp8(x, None, x[0], 1e-5), lambda: G.fp8_linear((q, s), w),
                 lambda: G.fp8_gate_up((q, s), w, w)):
        with pytest.raises(ValueError, match='CUDA'):
            call()


def test_the_64_bit_forms_hold_for_the_plain_formula():
    """check_rows and check_product accept correct results and see a wrong scale, code or operand."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(5, 200, generator=gen).bfloat16()
    zero = torch.zeros(5, 200, dtype=torch.float64)
    a = F.torch_rows(x)
    F.check_rows(a, x.double(), zero)
    wrong = a[1].clone()
    wrong[2, 1] *= 1 + 1e-6
    with pytest.raises(AssertionError):
        F.check_rows((a[0], wrong), x.double(), zero)
    code = a[0].view(torch.uint8).clone()
    code[3, 150] ^= 3
    with pytest.raises(AssertionError):
        F.check_rows((code.view(torch.float8_e4m3fn), a[1]), x.double(), zero)
    w = F.torch_blocks(torch.randn(130, 200, generator=gen).bfloat16())
    out = (F.row_values(a) @ F.block_values(w).T).bfloat16()
    F.check_product(out, a, w)
    out[1, 129] *= 1.02
    with pytest.raises(AssertionError):
        F.check_product(out, a, w)
