"""CPU checks of the plan of the 8-bit products: what it refuses, and that the GPU tests' cases run every
kernel, stage count, split and form that it chooses anywhere."""
import ctypes

import pytest

import test_gpu_fp8_ops as ops
import test_gpu_fp8_plans as plans
from src import gpu_kernels as K

ROWS = [1, 5, 16, 17, 25, 32, 33, 48, 64, 65, 100, 129, 192, 256, 300, 512, 700, 1000, 1500, 2048, 4096, 8192, 20000]
OUTS = [16, 128, 256, 400, 960, 1600, 2560, 4096, 5120, 8192, 16384, 30000, 49280, 100000]
WIDTHS = [16, 128, 256, 400, 960, 2048, 2560, 4096, 8192, 16384]


def plan(m, n, k, bits):
    p = (ctypes.c_int32 * 4)()
    assert K.LIB.dkv_fp8_plan(m, n, k, bits, p) == K.DKV_OK, K.LIB.dkv_last_error()
    return tuple(p)


def kind(m, n, k, bits):
    tokens, blocks, stages, form = plan(m, n, k, bits)
    return bits, tokens, blocks > 1, stages, form


def _cases(test):
    return next(mark.args[1] for mark in test.pytestmark if mark.name == 'parametrize' and mark.args[0] == 'm,n,k')


def test_the_gpu_cases_reach_every_plan():
    linear = ops.SHAPES + ops.PAIRS + ops.HALVES + plans.LINEAR
    gate_up = [*_cases(ops.test_gate_up), *_cases(ops.test_gate_up_by_pairs), *plans.GATE_UP]
    tested = {kind(*c, bits) for c in linear for bits in (16, 32)} | {kind(*c, 8) for c in gate_up}
    reached = {}
    for m in ROWS:
        for k in WIDTHS:
            for n in OUTS:
                if n <= 16384:
                    reached.setdefault(kind(m, n, k, 8), (m, n, k))
                for odd in (0, 1):
                    for bits in (16, 32):
                        reached.setdefault(kind(m, n + odd, k, bits), (m, n + odd, k))
    assert len(reached) > 20  # bits, three tile sizes, splits, stages; pairs and their forms
    assert not {kind: case for kind, case in reached.items() if kind not in tested}


def test_a_plan_is_within_its_kernels_limits():
    for m in ROWS:
        for n in OUTS[:11]:
            for k in WIDTHS:
                for bits in (8, 16):
                    tokens, blocks, stages, form = plan(m, n, k, bits)
                    assert tokens in ((16, 32, 256) if bits == 8 else (16, 32, 64, 256))
                    assert 1 <= blocks <= 16 and blocks <= -(-k // 128)
                    assert stages in (3, 4) and (form == 0 or tokens == 256)


@pytest.mark.parametrize('args,text', [
    ((4, 960, 1000, 16), 'multiple of 16'), ((4, 960, 16400, 16), 'multiple of 16'), ((4, 24, 960, 8), 'multiple of 16'),
    ((4, 960, 960, 64), 'e4m3'), ((0, 960, 960, 16), 'no rows'), ((-1, 960, 960, 16), 'rows'),
    (((1 << 21) + 1, 960, 960, 16), 'rows'), ((4, 0, 960, 32), 'weight rows'), ((4, (1 << 24) + 1, 960, 32), 'weight rows'),
])
def test_refusals(args, text):
    p = (ctypes.c_int32 * 4)()
    assert K.LIB.dkv_fp8_plan(*args, p) == K.DKV_EINVAL
    assert text in K.LIB.dkv_last_error().decode()
    assert K.LIB.dkv_fp8_plan(4, 960, 960, 16, None) == K.DKV_EINVAL
