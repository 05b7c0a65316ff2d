"""GPU checks of how the 8-bit products' blocks leave their SMs: nothing of one launch may reach
the barriers, shared memory or TMEM of the next block there."""
import pytest
import torch

import fp8_cases as F
from src import gpu_ops as G

pytestmark = pytest.mark.gpu


def _rows(gen, m, k):
    return F.torch_rows((torch.randn(m, k, generator=gen) * torch.exp(torch.randn(k, generator=gen))).cuda())


def _blocks(gen, n, k):
    return F.torch_blocks((torch.randn(n, k, generator=gen) * k ** -0.5).bfloat16().cuda())


# Pair kernels of one to three column groups, whose blocks leave soonest after their last products:
# one round of tiles, several, half tiles, rows stored by words, and gate/up.
SHORT = [(512, 4096, 16), (512, 4096, 272), (4096, 4096, 128), (4096, 2560, 384), (2049, 5000, 144), (2305, 4098, 256)]


def test_blocks_after_a_pair_kernel_find_their_own_barriers(cuda):
    """Short pair kernels back to back and beside the split kernel's blocks on another stream, which
    take over their SMs: every output is, bit for bit, what the same call gives alone."""
    gen = torch.Generator().manual_seed(21)
    calls = []
    for m, n, k in SHORT:
        a, w = _rows(gen, m, k), _blocks(gen, n, k)
        calls.append(lambda a=a, w=w: (G.fp8_linear(a, w),))
        if n % 16 == 0:
            calls.append(lambda a=a, w=w: tuple(G.fp8_gate_up(a, w, w)))
    small = [(_rows(gen, m, k), _blocks(gen, n, k)) for m, n, k in ((1, 1600, 960), (64, 960, 2560), (25, 2560, 960))]
    calls_small = [lambda a=a, w=w: (G.fp8_linear(a, w, torch.float32),) for a, w in small]

    def alone(call):
        out = call()
        torch.cuda.synchronize()
        return out

    bits = lambda out: [t.view(torch.uint8) for t in out]
    expected, expected_small = [alone(c) for c in calls], [alone(c) for c in calls_small]
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for turn in range(20):
        with torch.cuda.stream(streams[0]):
            got = [c() for c in calls]
        with torch.cuda.stream(streams[1]):
            got_small = [c() for c in calls_small * 4]
        torch.cuda.synchronize()
        for out, ref in zip(got + got_small, expected + expected_small * 4):
            assert all(torch.equal(x, y) for x, y in zip(bits(out), bits(ref))), turn


# Tiles of few tokens: fewer, as many and more column groups than stages (3 or 4), in one block and
# split over clusters, down to clusters whose last blocks have no token to add up.
FEW = [(1, 128, 16), (1, 40000, 144), (3, 130, 640), (40, 960, 400), (16, 128, 4096), (64, 30001, 528), (33, 20000, 1040)]


@pytest.mark.parametrize('m,n,k', FEW)
def test_split_kernel_ends_with_its_last_copies_and_products(cuda, m, n, k):
    """Back to back launches, each against the 64-bit product, the last as the first."""
    gen = torch.Generator().manual_seed(m + n + k)
    a, w = _rows(gen, m, k), _blocks(gen, n, k)
    out = [G.fp8_linear(a, w, torch.float32) for _ in range(20)]
    F.check_product(out[0], a, w)
    assert all(torch.equal(o, out[0]) for o in out[1:])


def test_products_of_every_kind_at_once_share_the_tensor_memory(cuda):
    """Three streams of products whose blocks share SMs and want more accumulator columns together
    than an SM has, beside the attention on a fourth: the ones that have to wait for columns, or for
    a block of their cluster that does, give what they give alone."""
    from src.gpu_cache import GPUCache
    gen = torch.Generator().manual_seed(5)
    past, heads, group, nq = 4096, 5, 3, 64
    cache = GPUCache(None, layers=1, heads=heads, max_tokens=past + nq)
    kv = torch.randn(1, heads, past, 64, generator=gen).bfloat16().cuda()
    cache.select(8, 0)
    cache.append(kv, kv, 0)
    q = torch.randn(1, heads * group, nq, 64, generator=gen).bfloat16().cuda()
    k = torch.randn(1, heads, nq, 64, generator=gen).bfloat16().cuda()
    attend = lambda: cache.attend(q, k, k, 0, past)
    linear = lambda m, n, k: (lambda a=_rows(gen, m, k), w=_blocks(gen, n, k): G.fp8_linear(a, w))
    gate_up = lambda m, n, k: (lambda a=_rows(gen, m, k), w=_blocks(gen, n, k): G.fp8_gate_up(a, w, w).q.view(torch.uint8))
    work = [[linear(64, 30001, 1040), linear(64, 960, 2560), linear(512, 1600, 960)],
            [gate_up(256, 2560, 960), gate_up(25, 2560, 960), gate_up(1, 8192, 528)],
            [linear(1, 1600, 960), linear(2048, 4096, 528), linear(25, 49280, 144)], [attend]]
    alone = [[call() for call in calls] for calls in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    for _ in range(10):
        got = [[] for _ in work]
        for _ in range(4):
            for s, calls, out in zip(streams, work, got):
                with torch.cuda.stream(s):
                    out.extend(call() for call in calls)
        torch.cuda.synchronize()
        for out, ref in zip(got, alone):
            assert all(torch.equal(a, b) for a, b in zip(out, ref * 4))
