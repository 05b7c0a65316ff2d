"""GPU checks of the 8-bit decoder operators against their 64-bit forms (fp8_cases)."""
import pytest
import torch

import fp8_cases as F
from src import gpu_ops as G

pytestmark = pytest.mark.gpu


def _bf16(gen, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen) * scale).bfloat16().cuda()


def _rows(gen, *shape):
    size = torch.exp(torch.randn(shape[-1], generator=gen))
    return F.torch_rows((torch.randn(*shape, generator=gen) * size).cuda())


def _blocks(gen, n, k):
    return F.torch_blocks(_bf16(gen, n, k, scale=k ** -0.5))


def _same(a, b):
    return all(torch.equal(x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x,
                           y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y) for x, y in zip(a, b))


@pytest.mark.parametrize('shape', [(1, 16), (1, 960), (3, 5, 144), (64, 960), (7, 2560), (513, 1040), (2, 16384)])
def test_quantize_rows_is_the_fp32_formula_bit_for_bit(cuda, shape):
    gen = torch.Generator().manual_seed(sum(shape))
    x = _bf16(gen, *shape, scale=3)
    a = G.fp8_quantize(x)
    assert a.q.shape == x.shape and a.scale.shape == (*shape[:-1], F.groups(shape[-1]))
    same = _same(a, F.torch_rows(x))
    assert same
    F.check_rows(a, x.double(), torch.zeros_like(x, dtype=torch.float64))


@pytest.mark.parametrize('n,k', [(1, 16), (128, 128), (129, 144), (1600, 960), (960, 2560), (77, 4112)])
def test_quantize_weight_is_the_fp32_formula_bit_for_bit(cuda, n, k):
    w = _bf16(torch.Generator().manual_seed(n + k), n, k, scale=0.02)
    a = G.fp8_quantize_weight(w)
    assert a.scale.shape == (F.groups(n), F.groups(k))
    assert _same(a, F.torch_blocks(w))


def test_quantize_reads_strided_rows_and_leaves_what_is_beside_them(cuda):
    gen = torch.Generator().manual_seed(5)
    wide = _bf16(gen, 33, 2 * 960)
    for x in (wide[:, :960], wide[:, 960:], wide[::3, 8:8 + 320], wide[:, 1:17], wide.T[:32].T):
        assert _same(G.fp8_quantize(x), F.torch_rows(x.contiguous()))
    assert _same(G.fp8_quantize_weight(wide[4:, 960:]), F.torch_blocks(wide[4:, 960:].contiguous()))


def test_quantize_extremes(cuda):
    """Zeros, the smallest and largest bf16 values and groups that mix them; a NaN or an
    infinity shows in its own group's scale and nowhere else."""
    x = torch.zeros(8, 256)
    x[1] = 1e-40  # subnormal in bf16: below the floor's reach
    x[2] = 3e38
    x[3, ::2] = -3e38
    x[4, 7] = 2.0 ** -120
    x[5, 3], x[6, 130], x[7, 200] = float('nan'), float('inf'), float('-inf')
    x = x.bfloat16().cuda()
    q, s = G.fp8_quantize(x)
    assert _same((q[:5], s[:5]), F.torch_rows(x[:5]))
    assert (q[0].float() == 0).all() and torch.isfinite(s[:5]).all()
    assert torch.isnan(s[5, 0]) and torch.isfinite(s[5, 1])
    assert torch.isinf(s[6, 1]) and torch.isfinite(s[6, 0]) and torch.isinf(s[7, 1])
    w = G.fp8_quantize_weight(torch.ones(16, 256, device='cuda').bfloat16())
    out = G.fp8_linear((q, s), w, torch.float32)
    assert torch.isfinite(out[[0, 1, 4]]).all() and torch.isnan(out[5:]).all()
    assert torch.isposinf(out[2]).all() and torch.isneginf(out[3]).all()  # 256 and 128 x 3e38: beyond fp32


@pytest.mark.parametrize('residual', [True, False])
@pytest.mark.parametrize('shape', [(1, 16), (1, 960), (5, 64, 960), (3, 1024), (4, 1040), (33, 2048), (9, 2576),
                                   (5, 4096), (3, 8192), (2, 8208), (2, 16384)])
def test_add_rms_norm(cuda, shape, residual):
    gen = torch.Generator().manual_seed(sum(shape))
    x, y = _bf16(gen, *shape, scale=3), _bf16(gen, *shape)
    weight = (1 + 0.2 * torch.randn(shape[-1], generator=gen)).bfloat16().cuda()
    total, a = G.add_rms_fp8(x, y if residual else None, weight, 1e-5)
    v = x + y if residual else x
    assert torch.equal(total.view(torch.int16), v.view(torch.int16))
    if not residual:
        assert total is x or total.data_ptr() == x.data_ptr()
    v = v.double()
    h = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * weight.double()
    # the mean: n roundings of positive terms, halved by the root; rsqrt 2 units; two products
    F.check_rows(a, h, h.abs() * ((shape[-1] / 2 + 8) * 2 ** -24))


def test_add_rms_norm_strided_rows_and_zero_rows(cuda):
    gen = torch.Generator().manual_seed(1)
    wide = _bf16(gen, 9, 4 * 320)
    x, y, w = wide[:, :320], wide[:, 640:960], _bf16(gen, 320)
    ref = G.add_rms_fp8(x.contiguous(), y.contiguous(), w, 1e-6)
    got = G.add_rms_fp8(x, y, w, 1e-6)
    assert torch.equal(got[0], ref[0]) and _same(got[1], ref[1])
    total, a = G.add_rms_fp8(x - x, None, w, 1e-6)  # a row of zeros stays zeros
    assert (a.q.float() == 0).all() and torch.isfinite(a.scale).all()


SHAPES = [(1, 1, 16), (1, 1600, 960), (2, 130, 144), (16, 128, 128), (17, 129, 1040), (25, 960, 2560), (31, 7, 4672),
          (33, 1001, 96), (64, 960, 2560), (65, 320, 960), (100, 2048, 8192), (128, 128, 16384), (129, 257, 400),
          (333, 1001, 1040), (512, 1600, 960), (1024, 1024, 512), (2048, 960, 960), (1500, 5000, 272)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k', SHAPES)
def test_linear(cuda, m, n, k, dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    a, w = _rows(gen, m, k), _blocks(gen, n, k)
    out = G.fp8_linear(a, w, dtype)
    assert out.shape == (m, n) and out.dtype == dtype and out.is_contiguous()
    F.check_product(out, a, w)
    assert torch.equal(G.fp8_linear(a, w, dtype), out)  # the same order of additions every time


def test_linear_row_does_not_depend_on_its_neighbours(cuda):
    """Rows of NaN beside a row, and weight rows of NaN beside a column, stay where they are."""
    gen = torch.Generator().manual_seed(3)
    a, w = _rows(gen, 40, 272), _blocks(gen, 300, 272)
    ref = G.fp8_linear(a, w)
    s = a[1].clone()
    s[::2] = float('nan')
    got = G.fp8_linear((a[0], s), w)
    assert torch.isnan(got[::2]).all() and torch.equal(got[1::2], ref[1::2])
    ws = w[1].clone()
    ws[1, 2] = float('nan')
    got = G.fp8_linear(a, (w[0], ws))
    assert torch.isnan(got[:, 128:256]).all()
    assert torch.equal(got[:, :128], ref[:, :128]) and torch.equal(got[:, 256:], ref[:, 256:])


def test_linear_leading_dimensions_strides_and_slices(cuda):
    gen = torch.Generator().manual_seed(4)
    a, w = _rows(gen, 3, 8, 320), _blocks(gen, 384, 320)
    ref = G.fp8_linear((a[0].view(24, 320), a[1].view(24, 3)), w)
    assert torch.equal(G.fp8_linear(a, w).view(24, 384), ref)
    padded = torch.zeros(24, 400, device='cuda').to(torch.float8_e4m3fn)
    padded.view(torch.uint8)[:, 16:336] = a[0].view(24, 320).view(torch.uint8)
    rows = padded[:, 16:336]
    assert torch.equal(G.fp8_linear((rows, a[1].view(24, 3)), w), ref)
    odd = torch.zeros(24, 337, device='cuda').to(torch.float8_e4m3fn)  # rows that start anywhere: copied
    odd.view(torch.uint8)[:, 17:] = rows.view(torch.uint8)
    assert torch.equal(G.fp8_linear((odd[:, 17:], a[1].view(24, 3)), w), ref)
    halves = [G.fp8_linear(a, (w[0][i:i + 128], w[1][i // 128:i // 128 + 1])) for i in (0, 128, 256)]
    assert torch.equal(torch.cat(halves, -1).view(24, 384), ref)


@pytest.mark.parametrize('m,n,k', [(1, 16, 16), (1, 2560, 960), (2, 128, 144), (16, 144, 960), (25, 2560, 960),
                                   (33, 400, 1040), (64, 2560, 960), (65, 272, 4096), (100, 8192, 512),
                                   (129, 128, 16384), (512, 2560, 960), (1100, 1040, 400), (2048, 2560, 960)])
def test_gate_up(cuda, m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    a, gate, up = _rows(gen, m, k), _blocks(gen, n, k), _blocks(gen, n, k)
    out = G.fp8_gate_up(a, gate, up)
    assert out.q.shape == (m, n) and out.scale.shape == (m, F.groups(n))
    F.check_gate_up(out, a, gate, up)
    assert _same(G.fp8_gate_up(a, gate, up), out)


def test_gate_up_of_joined_weights_large_gates_and_nan(cuda):
    gen = torch.Generator().manual_seed(9)
    x = _bf16(gen, 70, 512, scale=400)  # gates up to +-1e3: exp overflows on one side, vanishes on the other
    joined = _bf16(gen, 2 * 384, 512, scale=512 ** -0.5)
    a, w = G.fp8_quantize(x), G.fp8_quantize_weight(joined)
    gate, up = (w.q[:384], w.scale[:3]), (w.q[384:], w.scale[3:])
    out = G.fp8_gate_up(a, gate, up)
    F.check_gate_up(out, a, gate, up)
    s = a.scale.clone()
    s[5, 1] = float('nan')
    bad = G.fp8_gate_up((a.q, s), gate, up)
    assert torch.isnan(bad.scale[5]).all()
    keep = torch.arange(70) != 5
    assert _same((bad.q[keep], bad.scale[keep]), (out.q[keep], out.scale[keep]))


def test_no_rows(cuda):
    gen = torch.Generator().manual_seed(2)
    x, w = torch.empty(0, 256, device='cuda').bfloat16(), _blocks(gen, 144, 256)
    a = G.fp8_quantize(x)
    assert a.q.shape == (0, 256) and a.scale.shape == (0, 2)
    total, b = G.add_rms_fp8(x, x, torch.ones(256, device='cuda').bfloat16(), 1e-5)
    assert total.shape == b.q.shape == (0, 256)
    assert G.fp8_linear(a, w).shape == (0, 144)
    assert G.fp8_gate_up(a, w, w).q.shape == (0, 144)


def _mlp(x, y, weight, gate, up, down):
    """One decoder block's second half, as the decoder runs it."""
    x, h = G.add_rms_fp8(x, y, weight, 1e-5)
    return x, G.fp8_linear(G.fp8_gate_up(h, gate, up), down)


def _mlp_operands(m, seed):
    gen = torch.Generator().manual_seed(seed)
    return (_bf16(gen, m, 960, scale=2), _bf16(gen, m, 960), (1 + 0.1 * torch.randn(960, generator=gen)).bfloat16().cuda(),
            _blocks(gen, 2560, 960), _blocks(gen, 2560, 960), _blocks(gen, 960, 2560))


@pytest.mark.parametrize('m', [1, 25, 64, 512])
def test_operators_together_each_against_its_own_inputs(cuda, m):
    x, y, weight, gate, up, down = _mlp_operands(m, m)
    total, h = G.add_rms_fp8(x, y, weight, 1e-5)
    act = G.fp8_gate_up(h, gate, up)
    out = G.fp8_linear(act, down)
    F.check_gate_up(act, h, gate, up)
    F.check_product(out, act, down)
    # the bf16 block it stands for: e4m3 rounds each normed value, weight and activation by at most 2^-4,
    # and over hundreds of terms those errors average out: a tenth in the 2-norm is far from a wrong operand
    v = (x + y).double()
    n = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + 1e-5) * weight.double()
    g, u = n @ F.block_values(gate).T, n @ F.block_values(up).T
    ref = (g * torch.sigmoid(g) * u) @ F.block_values(down).T
    assert (out.double() - ref).norm() <= 0.1 * ref.norm()


def test_captured_steps_replay_on_new_inputs(cuda):
    """A block captured into a graph, beside eager calls of other sizes between its replays."""
    args = _mlp_operands(64, 1)
    other = _mlp_operands(64, 2)
    expected = [t.clone() for t in _mlp(*other)]
    x, y = args[0].clone(), args[1].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        _mlp(x, y, *other[2:])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = _mlp(x, y, *other[2:])
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(3):
        x.copy_(args[0]), y.copy_(args[1])
        graph.replay()
        _mlp(*_mlp_operands(5, 3))
        x.copy_(other[0]), y.copy_(other[1])
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_two_streams_at_once(cuda):
    sizes = [1, 64, 300, 17]
    operands = [_mlp_operands(m, m) for m in sizes]
    expected = [[t.clone() for t in _mlp(*o)] for o in operands]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    for _ in range(10):
        got = []
        for s, o in zip(streams, operands):
            with torch.cuda.stream(s):
                got.append(_mlp(*o))
        torch.cuda.synchronize()
        for g, e in zip(got, expected):
            assert all(torch.equal(a, b) for a, b in zip(g, e))


def test_a_chain_reads_what_the_launch_before_wrote(cuda):
    """Weights quantised right before the product that reads them, rows written right before
    theirs: every launch waits for the one before it."""
    gen = torch.Generator().manual_seed(6)
    x, w = _bf16(gen, 8, 960), [_bf16(gen, 960, 960, scale=0.03) for _ in range(6)]
    expected = x
    for m in w:
        expected = G.fp8_linear(F.torch_rows(expected), F.torch_blocks(m))
        torch.cuda.synchronize()
    for _ in range(20):
        h = x
        for m in w:
            h = G.fp8_linear(G.fp8_quantize(h), G.fp8_quantize_weight(m))
        assert torch.equal(h, expected)


def test_outputs_end_where_their_rows_do(cuda):
    """Through the C ABI into the middle of larger buffers: nothing around the outputs changes."""
    from src import gpu_kernels as K
    gen = torch.Generator().manual_seed(8)
    m, n, k = 21, 400, 272
    a, w, u = _rows(gen, m, k), _blocks(gen, n, k), _blocks(gen, n, k)
    stream = torch.cuda.current_stream().cuda_stream
    out = torch.full((m + 2, n), 7.0, device='cuda')
    assert K.LIB.dkv_fp8_linear(a[0].data_ptr(), a[1].data_ptr(), w[0].data_ptr(), w[1].data_ptr(),
                                out[1].data_ptr(), 32, m, n, k, k, k, stream) == 0
    q = torch.full((m + 2, n), 9, dtype=torch.uint8, device='cuda')
    s = torch.full((m + 2, F.groups(n)), 5.0, device='cuda')
    assert K.LIB.dkv_fp8_gate_up(a[0].data_ptr(), a[1].data_ptr(), w[0].data_ptr(), w[1].data_ptr(), u[0].data_ptr(),
                                 u[1].data_ptr(), q[1].data_ptr(), s[1].data_ptr(), m, n, k, k, k, k, stream) == 0
    x = _bf16(gen, m, n)
    q2, s2 = q.clone().fill_(9), s.clone().fill_(5)
    assert K.LIB.dkv_fp8_quantize(x.data_ptr(), q2[1].data_ptr(), s2[1].data_ptr(), m, n, n, stream) == 0
    torch.cuda.synchronize()
    for t, v in ((out, 7), (q, 9), (s, 5), (q2, 9), (s2, 5)):
        assert (t[0] == v).all() and (t[-1] == v).all()
    assert torch.equal(out[1:-1], G.fp8_linear(a, w, torch.float32))
    assert torch.equal(q[1:-1], G.fp8_gate_up(a, w, u).q.view(torch.uint8))
    assert torch.equal(q2[1:-1], G.fp8_quantize(x).q.view(torch.uint8))


def test_refusals(cuda):
    gen = torch.Generator().manual_seed(7)
    a, w = _rows(gen, 4, 256), _blocks(gen, 144, 256)
    x = _bf16(gen, 4, 256)
    ones = torch.ones(256, device='cuda').bfloat16()
    bad = [
        (lambda: G.fp8_quantize(x.float()), 'bfloat16'),
        (lambda: G.fp8_quantize(x.cpu()), 'CUDA'),
        (lambda: G.fp8_quantize(x[:, :24]), 'multiple of 16'),
        (lambda: G.fp8_quantize(x[:, :0]), 'multiple of 16'),
        (lambda: G.fp8_quantize(torch.zeros(1, 16400, device='cuda').bfloat16()), 'multiple of 16'),
        (lambda: G.fp8_quantize(x.clone().requires_grad_()), 'backward'),
        (lambda: G.fp8_quantize_weight(x[0]), r'\[n, k\]'),
        (lambda: G.fp8_quantize_weight(x[:0]), 'rows'),
        (lambda: G.add_rms_fp8(x, x[:3], ones, 1e-5), 'match'),
        (lambda: G.add_rms_fp8(x, x.float(), ones, 1e-5), 'bfloat16'),
        (lambda: G.add_rms_fp8(x, None, ones[:128], 1e-5), 'weight'),
        (lambda: G.add_rms_fp8(x, None, ones, -1.0), 'eps'),
        (lambda: G.fp8_linear(a, w, torch.float16), 'bfloat16 or float32'),
        (lambda: G.fp8_linear((x, a[1]), w), 'float8_e4m3fn'),
        (lambda: G.fp8_linear((a[0], a[1][:, :1]), w), 'scales'),
        (lambda: G.fp8_linear((a[0], a[1].double()), w), 'scales'),
        (lambda: G.fp8_linear(a, (w[0], w[1][:1])), 'scales'),
        (lambda: G.fp8_linear(a, (w[0][:, :128], w[1][:, :1])), 'width'),
        (lambda: G.fp8_linear(a, (w[0].cpu(), w[1].cpu())), 'CUDA'),
        (lambda: G.fp8_gate_up(a, w, (w[0][:128], w[1][:1])), 'one shape'),
        (lambda: G.fp8_gate_up(a, _blocks(gen, 136, 256), _blocks(gen, 136, 256)), 'multiple of 16'),
    ]
    for call, text in bad:
        with pytest.raises(ValueError, match=text):
            call()
    torch.cuda.synchronize()


# Products with tokens enough for the pair kernel (256 x 256 tiles; more than 74 of them are several
# rounds of the grid): rows and columns that end inside a tile, column groups of every remainder, and
# every start of a row that the stores tell apart (n modulo 2, 4 and 8; bf16 and fp32).
PAIRS = [(4096, 4096, 256), (3000, 4104, 144), (2049, 5000, 272), (2305, 4098, 400), (2500, 4097, 1040),
         (5000, 2051, 528), (8192, 2052, 32), (2048, 2600, 2064)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k', PAIRS)
def test_linear_by_pairs(cuda, m, n, k, dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    a, w = _rows(gen, m, k), _blocks(gen, n, k)
    out = G.fp8_linear(a, w, dtype)
    F.check_product(out, a, w)
    assert torch.equal(G.fp8_linear(a, w, dtype), out)


# The last round's tiles cut into halves of 128 columns: all of them, some, the most that are cut (37),
# a second half of few columns and one of none.
HALVES = [(512, 4096, 4096), (500, 4040, 1040), (2048, 2560, 400), (2100, 2200, 2064), (9467, 664, 144),
          (9467, 608, 272)]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('m,n,k', HALVES)
def test_linear_by_halves(cuda, m, n, k, dtype):
    gen = torch.Generator().manual_seed(m + n + k)
    a, w = _rows(gen, m, k), _blocks(gen, n, k)
    out = G.fp8_linear(a, w, dtype)
    F.check_product(out, a, w)
    assert torch.equal(G.fp8_linear(a, w, dtype), out)


@pytest.mark.parametrize('m,n,block', [(2500, 4096, 30), (2500, 4096, 31), (500, 4040, 0), (500, 4040, 31)])
def test_halves_keep_weight_blocks_apart(cuda, m, n, block):
    """A NaN weight block reaches its own 128 columns: not the tile's other half, nor another group."""
    gen = torch.Generator().manual_seed(block)
    a, (wq, ws) = _rows(gen, m, 528), _blocks(gen, n, 528)
    ref = G.fp8_linear(a, (wq, ws))
    ws[block, 3] = float('nan')
    out = G.fp8_linear(a, (wq, ws))
    own = torch.arange(n, device='cuda') // 128 == block
    assert torch.isnan(out[:, own]).all()
    assert torch.equal(out[:, ~own], ref[:, ~own])


@pytest.mark.parametrize('m,n,k', [(4096, 2560, 960), (3001, 2576, 272), (2304, 1040, 2064), (700, 6416, 400)])
def test_gate_up_by_pairs(cuda, m, n, k):
    gen = torch.Generator().manual_seed(m + n + k)
    a, gate, up = _rows(gen, m, k), _blocks(gen, n, k), _blocks(gen, n, k)
    out = G.fp8_gate_up(a, gate, up)
    F.check_gate_up(out, a, gate, up)
    assert _same(G.fp8_gate_up(a, gate, up), out)


@pytest.mark.parametrize('n,dtype', [(4096, torch.bfloat16), (4097, torch.bfloat16), (4102, torch.bfloat16),
                                     (4096, torch.float32), (4099, torch.float32)])
def test_pairs_keep_rows_and_columns_apart(cuda, n, dtype):
    """NaN rows and a NaN weight block beside clean ones, in the middle of a larger buffer."""
    from src import gpu_kernels as K
    gen = torch.Generator().manual_seed(n)
    m, k = 2500, 272
    (q, s), (wq, ws) = _rows(gen, m, k), _blocks(gen, n, k)
    ref = G.fp8_linear((q, s), (wq, ws), dtype)
    s[::3], ws[3, 1] = float('nan'), float('nan')
    pad = 1 << 15  # keeps the output's start on 16 bytes
    flat = torch.full((m * n + 2 * pad,), 7.0, device='cuda', dtype=dtype)
    out = flat[pad:pad + m * n].view(m, n)
    rc = K.LIB.dkv_fp8_linear(q.data_ptr(), s.data_ptr(), wq.data_ptr(), ws.data_ptr(), out.data_ptr(),
                              out.element_size() * 8, m, n, k, k, k, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, K.LIB.dkv_last_error()
    torch.cuda.synchronize()
    assert (flat[:pad] == 7).all() and (flat[pad + m * n:] == 7).all()
    assert torch.isnan(out[::3]).all() and torch.isnan(out[:, 384:512]).all()
    clean = torch.ones(m, dtype=torch.bool, device='cuda')
    clean[::3] = False
    keep = torch.ones(n, dtype=torch.bool, device='cuda')
    keep[384:512] = False
    assert torch.equal(out[clean][:, keep], ref[clean][:, keep])


def test_threads_launch_different_shapes_at_once(cuda):
    """Four host threads, each on its own stream with its own shapes: no call changes another's."""
    import threading
    shapes = [(1, 1600, 960), (64, 960, 2560), (512, 960, 960), (2048, 1600, 960)]
    gen = torch.Generator().manual_seed(11)
    operands = [(_rows(gen, m, k), _blocks(gen, n, k)) for m, n, k in shapes]
    expected = [G.fp8_linear(*o) for o in operands]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                out = G.fp8_linear(*operands[i])
                torch.cuda.current_stream().synchronize()
                if not torch.equal(out, expected[i]):
                    failed.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
