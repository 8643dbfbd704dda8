"""Rows and matrices in 8 bits with a scale per block, and products of them, against their definitions in 64 bits."""
import math

import pytest
import torch

from llmserver_b200 import ops
from test_gpu_kernels import DEVICE, rand

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def finished():
    from llmserver_b200.ops.library import check_wait_errors
    torch.cuda.synchronize()
    check_wait_errors()


def e4m3_numbers():
    """All finite numbers of e4m3, ascending: sign, four bits of exponent (bias 7), three of mantissa; exponent 0 without the leading one."""
    positive = [(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8) if (e, m) != (15, 7)]
    return sorted({-v for v in positive} | set(positive))


def nearest(quotient):
    """The nearest of e4m3's numbers, ties to the one whose last mantissa bit is 0."""
    numbers = torch.tensor(e4m3_numbers(), dtype=torch.float64, device=quotient.device)
    even = torch.tensor([(i - 126) % 2 == 0 for i in range(253)], device=quotient.device)      # 0 is in the middle, and even
    above = torch.searchsorted(numbers, quotient.contiguous()).clamp(1, 252)
    below = above - 1
    up, down = numbers[above] - quotient, quotient - numbers[below]
    take_up = (up < down) | ((up == down) & even[above])
    return torch.where(take_up, numbers[above], numbers[below])


def quantized(x, block_rows):
    """(values, scales) of the definition, block by block."""
    rows, columns = x.shape
    x = x.double()
    values = torch.empty_like(x)
    scales = torch.empty((-(-rows // block_rows), -(-columns // 128)), dtype=torch.float64, device=x.device)
    for i in range(scales.shape[0]):
        for j in range(scales.shape[1]):
            part = x[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128]
            if not bool(torch.isfinite(part).all()):
                scales[i, j], scale = math.nan, math.nan
                values[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = math.nan
                continue
            largest = float(part.abs().max())
            exponent = -126
            if largest > 448 * 2.0 ** -126:
                exponent = math.frexp(largest / 448)[1] - 2
                while largest > 448 * 2.0 ** exponent:
                    exponent += 1
            scales[i, j] = 2.0 ** exponent
            values[i * block_rows:(i + 1) * block_rows, j * 128:(j + 1) * 128] = nearest(part / 2.0 ** exponent)
    return values, scales


def same(got, want):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got.nan_to_num(0.0), want.nan_to_num(0.0))


def matrix(cols, inner, seed):
    """A matrix in blocks of 128 x 128 whose scales are no powers of two, as checkpoints have them."""
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    values = (torch.randn((cols, inner), generator=generator, device=DEVICE) * 100).clamp(-448, 448).to(F8)
    scales = (0.5 + torch.rand((-(-cols // 128), -(-inner // 128)), generator=generator, device=DEVICE)) * 1e-4
    return ops.block_scaled(values, scales)


def product(rows, weight):
    """y of two ``BlockScaled`` in 64 bits, and the sum of the products' magnitudes."""
    x, w = wide(rows), wide(weight)
    return x @ w.t(), x.abs() @ w.abs().t()


def wide(operand):
    scales = operand.scales.double().repeat_interleave(128, dim=1)[:, :operand.values.shape[1]]
    return operand.values.double() * scales.repeat_interleave(operand.block_rows, dim=0)[:operand.values.shape[0]]


def close(got, rows, weight):
    """The bound: the 128 products of a block are exact and each of their additions is off by a unit in the last place of 24 bits at most (the tensor
    core may cut where it adds); the two scales' product, its product with the block's sum and the addition to the sums before it by
    half a unit each, G blocks one after the other; then one rounding to the output's type, by half a step."""
    want, size = product(rows, weight)
    blocks = weight.scales.shape[1]
    bound = (2 * 128 + 3 + blocks) * 2.0 ** -24 * size
    bound = bound + torch.finfo(got.dtype).eps / 2 * (want.abs() + bound)
    error = (got.double() - want).abs()
    assert got.shape == want.shape
    assert bool((error <= bound).all()), f"{float((error / bound.clamp(min=1e-300)).max()):.2f} of the bound"


@pytest.mark.parametrize("rows,columns", [(1, 1), (1, 128), (3, 130), (129, 127), (5, 1000), (300, 512), (130, 4099)])
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_in_8_bits(rows, columns, block_rows, dtype):
    x = rand((rows, columns), dtype, rows + columns)
    if rows > 2:
        x[0] = 0.0
        x[1] *= 1e-38          # below the least scale
        x[2, 0] = 3e38
    got = ops.quantize_blocks(x, block_rows)
    finished()
    want_values, want_scales = quantized(x, block_rows)
    same(got.scales, want_scales)
    same(got.values, want_values)
    assert got.values.stride(0) % 16 == 0
    same(got.widened(), (want_values * want_scales.repeat_interleave(128, 1)[:, :columns].repeat_interleave(block_rows, 0)[:rows]).float())


@pytest.mark.parametrize("block_rows", [1, 128])
def test_ties_borders_and_what_is_not_finite(block_rows):
    """Every midpoint between two of e4m3's numbers, 448 and what lies just above it, and blocks with an infinity or a NaN."""
    numbers = torch.tensor(e4m3_numbers(), dtype=torch.float64)
    middles = (numbers[1:] + numbers[:-1]) / 2
    x = torch.zeros((4, 5 * 128), dtype=torch.float32)
    x[0, :252] = middles.float()
    x[0, 252:254] = 448.0          # the scale is 1 in both blocks
    x[0, 127] = 448.0
    x[1, :128] = torch.linspace(440, 480, 128)
    x[2, 256], x[2, 384], x[3, 512] = math.inf, -math.inf, math.nan
    x[3, 10] = 2.0 ** -149
    x = x.to(DEVICE)
    got = ops.quantize_blocks(x, block_rows)
    finished()
    want_values, want_scales = quantized(x, block_rows)
    same(got.scales, want_scales)
    same(got.values, want_values)


def test_rows_that_begin_anywhere():
    """Operands that lie at odd addresses and end in the middle of four numbers."""
    for dtype in (torch.float32, torch.bfloat16):
        pool = rand((1 + 7 * 260,), dtype, 5)
        for columns in (258, 260):
            x = pool[1:1 + 7 * columns].view(7, columns)
            got = ops.quantize_blocks(x)
            finished()
            want_values, want_scales = quantized(x, 1)
            same(got.values, want_values)
            same(got.scales, want_scales)


# tokens on both sides of every tile, inner sizes that end inside a block of 128 and inside 16 bytes, columns that fill no tile, few
# and many blocks of k, more tiles than SMs
SIZES = [(1, 128, 128), (1, 1, 1), (2, 16, 5), (15, 127, 129), (16, 129, 128), (17, 500, 257), (32, 512, 1000), (33, 1000, 384), (64, 640, 130),
         (65, 2001, 300), (128, 384, 1111), (129, 1024, 128), (300, 700, 700), (1000, 256, 513), (1, 4096, 6144), (8, 12288, 4096), (61, 4096, 19000),
         (260, 8192, 260), (511, 1536, 2049), (66, 300, 40000), (1000, 384, 4100), (1290, 650, 5000), (4500, 130, 1300), (40000, 300, 100), (20001, 1500, 37),
         (1000, 100, 20000), (37900, 128, 128)]


@pytest.mark.parametrize("rows,inner,cols", SIZES)
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_products(rows, inner, cols, out_dtype):
    weight = matrix(cols, inner, 1)
    x = rand((rows, inner), torch.bfloat16 if inner % 2 else torch.float32, 2)
    got = ops.linear(x, weight, out_dtype=out_dtype)
    finished()
    close(got, ops.quantize_blocks(x), weight)


@pytest.mark.parametrize("rows", [1, 31, 200, 700])
def test_rows_in_8_bits_are_taken_as_they_are(rows):
    """The same rows for two products, scales that are no powers of two, and an output of the caller's."""
    inner = 900
    held = ops.quantize_blocks(rand((rows, inner), torch.bfloat16, 3))
    held.scales.mul_(torch.rand_like(held.scales) + 0.5)
    for cols, seed in ((320, 4), (1300, 5)):
        weight = matrix(cols, inner, seed)
        out = torch.full((rows, cols), math.nan, dtype=torch.bfloat16, device=DEVICE)
        assert ops.linear(held, weight, out=out) is out
        finished()
        close(out, held, weight)


def test_columns_of_a_wider_matrix():
    """Values whose rows lie apart, on both sides, with NaN around them."""
    pool = torch.full((300, 1024), 0x7F, dtype=torch.uint8, device=DEVICE)
    wide_matrix = matrix(300, 400, 6)
    pool[:, 16:416] = wide_matrix.values.view(torch.uint8)
    weight = ops.BlockScaled(pool.view(F8)[:, 16:416], wide_matrix.scales)
    rows_pool = torch.full((70, 512), 0x7F, dtype=torch.uint8, device=DEVICE)
    held = ops.quantize_blocks(rand((70, 400), torch.float32, 7))
    rows_pool[:, 32:432] = held.values.view(torch.uint8)
    rows = ops.BlockScaled(rows_pool.view(F8)[:, 32:432], held.scales, 1)
    got = ops.linear(rows, weight, out_dtype=torch.float32)
    finished()
    close(got, held, wide_matrix)
    assert torch.equal(got, ops.linear(held, wide_matrix, out_dtype=torch.float32))


@pytest.mark.parametrize("rows", [3, 100, 600])
def test_a_row_that_is_not_finite_stays_alone(rows):
    weight = matrix(200, 512, 8)
    x = rand((rows, 512), torch.bfloat16, 9)
    clean = ops.linear(x, weight)
    bad = x.clone()
    bad[1, 300], bad[2, 5] = math.nan, math.inf
    got = ops.linear(bad, weight)
    finished()
    assert bool(torch.isnan(got[1:3]).all())
    assert torch.equal(got[0], clean[0]) and torch.equal(got[3:], clean[3:])


@pytest.mark.parametrize("rows,inner,cols", [(1, 4096, 512), (40, 4096, 512), (120, 2048, 1024), (700, 1024, 1024)])
def test_the_same_call_gives_the_same_bits(rows, inner, cols):
    weight, x = matrix(cols, inner, 10), rand((rows, inner), torch.bfloat16, 11)
    first = ops.linear(x, weight, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(first, ops.linear(x, weight, out_dtype=torch.float32))
    finished()


def test_a_matrix_is_used_as_soon_as_it_is_made():
    """The kernel that makes the matrix runs right in front, into memory that another one filled before."""
    x = rand((5, 2048), torch.bfloat16, 12)
    sources = [rand((2048, 2048), torch.bfloat16, 20 + i, 2048 ** -0.5) for i in range(6)]
    want = [ops.linear(x, ops.quantize_blocks(source, 128), out_dtype=torch.float32) for source in sources]
    torch.cuda.synchronize()
    for _ in range(5):
        for source, expected in zip(sources, want):
            weight = ops.quantize_blocks(source, 128)
            got = ops.linear(x, weight, out_dtype=torch.float32)
            del weight
            assert torch.equal(got, expected)
            weight = ops.quantize_blocks(source, 128)
            assert torch.equal(ops.linear(ops.quantize_blocks(x), weight, out_dtype=torch.float32), expected)
    finished()


def test_no_rows_and_results_of_a_chain():
    weight = matrix(300, 256, 13)
    assert ops.linear(torch.empty((0, 256), dtype=torch.bfloat16, device=DEVICE), weight).shape == (0, 300)
    assert ops.quantize_blocks(torch.empty((0, 256), device=DEVICE)).scales.shape == (0, 2)
    # a feed-forward of two products in 8 bits
    down = matrix(256, 300, 14)
    x = rand((50, 256), torch.bfloat16, 15)
    hidden = ops.linear(x, weight)
    y = ops.linear(hidden, down)
    finished()
    close(hidden, ops.quantize_blocks(x), weight)
    close(y, ops.quantize_blocks(hidden), down)


@pytest.mark.parametrize("rows", [4, 90, 520])
def test_captured_and_replayed_on_another_stream(rows):
    """Two graphs of the same weight with operands of their own, replayed in turn, give what eager calls give."""
    weight = matrix(700, 1000, 16)
    inputs = [rand((rows, 1000), torch.bfloat16, 17 + i) for i in range(2)]
    want = [ops.linear(x, weight) for x in inputs]
    graphs, held, results = [], [], []
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for x in inputs:
            ops.linear(x, weight)
            fixed = torch.zeros_like(x)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                result = ops.linear(fixed, weight)
            graphs.append(graph), held.append(fixed), results.append(result)
        for turn in (0, 1, 1, 0):
            held[turn].copy_(inputs[turn])
            graphs[turn].replay()
            stream.synchronize()
            assert torch.equal(results[turn], want[turn])
            results[turn].zero_()
    finished()


def test_refusals_on_the_device():
    from llmserver_b200.ops import KernelError
    weight, x = matrix(256, 256, 18), rand((4, 256), torch.bfloat16, 19)
    cases = [
        (lambda: ops.linear(x[:, :128].contiguous(), weight), "columns"),
        (lambda: ops.linear(x.half(), weight), "float32 or bfloat16"),
        (lambda: ops.linear(x.t(), weight), "contiguous"),
        (lambda: ops.linear(x, weight, out_dtype=torch.float16), "writes float32 or bfloat16"),
        (lambda: ops.linear(x, weight, out=torch.empty((4, 255), dtype=torch.bfloat16, device=DEVICE)), "output"),
        (lambda: ops.linear(x, ops.quantize_blocks(rand((4, 256), torch.float32, 1))), "128 rows"),
        (lambda: ops.linear(weight, weight), "1 rows"),
        (lambda: ops.linear(x, ops.BlockScaled(weight.values, weight.scales[:1])), "scales"),
        (lambda: ops.linear(x, ops.BlockScaled(weight.values, weight.scales.double())), "float32 scales"),
        (lambda: ops.linear(x, ops.BlockScaled(weight.values.float(), weight.scales)), "float8_e4m3fn"),
        (lambda: ops.linear(x, ops.BlockScaled(weight.values.view(torch.uint8).view(-1)[1:1 + 255 * 256].view(F8).view(255, 256), weight.scales)), "16 bytes"),
        (lambda: ops.quantize_blocks(x, 64), "1 or 128"),
        (lambda: ops.quantize_blocks(x[0]), "matrix"),
        (lambda: ops.quantize_blocks(x.half()), "float32 or bfloat16"),
    ]
    for call, message in cases:
        with pytest.raises(KernelError, match=message):
            call()


def test_two_streams_at_once():
    """Products of every form, replayed on two streams side by side again and again: the same bits as alone."""
    shapes = [(1, 4096, 2048), (20, 2048, 1024), (64, 4096, 700), (100, 4096, 1024), (300, 1024, 3000), (900, 512, 6000)]
    work = [(rand((rows, inner), torch.bfloat16, rows), matrix(cols, inner, cols)) for rows, inner, cols in shapes]
    want = [ops.linear(x, weight, out_dtype=torch.float32) for x, weight in work]
    graphs, kept = [], []
    for order in (work, work[::-1]):
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                kept.append([ops.linear(x, weight, out_dtype=torch.float32) for _ in range(4) for x, weight in order])
        graphs.append((graph, stream))
    for _ in range(5):
        for graph, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
    for _, stream in graphs:
        stream.synchronize()
    finished()
    for results, order in zip(kept, (want, want[::-1])):
        for at, got in enumerate(results):
            assert torch.equal(got, order[at % len(order)]), at


def quantized_rows(x):
    """``quantized(x, 1)`` for many rows: all blocks at a time, finite numbers only."""
    rows, columns = x.shape
    groups = -(-columns // 128)
    blocks = torch.nn.functional.pad(x.double(), (0, groups * 128 - columns)).view(rows, groups, 128)
    mantissa, exponent = torch.frexp(blocks.abs().amax(2))      # 448 is 0.875 times 2^9
    exponent = torch.where(mantissa > 0.875, exponent - 8, torch.where(mantissa > 0, exponent - 9, -126)).clamp(min=-126)
    scales = torch.ldexp(torch.ones_like(mantissa), exponent)
    return nearest(blocks / scales[:, :, None]).reshape(rows, groups * 128)[:, :columns], scales


@pytest.mark.parametrize("rows,columns", [(7, 130), (2400, 4104), (19001, 504), (80000, 8), (77000, 100), (1300, 8200), (600, 12345)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_that_end_inside_a_block(rows, columns, dtype):
    """More groups than half warps run at a time, several times over."""
    x = rand((rows, columns), dtype, 31)
    x[rows // 2] = 0
    x[rows - 1, columns - 1] = 1e4
    got = ops.quantize_blocks(x)
    finished()
    want_values, want_scales = quantized_rows(x)
    if rows < 10:
        same(want_values, quantized(x, 1)[0].float())
        same(want_scales, quantized(x, 1)[1].float())
    same(got.values, want_values)
    same(got.scales, want_scales)
