"""Controls on logits, rounding to 8 bits and products at the sizes of a busy server's steps and of long prompts, whose slices, laps, lists and rounds of
tiles smaller sizes do not have.  (Slices, rounds and groups are named as 148 SMs make them.)"""
import math
import random

import pytest
import torch

from llmserver_b200 import ops
from test_gpu_block_scaled import close as product_close
from test_gpu_block_scaled import matrix, quantized_rows, same
from test_gpu_kernels import DEVICE, rand
from test_gpu_logit_controls import Request, close, controls_of, finished, logits_for, some_requests

pytestmark = pytest.mark.gpu


def drawn_of(rows, seed):
    """Temperatures (one row in five greedy), seeds and steps."""
    generator = torch.Generator().manual_seed(seed)
    return ((0.2 + torch.rand(rows, generator=generator)) * (torch.rand(rows, generator=generator) < 0.8)).to(DEVICE), \
        torch.randint(0, 1 << 62, (rows,), generator=generator).to(DEVICE), torch.randint(0, 5000, (rows,), generator=generator, dtype=torch.int32).to(DEVICE)


def whole_step(logits, requests, controls):
    """Returned, returned in place, drawn greedily and at temperatures."""
    rows = logits.shape[0]
    steered = ops.control_logits(logits, controls)
    finished()
    close(steered, logits, requests)
    nothing = (steered == -math.inf).all(dim=1)
    for drawn in ((), drawn_of(rows, 7)):
        got, want = ops.sample(logits, *drawn, controls=controls), ops.sample(steered, *drawn)
        finished()
        # (a row of which nothing is said draws as it would alone)
        assert torch.equal(got, torch.where(nothing, -1, want))
    assert ops.control_logits(logits, controls, out=logits) is logits
    finished()
    assert torch.equal(logits, steered)


# slices of 25344 tokens and 7 laps; of 25024, with a vocabulary that no four tokens divide; two rounds of blocks, one slice a row; slices that end 32
# tokens into their second lap; marks of 32 bits
@pytest.mark.parametrize("rows,vocab,length,biases", [(64, 151936, 4096, 50), (100, 100003, 3000, 20), (600, 9001, 500, 10), (150, 8196, 900, 10), (37, 130001, 20000, 300)])
def test_slices_of_many_laps(rows, vocab, length, biases):
    requests = some_requests(rows, vocab, length, rows + vocab, biases)
    whole_step(logits_for(rows, vocab, 50), requests, controls_of(requests, vocab))


@pytest.mark.parametrize("vocab", [151936, 100003])
def test_the_best_token_wherever_it_lies(vocab):
    """One far above the others, or two that are equal, in the first lap, in a middle one, in the last, at the ends of slices: marked or not."""
    rows = 64
    logits = logits_for(rows, vocab, 51)
    requests, want = [], []
    rng = random.Random(5)
    for row in range(rows):
        low, high = sorted((rng.choice((0, 4095, 4096, 8191, 16671, 16672, 25343, 25344, vocab - 1, rng.randrange(vocab))), rng.randrange(vocab)))
        logits[row, low] = logits[row, high] = 100.0
        held = [[], [low], [high], [low, high]][row % 4]
        # a presence penalty takes the marked one below its equal
        requests.append(Request([], held, presence=1.0))
        want.append(low if low == high or not (low in held and high not in held) else high)
    controls = controls_of(requests, vocab)
    got = ops.sample(logits, controls=controls)
    finished()
    assert got.tolist() == want
    whole_step(logits, requests, controls)


# slices of 10016 tokens, listed when they are marked first; of 3008, looked through
@pytest.mark.parametrize("rows,vocab", [(64, 60000), (200, 6000)])
@pytest.mark.parametrize("capacity", [16383, 16384])      # marks of 16 bits and of 32
def test_lists_of_marked_tokens_that_overflow(rows, vocab, capacity):
    """2047 to 2049 marked tokens in the first slice, all of its tokens, and few, side by side."""
    rng = random.Random(vocab + capacity)
    first = 10016 if rows == 64 else 3008
    requests = []
    for row in range(rows):
        kind = row % 6
        count = (2047, 2048, 2049, first, 5, 0)[kind]
        held = rng.sample(range(first), count)
        held += [rng.choice(held) for _ in range(100)] if held else []
        rng.shuffle(held)
        held += [rng.randrange(first, vocab) for _ in range(50)]
        bias = {rng.choice(held): 2.0 - row % 5 for _ in range(30)} if row % 2 else None
        allowed = torch.rand(vocab, generator=torch.Generator().manual_seed(row)) < 0.5 if row % 3 == 0 else None
        cut = rng.randrange(len(held) + 1)
        requests.append(Request(held[:cut], held[cut:], 1.0 + rng.random(), rng.random(), rng.random(), bias, allowed))
    whole_step(logits_for(rows, vocab, 52), requests, controls_of(requests, vocab, capacity=capacity))


@pytest.mark.parametrize("capacity", [16383, 16384, 40000])
@pytest.mark.parametrize("vocab", [3000, 60000])
def test_one_token_as_often_as_a_history_holds(capacity, vocab):
    """The times fill their bits beside the flags of the prompt, of a bias and of the neighbour that shares the word."""
    rows = 64
    requests = []
    for row in range(rows):
        token = row % 4 + 10
        prompt = [token ^ 1] if row % 2 else []
        answer = [token] * (capacity - len(prompt) - row % 3)
        requests.append(Request(prompt, answer, 1.5, 0.25, 2.0 ** -12, {token: 3.0, token ^ 1: -1.0} if row % 5 == 0 else None))
    whole_step(logits_for(rows, vocab, 53), requests, controls_of(requests, vocab, capacity=capacity))


# groups that lie one after the other, several at once for each half warp and once more
@pytest.mark.parametrize("rows,columns", [(20000, 512), (76001, 128), (37889, 256), (9473, 1024)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows_of_whole_groups(rows, columns, dtype):
    x = rand((rows, columns), dtype, 54)
    x[rows // 2] = 0
    x[rows - 1, columns - 1] = 1e4
    x[5] *= 1e-30
    got = ops.quantize_blocks(x)
    finished()
    want_values, want_scales = quantized_rows(x)
    same(got.values, want_values)
    same(got.scales, want_scales)


# tiles of 256 columns, several a block and several units of k each; with rows of x in more than one part of 32 MiB, for W of a down projection;
# ragged in all three sizes, in pieces that leave number by number
@pytest.mark.parametrize("rows,inner,cols", [(1500, 1024, 8192), (2900, 12288, 4096), (2817, 12300, 4100), (8192, 1152, 2304), (1025, 2001, 10241)])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
def test_products_of_prompts(rows, inner, cols, out_dtype):
    weight = matrix(cols, inner, 55)
    x = rand((rows, inner), torch.bfloat16, 56)
    got = ops.linear(x, weight, out_dtype=out_dtype)
    finished()
    product_close(got, ops.quantize_blocks(x), weight)


@pytest.mark.parametrize("rows", [1, 40, 300, 2000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_how_far_products_in_8_bits_lie_from_unrounded_ones(rows, dtype):
    """Both operands in 8 bits as the engine's matrices are.  A number of e4m3 is off by half a step: 2^-4 of it, or 2^-10 of its scale below the normal
    numbers; the products of what is off, and the sums' own errors on the rounded operands behind it."""
    inner, cols = 1000, 1400
    x, w = rand((rows, inner), dtype, 57), rand((cols, inner), dtype, 58, inner ** -0.5)
    weight, held = ops.quantize_blocks(w, 128), ops.quantize_blocks(x)
    got = ops.linear(x, weight, out_dtype=torch.float32)
    finished()

    def off(values, operand):
        scales = operand.scales.double().repeat_interleave(128, dim=1)[:, :inner].repeat_interleave(operand.block_rows, dim=0)[:values.shape[0]]
        return torch.maximum(values.double().abs() * 2.0 ** -4, scales * 2.0 ** -10)

    off_x, off_w = off(x, held), off(w, weight)
    size_x, size_w = x.double().abs(), w.double().abs()
    bound = size_x @ off_w.t() + off_x @ size_w.t() + off_x @ off_w.t()
    sums = (2 * 128 + 3 + 8) * 2.0 ** -24 * ((size_x + off_x) @ (size_w + off_w).t())
    want = x.double() @ w.double().t()
    assert bool(((got.double() - want).abs() <= bound + sums).all())
    assert float((got.double() - want).norm() / want.norm()) > 2.0 ** -8      # the rounding is there
