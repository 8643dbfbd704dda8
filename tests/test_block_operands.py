"""Operands of products in 8-bit blocks that the host refuses, seen without a GPU through tensors that only claim to lie on one."""
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.ops import KernelError
from llmserver_b200.ops.block_scaled import _checked, _sound

F8 = torch.float8_e4m3fn


class Claimed:
    """A host tensor that says it lies on a CUDA device."""

    def __init__(self, tensor, index):
        self.tensor, self.is_cuda, self.device = tensor, True, torch.device("cuda", index)

    def get_device(self):
        return self.device.index

    def float(self):
        return self

    def contiguous(self):
        return self

    def __getattr__(self, name):
        return getattr(self.tensor, name)


def operand(rows, columns, block_rows, values_on=0, scales_on=0):
    values = torch.zeros((rows, -(-columns // 16) * 16), dtype=F8)[:, :columns]
    return ops.BlockScaled(Claimed(values, values_on), Claimed(torch.ones((-(-rows // block_rows), -(-columns // 128))), scales_on), block_rows)


@pytest.mark.parametrize("rows,columns", [(256, 256), (130, 100), (1, 16)])
def test_scales_on_another_device_than_their_values_are_refused(rows, columns):
    weight = operand(rows, columns, 128, 0, 1)
    with pytest.raises(KernelError, match="cuda:0 and cuda:1"):
        ops.block_linear(Claimed(torch.zeros((3, columns)), 0), weight)
    with pytest.raises(KernelError, match="cuda:1 and cuda:0"):
        ops.block_linear(operand(3, columns, 1, 1, 0), operand(rows, columns, 128))
    with pytest.raises(KernelError, match="cuda:0 and cuda:1"):
        ops.block_scaled(weight.values, weight.scales)


@pytest.mark.parametrize("block_rows", [1, 128])
def test_both_looks_at_an_operand_agree(block_rows):
    """What the quick look lets through the thorough one does, and what it does not the thorough one refuses: but for the operands that it alone knows
    to be fine (no rows, one row or one column, whose strides do not matter)."""
    good = operand(200, 300, block_rows)
    assert _sound(good, block_rows) and _checked(good, block_rows, "x") is good
    wrong = [operand(200, 300, block_rows, 0, 1), ops.BlockScaled(good.values, good.scales, 129 - block_rows)]
    for values in (torch.zeros((200, 300), dtype=F8), torch.zeros((304, 200), dtype=F8).t()[:, :300], torch.zeros((200, 304), dtype=torch.uint8)[:, :300],
                   torch.zeros(200 * 304 + 1, dtype=F8)[1:].view(200, 304)[:, :300], torch.zeros((1, 304), dtype=F8).expand(200, 304)[:, :300]):
        wrong.append(ops.BlockScaled(Claimed(values, 0), good.scales, block_rows))
    shape = tuple(good.scales.shape)
    for scales in (torch.ones(shape, dtype=torch.float64), torch.ones((shape[0], shape[1] + 1)), torch.ones(shape[::-1]).t(), torch.ones(shape).view(-1)):
        if tuple(scales.shape) != shape or not scales.is_contiguous() or scales.dtype != torch.float32:
            wrong.append(ops.BlockScaled(good.values, Claimed(scales, 0), block_rows))
    for made in wrong:
        assert not _sound(made, block_rows)
        with pytest.raises(KernelError):
            _checked(made, block_rows, "x")


def claimed(shape, dtype, strides=None):
    """One of any size, without memory."""
    if strides is None:
        return Claimed(torch.empty(shape, dtype=dtype, device="meta"), 0)
    return Claimed(torch.empty_strided(shape, strides, dtype=dtype, device="meta"), 0)


HUGE = (1 << 32) + 3      # 3, where 32 bits are kept of it


def test_sizes_beyond_32_bits_are_refused():
    """They do not reach a launcher, whose whole numbers are of 32 bits."""
    for shape in ((HUGE, 1), (1, HUGE), ((1 << 31) - 1, 1), (1, (1 << 31) - 1)):
        with pytest.raises(KernelError, match="at most"):
            ops.quantize_blocks(claimed(shape, torch.bfloat16))
        with pytest.raises(KernelError, match="at most"):
            ops.control_logits(claimed(shape, torch.float32), ops.LogitControls())
        with pytest.raises(KernelError, match="at most"):
            ops.sample(claimed(shape, torch.float32), controls=ops.LogitControls())
    for rows, inner, cols in ((HUGE, 16, 16), (16, HUGE, 16), (16, 16, HUGE)):
        pitch = -(-inner // 16) * 16
        weight = ops.BlockScaled(claimed((cols, inner), F8, (pitch, 1)), claimed((-(-cols // 128), -(-inner // 128)), torch.float32))
        with pytest.raises(KernelError, match="at most"):
            ops.block_linear(claimed((rows, inner), torch.bfloat16), weight)


def test_launchers_refuse_places_that_32_bits_cannot_count():
    library, most = ops.library(), (1 << 31) - 1
    pitch = 1 << 31
    assert library.llm_quantize_blocks(0, 0, 0, 0, 1, most, pitch, 1, 0) == -1
    assert library.llm_quantize_blocks(0, 0, 0, 0, most, 16, 16, 1, 0) == -1
    for n, inner in ((most, 16), (16, most)):
        assert library.llm_block_linear(0, -1, pitch, 0, 0, pitch, 0, 0, 0, 1, n, inner, 0, 0, 0) == -1
    from llmserver_b200.ops.logit_controls import _DESCRIPTION
    said = _DESCRIPTION.pack(*[0] * 18)
    assert library.llm_control_logits(0, 0, 1, most, said, 0) == -1
    assert library.llm_control_sample(0, 0, 0, 0, 0, 1, most, said, 0, 0, 0, 0, 0, 0) == -1
    assert library.llm_control_logits(0, 0, 0, 0x7FFE0000, said, 0) == 0 and library.llm_block_linear(0, -1, pitch, 0, 0, pitch, 0, 0, 0, 0, 0x7FFFFF00, 16, 0, 0, 0) == 0
