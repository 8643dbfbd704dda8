"""What the products in 8-bit blocks refuse before anything is launched."""
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.ops import KernelError


def test_operands_on_the_host_are_refused():
    weight = ops.BlockScaled(torch.zeros((128, 128), dtype=torch.float8_e4m3fn), torch.ones((1, 1)))
    with pytest.raises(KernelError, match="no CPU path"):
        ops.linear(torch.zeros((1, 128)), weight)
    with pytest.raises(KernelError, match="CUDA device"):
        ops.quantize_blocks(torch.zeros((1, 128)))
    with pytest.raises(KernelError, match="CUDA device"):
        ops.block_scaled(torch.zeros((128, 100), dtype=torch.float8_e4m3fn), torch.ones((1, 1)))


def test_what_a_block_scaled_stands_for():
    values = torch.tensor([[1.0, -2.0, 448.0]]).to(torch.float8_e4m3fn)
    rows = ops.BlockScaled(values.repeat(1, 50)[:, :130], torch.tensor([[0.5, 3.0]]), 1)
    assert rows.shape == (1, 130) and rows.dtype == torch.float8_e4m3fn
    wide = rows.widened()
    assert wide[0, :3].tolist() == [0.5, -1.0, 224.0] and wide[0, 127:].tolist() == [-1.0, 1344.0, 3.0]
    whole = ops.BlockScaled(torch.ones((130, 2)).to(torch.float8_e4m3fn), torch.tensor([[2.0], [5.0]]))
    assert whole.widened()[127:129, 1].tolist() == [2.0, 5.0]


@pytest.mark.parametrize("rows,inner,pitch,block_rows", [(-1, 128, 128, 1), (1, 0, 16, 1), (1, 128, 112, 1), (1, 128, 136, 1), (1, 128, 128, 2)])
def test_the_launcher_refuses_sizes_it_cannot_take(rows, inner, pitch, block_rows):
    library = ops.library()
    assert library.llm_quantize_blocks(0, 0, 0, 0, rows, inner, pitch, block_rows, 0) == -1
    assert b"quantize_blocks" in library.llm_last_error()


def test_the_product_refuses_sizes_it_cannot_take():
    library = ops.library()

    def run(m=1, n=128, inner=128, x_pitch=128, w_pitch=128, x=0, w=0, scratch=0, dtype=-1):
        return library.llm_block_linear(x, dtype, x_pitch, 0, w, w_pitch, 0, 0, 0, m, n, inner, scratch, 0, 0)

    assert run(m=0) == 0
    for given in ({"m": -1}, {"n": 0}, {"inner": 0}, {"x_pitch": 120}, {"w_pitch": 120}, {"x_pitch": 112}, {"w_pitch": 112}, {"x": 8}, {"w": 4},
                  {"m": 65535 * 128 + 1}, {"scratch": 8}, {"dtype": 2}, {"dtype": 0}):
        assert run(**given) == -1, given
        assert library.llm_last_error()


def test_dtype_codes_are_checked_before_a_launch():
    assert ops.library().llm_quantize_blocks(0, 7, 0, 0, 1, 128, 128, 1, 0) == -1
