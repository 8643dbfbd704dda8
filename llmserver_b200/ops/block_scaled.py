"""Rows and matrices in 8 bits (e4m3) with a 32-bit scale for each block, and products of them.

A ``BlockScaled`` of ``block_rows`` 128 is a projection's matrix W [out, in] as checkpoints in 8 bits keep it: a scale for each
128 x 128.  One of ``block_rows`` 1 holds rows of activations: a scale for each row and 128 columns.  ``ops.linear`` takes the first
in place of a weight, and either a plain tensor (brought to 8 bits on the way) or the second as its rows:

    weight = ops.quantize_blocks(w, 128)                       # once, when the weights are loaded
    y = ops.linear(x, weight)                                  # x bfloat16 or float32 [N, in]
    rows = ops.quantize_blocks(x)                              # once for several products of the same rows
    a, b = ops.linear(rows, weight_a), ops.linear(rows, weight_b)
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from .library import KernelError, call, check, current_device, dtype_code, stream_handle, wait_error_flag

BLOCK = 128
MOST_ALONG = 0x7FFFFF00     # rows or columns: the kernels count places in 32 bits
FLOAT8 = torch.float8_e4m3fn


def _blocks(count: int, size: int = BLOCK) -> int:
    return -(-count // size)


def _pitch(inner: int) -> int:
    """Bytes from one row to the next: the copies of the product kernel begin at multiples of 16 bytes."""
    return -(-inner // 16) * 16


@dataclass
class BlockScaled:
    """``values`` (float8_e4m3fn [rows, columns]) times ``scales`` (float32 [ceil(rows / block_rows), ceil(columns / 128)]), each scale for
    ``block_rows`` (1 or 128) rows and 128 columns.  The rows of ``values`` may lie apart (``values.stride(0)``); the product kernel wants
    them at multiples of 16 bytes, which ``block_scaled`` sees to."""
    values: torch.Tensor
    scales: torch.Tensor
    block_rows: int = BLOCK

    @property
    def shape(self) -> torch.Size:
        return self.values.shape

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def dtype(self) -> torch.dtype:
        return self.values.dtype

    def widened(self) -> torch.Tensor:
        """The numbers that this stands for, float32."""
        rows, columns = self.values.shape
        wide = self.scales.repeat_interleave(BLOCK, dim=1)[:, :columns]
        return self.values.float() * (wide if self.block_rows == 1 else wide.repeat_interleave(self.block_rows, dim=0)[:rows])


def block_scaled(values: torch.Tensor, scales: torch.Tensor, block_rows: int = BLOCK) -> BlockScaled:
    """A ``BlockScaled`` of a checkpoint's tensors; ``values`` are copied into rows at multiples of 16 bytes where theirs are not, ``scales``
    are widened to float32."""
    result = BlockScaled(values, scales.float().contiguous(), block_rows)
    if values.dim() == 2 and values.dtype == FLOAT8 and values.shape[1] > 0 and (
            values.stride(1) != 1 or values.stride(0) % 16 or values.stride(0) < values.shape[1] or values.data_ptr() % 16):
        rows, columns = values.shape
        kept = torch.empty((rows, _pitch(columns)), dtype=FLOAT8, device=values.device)[:, :columns]
        kept.view(torch.uint8).copy_(values.view(torch.uint8))
        result.values = kept
    return _checked(result, block_rows, "block-scaled tensor")


def _checked(operand: BlockScaled, block_rows: int, name: str) -> BlockScaled:
    values, scales = operand.values, operand.scales
    if not (values.is_cuda and scales.is_cuda):
        raise KernelError(f"{name} must live on a CUDA device (there is no CPU path); it is on {values.device} and {scales.device}")
    if values.device != scales.device:
        raise KernelError(f"{name}: values and scales lie on {values.device} and {scales.device}")
    if values.dtype != FLOAT8 or scales.dtype != torch.float32 or values.dim() != 2:
        raise KernelError(f"{name} must be float8_e4m3fn [rows, columns] with float32 scales, got {values.dtype} {tuple(values.shape)} and {scales.dtype}")
    if operand.block_rows != block_rows:
        raise KernelError(f"{name}: scales for {block_rows} rows are needed, these are for {operand.block_rows}")
    rows, columns = values.shape
    if columns < 1 or (block_rows > 1 and rows < 1):
        raise KernelError(f"{name} is empty: {tuple(values.shape)}")
    if tuple(scales.shape) != (_blocks(rows, block_rows), _blocks(columns)) or not scales.is_contiguous():
        raise KernelError(f"{name}: {tuple(values.shape)} in blocks of {block_rows} x {BLOCK} has contiguous scales "
                          f"[{_blocks(rows, block_rows)}, {_blocks(columns)}], got {tuple(scales.shape)} with strides {scales.stride()}")
    stride = values.stride(0) if rows > 1 else max(values.stride(0), _pitch(columns))
    if (values.stride(1) != 1 and columns > 1) or stride % 16 or stride < columns or values.data_ptr() % 16:
        raise KernelError(f"{name}: rows must begin at multiples of 16 bytes (strides {values.stride()}, address {values.data_ptr():#x}); "
                          "block_scaled() copies them so")
    return operand


def _sound(operand: BlockScaled, block_rows: int) -> bool:
    """Whether an operand is as the product takes it, in a few looks (``_checked`` says what is wrong with one that is not)."""
    values, scales = operand.values, operand.scales
    rows, columns = values.shape
    stride, step = values.stride()
    return (values.dtype is FLOAT8 and scales.dtype is torch.float32 and operand.block_rows == block_rows and step == 1 and stride % 16 == 0
            and stride >= columns > 0 and rows > 0 and values.data_ptr() % 16 == 0 and scales.is_contiguous()
            and scales.shape == (-(-rows // block_rows), -(-columns // BLOCK)) and scales.get_device() == values.get_device() >= 0)


def _row_stride(values: torch.Tensor) -> int:
    """Bytes between rows; of a single row whatever the kernel may be told."""
    return values.stride(0) if values.shape[0] > 1 else _pitch(values.shape[1])


def quantize_blocks(x: torch.Tensor, block_rows: int = 1) -> BlockScaled:
    """``x`` (float32 or bfloat16 [rows, columns]) in 8 bits: with ``block_rows`` 1 a scale for each row and 128 columns, with 128 one for
    each 128 x 128.  A scale is 2^e with the least e (not below -126) for which no number of the block exceeds 448 * 2^e; the numbers
    are divided by it and rounded to the nearest of e4m3's, ties to the even one.  A block that holds an infinity or a NaN becomes NaN."""
    check(x, "x")
    if x.dim() != 2 or x.shape[1] < 1:
        raise KernelError(f"quantize_blocks takes a matrix, got {tuple(x.shape)}")
    if block_rows not in (1, BLOCK):
        raise KernelError(f"blocks have 1 or {BLOCK} rows, not {block_rows}")
    rows, columns = x.shape
    if max(rows, columns) > MOST_ALONG:
        raise KernelError(f"quantize_blocks takes at most {MOST_ALONG} rows and columns, got {rows} and {columns}")
    current_device(x, "x")
    pitch = _pitch(columns)
    values = x.new_empty((rows, pitch), dtype=FLOAT8)
    scales = x.new_empty((_blocks(rows, block_rows), _blocks(columns)), dtype=torch.float32)
    call("llm_quantize_blocks", x.data_ptr(), dtype_code(x.dtype), values.data_ptr(), scales.data_ptr(), rows, columns, pitch, int(block_rows),
         stream_handle())
    return BlockScaled(values if pitch == columns else values[:, :columns], scales, block_rows)


def block_linear(x, weight: BlockScaled, out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x W^T for W in 8 bits: what ``ops.linear`` does with a ``BlockScaled`` weight.  ``x`` [N, in]: float32 or bfloat16 (brought to 8
    bits as ``quantize_blocks`` does), or a ``BlockScaled`` of single rows.  Sums and scales are 32-bit, and so is the product of a block's two scales
    (below 2^-126 it loses digits); the result is rounded once to
    ``out_dtype`` (float32 or bfloat16; default: that of ``out``, or x's, or bfloat16 where x is in 8 bits)."""
    values = weight.values
    if values.dim() != 2 or not _sound(weight, BLOCK):
        _checked(weight, BLOCK, "weight")
    cols, inner = values.shape
    quantized = isinstance(x, BlockScaled)
    held = x.values if quantized else x
    if not quantized:
        check(x, "x")
    elif held.dim() != 2 or not _sound(x, 1):
        _checked(x, 1, "x")
    if held.dim() != 2:
        raise KernelError(f"block_linear takes rows [N, {inner}], got {tuple(held.shape)}")
    rows, columns = held.shape
    if columns != inner:
        raise KernelError(f"x has {columns} columns, the weight {inner}")
    if max(rows, inner, cols) > MOST_ALONG:
        raise KernelError(f"block_linear takes at most {MOST_ALONG} rows and columns, got {rows} rows and a weight [{cols}, {inner}]")
    index = values.get_device()
    if held.get_device() != index or (out is not None and out.get_device() != index):
        raise KernelError(f"the operands lie on {held.device} and {values.device}" + ("" if out is None else f", the output on {out.device}"))
    current_device(values, "weight")
    if out_dtype is None:
        out_dtype = out.dtype if out is not None else torch.bfloat16 if quantized else x.dtype
    if out_dtype is not torch.bfloat16 and out_dtype is not torch.float32:
        raise KernelError(f"block_linear writes float32 or bfloat16, not {out_dtype}")
    if out is None:
        out = held.new_empty((rows, cols), dtype=out_dtype)
    elif out.dtype != out_dtype or not out.is_contiguous() or tuple(out.shape) != (rows, cols):
        raise KernelError(f"block_linear: the output must be contiguous {out_dtype} [{rows}, {cols}], got {out.dtype} {tuple(out.shape)}")
    scratch = 0
    if quantized:
        kind, pitch, scales = -1, _row_stride(held), x.scales.data_ptr()
    else:
        kind, pitch, scales = dtype_code(x.dtype), _pitch(inner), 0
        room = held.new_empty(rows * (pitch + 4 * _blocks(inner)), dtype=torch.uint8)      # the rows in 8 bits, then their scales
        scratch = room.data_ptr()
    call("llm_block_linear", held.data_ptr(), kind, pitch, scales, values.data_ptr(), _row_stride(values), weight.scales.data_ptr(), out.data_ptr(),
         int(out_dtype is torch.float32), rows, cols, inner, scratch, wait_error_flag(values.device).data_ptr(), stream_handle())
    return out
