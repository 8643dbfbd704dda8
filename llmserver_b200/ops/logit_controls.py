"""Penalties for repeated tokens, biases and masks on a step's logits, and tokens drawn from the result.

``LogitControls`` says what holds for each row of a step's logits; ``control_logits`` returns the logits under it, and ``ops.sample``
with ``controls`` draws a token from them without writing them.  Token v of a row with logit l, each step rounded to 32 bits:

    v stands in the request, prompt or answer:   l <- l / repetition if l > 0 else l * repetition
    v stands c > 0 times in the answer:          l <- (l - c * frequency) - presence
    the row's list has a bias for v:             l <- l + bias
    the row's mask has no bit for v:             l <- -inf
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Mapping, Optional, Sequence

import torch

from .library import KernelError, call, check, current_device, library, pointer, stream_handle, wait_error_flag


@dataclass
class LogitControls:
    """Each of the three kinds may be absent (its ``*_rows`` None), and a row goes without one by the index -1.

    ``history`` int32 [H, capacity]: token ids of H requests, of which the first ``lengths[r]`` of row ``history_rows[r]`` belong to the
    request of logits row r and the first ``prompt_lengths[r]`` of those are its prompt; ``penalties`` float32 [R, 3]: repetition (positive; 1: none),
    presence and frequency (0: none).  Ids outside the vocabulary count nowhere.
    ``bias_starts`` int32 [B + 1], ``bias_ids`` int32, ``bias_values`` float32: list b holds entries bias_starts[b] .. bias_starts[b + 1] - 1,
    ids ascending and each once (``bias_lists`` makes them); ``bias_rows`` int32 [R].
    ``masks`` int32 [M, >= ceil(V / 32)]: bit v % 32 of word v / 32 set where token v is allowed (``token_masks`` makes them); ``mask_rows`` int32 [R].

    An index that names no history, list or mask sets the device's shared error flag to 8 and counts as -1."""
    penalties: Optional[torch.Tensor] = None
    history: Optional[torch.Tensor] = None
    history_rows: Optional[torch.Tensor] = None
    lengths: Optional[torch.Tensor] = None
    prompt_lengths: Optional[torch.Tensor] = None
    bias_starts: Optional[torch.Tensor] = None
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    bias_rows: Optional[torch.Tensor] = None
    masks: Optional[torch.Tensor] = None
    mask_rows: Optional[torch.Tensor] = None


class _Controls(ctypes.Structure):      # LlmControls of csrc/logit_controls.cu
    _fields_ = [("penalties", ctypes.c_void_p), ("history", ctypes.c_void_p), ("history_rows", ctypes.c_void_p), ("lengths", ctypes.c_void_p),
                ("prompt_lengths", ctypes.c_void_p), ("histories", ctypes.c_int), ("capacity", ctypes.c_int), ("bias_starts", ctypes.c_void_p),
                ("bias_ids", ctypes.c_void_p), ("bias_values", ctypes.c_void_p), ("bias_rows", ctypes.c_void_p), ("bias_lists", ctypes.c_int),
                ("bias_entries", ctypes.c_int), ("masks", ctypes.c_void_p), ("mask_rows", ctypes.c_void_p), ("mask_count", ctypes.c_int),
                ("mask_words", ctypes.c_int), ("error_flag", ctypes.c_void_p)]


MOST_HISTORY = (1 << 30) - 1        # tokens of a request that a 30-bit count can hold


def _checked(tensor, name: str, device: torch.device, dtype: torch.dtype, *shape) -> torch.Tensor:
    if tensor is None:
        raise KernelError(f"the controls lack {name}")
    check(tensor, name, dtype)
    if tensor.device != device:
        raise KernelError(f"{name} lies on {tensor.device}, the logits on {device}")
    if tensor.dim() != len(shape) or any(want is not None and have != want for have, want in zip(tensor.shape, shape)):
        raise KernelError(f"{name} must be [{', '.join('*' if want is None else str(want) for want in shape)}], got {tuple(tensor.shape)}")
    return tensor


def _described(logits: torch.Tensor, controls: LogitControls, note: bool = False) -> _Controls:
    """The kernel's view of the controls, checked."""
    check(logits, "logits", torch.float32)
    if logits.dim() != 2:
        raise KernelError(f"logits must be [rows, vocabulary], got {tuple(logits.shape)}")
    current_device(logits, "logits")
    rows, vocab = logits.shape
    device, whole = logits.device, torch.int32
    c, said = controls, _Controls()
    if c.history_rows is not None:
        history = _checked(c.history, "history", device, whole, None, None)
        if history.shape[1] > MOST_HISTORY:
            raise KernelError(f"a history holds at most {MOST_HISTORY} tokens, not {history.shape[1]}")
        said.history, said.histories, said.capacity = history.data_ptr(), history.shape[0], history.shape[1]
        said.history_rows = _checked(c.history_rows, "history_rows", device, whole, rows).data_ptr()
        said.lengths = _checked(c.lengths, "lengths", device, whole, rows).data_ptr()
        said.prompt_lengths = _checked(c.prompt_lengths, "prompt_lengths", device, whole, rows).data_ptr()
        if c.penalties is not None:
            said.penalties = _checked(c.penalties, "penalties", device, torch.float32, rows, 3).data_ptr()
    elif c.penalties is not None or note:
        raise KernelError("penalties and noted tokens go with a history (history_rows)")
    if c.bias_rows is not None:
        starts = _checked(c.bias_starts, "bias_starts", device, whole, None)
        if starts.numel() < 1:
            raise KernelError("bias_starts holds one number more than there are lists")
        ids = _checked(c.bias_ids, "bias_ids", device, whole, None)
        said.bias_starts, said.bias_ids = starts.data_ptr(), ids.data_ptr()
        said.bias_values = _checked(c.bias_values, "bias_values", device, torch.float32, ids.numel()).data_ptr()
        said.bias_rows = _checked(c.bias_rows, "bias_rows", device, whole, rows).data_ptr()
        said.bias_lists, said.bias_entries = starts.numel() - 1, ids.numel()
    if c.mask_rows is not None:
        masks = _checked(c.masks, "masks", device, whole, None, None)
        if masks.shape[1] * 32 < vocab:
            raise KernelError(f"masks of {masks.shape[1]} words do not cover {vocab} tokens")
        said.masks, said.mask_count, said.mask_words = masks.data_ptr(), masks.shape[0], masks.shape[1]
        said.mask_rows = _checked(c.mask_rows, "mask_rows", device, whole, rows).data_ptr()
    said.error_flag = wait_error_flag(device).data_ptr()
    return said


def control_logits(logits: torch.Tensor, controls: LogitControls, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits (float32 [R, V]) under ``controls``, in a new tensor or in ``out``, which may be ``logits`` itself."""
    said = _described(logits, controls)
    if out is None:
        out = torch.empty_like(logits)
    else:
        check(out, "controlled logits", torch.float32)
        if out.shape != logits.shape or out.device != logits.device:
            raise KernelError(f"the controlled logits {tuple(out.shape)} do not match {tuple(logits.shape)}")
    rows, vocab = logits.shape
    call("llm_control_logits", logits.data_ptr(), out.data_ptr(), rows, vocab, ctypes.byref(said), stream_handle())
    return out


def sample_controlled(logits: torch.Tensor, temperatures, seeds, steps, out: torch.Tensor, flags, controls: LogitControls, note: bool) -> torch.Tensor:
    """``ops.sample`` with controls (the types of its other arguments are checked there)."""
    said = _described(logits, controls, note)
    rows, vocab = logits.shape
    for name, tensor, size in (("temperatures", temperatures, rows), ("seeds", seeds, rows), ("steps", steps, rows), ("tokens", out, rows + (2 if flags else 0))):
        if tensor is not None and (tensor.numel() != size or tensor.device != logits.device):
            raise KernelError(f"{rows} rows of logits on {logits.device} and {tensor.numel()} {name} on {tensor.device}")
    slices = library().llm_control_slices(rows, vocab, said.capacity)
    scratch = torch.empty((2, rows, slices), dtype=torch.float32, device=logits.device)
    call("llm_control_sample", logits.data_ptr(), pointer(temperatures), pointer(seeds), pointer(steps), out.data_ptr(), rows, vocab, ctypes.byref(said),
         controls.history.data_ptr() if note else 0, scratch.data_ptr(), scratch.data_ptr() + 4 * rows * slices,
         *((flags[0].data_ptr(), flags[1].data_ptr()) if flags else (0, 0)), stream_handle())
    return out


def bias_lists(biases: Sequence[Mapping[int, float]], vocab: int, device) -> dict:
    """``bias_starts``, ``bias_ids`` and ``bias_values`` of ``LogitControls`` for one mapping (token -> bias) per list."""
    starts, ids, values = [0], [], []
    for index, entries in enumerate(biases):
        for token in sorted(entries):
            if not 0 <= int(token) < vocab:
                raise KernelError(f"bias list {index}: token {token} is outside the vocabulary of {vocab}")
            ids.append(int(token))
            values.append(float(entries[token]))
        starts.append(len(ids))
    return {"bias_starts": torch.tensor(starts, dtype=torch.int32, device=device), "bias_ids": torch.tensor(ids, dtype=torch.int32, device=device),
            "bias_values": torch.tensor(values, dtype=torch.float32, device=device)}


def token_masks(allowed: torch.Tensor) -> torch.Tensor:
    """``masks`` of ``LogitControls`` from truth values [M, V] (on any device, where the result lies too)."""
    if allowed.dim() != 2 or allowed.dtype != torch.bool:
        raise KernelError(f"token_masks takes truth values [masks, vocabulary], got {allowed.dtype} {tuple(allowed.shape)}")
    count, vocab = allowed.shape
    words = -(-vocab // 32)
    bits = torch.nn.functional.pad(allowed, (0, words * 32 - vocab)).view(count, words, 32).to(torch.int64)
    packed = (bits << torch.arange(32, device=allowed.device)).sum(2)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)
