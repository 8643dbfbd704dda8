"""Penalties for repeated tokens, biases and masks on a step's logits, and tokens drawn from the result.

``LogitControls`` says what holds for each row of a step's logits; ``control_logits`` returns the logits under it, and ``ops.sample``
with ``controls`` draws a token from them without writing them.  Token v of a row with logit l, each step rounded to 32 bits:

    v stands in the request, prompt or answer:   l <- l / repetition if l > 0 else l * repetition
    v stands c > 0 times in the answer:          l <- (l - c * frequency) - presence
    the row's list has a bias for v:             l <- l + bias
    the row's mask has no bit for v:             l <- -inf
"""
from __future__ import annotations

import struct
from dataclasses import dataclass
from typing import Dict, Mapping, Optional, Sequence

import torch

from .library import KernelError, call, check, current_device, pointer, stream_handle, wait_error_flag


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


# LlmControls of csrc/logit_controls.cu: penalties, history, history_rows, lengths, prompt_lengths, how many histories and how long; starts, ids,
# values and rows of the biases, how many lists and entries; masks, mask_rows, how many masks and words; the error flag
_DESCRIPTION = struct.Struct("@PPPPPiiPPPPiiPPiiP")
_LEAST_SLICE = 2048        # a row is scanned in no more slices than of so many tokens
MOST_LOGITS = 0x7FFE0000   # rows or tokens: the kernels count places in 32 bits
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


def _described(logits: torch.Tensor, controls: LogitControls, note: bool = False) -> bytes:
    """The kernel's view of the controls.  Everything is looked over in one go; where something is not as it should be, ``_complaint`` says
    what."""
    check(logits, "logits", torch.float32)
    if logits.dim() != 2:
        raise KernelError(f"logits must be [rows, vocabulary], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if max(rows, vocab) > MOST_LOGITS:
        raise KernelError(f"logits of at most {MOST_LOGITS} rows and tokens, got {rows} and {vocab}")
    current_device(logits, "logits")
    index, whole = logits.get_device(), torch.int32
    c = controls
    history = lengths = prompts = history_rows = penalties = histories = capacity = 0
    starts = ids = values = bias_rows = lists = entries = 0
    masks = mask_rows = mask_count = words = 0

    def plain(tensor, dtype, size) -> bool:
        return tensor is not None and tensor.dtype is dtype and tensor.get_device() == index and tensor.is_contiguous() and tensor.shape == size

    row = (rows,)
    if c.history_rows is not None:
        held = c.history
        if (held is None or held.dtype is not whole or held.get_device() != index or not held.is_contiguous() or held.dim() != 2
                or held.shape[1] > MOST_HISTORY or not plain(c.history_rows, whole, row) or not plain(c.lengths, whole, row)
                or not plain(c.prompt_lengths, whole, row) or (c.penalties is not None and not plain(c.penalties, torch.float32, (rows, 3)))):
            _complaint(logits, c)
        history, (histories, capacity), history_rows = held.data_ptr(), held.shape, c.history_rows.data_ptr()
        lengths, prompts = c.lengths.data_ptr(), c.prompt_lengths.data_ptr()
        if c.penalties is not None:
            penalties = c.penalties.data_ptr()
    elif c.penalties is not None or note:
        raise KernelError("penalties and noted tokens go with a history (history_rows)")
    if c.bias_rows is not None:
        tokens, first = c.bias_ids, c.bias_starts
        if (tokens is None or first is None or not plain(tokens, whole, tokens.shape[:1]) or not plain(first, whole, first.shape[:1]) or first.numel() < 1
                or not plain(c.bias_values, torch.float32, tokens.shape) or not plain(c.bias_rows, whole, row)):
            _complaint(logits, c)
        starts, ids, values, bias_rows = first.data_ptr(), tokens.data_ptr(), c.bias_values.data_ptr(), c.bias_rows.data_ptr()
        lists, entries = first.numel() - 1, tokens.numel()
    if c.mask_rows is not None:
        bits = c.masks
        if (bits is None or bits.dtype is not whole or bits.get_device() != index or not bits.is_contiguous() or bits.dim() != 2
                or bits.shape[1] * 32 < vocab or not plain(c.mask_rows, whole, row)):
            _complaint(logits, c)
        masks, (mask_count, words), mask_rows = bits.data_ptr(), bits.shape, c.mask_rows.data_ptr()
    if max(histories, lists, entries, mask_count, words) >= 1 << 31:
        raise KernelError(f"the controls hold {histories} histories, {lists} lists of {entries} biases and {mask_count} masks of {words} words; 32 bits count them")
    return _DESCRIPTION.pack(penalties, history, history_rows, lengths, prompts, histories, capacity, starts, ids, values, bias_rows, lists, entries,
                             masks, mask_rows, mask_count, words, wait_error_flag(logits.device).data_ptr())


def _complaint(logits: torch.Tensor, c: LogitControls) -> None:
    """Raises for the first tensor of the controls that is not as it should be."""
    rows, vocab = logits.shape
    device, whole = logits.device, torch.int32
    if c.history_rows is not None:
        history = _checked(c.history, "history", device, whole, None, None)
        if history.shape[1] > MOST_HISTORY:
            raise KernelError(f"a history holds at most {MOST_HISTORY} tokens, not {history.shape[1]}")
        for name in ("history_rows", "lengths", "prompt_lengths"):
            _checked(getattr(c, name), name, device, whole, rows)
        if c.penalties is not None:
            _checked(c.penalties, "penalties", device, torch.float32, rows, 3)
    if c.bias_rows is not None:
        if _checked(c.bias_starts, "bias_starts", device, whole, None).numel() < 1:
            raise KernelError("bias_starts holds one number more than there are lists")
        ids = _checked(c.bias_ids, "bias_ids", device, whole, None)
        _checked(c.bias_values, "bias_values", device, torch.float32, ids.numel())
        _checked(c.bias_rows, "bias_rows", device, whole, rows)
    if c.mask_rows is not None:
        if _checked(c.masks, "masks", device, whole, None, None).shape[1] * 32 < vocab:
            raise KernelError(f"masks of {c.masks.shape[1]} words do not cover {vocab} tokens")
        _checked(c.mask_rows, "mask_rows", device, whole, rows)
    raise KernelError("the controls do not fit the logits")


def control_logits(logits: torch.Tensor, controls: LogitControls, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The logits (float32 [R, V]) under ``controls``, in a new tensor or in ``out``, which may be ``logits`` itself."""
    said = _described(logits, controls)
    if out is None:
        out = torch.empty_like(logits)
    else:
        check(out, "controlled logits", torch.float32)
        if out.shape != logits.shape or out.device != logits.device:
            raise KernelError(f"the controlled logits {tuple(out.shape)} do not match {tuple(logits.shape)}")
        apart = abs(out.data_ptr() - logits.data_ptr())
        if 0 < apart < logits.numel() * 4:
            raise KernelError("the controlled logits go to the logits' own place or to another, not to one that overlaps it")
    rows, vocab = logits.shape
    call("llm_control_logits", logits.data_ptr(), out.data_ptr(), rows, vocab, said, stream_handle())
    return out


def sample_controlled(logits: torch.Tensor, temperatures, seeds, steps, out: Optional[torch.Tensor], flags, controls: LogitControls, note: bool) -> torch.Tensor:
    """``ops.sample`` with controls."""
    said = _described(logits, controls, note)
    rows, vocab = logits.shape
    index, device = logits.get_device(), logits.device
    if temperatures is not None:
        for name, tensor, dtype in (("temperatures", temperatures, torch.float32), ("seeds", seeds, torch.int64), ("steps", steps, torch.int32)):
            if tensor is None:
                raise KernelError("temperature sampling needs seeds and steps")
            if tensor.dtype is not dtype or tensor.get_device() != index or not tensor.is_contiguous() or tensor.numel() != rows:
                check(tensor, name, dtype)
                raise KernelError(f"{rows} rows of logits on {device} and {tensor.numel()} {name} on {tensor.device}")
    if flags:
        for flag in flags:
            check(flag, "flag", torch.int32, 1)
            if flag.get_device() != index:
                raise KernelError(f"a flag lies on {flag.device}, the logits on {device}")
        if rows == 0:
            raise KernelError("no tokens and two flags")
    if out is None:
        out = logits.new_empty(rows + (2 if flags else 0), dtype=torch.int32)
    else:
        check(out, "sampled tokens", torch.int32)
        if out.numel() != rows + (2 if flags else 0) or out.get_device() != index:
            raise KernelError(f"{rows} tokens{' and two flags' if flags else ''} do not fit {out.numel()} elements on {out.device}")
    most = rows * -(-vocab // _LEAST_SLICE)       # a score and a token for each slice of each row
    scratch = logits.new_empty(2 * most)
    call("llm_control_sample", logits.data_ptr(), pointer(temperatures), pointer(seeds), pointer(steps), out.data_ptr(), rows, vocab, said,
         controls.history.data_ptr() if note else 0, scratch.data_ptr(), scratch.data_ptr() + 4 * most,
         *((flags[0].data_ptr(), flags[1].data_ptr()) if flags else (0, 0)), stream_handle())
    return out


def biases_by_token(entries: Mapping, vocab: int) -> Dict[int, float]:
    """Token -> bias in ascending order.  The keys are whole numbers, or texts of such, which JSON makes of them; raises ValueError for any
    other, for tokens outside the vocabulary and for a token that is named twice."""
    found = {}
    for key, value in entries.items():
        try:
            token = int(key)
        except (TypeError, ValueError, OverflowError):
            token = None
        if token is None or (not isinstance(key, str) and token != key):
            raise ValueError(f"a bias for {key!r}, which is no token")
        if not 0 <= token < vocab:
            raise ValueError(f"a bias for token {token}, which is outside the vocabulary of {vocab}: tokens are 0 to {vocab - 1}")
        if token in found:
            raise ValueError(f"two biases for token {token}")
        found[token] = float(value)
    return dict(sorted(found.items()))


def bias_lists(biases: Sequence[Mapping[int, float]], vocab: int, device) -> dict:
    """``bias_starts``, ``bias_ids`` and ``bias_values`` of ``LogitControls`` for one mapping (token -> bias) per list."""
    starts, ids, values = [0], [], []
    for index, entries in enumerate(biases):
        try:
            whole = biases_by_token(entries, vocab)
        except ValueError as error:
            raise KernelError(f"bias list {index}: {error}") from error
        ids.extend(whole)
        values.extend(whole.values())
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
