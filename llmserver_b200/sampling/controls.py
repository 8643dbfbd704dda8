"""What a request may say about its logits beside temperature and seed, and the table that keeps it on the device.

``RequestControls`` holds a request's penalties for repeated tokens, its biases and its grammar (a function of the tokens generated so
far); ``ControlTable`` keeps the histories of such requests on the device and describes a step's rows for ``ops.sample``, which applies the
controls, draws a token and notes it.  The reference samples greedily without any of these (utils/engine.py:295-297).
"""
from __future__ import annotations

import math
from dataclasses import dataclass, replace
from typing import Callable, Dict, List, Mapping, Optional, Sequence

import numpy as np
import torch

from .. import ops
from ..ops.logit_controls import biases_by_token


def _in_32_bits(value: float) -> float:
    with np.errstate(over="ignore"):
        return float(np.float32(value))


@dataclass(frozen=True)
class RequestControls:
    """``repetition_penalty`` (positive): logits of tokens that stand in the prompt or the answer are divided by it where they are positive and
    multiplied where not.  ``frequency_penalty`` times the times a token stands in the answer, and ``presence_penalty`` where it stands
    there at all, are taken off.  ``logit_bias``: token (a whole number, or the text of one) -> what is added to its logit.
    ``allowed_tokens``: a function of the list of tokens generated so far that gives the tokens allowed next, as ids or as truth values for the
    whole vocabulary, or None where all are."""
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Mapping[int, float]] = None
    allowed_tokens: Optional[Callable[[List[int]], object]] = None

    def check(self, vocab: int) -> "RequestControls":
        """The same with the biases by whole numbers, in a mapping of its own; raises ValueError for what cannot be meant."""
        # (as the device holds them)
        if not (math.isfinite(_in_32_bits(self.repetition_penalty)) and _in_32_bits(self.repetition_penalty) > 0):
            raise ValueError(f"a repetition penalty is a positive number of 32 bits (1: none), not {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not math.isfinite(_in_32_bits(getattr(self, name))):
                raise ValueError(f"{name} must be a finite number of 32 bits, not {getattr(self, name)}")
        biases = biases_by_token(self.logit_bias or {}, vocab)
        for token, value in biases.items():
            if math.isnan(value):
                raise ValueError(f"a bias of {value} for token {token}: biases are numbers")
        if self.allowed_tokens is not None and not callable(self.allowed_tokens):
            raise ValueError("allowed_tokens is a function of the tokens generated so far")
        return replace(self, logit_bias=biases or None)

    @property
    def penalises(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    @property
    def active(self) -> bool:
        return self.penalises or bool(self.logit_bias) or self.allowed_tokens is not None


def mask_words(allowed, vocab: int) -> np.ndarray:
    """The int32 words of a mask from ids or from truth values for the whole vocabulary.  (A step waits for it: packed bits of 151936 truth values
    take 0.02 ms, ids or-ed one by one took 2.)"""
    if isinstance(allowed, torch.Tensor):
        given = allowed.cpu().numpy()
    elif isinstance(allowed, range):
        given = np.arange(allowed.start, allowed.stop, allowed.step)
    else:
        given = np.asarray(allowed if isinstance(allowed, (np.ndarray, list, tuple)) else list(allowed))
    truth = np.zeros(-(-vocab // 32) * 32, dtype=np.bool_)
    if given.dtype == np.bool_:
        if given.shape != (vocab,):
            raise ValueError(f"truth values for {given.shape} tokens, the vocabulary has {vocab}")
        truth[:vocab] = given
    elif given.size:
        if given.dtype.kind not in "iuf" or (given.dtype.kind == "f" and not (given == np.floor(given)).all()):
            raise ValueError(f"allowed tokens are whole numbers, not {given.reshape(-1)[0]!r} and the like")
        if given.min() < 0 or given.max() >= vocab:
            raise ValueError(f"an allowed token is outside the vocabulary of {vocab}")
        truth[given.reshape(-1).astype(np.int64)] = True
    return np.packbits(truth, bitorder="little").view("<i4")


class ControlTable:
    """Histories on the device, a row per request that has penalties: the prompt and the answer so far.  The sampling kernel notes each token
    it draws, so a row is copied only when a request is seen first, or again after the table grew or the request was put out."""

    def __init__(self, device, vocab: int):
        self.device, self.vocab = torch.device(device), int(vocab)
        self.history = torch.zeros((0, 0), dtype=torch.int32, device=self.device)
        self.places: Dict[object, int] = {}
        self.noted: Dict[object, int] = {}       # tokens of the request that its row holds
        self._biased: tuple = ()
        self._bias_lists: dict = {}

    def forget(self, request_id) -> None:
        self.places.pop(request_id, None)
        self.noted.pop(request_id, None)

    def _on_device(self, values: np.ndarray) -> torch.Tensor:
        host = torch.empty(values.shape, dtype=torch.int32, pin_memory=self.device.type == "cuda")
        host.numpy()[...] = values
        return host.to(self.device, non_blocking=True)

    def _place(self, request, needed: int) -> int:
        """The row of a request's history, with room for ``needed`` tokens."""
        if request.request_id not in self.places:
            taken = set(self.places.values())
            self.places[request.request_id] = next(place for place in range(len(taken) + 1) if place not in taken)
            self.noted.pop(request.request_id, None)
        place = self.places[request.request_id]
        rows, capacity = self.history.shape
        if place >= rows or needed > capacity:
            # a larger table; the rows of the old one are copied anew when they are next needed
            self.history = torch.zeros((max(rows, 4, 2 * place), max(capacity, 256, 1 << (needed - 1).bit_length())), dtype=torch.int32, device=self.device)
            self.noted.clear()
        return place

    def allowed(self, requests: Sequence) -> List[Optional[np.ndarray]]:
        """Asks the grammars of a step's rows: per row the words of its mask, or None where all tokens are allowed.  What a grammar raises goes on
        to the caller with a note that names the request; nothing has changed here by then.  A grammar that gives what is no token leaves its
        request nothing to draw from, and ``request.error`` says why."""
        found: List[Optional[np.ndarray]] = []
        for request in requests:
            words = None
            if request is not None and request.controls.allowed_tokens is not None:
                try:
                    given = request.controls.allowed_tokens(list(request.generated_token_ids))
                except Exception as error:
                    error.add_note(f"raised by allowed_tokens of request {request.request_id!r}")
                    raise
                try:
                    words = None if given is None else mask_words(given, self.vocab)
                except (TypeError, ValueError, OverflowError) as error:      # no mask can be made of it: the request ends, the others go on
                    request.error = f"allowed_tokens: {error}"
                    words = np.zeros(-(-self.vocab // 32), dtype=np.int32)
            found.append(words)
        return found

    def describe(self, requests: Sequence, allowed: Optional[Sequence] = None) -> ops.LogitControls:
        """The controls of a step's rows; ``requests``: per row a request with ``controls``, ``request_id``, ``prompt_token_ids`` and
        ``generated_token_ids``, or None for a row without controls.  ``allowed``: what ``allowed`` gave for them (default: it is asked)."""
        if allowed is None:
            allowed = self.allowed(requests)
        count = len(requests)
        packed = np.zeros((8, count), dtype=np.int32)      # history, bias and mask rows, length, prompt length, then the penalties
        packed[:3] = -1
        penalties = packed[5:].reshape(-1).view(np.float32).reshape(count, 3)
        penalties[:] = (1.0, 0.0, 0.0)
        biased = tuple(request for request in requests if request is not None and request.controls.logit_bias)
        masks, placed = [], []
        for row, request in enumerate(requests):
            if request is None:
                continue
            controls = request.controls
            if controls.penalises:
                held = len(request.prompt_token_ids) + len(request.generated_token_ids)
                packed[0, row] = self._place(request, held + 1)
                packed[3, row], packed[4, row] = held, len(request.prompt_token_ids)
                penalties[row] = (controls.repetition_penalty, controls.presence_penalty, controls.frequency_penalty)
                placed.append((request, held))
            if controls.logit_bias:
                packed[1, row] = biased.index(request)
            if allowed[row] is not None:
                packed[2, row] = len(masks)
                masks.append(allowed[row])
        for request, held in placed:      # (behind all rows: the table may have grown)
            if self.noted.get(request.request_id) != held:
                tokens = np.asarray(list(request.prompt_token_ids) + list(request.generated_token_ids), dtype=np.int32)
                self.history[self.places[request.request_id], :held].copy_(self._on_device(tokens))
            self.noted[request.request_id] = held + 1      # the draw notes one more
        on_device = self._on_device(packed.reshape(-1))
        result = ops.LogitControls()
        if placed:
            result.history, result.history_rows = self.history, on_device[:count]
            result.lengths, result.prompt_lengths = on_device[3 * count:4 * count], on_device[4 * count:5 * count]
            result.penalties = on_device[5 * count:].view(torch.float32).view(count, 3)
        if biased:
            if biased != self._biased:
                self._biased, self._bias_lists = biased, ops.bias_lists([request.controls.logit_bias for request in biased], self.vocab, self.device)
            for name, tensor in self._bias_lists.items():
                setattr(result, name, tensor)
            result.bias_rows = on_device[count:2 * count]
        else:
            self._biased, self._bias_lists = (), {}
        if masks:
            result.masks, result.mask_rows = self._on_device(np.stack(masks)), on_device[2 * count:3 * count]
        return result
