"""The host's side of controls on logits: lists and masks from what a request says, and what is refused before a launch."""
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.ops import KernelError
from llmserver_b200.ops.logit_controls import _DESCRIPTION


def test_lists_ascend_and_stay_apart():
    made = ops.bias_lists([{7: 1.5, 2: -1.0}, {}, {0: 3.0}], 8, "cpu")
    assert made["bias_starts"].tolist() == [0, 2, 2, 3] and made["bias_ids"].tolist() == [2, 7, 0] and made["bias_values"].tolist() == [-1.0, 1.5, 3.0]
    assert made["bias_ids"].dtype == torch.int32 and ops.bias_lists([], 8, "cpu")["bias_starts"].tolist() == [0]
    for token in (-1, 8):
        with pytest.raises(KernelError, match="outside the vocabulary"):
            ops.bias_lists([{token: 1.0}], 8, "cpu")


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 100])
def test_masks_bit_by_bit(vocab):
    allowed = torch.rand((3, vocab), generator=torch.Generator().manual_seed(vocab)) < 0.5
    allowed[0], allowed[1] = True, False
    masks = ops.token_masks(allowed)
    assert masks.dtype == torch.int32 and masks.shape == (3, -(-vocab // 32))
    for row in range(3):
        for token in range(vocab):
            assert bool((int(masks[row, token // 32]) >> (token % 32)) & 1) == bool(allowed[row, token])
    for wrong in (allowed[0], allowed.int()):
        with pytest.raises(KernelError, match="truth values"):
            ops.token_masks(wrong)


def test_logits_on_the_host_are_refused():
    for run in (ops.control_logits, lambda l, c: ops.sample(l, controls=c)):
        with pytest.raises(KernelError, match="CUDA device"):
            run(torch.zeros((1, 5)), ops.LogitControls())


def test_the_launchers_refuse_sizes_they_cannot_take():
    library = ops.library()
    said = _DESCRIPTION.pack(*[0] * 18)
    for rows, vocab in ((-1, 5), (65536, 5), (1, 0)):
        assert library.llm_control_logits(0, 0, rows, vocab, said, 0) == -1
        assert library.llm_control_sample(0, 0, 0, 0, 0, rows, vocab, said, 0, 0, 0, 0, 0, 0) == -1
    said = _DESCRIPTION.pack(*[0] * 13, 16, 0, 1, 3, 0)
    assert library.llm_control_logits(0, 0, 1, 97, said, 0) == -1 and b"words" in library.llm_last_error()
    assert library.llm_control_logits(0, 0, 0, 96, said, 0) == 0
