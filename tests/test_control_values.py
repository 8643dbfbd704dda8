"""What requests may say about their logits and in what form it reaches the device."""
import numpy as np
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.engine.engine import Engine
from llmserver_b200.ops import KernelError
from llmserver_b200.sampling import ControlTable, RequestControls
from stubs import VOCAB, ArgmaxSampler, StubModel
from test_request_controls import Held


@pytest.mark.parametrize("biases", [{"9": -100.0, "17": 5.0}, {17: 5.0, 9: -100.0}, {9.0: -100.0, "17": 5.0}, {np.int64(17): 5.0, np.int32(9): -100.0}])
def test_tokens_of_a_bias_are_whole_numbers_in_ascending_order(biases):
    """Texts are what JSON makes of whole numbers as keys."""
    made = ops.bias_lists([biases], 50, "cpu")
    assert made["bias_starts"].tolist() == [0, 2] and made["bias_ids"].tolist() == [9, 17] and made["bias_values"].tolist() == [-100.0, 5.0]
    assert RequestControls(logit_bias=biases).check(50).logit_bias == {9: -100.0, 17: 5.0}
    engine = Engine(StubModel(), kv_cache_num_blocks=8, cuda_graphs=False, max_context=64, sampler=ArgmaxSampler())
    request = engine.add_request(prompt_token_ids=[1], logit_bias=biases)
    described = ControlTable("cpu", VOCAB).describe([request])
    assert described.bias_ids.tolist() == [9, 17] and described.bias_values.tolist() == [-100.0, 5.0]


@pytest.mark.parametrize("biases", [{9.7: 1.0}, {"9.7": 1.0}, {"nine": 1.0}, {None: 1.0}, {"9": 1.0, 9: 2.0}, {"50": 1.0}, {-1.0: 1.0}, {float("inf"): 1.0}, {(1,): 2.0}])
def test_a_bias_for_what_is_no_token_is_refused(biases):
    with pytest.raises(ValueError, match="token"):
        RequestControls(logit_bias=biases).check(50)
    with pytest.raises(KernelError, match="token"):
        ops.bias_lists([{}, biases], 50, "cpu")


def test_a_request_keeps_the_biases_it_came_with():
    """The caller's mapping may change behind the request."""
    engine = Engine(StubModel(), kv_cache_num_blocks=8, cuda_graphs=False, max_context=64, sampler=ArgmaxSampler())
    biases = {3: 1.0}
    request = engine.add_request(prompt_token_ids=[1], logit_bias=biases)
    biases[VOCAB + 5] = 2.0
    del biases[3]
    assert request.controls.logit_bias == {3: 1.0}


@pytest.mark.parametrize("given,message", [({"repetition_penalty": 1e-46}, "positive"), ({"repetition_penalty": 1e39}, "positive"), ({"presence_penalty": 1e300}, "finite"),
                                           ({"presence_penalty": -1e39}, "finite"), ({"frequency_penalty": 3.5e38}, "finite")])
def test_what_32_bits_cannot_hold_is_refused(given, message):
    """The device holds penalties in 32 bits, where these are zero or infinite."""
    with pytest.raises(ValueError, match=message):
        RequestControls(**given).check(50)


def test_what_32_bits_can_hold_is_taken():
    for given in ({"repetition_penalty": 1e-45}, {"repetition_penalty": 3.4e38}, {"presence_penalty": -3.4e38}, {"frequency_penalty": 1e-300}):
        RequestControls(**given).check(50)
    # a bias may be infinite, and one beyond 32 bits is that
    biases = RequestControls(logit_bias={3: float("-inf"), 4: -1e300}).check(50).logit_bias
    assert ops.bias_lists([biases], 50, "cpu")["bias_values"].tolist() == [-float("inf")] * 2
