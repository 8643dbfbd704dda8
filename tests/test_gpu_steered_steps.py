"""Requests' controls through the engine beside what can go wrong in a step, on the device."""
import math

import pytest
import torch

from dikusun_configs import DIKUSUN
from llmserver_b200 import ops
from llmserver_b200.engine.engine import Engine
from test_gpu_kernels import DEVICE
from test_gpu_logit_controls import Request as Row
from test_gpu_logit_controls import controls_of, finished, logits_for

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,cuda_graphs", [("gla_only", False), ("all_kinds", False), ("all_kinds", True)])
def test_a_grammar_that_raises_leaves_no_token_in_a_recurrent_state(name, cuda_graphs):
    """The step is run again: the answers of every request in it are those of a run in which nothing raised (the 32-bit path gives the
    same logits whatever else a step holds)."""
    from llmserver_b200.config import DikusunConfig
    from llmserver_b200.models import random_model
    raw, seed = DIKUSUN[name]
    model = random_model(DikusunConfig.from_dict(raw), seed, "float32", DEVICE)
    prompts = [[5, 3, 8, 1], [9, 2], [4, 4, 7]]

    def run(fails_at):
        engine = Engine(model, max_new_tokens=16, max_batch_size=4, max_context=64, ignore_eos=True, cuda_graphs=cuda_graphs, prefix_caching=False)
        failed = []

        def grammar(sofar):
            if len(sofar) in fails_at and len(sofar) not in failed:
                failed.append(len(sofar))
                raise RuntimeError("no grammar today")
            return None

        requests = [engine.add_request(prompt_token_ids=prompts[0], allowed_tokens=grammar, temperature=0.8, seed=1),
                    engine.add_request(prompt_token_ids=prompts[1], temperature=0.8, seed=2),
                    engine.add_request(prompt_token_ids=prompts[2], frequency_penalty=0.5, temperature=0.8, seed=3)]
        while True:
            try:
                if not engine.step():
                    break
            except RuntimeError as error:
                assert "no grammar" in str(error)
        assert failed == list(fails_at) and (not cuda_graphs or engine.step_function.graph_steps > 0)
        return [request.generated_token_ids for request in requests]

    assert run((0, 1, 2, 7, 11)) == run(())


@pytest.mark.parametrize("vocab", [700, 3000, 50000])
@pytest.mark.parametrize("warm", [False, True])
def test_a_row_without_controls_draws_as_it_would_alone(vocab, warm):
    """Logits that are all NaN, all -inf or partly so, beside rows that are steered."""
    logits = logits_for(8, vocab, 40)
    logits[1], logits[2] = math.nan, -math.inf
    logits[3, ::2], logits[3, 1::2] = math.nan, -math.inf
    logits[4] = math.inf
    logits[5, 9:] = -math.inf
    none = torch.zeros(vocab, dtype=torch.bool)
    requests = [Row([1, 2], [3], 1.5, 0.5, 0.5), Row(), Row(), Row(), Row(), Row(), Row(allowed=none), Row(bias={4: 1.0})]
    controls = controls_of(requests, vocab)
    for row in range(1, 6):
        controls.history_rows[row] = -1
    drawn = (torch.full((8,), 0.7, device=DEVICE), torch.arange(8, device=DEVICE), torch.arange(8, dtype=torch.int32, device=DEVICE)) if warm else ()
    for note in (False, True):
        got = ops.sample(logits, *drawn, controls=controls, note=note)
        finished()
        alone = [int(ops.sample(logits[row:row + 1], *(part[row:row + 1] for part in drawn))) for row in range(8)]
        assert got.tolist()[1:6] == alone[1:6] and int(got[6]) == -1
    # controls that say something leave nothing of such a row
    controls.history_rows[1:4] = controls.history_rows[0]
    got = ops.sample(logits, *drawn, controls=controls)
    finished()
    assert got.tolist()[1:4] == [-1, -1, -1]


def test_a_score_that_32_bits_cannot_hold_is_still_a_token():
    """A temperature below the normal numbers makes every quotient -inf: the lowest of the tokens that the mask leaves."""
    vocab = 5000
    logits = -1 - logits_for(3, vocab, 41).abs()
    few = torch.zeros(vocab, dtype=torch.bool)
    few[[37, 4100]] = True
    controls = controls_of([Row(allowed=few), Row([1], [], 1.5), Row(allowed=few & False)], vocab)
    for temperature in (1e-39, 2e-39):
        got = ops.sample(logits, torch.full((3,), temperature, device=DEVICE), torch.arange(3, device=DEVICE), torch.zeros(3, dtype=torch.int32, device=DEVICE), controls=controls)
        finished()
        assert got.tolist() == [37, 0, -1]


def test_a_history_that_does_not_exist_is_reported_with_the_step():
    """The flag behind the tokens is that of this step, whichever row is at fault, and with penalties or without."""
    from llmserver_b200.ops.library import KernelError, check_wait_errors, wait_error_flag
    vocab, rows = 300, 400
    logits = logits_for(rows, vocab, 42)
    controls = controls_of([Row([row % vocab], [], 1.2) for row in range(rows)], vocab, capacity=6)
    flag, own = wait_error_flag(torch.device(DEVICE)), torch.full((1,), 5, dtype=torch.int32, device=DEVICE)
    good = controls.history_rows.clone()
    for penalties in (controls.penalties, None):
        controls.penalties = penalties
        for bad in (0, 1, rows - 1):
            controls.history_rows.copy_(good)
            controls.history_rows[bad] = rows + 2
            for note in (True, False):
                got = ops.sample(logits, controls=controls, flags=(own, flag), note=note)
                torch.cuda.synchronize()
                assert got.tolist()[rows:] == [5, 8]
                with pytest.raises(KernelError, match="does not exist"):
                    check_wait_errors()
            ops.control_logits(logits, controls)
            torch.cuda.synchronize()
            with pytest.raises(KernelError, match="does not exist"):
                check_wait_errors()
    finished()
