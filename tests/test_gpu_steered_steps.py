"""Requests' controls through the engine beside what can go wrong in a step, on the device."""
import pytest
import torch

from dikusun_configs import DIKUSUN
from llmserver_b200.engine.engine import Engine
from test_gpu_kernels import DEVICE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cuda_graphs", [False, True])
@pytest.mark.parametrize("name", ["gla_only", "all_kinds"])
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
