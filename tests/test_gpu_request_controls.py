"""Controls and products in 8 bits through the engine, on the device."""
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.engine.engine import Engine
from llmserver_b200.engine.request import RequestFinishReason
from test_gpu_kernels import DEVICE, rand
from test_gpu_logit_controls import Request as Row
from test_gpu_logit_controls import formula

pytestmark = pytest.mark.gpu


def tiny(name="b", dtype="float32", products="same"):
    from llmserver_b200.config import Qwen3Config
    from llmserver_b200.models import random_model
    from tiny_configs import TINY
    raw, seed = TINY[name]
    return random_model(Qwen3Config.from_dict(raw), seed, dtype, DEVICE, products=products)


CONTROLS = [{}, {"repetition_penalty": 1.4}, {"presence_penalty": 0.5, "frequency_penalty": 0.3}, {"logit_bias": {3: 4.0, 7: -100.0}},
            {"repetition_penalty": 1.2, "frequency_penalty": 0.2, "logit_bias": {11: 2.0}, "allowed_tokens": lambda sofar: range(len(sofar) % 2, 200, 2)},
            {"allowed_tokens": lambda sofar: None if len(sofar) % 3 else [5, 9, 13, 77]}]


def answers(model, cuda_graphs, together=True, temperature=0.0, count=20):
    prompts = [[(7 * row + 3 * place) % 150 for place in range(5 + row)] for row in range(len(CONTROLS))]
    found = []
    for group in ([range(len(CONTROLS))] if together else [[row] for row in range(len(CONTROLS))]):
        engine = Engine(model, max_new_tokens=count, max_batch_size=len(CONTROLS), max_context=64, kv_cache_block_size=16, ignore_eos=True, cuda_graphs=cuda_graphs)
        requests = [engine.add_request(prompt_token_ids=prompts[row], temperature=temperature, seed=row, **CONTROLS[row]) for row in group]
        while engine.step():
            pass
        assert not engine.step_function.controls or not engine.step_function.controls.places
        if cuda_graphs:
            assert engine.step_function.graph_steps > 0
        found += [request.generated_token_ids for request in requests]
    return prompts, found


@pytest.mark.parametrize("temperature", [0.0, 0.9])
def test_answers_are_the_same_alone_together_and_replayed(temperature):
    """The 32-bit path gives the same logits whoever shares a step, so the answers must not depend on it either."""
    model = tiny()
    _, together = answers(model, False, temperature=temperature)
    assert together == answers(model, True, temperature=temperature)[1]
    assert together == answers(model, False, together=False, temperature=temperature)[1]
    assert together == answers(model, True, together=False, temperature=temperature)[1]


def test_answers_follow_the_formulas():
    """Token by token, from the logits of the same model behind the same tokens, in 64 bits; wherever the two best lie further apart than
    the roundings of the controls can reach."""
    model = tiny()
    prompts, found = answers(model, True)
    vocab, clear = model.spec.vocab_size, 0
    for row, (prompt, answer) in enumerate(zip(prompts, found)):
        engine = Engine(model, max_batch_size=1, max_context=64, cuda_graphs=False)
        engine.step_function.admit("whole")
        held = prompt + answer[:-1]
        logits = engine.step_function.run([("whole", held, list(range(len(prompt) - 1, len(held))))])
        for place, token in enumerate(answer):
            given = {name: value for name, value in CONTROLS[row].items() if name.endswith("penalty")}
            grammar = CONTROLS[row].get("allowed_tokens")
            allowed = grammar(answer[:place]) if grammar else None
            truth = None
            if allowed is not None:
                truth = torch.zeros(vocab, dtype=torch.bool)
                truth[[t for t in allowed if t < vocab]] = True
            request = Row(prompt, answer[:place], given.get("repetition_penalty", 1.0), given.get("presence_penalty", 0.0), given.get("frequency_penalty", 0.0),
                          CONTROLS[row].get("logit_bias"), truth)
            want, largest = formula(logits[place:place + 1], [request])
            best = want[0].topk(2)
            if float(best.values[0] - best.values[1]) > 2 * 6 * 2.0 ** -24 * float(largest.max()):
                clear += 1
                assert token == int(best.indices[0]), (row, place)
    assert clear > 100


def test_nothing_left_in_a_replayed_step():
    model = tiny()
    engine = Engine(model, max_new_tokens=12, max_batch_size=2, max_context=64, ignore_eos=True)
    engine.warmup([2])
    stuck = engine.add_request(prompt_token_ids=[1, 2, 3], allowed_tokens=lambda sofar: [4] if len(sofar) < 5 else [])
    free = engine.add_request(prompt_token_ids=[1, 2, 3])
    while engine.step():
        pass
    assert stuck.finish_reason is RequestFinishReason.ERROR and stuck.generated_token_ids == [4] * 5
    assert free.finish_reason is RequestFinishReason.LENGTH and len(free.generated_token_ids) == 12
    assert engine.step_function.graph_steps > 5


def test_answers_survive_being_put_out():
    """A cache too small for all: histories are copied again when a request comes back."""
    model = tiny()
    prompts = [[(row + place) % 100 for place in range(20)] for row in range(3)]

    def run(blocks):
        engine = Engine(model, max_new_tokens=30, max_batch_size=3, max_context=64, kv_cache_num_blocks=blocks, kv_cache_block_size=16, ignore_eos=True, prefix_caching=False)
        requests = [engine.add_request(prompt_token_ids=prompt, repetition_penalty=1.3, frequency_penalty=0.4) for prompt in prompts]
        while engine.step():
            pass
        return [request.generated_token_ids for request in requests], engine.stats["preemptions"]

    roomy, none = run(64)
    tight, some = run(9)
    assert none == 0 and some > 0 and roomy == tight


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_products_in_8_bits_through_the_engine(dtype):
    """The feed-forward is its two products and the activation; the head's logits are the product's; graphs and eager steps agree."""
    from llmserver_b200.parts import FEED_FORWARDS, Runtime
    torch_dtype = torch.float32 if dtype == "float32" else torch.bfloat16
    weights = {"gate_proj.weight": rand((200, 96), torch_dtype, 1, 0.1), "up_proj.weight": rand((200, 96), torch_dtype, 2, 0.1), "down_proj.weight": rand((96, 200), torch_dtype, 3, 0.1)}
    part = FEED_FORWARDS.get("swiglu")({"hidden": 96, "intermediate": 200}, weights, Runtime(torch_dtype, torch.device(DEVICE), "float8"))
    assert not part.takes_unscaled
    for rows in (1, 30, 90):
        x = rand((rows, 96), torch_dtype, 4)
        gate_up = ops.quantize_blocks(torch.cat([weights["gate_proj.weight"], weights["up_proj.weight"]]), 128)
        hidden = ops.silu_mul(ops.linear(x, gate_up))
        assert torch.equal(part.forward(x), ops.linear(hidden, ops.quantize_blocks(weights["down_proj.weight"], 128)))
    model = tiny(dtype=dtype, products="float8")
    assert isinstance(model.head, ops.BlockScaled) and model.embedding.dtype == torch_dtype
    prompts = [[5, 6, 7, 8], [9, 10], [11]]
    eager = Engine(model, max_new_tokens=12, max_batch_size=4, max_context=64, ignore_eos=True, cuda_graphs=False).generate(prompts, presence_penalty=0.3)
    replayed = Engine(model, max_new_tokens=12, max_batch_size=4, max_context=64, ignore_eos=True, cuda_graphs=True).generate(prompts, presence_penalty=0.3)
    assert all(len(answer) == 12 for answer in eager)
    if dtype == "float32":
        assert eager == replayed


def test_products_are_named_once():
    from llmserver_b200.parts import Runtime
    with pytest.raises(ValueError, match="float8"):
        Runtime(torch.float32, torch.device(DEVICE), "int4")
    with pytest.raises(ValueError, match="loaded with"):
        Engine(tiny(), products="float8", max_context=64)
