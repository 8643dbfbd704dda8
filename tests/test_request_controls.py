"""What requests say about their logits: checked, kept in the table of histories, and carried through the engine, without a GPU."""
import collections
import random

import numpy as np
import pytest
import torch

from llmserver_b200 import ops
from llmserver_b200.engine.engine import Engine
from llmserver_b200.engine.request import RequestFinishReason
from llmserver_b200.sampling import ControlTable, RequestControls
from llmserver_b200.sampling.controls import mask_words
from stubs import VOCAB, ArgmaxSampler, StubModel


@pytest.mark.parametrize("given,message", [({"repetition_penalty": 0.0}, "positive"), ({"repetition_penalty": float("nan")}, "positive"),
                                           ({"presence_penalty": float("inf")}, "finite"), ({"frequency_penalty": float("nan")}, "finite"),
                                           ({"logit_bias": {50: 1.0}}, "tokens are"), ({"logit_bias": {-1: 1.0}}, "tokens are"),
                                           ({"logit_bias": {1: float("nan")}}, "numbers"), ({"allowed_tokens": [1, 2]}, "function")])
def test_what_cannot_be_meant_is_refused(given, message):
    with pytest.raises(ValueError, match=message):
        RequestControls(**given).check(50)
    engine = Engine(StubModel(), kv_cache_num_blocks=8, cuda_graphs=False, max_context=64, sampler=ArgmaxSampler())
    with pytest.raises(ValueError, match=message):
        engine.add_request(prompt_token_ids=[1], **given)
    assert not engine.active_requests and not engine.scheduler.waiting


def test_controls_that_change_nothing_are_none():
    assert not RequestControls().active and not RequestControls(logit_bias={}).active
    assert RequestControls(logit_bias={3: 0.0}).active and RequestControls(presence_penalty=-1.0).check(50).penalises
    engine = Engine(StubModel(), kv_cache_num_blocks=8, cuda_graphs=False, max_context=64, sampler=ArgmaxSampler())
    assert engine.add_request(prompt_token_ids=[1], repetition_penalty=1.0, logit_bias={}).controls is None
    with pytest.raises(TypeError):
        engine.add_request(prompt_token_ids=[1], no_such_penalty=1.0)


@pytest.mark.parametrize("vocab", [1, 32, 33, 77])
def test_masks_from_ids_and_from_truth_values(vocab):
    rng = random.Random(vocab)
    ids = sorted(rng.sample(range(vocab), rng.randint(1, vocab)))
    truth = torch.zeros(vocab, dtype=torch.bool)
    truth[ids] = True
    want = ops.token_masks(truth[None])[0].tolist()
    for given in (ids, set(ids), iter(ids), np.array(ids), torch.tensor(ids), truth, truth.numpy()):
        assert mask_words(given, vocab).tolist() == want
    assert mask_words([], vocab).tolist() == [0] * len(want)
    for wrong in ([vocab], [-1], torch.zeros(vocab + 1, dtype=torch.bool)):
        with pytest.raises(ValueError):
            mask_words(wrong, vocab)


class Held:
    def __init__(self, request_id, prompt, **controls):
        self.request_id, self.prompt_token_ids, self.generated_token_ids = request_id, list(prompt), []
        self.controls = RequestControls(**controls)


def history_of(described, row):
    place, length = int(described.history_rows[row]), int(described.lengths[row])
    return described.history[place, :length].tolist()


def test_histories_follow_their_requests():
    """A few hundred steps of requests that come, go, come back under their name and outgrow the table; what a draw notes is written as the
    kernel would, or lost where the step failed."""
    rng = random.Random(1)
    table, live, count = ControlTable("cpu", VOCAB), [], 0
    for step in range(400):
        if len(live) < 9 and rng.random() < 0.4:
            live.append(Held(f"r{count if rng.random() < 0.9 else 0}", [rng.randrange(VOCAB) for _ in range(rng.randint(1, 300 if step > 200 else 20))],
                             repetition_penalty=rng.choice((1.0, 1.5)), frequency_penalty=rng.choice((0.0, 0.5)), logit_bias={count % VOCAB: 1.0 + count} if rng.random() < 0.3 else None))
            count += 1
            if sum(held.request_id == live[-1].request_id for held in live) > 1:
                live.pop()
                continue
            table.forget(live[-1].request_id)
        if live and rng.random() < 0.15:
            table.forget(live.pop(rng.randrange(len(live))).request_id)
        rows = [held if held is None or held.controls.active else None for held in rng.sample(live, rng.randint(0, len(live))) + [None] * rng.randint(0, 2)]
        if not rows:
            continue
        described = table.describe(rows)
        for row, held in enumerate(rows):
            if held is None or not held.controls.penalises:
                assert described.history_rows is None or int(described.history_rows[row]) == -1
            else:
                assert history_of(described, row) == held.prompt_token_ids + held.generated_token_ids
                assert int(described.prompt_lengths[row]) == len(held.prompt_token_ids) and described.history.shape[1] > int(described.lengths[row])
                assert described.penalties[row].tolist() == [held.controls.repetition_penalty, 0.0, held.controls.frequency_penalty]
            if held is not None and held.controls.logit_bias:
                at = int(described.bias_rows[row])
                first, last = described.bias_starts[at:at + 2].tolist()
                assert dict(zip(described.bias_ids[first:last].tolist(), described.bias_values[first:last].tolist())) == held.controls.logit_bias
            elif described.bias_rows is not None:
                assert int(described.bias_rows[row]) == -1
        if rng.random() < 0.1:
            continue                     # the step failed behind the description: nothing was drawn
        for row, held in enumerate(rows):
            if held is not None:
                token = rng.randrange(VOCAB)
                held.generated_token_ids.append(token)
                if held.controls.penalises:
                    described.history[int(described.history_rows[row]), int(described.lengths[row])] = token
    places = list(table.places.values())
    assert len(set(places)) == len(places) and max(places) < table.history.shape[0] <= 32


def steer(logits, request):
    """The formula, on the host."""
    logits, controls = logits.double().clone(), request.controls
    seen = set(request.prompt_token_ids + request.generated_token_ids)
    for token in seen:
        logits[token] = logits[token] / controls.repetition_penalty if logits[token] > 0 else logits[token] * controls.repetition_penalty
    for token, times in collections.Counter(request.generated_token_ids).items():
        logits[token] -= times * controls.frequency_penalty + controls.presence_penalty
    for token, value in (controls.logit_bias or {}).items():
        logits[token] += value
    allowed = controls.allowed_tokens(request.generated_token_ids) if controls.allowed_tokens else None
    if allowed is not None:
        logits[[token for token in range(VOCAB) if token not in set(allowed)]] = -float("inf")
    return logits


class HostSampler:
    """What the device's sampler does, from what the table describes and nothing else."""

    def from_batch(self, logits, batch):
        return torch.argmax(logits, dim=-1).to(torch.int32)

    def steered_from_batch(self, logits, batch, described):
        tokens = []
        for row in range(logits.shape[0]):
            line = logits[row].double().clone()
            if described.history_rows is not None and int(described.history_rows[row]) >= 0:
                held, cut = history_of(described, row), int(described.prompt_lengths[row])
                repetition, presence, frequency = described.penalties[row].tolist()
                for token in set(held):
                    line[token] = line[token] / repetition if line[token] > 0 else line[token] * repetition
                for token, times in collections.Counter(held[cut:]).items():
                    line[token] -= times * frequency + presence
            if described.bias_rows is not None and int(described.bias_rows[row]) >= 0:
                at = int(described.bias_rows[row])
                for entry in range(int(described.bias_starts[at]), int(described.bias_starts[at + 1])):
                    line[int(described.bias_ids[entry])] += float(described.bias_values[entry])
            if described.mask_rows is not None and int(described.mask_rows[row]) >= 0:
                words = described.masks[int(described.mask_rows[row])].tolist()
                line[[token for token in range(VOCAB) if not (words[token // 32] >> (token % 32)) & 1]] = -float("inf")
            token = -1 if bool((line == -float("inf")).all()) else int(torch.argmax(line))
            tokens.append(token)
            if token >= 0 and described.history_rows is not None and int(described.history_rows[row]) >= 0:
                described.history[int(described.history_rows[row]), int(described.lengths[row])] = token
        return torch.tensor(tokens, dtype=torch.int32)


def expected(request, count):
    """The stub model's answer under the request's controls."""
    class Sofar:
        controls, prompt_token_ids, generated_token_ids = request.controls, request.prompt_token_ids, []
    sofar = Sofar()
    sofar.generated_token_ids = []
    for _ in range(count):
        held = sofar.prompt_token_ids + sofar.generated_token_ids
        logits = torch.zeros(VOCAB)
        logits[(held[-1] + 1 + len(held) - 1) % VOCAB] = 1.0
        line = steer(logits, sofar) if request.controls else logits
        if bool((line == -float("inf")).all()):
            break
        sofar.generated_token_ids.append(int(torch.argmax(line)))
    return sofar.generated_token_ids


def test_the_engine_steers_each_request_by_its_own_controls_through_preemption(monkeypatch):
    """Requests with and without controls in the same steps, in a cache too small for all of them."""
    monkeypatch.setattr("llmserver_b200.engine.step.wait_error_flag", lambda device: torch.zeros(1, dtype=torch.int32))
    put_out = 0
    for seed in range(25):
        rng = random.Random(seed)
        engine = Engine(StubModel(), max_new_tokens=16, max_batch_size=4, max_num_batched_tokens=24, kv_cache_num_blocks=rng.randint(9, 14),
                        kv_cache_block_size=4, ignore_eos=True, prefix_caching=False, sampler=HostSampler(), cuda_graphs=False, max_context=64)
        requests = []
        for index in range(8):
            kind = rng.randrange(4)
            controls = {} if kind == 0 else {"repetition_penalty": rng.choice((1.0, 2.0)), "presence_penalty": rng.choice((0.0, 2.0)), "frequency_penalty": rng.choice((0.0, 0.75)),
                                             "logit_bias": {rng.randrange(VOCAB): rng.choice((0.5, 3.0, -5.0))} if rng.random() < 0.5 else None,
                                             "allowed_tokens": (lambda sofar, odd=rng.randrange(2): range(len(sofar) % 3 + odd, VOCAB, 2)) if kind == 2 else None}
            requests.append(engine.add_request(prompt_token_ids=[rng.randrange(VOCAB) for _ in range(rng.randint(1, 12))], max_new_tokens=rng.randint(1, 16), **controls))
        while engine.step():
            pass
        for request in requests:
            assert request.generated_token_ids == expected(request, request.max_new_tokens) and request.finish_reason is RequestFinishReason.LENGTH
        put_out += sum(request.times_put_out > 0 and request.controls is not None for request in requests)
        assert engine.step_function.controls is None or not engine.step_function.controls.places
    assert put_out > 5


def test_a_request_with_nothing_left_to_draw_ends_and_the_others_go_on(monkeypatch):
    monkeypatch.setattr("llmserver_b200.engine.step.wait_error_flag", lambda device: torch.zeros(1, dtype=torch.int32))
    engine = Engine(StubModel(), max_batch_size=4, kv_cache_num_blocks=40, ignore_eos=True, sampler=HostSampler(), cuda_graphs=False, max_context=64)
    stuck = engine.add_request(prompt_token_ids=[1, 2], max_new_tokens=10, allowed_tokens=lambda sofar: None if len(sofar) < 3 else [])
    other = engine.add_request(prompt_token_ids=[5], max_new_tokens=10)
    while engine.step():
        pass
    assert stuck.finish_reason is RequestFinishReason.ERROR and stuck.generated_token_ids == expected(other, 0) + stuck.generated_token_ids[:3]
    assert len(stuck.generated_token_ids) == 3 and other.generated_token_ids == expected(other, 10)
    assert not engine.cache.requests


def test_a_grammar_that_raises_stops_the_step_and_it_can_be_run_again(monkeypatch):
    monkeypatch.setattr("llmserver_b200.engine.step.wait_error_flag", lambda device: torch.zeros(1, dtype=torch.int32))
    engine = Engine(StubModel(), max_batch_size=4, kv_cache_num_blocks=40, ignore_eos=True, sampler=HostSampler(), cuda_graphs=False, max_context=64)
    calls = []

    def allowed(sofar):
        calls.append(len(sofar))
        if calls == [0, 1]:
            raise RuntimeError("no grammar today")
        return None

    request = engine.add_request(prompt_token_ids=[3], max_new_tokens=4, allowed_tokens=allowed)
    engine.step()
    with pytest.raises(RuntimeError, match="no grammar"):
        engine.step()
    while engine.step():
        pass
    assert request.generated_token_ids == expected(engine.finished_requests[request.request_id], 0) + request.generated_token_ids and len(request.generated_token_ids) == 4
    held = [3]
    for _ in range(4):
        held.append((held[-1] + 1 + len(held) - 1) % VOCAB)
    assert request.generated_token_ids == held[1:]


def test_a_sampler_that_knows_no_controls_is_refused():
    engine = Engine(StubModel(), kv_cache_num_blocks=8, cuda_graphs=False, max_context=64, sampler=ArgmaxSampler())
    engine.add_request(prompt_token_ids=[1], presence_penalty=1.0)
    with pytest.raises(ValueError, match="controls"):
        engine.step()
