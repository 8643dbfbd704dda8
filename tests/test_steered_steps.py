"""Steps whose requests say something about their logits, with a model that keeps a state: what a failing step may leave behind."""
from types import SimpleNamespace

import pytest
import torch

from llmserver_b200.engine.engine import Engine
from llmserver_b200.engine.graphs import DecodeGraphs
from llmserver_b200.engine.request import RequestFinishReason
from stubs import VOCAB, StubModel
from test_request_controls import HostSampler

FLAG = "llmserver_b200.engine.step.wait_error_flag"


class SummingModel(StubModel):
    """Keeps the sum of the tokens that a request fed, replaced in place by every step as recurrent states are: the next token is that sum + 1, so
    a token that goes in twice is in every answer from then on.  A request is told by its first page."""

    def __init__(self):
        super().__init__()
        self.sums = {}

    def step(self, batch):
        tables = batch.block_tables[0].view(batch.n_seqs, -1)
        logits, at = torch.zeros((batch.n_logits, VOCAB)), 0
        wanted = batch.logit_rows.tolist()
        for place in range(batch.n_tokens):
            page = int(tables[int(batch.seq_of_token[place]), 0])
            before = self.sums.get(page, 0) if int(batch.positions[place]) else 0
            self.sums[page] = before + int(batch.token_ids[place])
            if place in wanted:
                logits[at, (self.sums[page] + 1) % VOCAB] = 1.0
                at += 1
        return logits


class HostGraph:
    """A replayed step that runs the model where the real one replays."""

    def __init__(self, owner, size):
        self.owner, self.batch, self.meanwhile = owner, None, None
        self.layout, self.rows = SimpleNamespace(total=0), SimpleNamespace(forget=lambda: None)

    def run(self, slices, sampling, phases=None):
        from llmserver_b200.engine.batch import build_batch
        self.began = 0.0
        batch = build_batch(slices, len(self.owner.cache.groups), torch.device("cpu"), VOCAB, sampling=sampling)
        self.logits = self.owner.model.step(batch)
        self.owner.replays += 1
        if self.meanwhile is not None:
            self.meanwhile()
        return torch.argmax(self.logits, dim=-1).tolist() + [0, 0]


class HostGraphs(DecodeGraphs):
    replays = 0

    def capture(self, size):
        return HostGraph(self, size)


def engine_of(model, monkeypatch, replayed):
    monkeypatch.setattr(FLAG, lambda device: torch.zeros(1, dtype=torch.int32))
    engine = Engine(model, max_new_tokens=8, max_batch_size=4, kv_cache_num_blocks=40, kv_cache_block_size=16, ignore_eos=True, prefix_caching=False,
                    sampler=HostSampler(), cuda_graphs=False, max_context=64)
    if replayed:
        engine.step_function.graphs = HostGraphs(model, engine.cache, 64, 4)
    return engine


def answer(prompt, count):
    held = list(prompt)
    for _ in range(count):
        held.append((sum(held) + 1) % VOCAB)
    return held[len(prompt):]


PROMPTS = [[3, 5], [7], [1, 2, 4]]


@pytest.mark.parametrize("replayed", [False, True])
@pytest.mark.parametrize("when", [0, 1, 4])
def test_a_grammar_that_raises_leaves_no_token_in_a_state(monkeypatch, replayed, when):
    """One request's grammar raises once; the same step is run again, and no request of it, steered or not, shows that."""
    model = SummingModel()
    engine = engine_of(model, monkeypatch, replayed)
    failed = []

    def grammar(sofar):
        if len(sofar) == when and not failed:
            failed.append(when)
            raise RuntimeError("no grammar today")
        return None

    requests = [engine.add_request(prompt_token_ids=PROMPTS[0], allowed_tokens=grammar), engine.add_request(prompt_token_ids=PROMPTS[1]),
                engine.add_request(prompt_token_ids=PROMPTS[2], presence_penalty=0.0, logit_bias={0: 0.0})]
    notes = []
    while True:
        try:
            if not engine.step():
                break
        except RuntimeError as error:
            assert "no grammar" in str(error)
            notes.append(getattr(error, "__notes__", []))
    assert [request.generated_token_ids for request in requests] == [answer(prompt, 8) for prompt in PROMPTS]
    assert len(notes) == 1 and requests[0].request_id in notes[0][0]      # the caller hears whose it was
    assert not replayed or engine.step_function.graphs.replays > 0


@pytest.mark.parametrize("replayed", [False, True])
def test_the_request_whose_grammar_raises_can_be_cancelled(monkeypatch, replayed):
    model = SummingModel()
    engine = engine_of(model, monkeypatch, replayed)

    def grammar(sofar):
        if len(sofar) >= 4:
            raise KeyError("state")
        return None

    bad, good = engine.add_request(prompt_token_ids=PROMPTS[0], allowed_tokens=grammar), engine.add_request(prompt_token_ids=PROMPTS[1], logit_bias={0: 0.0})
    for _ in range(3):
        with pytest.raises(KeyError, match="state"):
            while engine.step():
                pass
    assert engine.cancel_request(bad.request_id)
    while engine.step():
        pass
    assert bad.finish_reason is RequestFinishReason.CANCELLED and bad.generated_token_ids == answer(PROMPTS[0], 4)
    assert good.generated_token_ids == answer(PROMPTS[1], 8)


@pytest.mark.parametrize("replayed", [False, True])
@pytest.mark.parametrize("given,said", [([1, VOCAB], "outside"), ([-1], "outside"), (torch.ones(VOCAB + 1, dtype=torch.bool), "truth values"), ([1.5], "whole"), (7, "iterable"),
                                        (["a"], "whole"), ([1 << 70], "whole")])
def test_a_request_whose_grammar_gives_what_is_no_token_ends_alone(monkeypatch, replayed, given, said):
    model = SummingModel()
    engine = engine_of(model, monkeypatch, replayed)
    bad = engine.add_request(prompt_token_ids=PROMPTS[0], allowed_tokens=lambda sofar: given if len(sofar) == 5 else None)
    others = [engine.add_request(prompt_token_ids=PROMPTS[1], frequency_penalty=0.0, logit_bias={0: 0.0}), engine.add_request(prompt_token_ids=PROMPTS[2])]
    while engine.step():
        pass
    assert bad.finish_reason is RequestFinishReason.ERROR and bad.generated_token_ids == answer(PROMPTS[0], 5) and said in bad.error
    for request, prompt in zip(others, PROMPTS[1:]):
        assert request.finish_reason is RequestFinishReason.LENGTH and request.generated_token_ids == answer(prompt, 8) and request.error is None
    assert not engine.cache.requests


def test_masks_take_whole_numbers_only():
    from llmserver_b200.sampling.controls import mask_words
    import numpy as np
    for given in ([2.0, 5.0], np.array([2, 5], dtype=np.uint8), torch.tensor([5, 2], dtype=torch.int32), (2, 5), {2: "a", 5: "b"}, torch.tensor([[2], [5]])):
        assert mask_words(given, 40).tolist() == [(1 << 2) | (1 << 5), 0]
    for wrong in ([2.5], [float("nan")], [None], ["2"], [1 + 2j]):
        with pytest.raises(ValueError, match="whole"):
            mask_words(wrong, 40)


@pytest.mark.parametrize("replayed", [False, True])
@pytest.mark.parametrize("none", [[], torch.zeros(VOCAB, dtype=torch.bool), range(0)])
def test_a_request_with_nothing_left_keeps_what_it_has_drawn(monkeypatch, replayed, none):
    engine = engine_of(SummingModel(), monkeypatch, replayed)
    stuck, other = engine.add_request(prompt_token_ids=PROMPTS[0], allowed_tokens=lambda sofar: none if len(sofar) == 3 else None), engine.add_request(prompt_token_ids=PROMPTS[1])
    while engine.step():
        pass
    assert stuck.finish_reason is RequestFinishReason.ERROR and stuck.generated_token_ids == answer(PROMPTS[0], 3) and stuck.error is None
    assert other.finish_reason is RequestFinishReason.LENGTH and other.generated_token_ids == answer(PROMPTS[1], 8)
