"""Penalties, biases and masks on logits, and tokens drawn under them, against the formulas in 64 bits."""
import collections
import math
import random

import pytest
import torch

from llmserver_b200 import ops
from test_gpu_kernels import DEVICE

pytestmark = pytest.mark.gpu


def finished():
    from llmserver_b200.ops.library import check_wait_errors
    torch.cuda.synchronize()
    check_wait_errors()


class Request:
    """What holds for one row of logits, on the host."""

    def __init__(self, prompt=(), answer=(), repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None):
        self.prompt, self.answer = list(prompt), list(answer)
        self.penalties = (repetition, presence, frequency)
        self.bias, self.allowed = bias, allowed


def controls_of(requests, vocab, capacity=None, seed=0):
    """``LogitControls`` of the requests, their histories in a shuffled table with rows of rubbish between them."""
    count = len(requests)
    capacity = capacity or max(1, max(len(r.prompt) + len(r.answer) for r in requests) + 2)
    places = list(range(count + 2))
    random.Random(seed).shuffle(places)
    history = torch.randint(0, vocab, (count + 2, capacity), generator=torch.Generator().manual_seed(seed), dtype=torch.int32)
    for request, place in zip(requests, places):
        held = request.prompt + request.answer
        history[place, :len(held)] = torch.tensor(held, dtype=torch.int32)
    lists = [request.bias for request in requests if request.bias is not None]
    masks = [request.allowed for request in requests if request.allowed is not None]

    def index(of):
        at, found = 0, []
        for request in requests:
            found.append(-1 if of(request) is None else at)
            at += of(request) is not None
        return torch.tensor(found, dtype=torch.int32, device=DEVICE)

    def whole(values):
        return torch.tensor(list(values), dtype=torch.int32, device=DEVICE)

    made = ops.LogitControls(penalties=torch.tensor([r.penalties for r in requests], dtype=torch.float32, device=DEVICE), history=history.to(DEVICE),
                             history_rows=whole(places[:count]), lengths=whole(len(r.prompt) + len(r.answer) for r in requests),
                             prompt_lengths=whole(len(r.prompt) for r in requests))
    if lists:
        for name, tensor in ops.bias_lists(lists, vocab, DEVICE).items():
            setattr(made, name, tensor)
        made.bias_rows = index(lambda r: r.bias)
    if masks:
        made.masks = ops.token_masks(torch.stack(masks)).to(DEVICE)
        made.mask_rows = index(lambda r: r.allowed)
    return made


def formula(logits, requests):
    """(controlled logits, the largest magnitude on the way to each) in 64 bits."""
    out = logits.double().cpu().clone()
    largest = out.abs().clone()
    for row, request in enumerate(requests):
        line = out[row]
        repetition, presence, frequency = (float(torch.tensor(p, dtype=torch.float32)) for p in request.penalties)

        def seen(ids):
            return torch.tensor(sorted({i for i in ids if 0 <= i < line.numel()}), dtype=torch.long)

        ids = seen(request.prompt + request.answer)
        line[ids] = torch.where(line[ids] > 0, line[ids] / repetition, line[ids] * repetition)
        largest[row] = torch.maximum(largest[row], line.abs())
        ids = seen(request.answer)
        counted = collections.Counter(request.answer)
        times = torch.tensor([counted[int(i)] for i in ids], dtype=torch.float64)
        line[ids] -= times * frequency
        largest[row, ids] = largest[row, ids] + times * abs(frequency) + abs(presence)
        line[ids] -= presence
        for token, value in (request.bias or {}).items():
            line[token] += float(torch.tensor(value, dtype=torch.float32))
            largest[row, token] += abs(value)
        if request.allowed is not None:
            line[~request.allowed.cpu()] = -math.inf
    return out, largest


def close(got, logits, requests):
    """Six roundings to 24 bits (quotient, product, two differences, sum, and the product of times and penalty), each by half a unit
    of a number no larger than the largest on the way."""
    want, largest = formula(logits, requests)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want.sign() * math.inf, want)      # what 32 bits cannot hold
    got = got.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    same = (got == want) | torch.isnan(want)
    assert bool((same | ((got - want).abs() <= 6 * 2.0 ** -24 * largest)).all())


def some_requests(count, vocab, length, seed, biases=20):
    rng = random.Random(seed)
    made = []
    for _ in range(count):
        held = [min(vocab - 1, int(vocab * rng.random() ** 3)) for _ in range(rng.randrange(length + 1))]
        cut = rng.randrange(len(held) + 1)
        pick = lambda value: value if rng.random() < 0.7 else None
        allowed = pick(rng.choice((0.9, 0.3, 0.01)))
        made.append(Request(held[:cut], held[cut:], pick(1.0 + rng.random()) or 1.0, pick(2 * rng.random()) or 0.0, pick(rng.random()) or 0.0,
                            pick({rng.randrange(vocab): rng.choice((-100.0, 5 * rng.gauss(0, 1))) for _ in range(rng.randrange(biases + 1))}),
                            None if allowed is None else torch.rand(vocab, generator=torch.Generator().manual_seed(rng.randrange(1 << 30))) < allowed))
    return made


def logits_for(rows, vocab, seed):
    return torch.randn((rows, vocab), generator=torch.Generator(device=DEVICE).manual_seed(seed), device=DEVICE) * 3


# one token, words of a mask that end early, one slice and many, more rows than SMs, long histories, many biases
SIZES = [(1, 1, 0, 0), (1, 33, 5, 3), (2, 2048, 0, 5), (3, 2049, 100, 20), (5, 50257, 700, 30), (1, 151936, 5000, 300), (17, 32001, 2000, 0), (200, 5003, 300, 10),
         (700, 513, 30, 2), (2, 300001, 40000, 2000)]


@pytest.mark.parametrize("rows,vocab,length,biases", SIZES)
def test_controlled_logits(rows, vocab, length, biases):
    requests = some_requests(rows, vocab, length, rows + vocab, biases)
    logits = logits_for(rows, vocab, 1)
    controls = controls_of(requests, vocab)
    before = logits.clone()
    got = ops.control_logits(logits, controls)
    finished()
    assert torch.equal(logits, before)
    close(got, logits, requests)
    assert ops.control_logits(logits, controls, out=logits) is logits      # in place
    finished()
    assert torch.equal(logits, got)


@pytest.mark.parametrize("rows,vocab,length,biases", SIZES)
@pytest.mark.parametrize("warm", [False, True])
def test_tokens_are_those_of_the_controlled_logits(rows, vocab, length, biases, warm):
    requests = some_requests(rows, vocab, length, rows * 3 + vocab, biases)
    logits = logits_for(rows, vocab, 2)
    controls = controls_of(requests, vocab)
    drawn = ()
    if warm:
        generator = torch.Generator().manual_seed(3)
        drawn = ((torch.rand(rows, generator=generator) * 2 * (torch.rand(rows, generator=generator) < 0.8)).to(DEVICE),
                 torch.randint(0, 1 << 62, (rows,), generator=generator).to(DEVICE), torch.randint(0, 5000, (rows,), generator=generator, dtype=torch.int32).to(DEVICE))
    got = ops.sample(logits, *drawn, controls=controls)
    steered = ops.control_logits(logits, controls)
    want = ops.sample(steered, *drawn)
    finished()
    nothing = (steered == -math.inf).all(dim=1)
    assert torch.equal(got, torch.where(nothing, -1, want))


def test_the_order_of_the_steps_by_hand():
    vocab = 8
    logits = torch.tensor([[2.0, -2.0, 0.0, 4.0, 1.0, 1.0, -1.0, 3.0]] * 2, device=DEVICE)
    allowed = torch.ones(vocab, dtype=torch.bool)
    allowed[7] = False
    requests = [Request([0, 1, 6], [3, 3, 1], 2.0, 0.25, 0.5, {3: 10.0, 5: -1.0, 7: 50.0}, allowed), Request()]
    got = ops.control_logits(logits, controls_of(requests, vocab))
    finished()
    assert got[0].tolist() == [1.0, -4.0 - 0.5 - 0.25, 0.0, 2.0 - 1.0 - 0.25 + 10.0, 1.0, 0.0, -2.0, -math.inf]
    assert torch.equal(got[1], logits[1])


def test_rows_with_nothing_left_infinities_and_nan():
    vocab, rows = 3000, 6
    logits = logits_for(rows, vocab, 4)
    logits[1] = -math.inf
    logits[2, 5], logits[2, 7] = math.nan, math.inf
    logits[3] = math.nan
    logits[4, :] = torch.finfo(torch.float32).min
    none, few = torch.zeros(vocab, dtype=torch.bool), torch.zeros(vocab, dtype=torch.bool)
    few[[5, 2999]] = True
    held = list(range(0, 40))
    requests = [Request(allowed=none), Request([1], [2], 1.5, 1.0, 1.0), Request([5, 7], [7], 1.5, 1.0, 1.0), Request(allowed=few),
                Request(held, held, 2.0, 1.0, 1.0, allowed=few), Request(held, held, 1.5, 0.5, 0.5, {2999: math.inf}, few)]
    controls = controls_of(requests, vocab)
    got = ops.control_logits(logits, controls)
    tokens = ops.sample(logits, controls=controls)
    finished()
    close(got, logits, requests)
    # the lowest number of the type, doubled, is -inf: token 2999 alone is left in row 4
    assert tokens.tolist() == [-1, -1, 7, -1, 2999, 2999]


def test_tokens_are_noted_once_all_histories_are_read():
    """Rows that share a history, one that is full, one without a history, one with nothing left: only what may be written changes."""
    vocab = 5000
    logits = logits_for(5, vocab, 5)
    none = torch.zeros(vocab, dtype=torch.bool)
    requests = [Request([1, 2], [3], 1.3, 0.4, 0.2), Request([1, 2], [3, 4], 1.3, 0.4, 0.2), Request([9] * 4, [8] * 3, 1.1, 0.1, 0.1), Request(), Request(allowed=none)]
    controls = controls_of(requests, vocab, capacity=7)
    shared, other = int(controls.history_rows[0]), int(controls.history_rows[1])
    controls.history[shared, :4] = controls.history[other, :4]
    controls.history_rows[1] = shared
    controls.history_rows[3] = -1
    before, alone = controls.history.clone(), ops.sample(logits, controls=controls)
    for _ in range(3):      # a repeated call finds what it found
        tokens = ops.sample(logits, controls=controls, note=True)
        finished()
        assert torch.equal(tokens, alone)
        want = before.clone()
        want[shared, 3], want[shared, 4] = tokens[0], tokens[1]
        assert torch.equal(controls.history, want)
        controls.history.copy_(before)


def test_ids_and_lengths_that_do_not_fit_are_read_as_far_as_they_do():
    vocab = 1000
    logits = logits_for(2, vocab, 6)
    requests = [Request([5, 6, 7], [8, 9], 1.5, 0.5, 0.5), Request([5], [6], 1.5, 0.5, 0.5)]
    controls = controls_of(requests, vocab, capacity=5)
    place = int(controls.history_rows[0])
    controls.history[place] = torch.tensor([5, -1, 1 << 30, 8, -(1 << 31)], dtype=torch.int32)
    controls.lengths[0], controls.prompt_lengths[0] = 1000, -3        # all five, none of them the prompt
    controls.lengths[1] = -2                                            # nothing
    got = ops.control_logits(logits, controls)
    finished()
    close(got, logits, [Request([], [5, 8], 1.5, 0.5, 0.5), Request()])


def test_an_index_of_something_that_does_not_exist_is_reported():
    from llmserver_b200.ops.library import KernelError, check_wait_errors
    vocab = 100
    logits = logits_for(2, vocab, 7)
    allowed = torch.rand(vocab) < 0.5
    requests = [Request([5], [6], 1.5, 0.5, 0.5, {3: 1.0}, allowed)] * 2
    for name in ("history_rows", "bias_rows", "mask_rows"):
        controls = controls_of(requests, vocab)
        getattr(controls, name)[1] = 1000
        got = ops.control_logits(logits, controls)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match="does not exist"):
            check_wait_errors()
        close(got[:1], logits[:1], requests[:1])
        finished()


def test_each_kind_alone_and_flags_behind_the_tokens():
    from llmserver_b200.ops.library import wait_error_flag
    vocab = 4000
    logits = logits_for(3, vocab, 8)
    requests = some_requests(3, vocab, 50, 9)
    whole = controls_of(requests, vocab)
    only = {"penalties": ("penalties", "history", "history_rows", "lengths", "prompt_lengths"), "bias": ("bias_starts", "bias_ids", "bias_values", "bias_rows"),
            "mask": ("masks", "mask_rows"), "nothing": ()}
    for kind, names in only.items():
        part = ops.LogitControls(**{name: getattr(whole, name) for name in names})
        kept = [Request(r.prompt, r.answer, *(r.penalties if kind == "penalties" else ()), bias=r.bias if kind == "bias" else None,
                        allowed=r.allowed if kind == "mask" else None) for r in requests]
        got = ops.control_logits(logits, part)
        finished()
        close(got, logits, kept)
    flag = torch.full((1,), 41, dtype=torch.int32, device=DEVICE)
    tokens = ops.sample(logits, controls=whole, flags=(flag, wait_error_flag(torch.device(DEVICE))))
    finished()
    assert tokens.tolist()[3:] == [41, 0] and torch.equal(tokens[:3], ops.sample(logits, controls=whole))
    assert ops.sample(logits[:0], controls=ops.LogitControls()).numel() == 0 and ops.control_logits(logits[:0], ops.LogitControls()).shape == (0, vocab)


def test_captured_and_replayed():
    """A step of sampling and noting in a graph: the lengths move on from replay to replay, as the eager steps do."""
    vocab, steps = 2500, 6
    requests = some_requests(4, vocab, 30, 10)
    logits = [logits_for(4, vocab, 20 + i) for i in range(steps)]

    def eager():
        controls = controls_of(requests, vocab, capacity=64)
        tokens = []
        for line in logits:
            tokens.append(ops.sample(line, controls=controls, note=True))
            controls.lengths += 1
        finished()
        return torch.stack(tokens), controls.history

    want_tokens, want_history = eager()
    controls = controls_of(requests, vocab, capacity=64)
    fixed = torch.zeros_like(logits[0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = ops.sample(fixed, controls=controls, note=True)
            controls.lengths += 1
        got = []
        for line in logits:
            fixed.copy_(line)
            graph.replay()
            got.append(out.clone())
        stream.synchronize()
    finished()
    assert torch.equal(torch.stack(got), want_tokens) and torch.equal(controls.history, want_history)


def test_from_a_norm_to_tokens():
    """The head's product in 8 bits, the controls and the draw one after the other for a few steps, against 64 bits: the tokens wherever
    the two best of a row lie further apart than the errors can reach."""
    rows, inner, vocab, steps = 9, 384, 7001, 5
    generator = torch.Generator(device=DEVICE).manual_seed(11)
    head = ops.quantize_blocks(torch.randn((vocab, inner), generator=generator, device=DEVICE) * inner ** -0.5, 128)
    requests = some_requests(rows, vocab, 40, 12)
    requests = [r for r in requests if r.allowed is None or bool(r.allowed.any())]
    rows = len(requests)
    controls = controls_of(requests, vocab, capacity=64)
    for step in range(steps):
        x = torch.randn((rows, inner), generator=generator, device=DEVICE).to(torch.bfloat16) * 3
        logits = ops.linear(x, head, out_dtype=torch.float32)
        tokens = ops.sample(logits, controls=controls, note=True)
        finished()
        held = ops.quantize_blocks(x)
        exact = held.widened().double() @ head.widened().double().t()
        size = held.widened().double().abs() @ head.widened().double().abs().t()
        want, largest = formula(exact, requests)
        slack = 2 * ((2 * 128 + 8) * 2.0 ** -24 * 2 * size.cpu().amax(1) + 6 * 2.0 ** -24 * largest.amax(1))      # repetition at most doubles an error
        best = want.topk(2, dim=1)
        clear = (best.values[:, 0] - best.values[:, 1]) > slack
        assert bool(clear.any()) and torch.equal(tokens.cpu().long()[clear], best.indices[:, 0][clear])
        for request, token in zip(requests, tokens.tolist()):
            request.answer.append(token)
        controls.lengths += 1


def test_refusals_on_the_device():
    from llmserver_b200.ops import KernelError
    vocab = 100
    logits = logits_for(2, vocab, 13)
    good = lambda: controls_of([Request([1], [2], 1.5, 0.5, 0.5, {3: 1.0}, torch.rand(vocab) < 0.5)] * 2, vocab)

    def changed(**fields):
        controls = good()
        for name, value in fields.items():
            setattr(controls, name, value)
        return controls

    whole = lambda *size: torch.zeros(size, dtype=torch.int32, device=DEVICE)
    for fields, message in (({"history_rows": None}, "history"), ({"lengths": whole(3)}, "lengths"), ({"penalties": torch.ones((2, 2), device=DEVICE)}, "penalties"),
                            ({"history": torch.zeros((4, 4), dtype=torch.int64, device=DEVICE)}, "int32"), ({"bias_values": torch.ones(1, device=DEVICE)}, "bias_values"),
                            ({"bias_starts": whole(0)}, "bias_starts"), ({"masks": whole(1, 3)}, "words"), ({"mask_rows": whole(1)}, "mask_rows"),
                            ({"prompt_lengths": None}, "prompt_lengths"), ({"history": whole(4, 8).t()}, "contiguous"), ({"history": whole(4, 4).cpu()}, "CUDA")):
        for run in (ops.control_logits, lambda l, c: ops.sample(l, controls=c)):
            with pytest.raises(KernelError, match=message):
                run(logits, changed(**fields))
    with pytest.raises(KernelError, match="noted"):
        ops.sample(logits, note=True)
    with pytest.raises(KernelError, match="history"):
        ops.sample(logits, controls=ops.LogitControls(), note=True)
    with pytest.raises(KernelError, match="float32"):
        ops.control_logits(logits.half(), good())
    with pytest.raises(KernelError, match="match"):
        ops.control_logits(logits, good(), out=torch.empty((2, 99), device=DEVICE))
    with pytest.raises(KernelError, match="temperatures"):
        ops.sample(logits, torch.ones(3, device=DEVICE), torch.zeros(3, dtype=torch.int64, device=DEVICE), whole(3), controls=good())


def test_of_rows_with_one_place_the_last_notes_its_token():
    """Forty rows, three of them and the last two with the same history and length; one that names no history is reported."""
    from llmserver_b200.ops.library import KernelError, check_wait_errors
    vocab, rows = 3000, 40
    logits = logits_for(rows, vocab, 17)
    controls = controls_of([Request([row], [row + 1], 1.2, 0.3, 0.1) for row in range(rows)], vocab, capacity=6)
    for row in (9, 35):
        controls.history_rows[row] = controls.history_rows[2]
    controls.history_rows[rows - 2] = controls.history_rows[rows - 1]
    before = controls.history.clone()
    for _ in range(2):
        controls.history.copy_(before)
        tokens = ops.sample(logits, controls=controls, note=True)
        finished()
        want = before.clone()
        for row in range(rows):      # in order, so that the last stays
            want[int(controls.history_rows[row]), 2] = tokens[row]
        assert torch.equal(controls.history, want)
    controls.history.copy_(before)
    controls.penalties, controls.history_rows[4] = None, 1000      # penalties or none: a bad index is reported
    tokens = ops.sample(logits, controls=controls, note=True)
    torch.cuda.synchronize()
    with pytest.raises(KernelError, match="does not exist"):
        check_wait_errors()
    want = before.clone()
    for row in range(rows):
        if row != 4:
            want[int(controls.history_rows[row]), 2] = tokens[row]
    assert torch.equal(controls.history, want)
    finished()


def test_logits_that_overlap_their_result_are_refused():
    from llmserver_b200.ops import KernelError
    vocab = 100
    room = torch.randn(300, device=DEVICE)
    controls = controls_of([Request([1], [2], 1.5)] * 2, vocab)
    with pytest.raises(KernelError, match="overlaps"):
        ops.control_logits(room[:200].view(2, vocab), controls, out=room[50:250].view(2, vocab))
    with pytest.raises(KernelError, match="overlaps"):
        ops.control_logits(room[100:].view(2, vocab), controls, out=room[:200].view(2, vocab))
    want = ops.control_logits(room[:200].view(2, vocab), controls)
    got = ops.control_logits(room[:200].view(2, vocab), controls, out=room[:200].view(2, vocab))
    finished()
    assert torch.equal(got, want) and got.data_ptr() == room.data_ptr()


@pytest.mark.parametrize("temperature", [1e-39, 1e-30, 1e-3, 0.3, 30.0, 1e30])
@pytest.mark.parametrize("shift,scale", [(0.0, 3.0), (-1e4, 1.0), (1e6, 50.0), (-1e-3, 1e-4)])
def test_draws_at_any_temperature_are_those_without_controls(temperature, shift, scale):
    """Controls that change nothing: tokens are passed over by a bound of their scores here and worked out one by one there."""
    rows, vocab = 6, 20000
    logits = logits_for(rows, vocab, 23) * scale + shift
    temperatures = torch.full((rows,), temperature, dtype=torch.float32, device=DEVICE)
    seeds, steps = torch.arange(rows, device=DEVICE), torch.arange(rows, dtype=torch.int32, device=DEVICE)
    want = ops.sample(logits, temperatures, seeds, steps)
    everything = torch.ones(vocab, dtype=torch.bool)
    got = ops.sample(logits, temperatures, seeds, steps, controls=controls_of([Request(allowed=everything)] * rows, vocab))
    finished()
    scores = logits.double() / float(temperatures[0])
    drawn = (scores.abs().max(1).values < torch.finfo(torch.float32).max).tolist()      # where no score is infinite
    assert [int(g) for g, d in zip(got, drawn) if d] == [int(w) for w, d in zip(want, drawn) if d]
