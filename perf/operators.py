"""Operators of serving and what they are measured on: cases, inputs, one pass, what a pass has to move and compute, and the same
results in 64 bits.

``linear``    y = x W^T with W in 8 bits (e4m3) and a 32-bit scale for each block of 128 x 128; a row of x is brought to 8 bits in
              groups of 128 with a power of two as each group's scale.
``quantize``  that step alone: the 8-bit numbers and the scales of rows in groups of 128, or of a matrix in blocks of 128 x 128.
``control``   a step's logits after penalties for repeated tokens, biases and grammar masks.
``sample``    the token drawn from such logits, noted in its request's history.
"""
import math

import torch

own = False

DEVICE = "cuda:0"
BLOCK = 128
LARGEST = 448.0                    # of e4m3
F8 = torch.float8_e4m3fn
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def _linear(name, rows, inner, cols, dtype="bfloat16", out="bfloat16"):
    return {"name": name, "op": "linear", "rows": rows, "inner": inner, "cols": cols, "dtype": dtype, "out": out}


def _quantize(name, rows, inner, block_rows, dtype="bfloat16"):
    return {"name": name, "op": "quantize", "rows": rows, "inner": inner, "block_rows": block_rows, "dtype": dtype}


def _logits(name, op, rows, vocab, history, biases, masks):
    return {"name": name, "op": op, "rows": rows, "vocab": vocab, "history": history, "biases": biases, "masks": masks}


def listed():
    return [
        # one chat user's token through the gate and up projections of the 8B shape: latency, and W from memory
        _linear("linear 1 gate-up", 1, 4096, 24576),
        # eight requests' logits, straight from the 32-bit sums
        _linear("linear 8 head", 8, 4096, 151936, out="float32"),
        # a batch that fills no tile, in 32 bits, over sizes that no block divides
        _linear("linear 61 odd", 61, 2001, 1111, dtype="float32", out="float32"),
        # a chunk of a prompt through the output projection
        _linear("linear 500 output", 500, 4096, 4096),
        # the engine's largest step of prompt tokens through the gate and up projections
        _linear("linear 8192 gate-up", 8192, 4096, 24576),
        # a decode step's rows, for several products that read the same ones
        _quantize("quantize 8 rows", 8, 4096, 1),
        # a projection's matrix, as it is loaded
        _quantize("quantize matrix", 24576, 4096, 128),
        # a few requests behind short contexts, with a vocabulary of odd size
        _logits("control 3 odd", "control", 3, 50257, 200, 11, 1),
        # a busy server's step
        _logits("control 64", "control", 64, 151936, 4096, 50, 8),
        # one chat user with a grammar
        _logits("sample 1", "sample", 1, 151936, 2048, 0, 1),
        # a busy server's step
        _logits("sample 64", "sample", 64, 151936, 4096, 50, 8),
        # few requests far into long documents
        _logits("sample 5 long", "sample", 5, 151936, 32768, 300, 2),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("linear", "linear", "quantize", "control", "sample"))
    if op == "linear":
        rows, inner, cols = _spread(rng, 1, 8192), _spread(rng, 64, 16384), _spread(rng, 64, 151936)
        while rows * inner * cols > 8192 * 4096 * 24576 or inner * cols > 4096 * 151936 or rows * cols > 8192 * 24576:
            rows, cols = max(1, rows // 2), max(64, cols * 3 // 4)
        case = _linear("", rows, inner, cols, rng.choice(("bfloat16", "bfloat16", "float32")), rng.choice(("bfloat16", "float32")))
    elif op == "quantize":
        case = _quantize("", _spread(rng, 1, 16384), _spread(rng, 16, 6144), rng.choice((1, 128)), rng.choice(("bfloat16", "float32")))
    else:
        rows = _spread(rng, 1, 96)
        case = _logits("", op, rows, _spread(rng, 500, 151936 if rows > 64 else 200000), _spread(rng, 1, 32768 if rows < 8 else 4096),
                       rng.choice((0, 1, _spread(rng, 1, 300))), rng.choice((0, 1, rng.randint(1, 9))))
    return {key: value for key, value in case.items() if key != "name"}


# ------------------------------------------------------------------------------------------------------ inputs
def _blocks(count, size=BLOCK):
    return -(-count // size)


def _activations(generator, rows, inner, dtype):
    """Rows as a norm leaves them: most channels alike, a few far larger, some tokens larger than others."""
    x = torch.randn((rows, inner), generator=generator, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=generator, device=DEVICE))
    loud = torch.rand((inner,), generator=generator, device=DEVICE) < 0.003
    return (x * torch.where(loud, 20.0, 1.0)).to(dtype)


def _matrix_in_blocks(generator, cols, inner):
    """(values, scales) of a matrix as checkpoints keep it: the largest of a block of 128 x 128 becomes 448.  Rows lie a multiple of
    16 bytes apart."""
    weight = torch.randn((cols, inner), generator=generator, device=DEVICE) * inner ** -0.5
    rows_of, cols_of = _blocks(cols), _blocks(inner)
    padded = torch.nn.functional.pad(weight, (0, cols_of * BLOCK - inner, 0, rows_of * BLOCK - cols)).view(rows_of, BLOCK, cols_of, BLOCK)
    scales = padded.abs().amax((1, 3)) / LARGEST
    values = (padded / scales[:, None, :, None]).to(F8).view(rows_of * BLOCK, cols_of * BLOCK)
    kept = torch.zeros((cols, _blocks(inner, 16) * 16), dtype=F8, device=DEVICE)
    kept.view(torch.uint8)[:, :inner] = values.view(torch.uint8)[:cols, :inner]
    return kept[:, :inner], scales


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    state = dict(case)
    if case["op"] in ("linear", "quantize"):
        state["x"] = _activations(generator, case["rows"], case["inner"], TYPES[case["dtype"]])
        if case["op"] == "linear":
            state["values"], state["scales"] = _matrix_in_blocks(generator, case["cols"], case["inner"])
        return state
    rows, vocab, most = case["rows"], case["vocab"], case["history"]

    def integers(low, high, size):
        return torch.randint(low, high, size, generator=generator, device=DEVICE, dtype=torch.int32)

    def uniform(size):
        return torch.rand(size, generator=generator, device=DEVICE)

    state["logits"] = torch.randn((rows, vocab), generator=generator, device=DEVICE) * 2.5
    # one row in four leaves a penalty out
    penalties = torch.stack([1.0 + 0.5 * uniform((rows,)), 1.5 * uniform((rows,)), 0.5 * uniform((rows,))], dim=1)
    off = uniform((rows, 3)) < 0.25
    state["penalties"] = torch.where(off, torch.tensor([1.0, 0.0, 0.0], device=DEVICE), penalties)
    # histories: frequent tokens come often; requests lie in any order in a table with room for more of them
    ids = (vocab * uniform((rows + 3, most + 1)) ** 3).to(torch.int32).clamp_(max=vocab - 1)
    state["history"] = ids
    state["history_rows"] = torch.randperm(rows + 3, generator=generator, device=DEVICE)[:rows].to(torch.int32)
    state["lengths"] = integers(most // 2, most + 1, (rows,))
    state["prompt_lengths"] = (state["lengths"] * uniform((rows,))).to(torch.int32)
    # biases: per request a list of ids that ascend, some bans among them
    count = min(case["biases"], vocab)
    lists = torch.sort(torch.rand((rows, vocab), generator=generator, device=DEVICE).topk(count, dim=1).indices, dim=1).values if count else ids[:rows, :0]
    state["bias_starts"] = torch.arange(rows + 1, device=DEVICE, dtype=torch.int32) * count
    state["bias_ids"] = lists.reshape(-1).to(torch.int32).contiguous()
    values = torch.randn((rows * count,), generator=generator, device=DEVICE) * 4
    state["bias_values"] = torch.where(uniform((rows * count,)) < 0.1, -100.0, values)
    state["bias_rows"] = torch.arange(rows, device=DEVICE, dtype=torch.int32).flip(0).contiguous()
    # masks: a grammar allows almost everything, a few tokens or, where there are four and more, in one state nothing
    words, masks = _blocks(vocab, 32), case["masks"]
    chance = torch.tensor([0.9, 0.001, 0.5, 0.0][:masks] + [0.01] * (masks - 4), device=DEVICE)
    allowed = torch.rand((masks, words, 32), generator=generator, device=DEVICE) < chance[:, None, None]
    bits = (allowed.to(torch.int64) << torch.arange(32, device=DEVICE)).sum(2)
    state["masks"] = torch.where(bits >= 1 << 31, bits - (1 << 32), bits).to(torch.int32)
    state["mask_rows"] = integers(0, masks + 1, (rows,)) - 1 if masks > 1 else torch.full((rows,), masks - 1, dtype=torch.int32, device=DEVICE)
    if case["op"] == "sample":
        # one request in three is greedy
        state["temperatures"] = torch.where(uniform((rows,)) < 0.33, 0.0, 0.5 + uniform((rows,)))
        state["seeds"] = torch.randint(0, 1 << 62, (rows,), generator=generator, device=DEVICE)
        state["steps"] = state["lengths"] - state["prompt_lengths"]
    return state


# ------------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "linear":
        values, scales = _quantize_plain(state["x"], 1)
        x = _widen(values, scales, 1)
        return (x @ _widen(state["values"], state["scales"], BLOCK).t()).to(TYPES[state["out"]])
    if state["op"] == "quantize":
        return list(_quantize_plain(state["x"], state["block_rows"]))
    logits = _control_plain(state)
    return logits if state["op"] == "control" else _sample_plain(state, logits)


def _run_own(state):
    from llmserver_b200 import ops
    if state["op"] == "linear":
        return ops.linear(state["x"], ops.BlockScaled(state["values"], state["scales"], BLOCK), out_dtype=TYPES[state["out"]])
    if state["op"] == "quantize":
        result = ops.quantize_blocks(state["x"], state["block_rows"])
        return [result.values, result.scales]
    controls = ops.LogitControls(
        penalties=state["penalties"], history=state["history"], history_rows=state["history_rows"], lengths=state["lengths"],
        prompt_lengths=state["prompt_lengths"], bias_starts=state["bias_starts"], bias_ids=state["bias_ids"], bias_values=state["bias_values"],
        bias_rows=state["bias_rows"], masks=state["masks"], mask_rows=state["mask_rows"])
    if state["op"] == "control":
        return ops.control_logits(state["logits"], controls)
    tokens = ops.sample(state["logits"], state["temperatures"], state["seeds"], state["steps"], controls=controls, note=True)
    return [tokens, state["history"]]


def _quantize_plain(x, block_rows):
    rows, inner = x.shape
    high, wide = _blocks(rows, block_rows), _blocks(inner)
    x = torch.nn.functional.pad(x.float(), (0, wide * BLOCK - inner, 0, high * block_rows - rows)).view(high, block_rows, wide, BLOCK)
    bits = x.abs().amax((1, 3)).view(torch.int32)
    # the smallest power of two that brings the largest to 448 (mantissa 0x600000) or below
    exponent = ((bits + 0x1FFFFF) >> 23).sub(8).clamp(min=1)
    finite = bits < 0x7F800000
    scales = torch.where(finite, (exponent << 23).view(torch.float32), math.nan)
    inverse = torch.where(finite, ((254 - exponent) << 23).view(torch.float32), math.nan)
    values = (x * inverse[:, None, :, None]).reshape(high * block_rows, wide * BLOCK)[:rows, :inner]
    return values.to(F8), scales


def _widen(values, scales, block_rows):
    rows, inner = values.shape
    wide = scales.repeat_interleave(BLOCK, dim=1)[:, :inner]
    return values.float() * (wide if block_rows == 1 else wide.repeat_interleave(block_rows, dim=0)[:rows])


def _counts(state):
    """How often each token stands in a request's answer so far, and whether it stands in the request at all."""
    rows, vocab = state["logits"].shape
    ids = state["history"][state["history_rows"].long()].long()
    place = torch.arange(ids.shape[1], device=ids.device)
    seen, generated = place < state["lengths"][:, None], place >= state["prompt_lengths"][:, None]
    counts = torch.zeros((2, rows, vocab + 1), dtype=torch.int32, device=ids.device)
    ones = torch.ones_like(ids, dtype=torch.int32)
    counts[0].scatter_add_(1, torch.where(seen & generated, ids, vocab), ones)
    counts[1].scatter_add_(1, torch.where(seen, ids, vocab), ones)
    return counts[0, :, :vocab], counts[1, :, :vocab] > 0


def _control_plain(state):
    logits = state["logits"]
    rows, vocab = logits.shape
    counts, seen = _counts(state)
    repetition, presence, frequency = state["penalties"].unbind(1)
    divided = torch.where(logits > 0, logits / repetition[:, None], logits * repetition[:, None])
    logits = torch.where(seen, divided, logits)
    logits = logits - counts * frequency[:, None]
    logits = torch.where(counts > 0, logits - presence[:, None], logits)
    count = state["bias_ids"].numel() // rows
    if count:
        lists = state["bias_rows"].long()
        ids, values = state["bias_ids"].view(rows, count)[lists].long(), state["bias_values"].view(rows, count)[lists]
        logits.scatter_(1, ids, logits.gather(1, ids) + values)
    if state["masks"].numel():
        which = state["mask_rows"].long()
        allowed = (state["masks"][:, :, None] >> torch.arange(32, device=logits.device, dtype=torch.int32)) & 1
        allowed = allowed.view(allowed.shape[0], -1)[:, :vocab].bool()
        logits = torch.where(allowed[which.clamp(min=0)] | (which < 0)[:, None], logits, -math.inf)
    return logits


def _mix(word):
    word = ((word ^ (word >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    word = ((word ^ (word >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return word ^ (word >> 16)


def _sample_plain(state, logits):
    rows, vocab = logits.shape
    seeds = state["seeds"]
    word = _mix((seeds & 0xFFFFFFFF) ^ 0x9E3779B9)
    word = _mix(word ^ (seeds >> 32))
    word = _mix(word ^ state["steps"].long())
    place = torch.arange(vocab, device=logits.device)
    uniform = ((_mix(word[:, None] ^ place) >> 9).float() + 0.5) * 2.0 ** -23
    warm = (state["temperatures"] > 0)[:, None]
    scores = torch.where(warm, logits / torch.where(warm, state["temperatures"][:, None], 1.0) - torch.log(-torch.log(uniform)), logits)
    best = scores.amax(1, keepdim=True)
    first = torch.where(scores == best, place, vocab).amin(1)
    tokens = torch.where(best[:, 0] == -math.inf, -1, first).to(torch.int32)
    # the token is noted behind what the history holds, where one was drawn and there is room
    table, at = state["history_rows"].long(), state["lengths"].long()
    at_most = at.clamp(max=state["history"].shape[1] - 1)
    noted = torch.where((tokens >= 0) & (at == at_most), tokens, state["history"][table, at_most])
    state["history"][table, at_most] = noted
    return [tokens, state["history"]]


# ------------------------------------------------------------------------------------------------------ what a pass needs
def work(case):
    if case["op"] in ("linear", "quantize"):
        rows, inner, size = case["rows"], case["inner"], TYPES[case["dtype"]].itemsize
        if case["op"] == "quantize":
            scales = 4 * _blocks(rows, case["block_rows"]) * _blocks(inner)
            return {"bytes": rows * inner * (size + 1) + scales, "flops": 2 * rows * inner}
        cols = case["cols"]
        scales = 4 * _blocks(cols) * _blocks(inner)
        return {"bytes": rows * inner * size + cols * inner + scales + rows * cols * TYPES[case["out"]].itemsize, "flops": 2 * rows * inner * cols}
    rows, vocab = case["rows"], case["vocab"]
    # three quarters of a history on average; a mask is read once
    small = rows * (3 * case["history"] + 8 * case["biases"] + 40) + 4 * _blocks(vocab, 32) * case["masks"]
    if case["op"] == "control":
        return {"bytes": 8 * rows * vocab + small, "flops": 6 * rows * vocab}
    return {"bytes": 4 * rows * vocab + small, "flops": 20 * rows * vocab}


# ------------------------------------------------------------------------------------------------------ in 64 bits
def _to_8_bits(x, block_rows):
    """The numbers that the 8 bits stand for and the scales, from the definition: scale = 2^e with the least e for which no number of
    the block exceeds 448 2^e (not below 2^-126), each quotient to the nearest of e4m3's numbers, ties to the even one."""
    rows, inner = x.shape
    high, wide = _blocks(rows, block_rows), _blocks(inner)
    whole = torch.zeros((high * block_rows, wide * BLOCK), dtype=torch.float64, device=x.device)
    whole[:rows, :inner] = x.double()
    whole = whole.view(high, block_rows, wide, BLOCK)
    fraction, exponent = torch.frexp(whole.abs().amax((1, 3)))
    exponent = torch.where(fraction == 0, -126, exponent - torch.where(fraction <= 0.875, 9, 8)).clamp(min=-126)
    scales = torch.ldexp(torch.ones((), dtype=torch.float64, device=x.device), exponent)
    quotient = whole / scales[:, None, :, None]
    step = torch.ldexp(torch.ones((), dtype=torch.float64, device=x.device), (torch.frexp(quotient).exponent - 1).clamp(min=-6) - 3)
    return (torch.round(quotient / step) * step), scales


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] in ("linear", "quantize"):
        block_rows = 1 if case["op"] == "linear" else case["block_rows"]
        rows, inner = case["rows"], case["inner"]
        values, scales = _to_8_bits(state["x"], block_rows)
        if case["op"] == "quantize":
            return [values.reshape(-1, values.shape[2] * BLOCK)[:rows, :inner], scales]
        x = (values * scales[:, None, :, None]).view(rows, -1)[:, :inner]
        result = torch.empty((rows, case["cols"]), dtype=torch.float64, device=DEVICE)
        for first in range(0, case["cols"], 128 * BLOCK):       # a part of the matrix at a time
            part = state["values"][first:first + 128 * BLOCK].double()
            for block in range(_blocks(part.shape[0])):
                scale = state["scales"][first // BLOCK + block].double().repeat_interleave(BLOCK)[:inner]
                part[block * BLOCK:(block + 1) * BLOCK] *= scale
            result[:, first:first + 128 * BLOCK] = x @ part.t()
        return result
    if case["op"] == "sample":
        return None          # tokens are whole numbers
    logits = state["logits"].double()
    repetition, presence, frequency = state["penalties"].double().unbind(1)
    for row in range(case["rows"]):
        at, length = int(state["history_rows"][row]), int(state["lengths"][row])
        ids = state["history"][at, :length].long()
        present = ids.unique()
        old = logits[row, present]
        logits[row, present] = torch.where(old > 0, old / repetition[row], old * repetition[row])
        answer, times = ids[int(state["prompt_lengths"][row]):].unique(return_counts=True)
        logits[row, answer] -= presence[row] + times * frequency[row]
        table = int(state["bias_rows"][row])
        first, last = int(state["bias_starts"][table]), int(state["bias_starts"][table + 1])
        logits[row, state["bias_ids"][first:last].long()] += state["bias_values"][first:last].double()
        mask = int(state["mask_rows"][row])
        if mask >= 0:
            place = torch.arange(case["vocab"], device=DEVICE)
            logits[row, (state["masks"][mask][place // 32] >> (place % 32)) & 1 == 0] = -math.inf
    return logits
