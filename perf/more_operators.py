"""The operators of a model's step around the attention over a paged cache, as they
are timed: products of 8-bit integers with a scale for each token and each channel,
the norms before and after a block with its gate and residual, rotated positions on
the way into the cache, and what is done to logits before drafts are verified.

Sizes are those of the library's models (width 1024, 16 x 64 heads, alphabet 1024, up
to 3 lanes of about a thousand frames) and, since none of the operators is tied to
them, generic ones of serving: grouped heads, contexts of thousands of tokens,
alphabets of tens of thousands.

`own` false: elementary torch operations in 32 bits, 64 where whole numbers are
decided and for angles. `own` true: the library's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
SIZES = {"bfloat16": 2, "float16": 2, "float32": 4}
EPSILON = 1e-5


def listed():
    return [
        # One frame of three lanes through the wide model's first feed-forward projection: the smallest call.
        {"name": "product_lanes", "kind": "product", "rows": 3, "inputs": 1024, "outputs": 4096, "bias": True,
         "type": "bfloat16", "out_type": "bfloat16"},
        # A batch of single tokens: the weights are what is read.
        {"name": "product_tokens", "kind": "product", "rows": 48, "inputs": 8192, "outputs": 8192, "bias": False,
         "type": "float16", "out_type": "float16"},
        # Logits of a batch's drafted nodes, odd sizes.
        {"name": "product_logits", "kind": "product", "rows": 190, "inputs": 2043, "outputs": 32003, "bias": False,
         "type": "bfloat16", "out_type": "float32"},
        # Prompts: many rows of a large projection.
        {"name": "product_prompt", "kind": "product", "rows": 8190, "inputs": 8192, "outputs": 8192, "bias": True,
         "type": "bfloat16", "out_type": "bfloat16"},
        # Behind a block of the wide model, three lanes of 12 nodes: residual, then the next block's norm.
        {"name": "norm_lanes", "kind": "norm", "rows": 36, "width": 1024, "post": "none", "norm": "layer",
         "gate": "none", "residual": "bfloat16", "type": "bfloat16"},
        # Prompts: a norm behind the block, a gate for each channel, the residual in 32 bits, a norm before the next.
        {"name": "norm_prompt", "kind": "norm", "rows": 8190, "width": 8192, "post": "rms", "norm": "rms",
         "gate": "channel", "residual": "float32", "type": "bfloat16"},
        # A drafted tree of each of three lanes at the wide model's heads.
        {"name": "append_lanes", "kind": "append", "sequences": 3, "longest": 1021, "nodes": 12, "tree": True,
         "heads": 16, "kv_heads": 16, "head_width": 64, "rotary": 64, "interleaved": False, "page_rows": 16,
         "type": "bfloat16"},
        # A full batch of trees, grouped heads, a part of each head rotated.
        {"name": "append_batch", "kind": "append", "sequences": 64, "longest": 4091, "nodes": 32, "tree": True,
         "heads": 32, "kv_heads": 8, "head_width": 128, "rotary": 96, "interleaved": True, "page_rows": 64,
         "type": "float16"},
        # A chunk of a long prompt behind what is cached of it.
        {"name": "append_prompt", "kind": "append", "sequences": 1, "longest": 131001, "nodes": 8191, "tree": False,
         "heads": 32, "kv_heads": 8, "head_width": 128, "rotary": 128, "interleaved": False, "page_rows": 128,
         "type": "bfloat16"},
        # The codec's alphabet, three trees.
        {"name": "logits_lanes", "kind": "logits", "sequences": 3, "nodes": 12, "history": 1021, "alphabet": 1024,
         "biases": 0, "grammar": False, "probabilities": True, "type": "bfloat16", "out_type": "bfloat16"},
        # A full batch of trees with grammars.
        {"name": "logits_batch", "kind": "logits", "sequences": 32, "nodes": 32, "history": 4093, "alphabet": 32000,
         "biases": 30, "grammar": True, "probabilities": True, "type": "bfloat16", "out_type": "float16"},
        # One token of each sequence of a batch, a wide alphabet in 32 bits.
        {"name": "logits_wide", "kind": "logits", "sequences": 24, "nodes": 1, "history": 16381, "alphabet": 128001,
         "biases": 300, "grammar": False, "probabilities": True, "type": "float32", "out_type": "float32"},
    ]


def _spread(rng, low, high):
    """A whole number, uniform in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["product", "product", "norm", "append", "logits"])
    type_ = rng.choice(["bfloat16", "float16"])
    if kind == "product":
        rows, inputs = _spread(rng, 1, 8190), _spread(rng, 33, 12289)
        # At most the prompt's products and outputs.
        outputs = _spread(rng, 33, min(32003, 8190 * 8192 * 8192 // (rows * inputs)))
        return {"kind": kind, "rows": rows, "inputs": inputs, "outputs": outputs, "bias": rng.random() < 0.5,
                "type": rng.choice([type_, type_, "float32"]), "out_type": rng.choice([type_, type_, "float32"])}
    if kind == "norm":
        width = _spread(rng, 33, 16385)
        return {"kind": kind, "rows": _spread(rng, 1, min(30960, 8190 * 8192 // width)), "width": width,
                "post": rng.choice(["none", "rms", "layer"]), "norm": rng.choice(["rms", "layer"]),
                "gate": rng.choice(["none", "channel", "row"]), "residual": rng.choice([type_, "float32"]), "type": type_}
    if kind == "append":
        heads, kv_heads, width = rng.choice([(16, 16, 64), (4, 4, 128), (32, 8, 128), (16, 2, 64), (8, 1, 128)])
        tree = rng.random() < 0.5
        nodes, longest = _spread(rng, 2, 64) if tree else _spread(rng, 1, 8191), _spread(rng, 1, 131001)
        # At most the long prompt's cache and its rows.
        most = min(139192 * 8 * 128 // ((longest + nodes) * kv_heads * width), 8191 * 32 * 128 // (nodes * heads * width))
        return {"kind": kind, "sequences": _spread(rng, 1, max(1, min(most, 64))), "longest": longest, "nodes": nodes,
                "tree": tree, "heads": heads, "kv_heads": kv_heads, "head_width": width,
                "rotary": rng.choice([width, width // 2, 2 * rng.randint(1, width // 2)]),
                "interleaved": rng.random() < 0.5, "page_rows": rng.choice([16, 32, 64, 128, 256]), "type": type_}
    alphabet, nodes = _spread(rng, 2, 128001), _spread(rng, 1, 32)
    most = min(64, 32 * 32 * 32000 // (alphabet * nodes))
    return {"kind": kind, "sequences": _spread(rng, 1, max(1, most)), "nodes": nodes, "history": _spread(rng, 1, 16381),
            "alphabet": alphabet, "biases": rng.choice([0, _spread(rng, 1, 300)]), "grammar": rng.random() < 0.5,
            "probabilities": rng.random() < 0.6, "type": rng.choice(["bfloat16", "float16", "float32"]),
            "out_type": rng.choice(["bfloat16", "float16", "float32"])}


# ---------------------------------------------------------------- inputs

def _ragged(count, most, step, low):
    """`count` sizes of at most `most`, the first of them `most`, none below `low`."""
    return [max(low, most - (i * step) % (most // 4 + 1)) for i in range(count)]


def _starts(counts):
    return [0] + np.cumsum(counts).tolist()


def _device(values, kind=torch.int32):
    return torch.tensor(np.asarray(values), dtype=kind, device="cuda")


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, seed, kind, scale=1.0):
    return torch.randn(shape, generator=_generator(seed), device="cuda", dtype=torch.float32).mul_(scale).to(kind)


def _pitched(values):
    """Rows that begin at whole vectors, as a program lays out rows of an odd width."""
    rows, width = values.shape
    held = torch.zeros(rows, -(-width // 16) * 16, dtype=values.dtype, device=values.device)
    held[:, :width] = values
    return held[:, :width]


def _empty(rows, width, kind):
    return torch.zeros(rows, -(-width // 16) * 16, dtype=kind, device="cuda")[:, :width]


def _tree(rng, nodes, children):
    """Parents of a random tree in which a parent precedes its children; at most `children` each."""
    parents, free = [-1], [0] * children
    for i in range(1, nodes):
        # Mostly near the front of what is open, so that trees are both wide and deep.
        parents.append(free.pop(int(len(free) * rng.random() ** 2)))
        free += [i] * children
    return parents


def _lines(trees, words):
    """Ancestor bits of every node of all trees, itself among them: int64 [nodes][words]."""
    rows = []
    for parents in trees:
        lines = []
        for i, p in enumerate(parents):
            lines.append((lines[p] if p >= 0 else 0) | 1 << i)
        rows += [[line >> 64 * w & (1 << 64) - 1 for w in range(words)] for line in lines]
    return _device(np.array(rows, np.uint64).reshape(-1, words).view(np.int64), torch.int64)


def prepare(case, seed):
    state = dict(case)
    {"product": _prepare_product, "norm": _prepare_norm, "append": _prepare_append,
     "logits": _prepare_logits}[case["kind"]](state, seed, np.random.default_rng(seed))
    return state


def _prepare_product(state, seed, rng):
    rows, inputs, outputs = state["rows"], state["inputs"], state["outputs"]
    # Activations have a few large channels; weights are about normal, quantised by channel.
    x = _normal((rows, inputs), 7 * seed + 1, torch.float32)
    x *= 1 + 8 * (torch.rand(inputs, generator=_generator(7 * seed + 2), device="cuda") < 0.01).float()
    state["x"] = _pitched(x.to(TYPES[state["type"]]))
    state["weights"] = _normal((outputs, inputs), 7 * seed + 3, torch.float32, 32.0).round_().clamp_(-127, 127).to(torch.int8)
    state["channel_scales"] = (0.5 + torch.rand(outputs, generator=_generator(7 * seed + 4), device="cuda")) / (
        32 * math.sqrt(inputs))
    state["offsets"] = _normal((outputs,), 7 * seed + 5, torch.float32) if state["bias"] else None
    state["q"] = _empty(rows, inputs, torch.int8)
    state["token_scales"] = torch.zeros(rows, device="cuda")
    state["out"] = _empty(rows, outputs, TYPES[state["out_type"]])
    if own:
        _linear(state)


def _prepare_norm(state, seed, rng):
    rows, width, kind = state["rows"], state["width"], TYPES[state["type"]]
    state["x"] = _pitched(_normal((rows, width), 7 * seed + 1, kind))
    state["r"] = _pitched(_normal((rows, width), 7 * seed + 2, TYPES[state["residual"]], 3.0))
    for i, name in enumerate(("post_gain", "post_bias", "gain", "bias")):
        state[name] = _normal((width,), 7 * seed + 3 + i, torch.float32, 0.2).add_(0.0 if "bias" in name else 1.0).to(kind)
    if state["post"] != "layer":
        state["post_bias"] = None
    if state["post"] == "none":
        state["post_gain"] = None
    if state["norm"] != "layer":
        state["bias"] = None
    state["gates"] = None
    if state["gate"] != "none":
        state["gates"] = _pitched(_normal((rows if state["gate"] == "row" else 1, width), 7 * seed + 7, kind, 0.5))
    state["scale"] = 0.7
    state["sum"] = _empty(rows, width, TYPES[state["residual"]])
    state["out"] = _empty(rows, width, kind)


def _frequencies(rotary):
    """Radians a position of each pair: a long context's, in which pairs of fewer than 1 turn over 8192 positions
    are 8 times slower, those of more than 4 as they were, and the others in between."""
    f = 500000.0 ** (-np.arange(0, rotary, 2) / rotary)
    keep = np.clip((8192 * f / (2 * math.pi) - 1) / (4 - 1), 0, 1)
    return f * (keep + (1 - keep) / 8)


def _prepare_append(state, seed, rng):
    n, kv, width, rows = state["sequences"], state["kv_heads"], state["head_width"], state["page_rows"]
    kind = TYPES[state["type"]]
    lengths, counts = _ragged(n, state["longest"], 37, 1), _ragged(n, state["nodes"], 5, 1)
    held = [-(-(a + b) // rows) for a, b in zip(lengths, counts)]
    order = rng.permutation(sum(held) + 5)
    table = -np.ones((n, max(held) + 2), np.int32)
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    references = np.zeros(len(order), np.int32)
    references[order[:at]] = 1
    state.update(table=_device(table), held=_device(held), lengths=_device(lengths), references=_device(references))
    starts = _starts(counts)
    state["starts"], state["most"], state["total"] = _device(starts), max(counts), starts[-1]
    shape = (1, len(order), rows, kv, width)
    state["keys"], state["values"] = _normal(shape, 7 * seed + 1, kind), _normal(shape, 7 * seed + 2, kind)
    # Queries, keys and values are the parts of the projection's output rows.
    qkv = _normal((starts[-1], state["heads"] + 2 * kv, width), 7 * seed + 3, kind)
    state["query"] = qkv[:, :state["heads"]]
    state["new_keys"] = qkv[:, state["heads"]:state["heads"] + kv]
    state["new_values"] = qkv[:, state["heads"] + kv:]
    state["rotated"] = torch.zeros(starts[-1], state["heads"], width, dtype=kind, device="cuda")
    state["frequencies"] = _device(_frequencies(state["rotary"]), torch.float64)
    state["amplitude"] = 1.2
    state["mask"] = None
    if state["tree"]:
        state["mask"] = _lines([_tree(rng, c, 3) for c in counts], -(-max(counts) // 64))


def _prepare_logits(state, seed, rng):
    n, alphabet = state["sequences"], state["alphabet"]
    counts = _ragged(n, state["nodes"], 5, 1)
    starts = _starts(counts)
    rows, most = starts[-1], max(counts)
    state["starts"], state["most"], state["total"] = _device(starts), most, rows
    state["logits"] = _pitched(_normal((rows, alphabet), 7 * seed + 1, TYPES[state["type"]], 3.0))
    # What a sequence has said: few tokens often, many seldom. Half of it is its prompt.
    lengths = _ragged(n, state["history"], 41, 1)
    state["history_tokens"] = (torch.rand(n, max(lengths), generator=_generator(7 * seed + 2), device="cuda") ** 3 *
                               (alphabet - 1)).int()
    state["history_lengths"], state["prompts"] = _device(lengths), _device([a // 2 for a in lengths])
    state["tokens"] = (torch.rand(rows, generator=_generator(7 * seed + 3), device="cuda") ** 3 * (alphabet - 1)).int()
    state["line"] = _lines([_tree(rng, c, 3) for c in counts], -(-most // 64))
    state["repetition"] = _device(1 + 0.3 * rng.random(n), torch.float32)
    state["presence"] = _device(0.5 * rng.random(n), torch.float32)
    state["frequency"] = _device(0.2 * rng.random(n), torch.float32)
    # One sequence in eight takes the likeliest token.
    state["temperature"] = _device([0.0 if i % 8 == 5 else 0.5 + 0.8 * rng.random() for i in range(n)], torch.float32)
    state["bias_starts"] = state["bias_tokens"] = state["bias_values"] = state["allowed"] = None
    if state["biases"]:
        sizes = [min(b, alphabet) for b in _ragged(n, state["biases"], 7, 0)]
        state["bias_starts"] = _device(_starts(sizes))
        state["bias_tokens"] = _device(np.concatenate([rng.choice(alphabet, b, replace=False) for b in sizes]))
        state["bias_values"] = _device(rng.normal(size=sum(sizes)) * 4, torch.float32)
    if state["grammar"]:
        # One row in three may go on with anything, the others with a quarter of the alphabet.
        words = torch.randint(-2 ** 31, 2 ** 31, (2, rows, -(-alphabet // 32)), generator=_generator(7 * seed + 4),
                              device="cuda").to(torch.int32)
        state["allowed"] = words[0] & words[1]
        state["allowed"][::3] = -1
    state["out"] = _empty(rows, alphabet, TYPES[state["out_type"]])


# ---------------------------------------------------------------- one pass

def run(state):
    return (OWN if own else PLAIN)[state["kind"]](state)


def _native():
    package = os.path.join(os.getcwd(), "tsac-metal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from tsac_hip import native

    return native


def _linear(state):
    """The projection's handle, which a program makes once from its weights."""
    if "linear" not in state:
        state["linear"] = _native().ChannelLinear(state["weights"], state["channel_scales"], state["offsets"])
    return state["linear"]


def _own_product(state):
    native = _native()
    native.quantize_tokens(state["x"], state["q"], state["token_scales"])
    _linear(state).apply(state["q"], state["token_scales"], state["out"])
    return state["out"]


def _own_norm(state):
    native = _native()
    kinds = {"none": native.NORM_NONE, "rms": native.NORM_RMS, "layer": native.NORM_LAYER}
    native.block_norm(state["x"], post=kinds[state["post"]], post_gain=state["post_gain"], post_bias=state["post_bias"],
                      gate=state["gates"], scale=state["scale"], residual=state["r"], sum=state["sum"],
                      norm=kinds[state["norm"]], gain=state["gain"], bias=state["bias"], epsilon=EPSILON,
                      out=state["out"])
    return state["sum"], state["out"]


def _own_append(state):
    if "cache" not in state:
        state["cache"] = _native().PagedCache(state["keys"], state["values"], state["table"], state["held"],
                                              state["lengths"], state["references"])
    state["cache"].append(0, state["query"], state["new_keys"], state["new_values"], state["starts"], state["most"],
                          state["frequencies"], state["rotated"], interleaved=state["interleaved"],
                          amplitude=state["amplitude"], mask=state["mask"])
    return state["rotated"], state["keys"], state["values"]


def _own_logits(state):
    _native().adjust_logits(
        state["logits"], state["out"], state["starts"], probabilities=state["probabilities"],
        history=state["history_tokens"], history_lengths=state["history_lengths"], prompt_lengths=state["prompts"],
        tokens=state["tokens"], mask=state["line"], repetition=state["repetition"], presence=state["presence"],
        frequency=state["frequency"], bias_starts=state["bias_starts"], bias_tokens=state["bias_tokens"],
        bias_values=state["bias_values"], allowed=state["allowed"],
        temperature=state["temperature"] if state["probabilities"] else None)
    return state["out"]


# ---------------------------------------------------------------- plain forms

def _places(starts, rows):
    """The sequence and the node of each row."""
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(starts, row.int(), right=True) - 1
    return sequence, row - starts[sequence]


def _bits(mask, count):
    """[rows][words] of 64 bits as truth values [rows][count]."""
    wide = mask[:, :, None] >> torch.arange(64, device="cuda") & 1
    return wide.flatten(1)[:, :count].bool()


def _plain_product(state):
    x = state["x"].float()
    scale = x.abs().amax(1) / 127
    q = torch.round(x.double() / scale.double()[:, None]).nan_to_num(0.0).float()
    out = torch.matmul(q, state["weights"].float().T) * (scale[:, None] * state["channel_scales"])
    if state["offsets"] is not None:
        out += state["offsets"]
    return out.to(state["out"].dtype)


def _plain_normed(x, kind, gain, bias):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPSILON) * gain.float()
    return x if bias is None else x + bias.float()


def _plain_norm(state):
    u = _plain_normed(state["x"].float(), state["post"], state["post_gain"], state["post_bias"])
    if state["gates"] is not None:
        u = u * state["gates"].float()
    total = state["r"].float() + state["scale"] * u
    out = _plain_normed(total, state["norm"], state["gain"], state["bias"])
    return total.to(state["sum"].dtype), out.to(state["out"].dtype)


def _plain_rotated(x, cos, sin, interleaved, rotary):
    half = rotary // 2
    cos, sin = cos[:, None], sin[:, None]
    x = x.float()
    a, b = (x[..., 0:rotary:2], x[..., 1:rotary:2]) if interleaved else (x[..., :half], x[..., half:rotary])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., rotary:]), -1)


def _plain_append(state):
    starts, rows = state["starts"], state["page_rows"]
    sequence, node = _places(starts, state["total"])
    length = state["lengths"][sequence].long()
    depth = node if state["mask"] is None else _bits(state["mask"], state["most"]).sum(1) - 1
    angle = (length + depth).double()[:, None] * state["frequencies"]
    cos, sin = ((f(angle) * state["amplitude"]).float() for f in (torch.cos, torch.sin))
    kind = state["rotated"].dtype
    place = length + node
    page, within = state["table"][sequence, place // rows].long(), place % rows
    turn = (cos, sin, state["interleaved"], state["rotary"])
    state["keys"][0, page, within] = _plain_rotated(state["new_keys"], *turn).to(kind)
    state["values"][0, page, within] = state["new_values"]
    return _plain_rotated(state["query"], *turn).to(kind), state["keys"], state["values"]


def _plain_logits(state):
    rows, alphabet, n = state["total"], state["alphabet"], state["sequences"]
    sequence, _ = _places(state["starts"], rows)
    length, prompt = state["history_lengths"][:, None], state["prompts"][:, None]
    at = torch.arange(state["history_tokens"].shape[1], device="cuda")
    index = state["history_tokens"].long()
    seen = torch.zeros(n, alphabet, device="cuda").scatter_add_(1, index, (at < length).float())
    said = torch.zeros(n, alphabet, device="cuda").scatter_add_(1, index, ((at < length) & (at >= prompt)).float())
    # The nodes on a row's line are said too.
    grid = (state["starts"][:-1, None] + torch.arange(state["most"], device="cuda")).clamp(max=rows - 1)
    line = torch.zeros(rows, alphabet, device="cuda")
    line.scatter_add_(1, state["tokens"].long()[grid][sequence], _bits(state["line"], state["most"]).float())
    said = said[sequence] + line
    seen = seen[sequence] + line > 0
    take = lambda name: state[name][sequence, None]  # noqa: E731
    x = state["logits"].float()
    r = take("repetition")
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - take("frequency") * said - take("presence") * (said > 0)
    if state["biases"]:
        bias = torch.zeros(n, alphabet, device="cuda")
        entry = torch.arange(len(state["bias_tokens"]), device="cuda", dtype=torch.int32)
        bias[torch.searchsorted(state["bias_starts"], entry, right=True) - 1, state["bias_tokens"].long()] = \
            state["bias_values"]
        x += bias[sequence]
    if state["grammar"]:
        token = torch.arange(alphabet, device="cuda")
        ok = state["allowed"][:, token // 32] >> (token % 32).int() & 1
        x = torch.where(ok == 1, x, -math.inf)
    if state["probabilities"]:
        t = take("temperature")
        top = x.amax(1, keepdim=True)
        weight = torch.where(x == -math.inf, 0.0, torch.exp((x - top) / torch.where(t == 0, 1.0, t)))
        total = weight.sum(1, keepdim=True)
        soft = torch.where(total == 0, 0.0, weight / total)
        first = (x == top).int().argmax(1, keepdim=True)
        hard = torch.zeros_like(x).scatter_(1, first, (top > -math.inf).float())
        x = torch.where(t == 0, hard, soft)
    return x.to(state["out"].dtype)


PLAIN = {"product": _plain_product, "norm": _plain_norm, "append": _plain_append, "logits": _plain_logits}
OWN = {"product": _own_product, "norm": _own_norm, "append": _own_append, "logits": _own_logits}


# ---------------------------------------------------------------- work

def work(case):
    size = SIZES[case["type"]]
    if case["kind"] == "product":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": m * k * size + n * k + n * 4 * (1 + case["bias"]) + m * n * SIZES[case["out_type"]],
                "flops": 2 * m * k * n}
    if case["kind"] == "norm":
        cells = case["rows"] * case["width"]
        gate = cells if case["gate"] == "row" else 0
        return {"bytes": cells * (2 * size + 2 * SIZES[case["residual"]]) + gate * size, "flops": 12 * cells}
    if case["kind"] == "append":
        rows = sum(_ragged(case["sequences"], case["nodes"], 5, 1))
        row = (case["heads"] + 2 * case["kv_heads"]) * case["head_width"]
        return {"bytes": 2 * rows * row * size, "flops": 3 * rows * (case["heads"] + case["kv_heads"]) * case["rotary"]}
    rows = sum(_ragged(case["sequences"], case["nodes"], 5, 1))
    cells = rows * case["alphabet"]
    return {"bytes": cells * (size + SIZES[case["out_type"]]) + case["grammar"] * cells // 8 +
            4 * sum(_ragged(case["sequences"], case["history"], 41, 1)), "flops": 8 * cells}


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    return {"product": _exact_product, "norm": _exact_norm, "append": _exact_append,
            "logits": _exact_logits}[case["kind"]](prepare(case, seed))


def _exact_product(state):
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    w = state["weights"].double()
    for i in range(0, state["rows"], 1024):
        x = state["x"][i:i + 1024].double()
        # A token's scale is a number of 32 bits.
        scale = (x.abs().max(1, keepdim=True).values / 127).float().double()
        q = torch.where(scale > 0, (x / scale).round(), 0.0)
        out[i:i + 1024] = (q @ w.t()) * scale * state["channel_scales"].double()
    return out if state["offsets"] is None else out + state["offsets"].double()


def _exact_norm(state):
    def normed(v, kind, gain, bias):
        if kind == "none":
            return v
        shift = v.mean(1, keepdim=True) if kind == "layer" else 0.0
        spread = ((v - shift) ** 2).sum(1, keepdim=True) / v.shape[1]
        v = (v - shift) / (spread + EPSILON).sqrt() * gain.double()
        return v + (0.0 if bias is None else bias.double())

    sums, outs = [], []
    for i in range(0, state["rows"], 2048):
        part = slice(i, i + 2048)
        v = normed(state["x"][part].double(), state["post"], state["post_gain"], state["post_bias"]) * state["scale"]
        if state["gates"] is not None:
            v = v * state["gates"][part if state["gate"] == "row" else slice(None)].double()
        sums.append(state["r"][part].double() + v)
        outs.append(normed(sums[-1], state["norm"], state["gain"], state["bias"]))
    return torch.cat(sums), torch.cat(outs)


def _exact_append(state):
    starts, lengths, table = (state[name].tolist() for name in ("starts", "lengths", "table"))
    rotary, rows, size = state["rotary"], state["page_rows"], state["head_width"]
    # A pair (a, b) as the number a + ib, times that of its angle.
    pairs = [(2 * j, 2 * j + 1) if state["interleaved"] else (j, j + rotary // 2) for j in range(rotary // 2)]
    a, b = ([p[i] for p in pairs] for i in (0, 1))
    rest = list(range(rotary, size))

    def turned(x, factor):
        x, out = x.double(), torch.zeros(x.shape, dtype=torch.float64, device="cuda")
        z = torch.complex(x[..., a], x[..., b]) * factor[:, None]
        out[..., a], out[..., b], out[..., rest] = z.real, z.imag, x[..., rest]
        return out

    query = torch.zeros(state["rotated"].shape, dtype=torch.float64, device="cuda")
    keys, values = state["keys"].double(), state["values"].double()
    for s, length in enumerate(lengths):
        first, end = starts[s], starts[s + 1]
        if state["mask"] is None:
            depth = list(range(end - first))
        else:
            depth = [sum(bin(w & (1 << 64) - 1).count("1") for w in line) - 1
                     for line in state["mask"][first:end].tolist()]
        angle = _device([length + d for d in depth], torch.float64)[:, None] * state["frequencies"]
        factor = torch.polar(torch.full_like(angle, state["amplitude"]), angle)
        query[first:end] = turned(state["query"][first:end], factor)
        where = [length + i for i in range(end - first)]
        page = _device([table[s][t // rows] for t in where], torch.int64)
        within = _device([t % rows for t in where], torch.int64)
        keys[0, page, within] = turned(state["new_keys"][first:end], factor)
        values[0, page, within] = state["new_values"][first:end].double()
    return query, keys, values


def _exact_logits(state):
    starts, alphabet = state["starts"].tolist(), state["alphabet"]
    out = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    names = ("repetition", "presence", "frequency", "temperature")
    for s in range(state["sequences"]):
        repetition, presence, frequency, temperature = (state[name][s].item() for name in names)
        length, prompt = state["history_lengths"][s].item(), state["prompts"][s].item()
        past = state["history_tokens"][s, :length].long()
        before = torch.bincount(past[:prompt], minlength=alphabet)
        after = torch.bincount(past[prompt:], minlength=alphabet)
        bias = torch.zeros(alphabet, dtype=torch.float64, device="cuda")
        if state["biases"]:
            mine = slice(*state["bias_starts"][s:s + 2].tolist())
            bias[state["bias_tokens"][mine].long()] = state["bias_values"][mine].double()
        own_tokens = state["tokens"][starts[s]:starts[s + 1]].long()
        for r in range(starts[s], starts[s + 1]):
            words = [w & (1 << 64) - 1 for w in state["line"][r].tolist()]
            nodes = [i for i in range(starts[s + 1] - starts[s]) if words[i // 64] >> i % 64 & 1]
            count = after + torch.bincount(own_tokens[nodes], minlength=alphabet)
            x = state["logits"][r].double()
            again = count + before > 0
            x = torch.where(again & (x > 0), x / repetition, torch.where(again, x * repetition, x))
            x = x - frequency * count - presence * (count > 0) + bias
            if state["grammar"]:
                word = state["allowed"][r].long()[:, None] >> torch.arange(32, device="cuda") & 1
                x = x.masked_fill(word.flatten()[:alphabet] == 0, -math.inf)
            if state["probabilities"]:
                if x.max() == -math.inf:
                    x = torch.zeros_like(x)
                elif temperature == 0:
                    x = torch.zeros_like(x).index_fill_(0, torch.nonzero(x == x.max())[0], 1.0)
                else:
                    x = torch.softmax(x / temperature, 0)
            out[r] = x
    return out
