"""The operators of drafted decoding, as they are timed: attention of drafted
tokens over a paged cache, verification of the drafts against the model's
probabilities, and the cache's pages before and after (branching, writing,
keeping what was accepted).

Sizes are those of the library's models (16 x 64 and 4 x 128 heads, alphabet
1024, 12 layers, up to 3 lanes of about a thousand frames) and, since none of the
operators is tied to them, generic ones of serving: grouped heads, contexts of
thousands of tokens, alphabets of tens of thousands.

`own` false: elementary torch operations in 32 bits, 64 where whole numbers are
decided. `own` true: the library's calls.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # One drafted tree over a lane's context at the wide model's heads, three lanes: the smallest call.
        {"name": "tree_lanes", "kind": "attention", "sequences": 3, "longest": 1021, "nodes": 12, "tree": True,
         "heads": 16, "kv_heads": 16, "head_width": 64, "page_rows": 16, "type": "bfloat16"},
        # One new token of each of eight sequences, grouped heads: the undrafted step.
        {"name": "token_step", "kind": "attention", "sequences": 8, "longest": 8190, "nodes": 1, "tree": False,
         "heads": 32, "kv_heads": 8, "head_width": 128, "page_rows": 64, "type": "float16"},
        # The rest of a prompt, 500 tokens, behind what is cached of it.
        {"name": "prompt_chunk", "kind": "attention", "sequences": 2, "longest": 2580, "nodes": 500, "tree": False,
         "heads": 16, "kv_heads": 16, "head_width": 64, "page_rows": 128, "type": "bfloat16"},
        # A full batch, each sequence with its own tree.
        {"name": "tree_batch", "kind": "attention", "sequences": 32, "longest": 4093, "nodes": 32, "tree": True,
         "heads": 32, "kv_heads": 8, "head_width": 128, "page_rows": 32, "type": "bfloat16"},
        # One sequence with a very long context and a large tree.
        {"name": "tree_long", "kind": "attention", "sequences": 1, "longest": 131001, "nodes": 64, "tree": True,
         "heads": 32, "kv_heads": 8, "head_width": 128, "page_rows": 256, "type": "bfloat16"},
        # A frame's twelve drafted tokens in three lanes over the model's alphabet: latency.
        {"name": "verify_lanes", "kind": "verify", "sequences": 3, "nodes": 12, "children": 1, "alphabet": 1024,
         "draft": True, "type": "bfloat16"},
        # A batch of sampled trees over an ordinary alphabet.
        {"name": "verify_batch", "kind": "verify", "sequences": 32, "nodes": 32, "children": 3, "alphabet": 32000,
         "draft": True, "type": "bfloat16"},
        # Drafts of a table or a greedy drafter (no distribution of their own), a wide odd alphabet, 32 bits.
        {"name": "verify_wide", "kind": "verify", "sequences": 4, "nodes": 24, "children": 4, "alphabet": 128001,
         "draft": False, "type": "float32"},
        # Three lanes branch off one and take room for a draft, at the reference geometry.
        {"name": "branch_lanes", "kind": "branch", "sources": 1, "targets": 3, "longest": 1021, "rows": 12,
         "layers": 12, "kv_heads": 4, "head_width": 128, "page_rows": 16, "type": "bfloat16"},
        # A batch of alternatives branches off eight long sequences.
        {"name": "branch_batch", "kind": "branch", "sources": 8, "targets": 64, "longest": 4091, "rows": 32,
         "layers": 12, "kv_heads": 8, "head_width": 128, "page_rows": 64, "type": "float16"},
        # A frame's drafted rows into the cache of three lanes, and what was accepted of them kept.
        {"name": "draft_lanes", "kind": "draft", "sequences": 3, "nodes": 12, "longest": 1021, "layers": 12,
         "kv_heads": 4, "head_width": 128, "page_rows": 16, "type": "bfloat16"},
        # The same for a batch of trees.
        {"name": "draft_batch", "kind": "draft", "sequences": 64, "nodes": 32, "longest": 2045, "layers": 12,
         "kv_heads": 8, "head_width": 128, "page_rows": 32, "type": "float16"},
    ]


def _spread(rng, low, high):
    """A whole number, uniform in its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "verify", "verify", "branch", "draft"])
    type_ = rng.choice(["bfloat16", "float16"])
    if kind == "attention":
        heads, kv_heads, width = rng.choice([(16, 16, 64), (4, 4, 128), (32, 8, 128), (16, 2, 64), (8, 1, 128)])
        tree = rng.random() < 0.5
        nodes = _spread(rng, 2, 64) if tree else rng.choice([1, _spread(rng, 1, 500)])
        longest = _spread(rng, 1, 131001)
        # At most the long tree's cache and scores.
        most = min(131001 * 8 * 128 // (longest * kv_heads * width), 64 * 32 * 131001 // (nodes * heads * longest), 48)
        return {"kind": kind, "sequences": _spread(rng, 1, max(1, most)), "longest": longest, "nodes": nodes,
                "tree": tree, "heads": heads, "kv_heads": kv_heads, "head_width": width,
                "page_rows": rng.choice([16, 32, 64, 128, 256]), "type": type_}
    if kind == "verify":
        alphabet, nodes = _spread(rng, 2, 128001), _spread(rng, 1, 48)
        most = min(48, 32 * 32 * 32000 // (alphabet * nodes))
        return {"kind": kind, "sequences": _spread(rng, 1, max(1, most)), "nodes": nodes,
                "children": rng.randint(1, 4), "alphabet": alphabet, "draft": rng.random() < 0.6,
                "type": rng.choice(["bfloat16", "float16", "float32"])}
    heads, width = rng.choice([(4, 128), (16, 64), (8, 128), (1, 64)])
    layers, page_rows = rng.randint(1, 12), rng.choice([16, 32, 64])
    case = {"kind": kind, "longest": _spread(rng, 1, 4091), "layers": layers, "kv_heads": heads, "head_width": width,
            "page_rows": page_rows, "type": type_}
    if kind == "branch":
        return dict(case, sources=rng.randint(1, 8), targets=_spread(rng, 1, 64), rows=_spread(rng, 1, 32))
    return dict(case, sequences=_spread(rng, 1, 32), nodes=_spread(rng, 1, 32))


# ---------------------------------------------------------------- inputs

def _ragged(count, most, step, low):
    """`count` sizes of at most `most`, the first of them `most`, none below `low`."""
    return [max(low, most - (i * step) % (most // 4 + 1)) for i in range(count)]


def _starts(counts):
    return [0] + np.cumsum(counts).tolist()


def _ints(values, kind=torch.int32):
    return torch.tensor(np.asarray(values), dtype=kind, device="cuda")


def _normal(shape, seed, kind, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(scale).to(kind)


def _pool(shape, seed, kind):
    """Keys or values of a whole cache, made layer by layer."""
    pool = torch.empty(shape, dtype=kind, device="cuda")
    for layer in range(shape[0]):
        pool[layer] = _normal(shape[1:], seed + 1000 * layer, kind)
    return pool


def _tree(rng, nodes, children):
    """Parents of a random tree in which a parent precedes its children; at most `children` each."""
    parents, free = [-1], [0] * children
    for i in range(1, nodes):
        # Mostly near the front of what is open, so that trees are both wide and deep.
        at = int(len(free) * rng.random() ** 2) if children > 1 else 0
        parents.append(free.pop(at))
        free += [i] * children
    return parents


def _ancestors(parents):
    lines = []
    for i, p in enumerate(parents):
        lines.append((lines[p] if p >= 0 else 0) | 1 << i)
    return lines


def _counts(case):
    """(context lengths, drafted rows) of each sequence of an attention or draft case."""
    n = case["sequences"]
    return _ragged(n, case["longest"], 37, 1), _ragged(n, case["nodes"], 5, 1)


def _pages(case, lengths, room, rng, spare):
    """A table of pages in no order, what each sequence holds of it, and the reference counts."""
    rows = case["page_rows"]
    held = [-(-n // rows) for n in room]
    order = rng.permutation(sum(held) + spare)
    table = -np.ones((len(lengths), max(held) + 2), np.int32)
    at = 0
    for s, h in enumerate(held):
        table[s, :h] = order[at:at + h]
        at += h
    references = np.zeros(len(order), np.int32)
    references[order[:at]] = 1
    return {"table": _ints(table), "held": _ints(held), "lengths": _ints(lengths), "references": _ints(references)}


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    kind = TYPES[case["type"]]
    state = dict(case)
    if case["kind"] == "verify":
        return _prepare_verify(case, state, seed, rng, kind)
    kv, width, layers = case["kv_heads"], case["head_width"], case.get("layers", 1)
    if case["kind"] == "branch":
        lengths = _ragged(case["sources"], case["longest"], 37, 1) + [0] * case["targets"]
        need = case["targets"] * (2 + case["rows"] // case["page_rows"])
        state.update(_pages(case, lengths, lengths, rng, need + 17))
        # Room for what a branch holds: its source's pages and those of the new rows.
        wide = -torch.ones((len(lengths), state["table"].shape[1] + 2 + case["rows"] // case["page_rows"]),
                           dtype=torch.int32, device="cuda")
        wide[:, :state["table"].shape[1]] = state["table"]
        state["table"] = wide
        state["source"] = _ints([i % case["sources"] for i in range(case["targets"])])
        state["target"] = _ints([case["sources"] + i for i in range(case["targets"])])
        state["more"] = _ints([case["rows"]] * case["targets"])
    else:
        lengths, counts = _counts(case)
        state.update(_pages(case, lengths, [a + b for a, b in zip(lengths, counts)], rng, 5))
        starts = _starts(counts)
        state["starts"], state["rows"], state["most"] = _ints(starts), starts[-1], max(counts)
        children = 3 if case.get("tree", True) else 1
        trees = [_tree(rng, n, children) for n in counts]
        state["parents"] = _ints(sum(trees, []))
        state["words"] = -(-state["most"] // 64)
    pages = state["references"].numel()
    shape = (layers, pages, case["page_rows"], kv, width)
    state["keys"], state["values"] = _pool(shape, 7 * seed + 1, kind), _pool(shape, 7 * seed + 2, kind)
    if case["kind"] == "attention":
        state["longest_row"] = max(a + b for a, b in zip(lengths, counts))
        # Queries are the first part of the projection's output rows.
        qkv = _normal((state["rows"], case["heads"] + 2 * kv, width), 7 * seed + 3, kind)
        state["query"] = qkv[:, :case["heads"]]
        state["scale"] = 1 / math.sqrt(width)
        state["out"] = torch.zeros(state["rows"], case["heads"], width, dtype=kind, device="cuda")
        state["mask"] = None
        if case["tree"]:
            lines = sum([_ancestors(t) for t in trees], [])
            words = [[line >> 64 * w & (1 << 64) - 1 for w in range(state["words"])] for line in lines]
            state["mask"] = _ints(np.array(words, np.uint64).view(np.int64), torch.int64)
    elif case["kind"] == "draft":
        # Keys and values are the other parts of those rows, here of every layer.
        qkv = _normal((layers, state["rows"], 3 * kv, width), 7 * seed + 3, kind)
        state["new_keys"], state["new_values"] = qkv[:, :, kv:2 * kv], qkv[:, :, 2 * kv:]
        state["mask"] = torch.zeros(state["rows"], state["words"], dtype=torch.int64, device="cuda")
        state["after"] = torch.zeros_like(state["lengths"])
        path = -np.ones((case["sequences"], state["most"]), np.int32)
        accepted = []
        for s, parents in enumerate(trees):
            line = _ancestors(parents)[rng.integers(len(parents))]
            nodes = [i for i in range(len(parents)) if line >> i & 1]
            path[s, :len(nodes)] = nodes
            accepted.append(len(nodes))
        state["path"], state["accepted"] = _ints(path), _ints(accepted)
    return state


def _prepare_verify(case, state, seed, rng, kind):
    counts = _ragged(case["sequences"], case["nodes"], 5, 1)
    starts = _starts(counts)
    trees = [_tree(rng, n, case["children"]) for n in counts]
    rows, alphabet = starts[-1], case["alphabet"]
    pitch = -(-alphabet // 8) * 8  # rows begin at whole vectors
    logits = _normal((rows, alphabet), 7 * seed + 1, torch.float32, 3.0)
    target = torch.zeros(rows, pitch, dtype=kind, device="cuda")
    target[:, :alphabet] = torch.softmax(logits, 1).to(kind)
    state["target"], state["drafts"] = target[:, :alphabet], None
    parent_rows = _ints([max(p, 0) + b for t, b in zip(trees, starts) for p in t], torch.int64)
    if case["draft"]:
        logits += _normal((rows, alphabet), 7 * seed + 2, torch.float32, 0.7)
        draft = torch.zeros(rows, pitch, dtype=kind, device="cuda")
        draft[:, :alphabet] = torch.softmax(logits, 1).to(kind)
        state["drafts"] = draft[:, :alphabet]
        g = torch.Generator(device="cuda").manual_seed(7 * seed + 3)
        tokens = torch.multinomial(torch.softmax(logits, 1)[parent_rows], 1, generator=g)[:, 0]
    else:
        # The likeliest tokens after the parent, one for each of its children in order.
        rank = [sum(t[j] == t[i] for j in range(i)) for t in trees for i in range(len(t))]
        best = torch.topk(logits, min(case["children"], alphabet), 1).indices[parent_rows]
        tokens = best.gather(1, _ints(rank, torch.int64).clamp(max=best.shape[1] - 1)[:, None])[:, 0]
    state["tokens"] = tokens.to(torch.int32)
    state["parents"], state["starts"], state["most"] = _ints(sum(trees, [])), _ints(starts), max(counts)
    state["uniforms"] = _ints(rng.random(rows, np.float32), torch.float32)
    state["draws"] = _ints(rng.random(case["sequences"], np.float32), torch.float32)
    n = case["sequences"]
    state["path"] = torch.zeros(n, state["most"], dtype=torch.int32, device="cuda")
    state["accepted"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    state["next"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return (OWN if own else PLAIN)[state["kind"]](state)


def _native():
    package = os.path.join(os.getcwd(), "tsac-metal_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from tsac_hip import native

    return native


def _cache(state):
    """The cache's handle, which a program keeps beside its tensors."""
    if "cache" not in state:
        state["cache"] = _native().PagedCache(state["keys"], state["values"], state["table"], state["held"],
                                              state["lengths"], state["references"])
    return state["cache"]


def _own_attention(state):
    _native().attention_paged(_cache(state), 0, state["query"], state["starts"], state["most"], state["longest_row"],
                              state["mask"], state["scale"], state["out"])
    return state["out"]


def _own_verify(state):
    _native().verify_drafts(state["target"], state["drafts"], state["tokens"], state["parents"], state["starts"],
                            state["most"], state["uniforms"], state["draws"], state["path"], state["accepted"],
                            state["next"])
    return state["path"], state["accepted"], state["next"]


def _own_branch(state):
    cache = _cache(state)
    cache.free(state["target"])
    cache.fork(state["source"], state["target"])
    cache.reserve(state["more"], state["target"])
    return tuple(state[name] for name in ("table", "held", "lengths", "references", "keys", "values"))


def _own_draft(state):
    cache = _cache(state)
    _native().tree_mask(state["parents"], state["starts"], state["most"], state["mask"])
    cache.write(state["new_keys"], state["new_values"], state["starts"], state["most"])
    cache.keep(state["starts"], state["path"], state["accepted"], state["after"])
    return tuple(state[name] for name in ("mask", "after", "keys", "values"))


# ---------------------------------------------------------------- plain forms

def _grid(starts, most):
    """Rows as a rectangle [sequence][node]: the row of each place, and whether it is one."""
    node = torch.arange(most, device="cuda")
    row = starts[:-1, None].long() + node
    there = row < starts[1:, None]
    return torch.where(there, row, starts[:-1, None].long()), there


def _places(starts, rows):
    """The sequence and the node of each row."""
    row = torch.arange(rows, device="cuda")
    sequence = torch.searchsorted(starts, row.int(), right=True) - 1
    return sequence, row - starts[sequence]


def _plain_attention(state):
    heads, kv, width = state["heads"], state["kv_heads"], state["head_width"]
    lengths, starts, most = state["lengths"].long(), state["starts"], state["most"]
    n, rows = len(lengths), state["page_rows"]
    row, there = _grid(starts, most)
    counts = there.sum(1)
    position = torch.arange(state["longest_row"], device="cuda")
    page = state["table"].long()[:, position // rows]
    inside = position < (lengths + counts)[:, None]
    page = torch.where(inside, page, state["table"][:, :1].long())
    keys = state["keys"][0][page, position % rows].permute(0, 2, 3, 1).float()  # [n][kv][width][position]
    values = state["values"][0][page, position % rows].permute(0, 2, 1, 3).float()
    query = state["query"][row].float().view(n, most, kv, heads // kv, width)
    query = query.permute(0, 2, 1, 3, 4).reshape(n, kv, -1, width)
    score = torch.matmul(query, keys).mul_(state["scale"]).view(n, kv, most, heads // kv, -1)
    drafted = position - lengths[:, None]
    if state["mask"] is None:
        seen = drafted[:, None] <= torch.arange(most, device="cuda")[:, None]
    else:
        bit = drafted.clamp(0, 64 * state["words"] - 1)
        word = state["mask"][row].gather(2, (bit // 64)[:, None].expand(n, most, -1))
        seen = (drafted < 0)[:, None] | (word >> (bit % 64)[:, None] & 1 == 1)
    live = (seen & inside[:, None])[:, None, :, None]
    score.masked_fill_(~live, -math.inf)
    top = score.amax(-1, keepdim=True)
    weight = score.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight.view(n, kv, -1, len(position)), values).view(n, kv, most, heads // kv, width)
    out = torch.where(total == 0, 0.0, out / total).permute(0, 2, 1, 3, 4).reshape(n, most, heads, width)
    return out[_places(starts, state["rows"])].to(state["out"].dtype)


def _plain_verify(state):
    """Every node decides between its children; the path is the nodes whose ancestors were all accepted."""
    starts, most, alphabet = state["starts"], state["most"], state["alphabet"]
    row, there = _grid(starts, most)
    places = _places(starts, len(state["tokens"]))
    n = len(there)
    parent = torch.where(there, state["parents"].long()[row], -1)
    token = state["tokens"].long()[row]
    node = torch.arange(most, device="cuda")
    earlier = (parent[:, :, None] == parent[:, None, :]) & (node < node[:, None]) & (parent >= 0)[:, :, None]
    rank = torch.where(parent >= 0, earlier.sum(2), -1)
    above = starts[:-1, None].long() + parent.clamp(min=0)
    p_token = state["target"][above, token].double()
    uniform = state["uniforms"][row].double()
    accept = torch.zeros_like(there)
    shift = torch.zeros(n, most, dtype=torch.float64, device="cuda")  # s and W of each node's own row
    weight = torch.ones_like(shift)
    done = torch.zeros_like(there)
    open_ = parent.clamp(min=0)
    if state["drafts"] is not None:
        q_token = state["drafts"][above, token].double()
    else:
        struck = (earlier & (token[:, :, None] == token[:, None, :])).any(2)
        p_token = torch.where(struck, 0.0, p_token)
    # Children are tried in order: each trial needs what the last one left.
    for k in range(state["children"]):
        trial = (rank == k) & ~done.gather(1, open_)
        s, w = shift.gather(1, open_), weight.gather(1, open_)
        if state["drafts"] is None:
            yes = trial & (uniform * w < p_token)
        else:
            yes = trial & (uniform * q_token * w < (p_token - s * q_token).clamp(min=0))
        accept |= yes
        at = torch.zeros(n, most, dtype=torch.int32, device="cuda")
        done |= at.scatter_add(1, open_, yes.int()) > 0
        failed = at.scatter_add(1, open_, (trial & ~yes).int()) > 0
        if state["drafts"] is None:
            lost = torch.zeros_like(weight).scatter_add(1, open_, torch.where(trial & ~yes, p_token, 0.0))
            weight = weight - lost
        else:
            shift = torch.where(failed, shift + weight, shift)
            if k + 1 < state["children"]:
                p, q = state["target"].double(), state["drafts"].double()
                total = (p - shift[places][:, None] * q).clamp_(min=0).sum(1)
                weight = torch.where(failed, total[row], weight)
    # (I + parents)^most has an entry above zero for every ancestor.
    step = torch.eye(most, dtype=torch.float64, device="cuda") + (parent[:, :, None] == node).double()
    lines = torch.linalg.matrix_power(step, most) > 0
    reached = (accept[:, None, :] | ~lines | (node == 0)).all(2) & there & ((parent >= 0) | (node == 0))
    accepted = reached.sum(1)
    path = torch.where(reached, node, most).sort(1).values
    path = torch.where(path == most, -1, path)
    stop = torch.where(reached, node, 0).amax(1)
    last = starts[:-1].long() + stop
    p = state["target"][last].double()
    if state["drafts"] is None:
        mine = (parent == stop[:, None]) & there
        gone = torch.zeros(n, alphabet, dtype=torch.int32, device="cuda")
        gone.scatter_add_(1, token, mine.int())
        left = torch.where(gone > 0, 0.0, p)
    else:
        left = (p - shift.gather(1, stop[:, None]) * state["drafts"][last].double()).clamp_(min=0)
    left = torch.where(left.sum(1, keepdim=True) > 0, left, p)
    sums = left.cumsum(1)
    chosen = (sums <= state["draws"].double()[:, None] * sums[:, -1:]).sum(1)
    return path.int(), accepted.int(), chosen.int()


def _lowest_free(references, rank):
    """The page of each rank among the free ones."""
    return torch.searchsorted((references == 0).cumsum(0), rank + 1)


def _plain_branch(state):
    table, held, lengths, references = (state[name] for name in ("table", "held", "lengths", "references"))
    source, target, rows = state["source"].long(), state["target"].long(), state["page_rows"]
    place = torch.arange(table.shape[1], device="cuda")
    # Free.
    mine = place < held[target, None]
    references.index_add_(0, table[target].clamp(min=0).long().view(-1), -mine.int().view(-1))
    table[target] = -1
    # Fork.
    full, rest = lengths[source].long() // rows, lengths[source].long() % rows
    shared = place < full[:, None]
    pages = table[source]
    references.index_add_(0, pages.clamp(min=0).long().view(-1), shared.int().view(-1))
    partial = rest > 0
    last = pages.long().gather(1, torch.where(partial, full, full - 1)[:, None])[:, 0]
    fresh = _lowest_free(references, partial.cumsum(0) - 1)
    fresh = torch.where(partial, fresh, last)
    fork = torch.where(shared, pages, -1)
    fork = torch.where((place == full[:, None]) & partial[:, None], fresh[:, None].int(), fork)
    references.index_add_(0, fresh, partial.int())
    keep = (torch.arange(rows, device="cuda") < rest[:, None])[:, :, None, None]
    for_whole = ~partial[:, None, None, None]
    state["keys"][:, fresh] = torch.where(keep | for_whole, state["keys"][:, last], state["keys"][:, fresh])
    state["values"][:, fresh] = torch.where(keep | for_whole, state["values"][:, last], state["values"][:, fresh])
    lengths[target] = lengths[source]
    # Reserve.
    has = full + partial
    need = ((lengths[target] + state["more"] + rows - 1) // rows - has).clamp(min=0)
    before = need.cumsum(0) - need
    new = (place >= has[:, None]) & (place < (has + need)[:, None])
    page = _lowest_free(references, torch.where(new, before[:, None] + place - has[:, None], 0))
    page = torch.where(new, page, 0)
    table[target] = torch.where(new, page.int(), fork)
    references.index_add_(0, page.view(-1), new.int().view(-1))
    held[target] = (has + need).int()
    return table, held, lengths, references, state["keys"], state["values"]


def _plain_draft(state):
    starts, most, rows = state["starts"], state["most"], state["page_rows"]
    row, there = _grid(starts, most)
    n, lengths = len(there), state["lengths"].long()
    node = torch.arange(most, device="cuda")
    parent = torch.where(there, state["parents"].long()[row], -1)
    step = torch.eye(most, dtype=torch.float64, device="cuda") + (parent[:, :, None] == node).double()
    lines = (torch.linalg.matrix_power(step, most) > 0).long()
    lines = torch.nn.functional.pad(lines, (0, 64 * state["words"] - most)).view(n, most, state["words"], 64)
    sequence, within = _places(starts, state["rows"])
    state["mask"].copy_((lines << torch.arange(64, device="cuda")).sum(3)[sequence, within])
    position = lengths[sequence] + within
    page = state["table"][sequence, position // rows].long()
    state["keys"][:, page, position % rows] = state["new_keys"]
    state["values"][:, page, position % rows] = state["new_values"]
    path, accepted = state["path"].long(), state["accepted"].long()
    kept = node < accepted[:, None]
    sequence = torch.arange(n, device="cuda")[:, None].expand(n, most)
    frm, to = lengths[:, None] + torch.where(kept, path, node), lengths[:, None] + node
    edge = state["held"].long()[:, None] * rows - 1
    frm, to = torch.minimum(frm, edge), torch.minimum(to, edge)
    page_from, page_to = state["table"][sequence, frm // rows].long(), state["table"][sequence, to // rows].long()
    pick = kept[None, :, :, None, None]
    state["keys"][:, page_to, to % rows] = torch.where(pick, state["keys"][:, page_from, frm % rows],
                                                       state["keys"][:, page_to, to % rows])
    state["values"][:, page_to, to % rows] = torch.where(pick, state["values"][:, page_from, frm % rows],
                                                         state["values"][:, page_to, to % rows])
    state["after"].copy_(state["lengths"] + state["accepted"])
    return state["mask"], state["after"], state["keys"], state["values"]


PLAIN = {"attention": _plain_attention, "verify": _plain_verify, "branch": _plain_branch, "draft": _plain_draft}
OWN = {"attention": _own_attention, "verify": _own_verify, "branch": _own_branch, "draft": _own_draft}


# ---------------------------------------------------------------- work

def work(case):
    if case["kind"] == "attention":
        lengths, counts = _counts(case)
        row = case["kv_heads"] * case["head_width"] * 2 * 2
        data = sum((a + b) * row + 2 * b * case["heads"] * case["head_width"] * 2 for a, b in zip(lengths, counts))
        pairs = sum(b * a + b * (b + 1) / 2 for a, b in zip(lengths, counts))
        return {"bytes": data, "flops": 4 * case["heads"] * case["head_width"] * pairs}
    size = 4 if case["type"] == "float32" else 2
    if case["kind"] == "verify":
        # One row of each distribution a sequence, for the draw; the nodes' own values.
        counts = _ragged(case["sequences"], case["nodes"], 5, 1)
        rows = 2 if case["draft"] else 1
        return {"bytes": case["sequences"] * (rows * case["alphabet"] * size + 12) + sum(counts) * (16 + rows * size),
                "flops": 3 * rows * case["sequences"] * case["alphabet"]}
    row = case["layers"] * 2 * case["kv_heads"] * case["head_width"] * size
    if case["kind"] == "branch":
        lengths = _ragged(case["sources"], case["longest"], 37, 1)
        copied = sum(lengths[i % case["sources"]] % case["page_rows"] for i in range(case["targets"]))
        shared = sum(lengths[i % case["sources"]] // case["page_rows"] + 1 for i in range(case["targets"]))
        return {"bytes": 2 * copied * row + 4 * 4 * shared, "flops": 0}
    _, counts = _counts(case)
    return {"bytes": 2 * sum(counts) * row, "flops": 0}


# ---------------------------------------------------------------- the definitions, in 64 bits

def exact(case, seed):
    return {"attention": _exact_attention, "verify": _exact_verify, "branch": _exact_branch,
            "draft": _exact_draft}[case["kind"]](prepare(case, seed))


def _exact_attention(state):
    table, starts, lengths = (state[name].tolist() for name in ("table", "starts", "lengths"))
    group = state["heads"] // state["kv_heads"]
    result = torch.zeros(state["out"].shape, dtype=torch.float64, device="cuda")
    for s, length in enumerate(lengths):
        first, count = starts[s], starts[s + 1] - starts[s]
        pages = table[s][:-(-(length + count) // state["page_rows"])]
        for g in range(state["kv_heads"]):
            k = torch.cat([state["keys"][0, p, :, g] for p in pages])[:length + count].double()
            v = torch.cat([state["values"][0, p, :, g] for p in pages])[:length + count].double()
            for i in range(0, count, 64):
                part = range(i, min(count, i + 64))
                ok = torch.zeros(len(part), length + count, dtype=torch.bool)
                ok[:, :length] = True
                for a, node in enumerate(part):
                    if state["mask"] is None:
                        ok[a, length:length + node + 1] = True
                    else:
                        words = state["mask"][first + node].tolist()
                        ok[a, length:] = torch.tensor([bool(words[j // 64] >> j % 64 & 1) for j in range(count)])
                ok = ok.cuda()[:, None]
                q = state["query"][first + i:first + i + len(part), g * group:(g + 1) * group].double()
                score = (q.reshape(-1, q.shape[2]) @ k.T * state["scale"]).view(len(part), group, -1)
                soft = torch.softmax(score.masked_fill(~ok, -math.inf), 2).nan_to_num(0.0)
                result[first + i:first + i + len(part), g * group:(g + 1) * group] = soft @ v
    return result


def _exact_verify(state):
    starts, most = state["starts"].tolist(), state["most"]
    parents, tokens = state["parents"].tolist(), state["tokens"].tolist()
    uniforms, draws = state["uniforms"].double().tolist(), state["draws"].double().tolist()
    paths, accepted, chosen = [], [], []
    for s, (first, end) in enumerate(zip(starts, starts[1:])):
        node, path = 0, [0]
        while True:
            p = state["target"][first + node].double().cpu().numpy()
            q = state["drafts"][first + node].double().cpu().numpy() if state["drafts"] is not None else None
            left, total, shift, taken = p.copy(), 1.0, 0.0, None
            for c in range(node + 1, end - first):
                if parents[first + c] != node:
                    continue
                x, u = tokens[first + c], uniforms[first + c]
                if u * (1.0 if q is None else q[x]) * total < left[x]:
                    taken = c
                    break
                if q is None:
                    total -= left[x]
                    left[x] = 0.0
                else:
                    shift += total
                    left = np.maximum(p - shift * q, 0.0)
                    total = left.sum()
            if taken is None:
                break
            node = taken
            path.append(node)
        if left.sum() == 0:
            left = p
        sums = np.cumsum(left)
        chosen.append(int(np.searchsorted(sums, draws[s] * sums[-1], side="right")))
        paths.append(path + [-1] * (most - len(path)))
        accepted.append(len(path))
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (paths, accepted, chosen))


def _exact_branch(state):
    table, held, lengths, references = (state[name].cpu().numpy().copy()
                                        for name in ("table", "held", "lengths", "references"))
    keys, values, rows = state["keys"].clone(), state["values"].clone(), state["page_rows"]
    source, target = state["source"].tolist(), state["target"].tolist()

    def take(s):
        page = int(np.flatnonzero(references == 0)[0])
        references[page] = 1
        table[s, held[s]] = page
        held[s] += 1
        return page

    for a, b in zip(source, target):
        full, rest = divmod(int(lengths[a]), rows)
        table[b, :full] = table[a, :full]
        references[table[a, :full]] += 1
        held[b], lengths[b] = full, lengths[a]
        if rest:
            page = take(b)
            keys[:, page, :rest] = keys[:, table[a, full], :rest]
            values[:, page, :rest] = values[:, table[a, full], :rest]
    for b, more in zip(target, state["more"].tolist()):
        while held[b] * rows < lengths[b] + more:
            take(b)
    return tuple(torch.from_numpy(x) for x in (table, held, lengths, references)) + (keys, values)


def _exact_draft(state):
    table, lengths, starts = (state[name].tolist() for name in ("table", "lengths", "starts"))
    parents, path, accepted = (state[name].tolist() for name in ("parents", "path", "accepted"))
    keys, values, rows = state["keys"].clone(), state["values"].clone(), state["page_rows"]
    mask = []
    for s, length in enumerate(lengths):
        first, end = starts[s], starts[s + 1]
        lines = _ancestors(parents[first:end])
        mask += [[line >> 64 * w & (1 << 64) - 1 for w in range(state["words"])] for line in lines]
        place = lambda i: (table[s][(length + i) // rows], (length + i) % rows)  # noqa: E731
        for i in range(end - first):
            page, at = place(i)
            keys[:, page, at], values[:, page, at] = state["new_keys"][:, first + i], state["new_values"][:, first + i]
        for k in range(accepted[s]):
            page, at = place(k)
            keys[:, page, at] = state["new_keys"][:, first + path[s][k]]
            values[:, page, at] = state["new_values"][:, first + path[s][k]]
    after = torch.tensor([a + b for a, b in zip(lengths, accepted)], dtype=torch.int32)
    return torch.from_numpy(np.array(mask, np.uint64).view(np.int64)), after, keys, values
