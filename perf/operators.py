"""What the speed of drafting, sharing and scoring is measured on: one call of an operator, case by case.

``tree``: attention of the nodes of drafted trees over the paged cache (one layer's call).  ``accept``: the walk down each
tree by what was drawn, and the cache rows of the accepted nodes moved together, for all layers at once.  ``copy``: cache
pages copied for all layers, as a fork of a sequence does.  ``logprobs``: log probabilities of given tokens, the entropy
and the top alternatives from a step's logits.  ``score``: log probabilities and entropy straight from the last hidden
rows and the head.

Sizes are those of the library's headline model (width 2560, 36 layers, 32 heads of 128 on 8, a vocabulary of 151,936) and
of its design comparisons (width 2048, 16 heads on 4), lengths and tree sizes are generic.
"""

import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
PAGE = 64


# ------------------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one conversation, a drafted chain of a few tokens: the least a step with drafts does
        dict(kind="tree", name="tree_one_chain", dtype="bf16", seqs=1, nodes=5, branch=1, past=1500, heads=32, kv_heads=8, dim=128, window=0),
        # a running batch with small trees, windowed layers of the narrower heads
        dict(kind="tree", name="tree_batch_window", dtype="bf16", seqs=8, nodes=24, branch=4, past=2000, heads=16, kv_heads=4, dim=64, window=1024),
        # a full batch with wide trees far into unequal sequences
        dict(kind="tree", name="tree_wide", dtype="bf16", seqs=16, nodes=64, branch=8, past=4096, heads=32, kv_heads=8, dim=128, window=0),
        # the 32-bit path
        dict(kind="tree", name="tree_float32", dtype="fp32", seqs=2, nodes=13, branch=4, past=300, heads=16, kv_heads=4, dim=128, window=0),
        # behind the tree attention of one conversation, and of a batch with wide trees
        dict(kind="accept", name="accept_one", dtype="bf16", seqs=1, nodes=8, branch=4, past=1000, taken=4, layers=36, kv_heads=8, dim=128),
        dict(kind="accept", name="accept_batch", dtype="bf16", seqs=16, nodes=64, branch=8, past=300, taken=6, layers=36, kv_heads=8, dim=128),
        # a fork copies the one page that is not full; a beam of many sequences copies one each
        dict(kind="copy", name="copy_one_page", dtype="bf16", pages=1, layers=8, kv_heads=4, dim=128),
        dict(kind="copy", name="copy_batch", dtype="bf16", pages=32, layers=36, kv_heads=8, dim=128),
        # a decode step of a batch whose requests want alternatives, and a portion of a prompt that is scored
        dict(kind="logprobs", name="logprobs_decode", dtype="fp32", rows=8, vocab=151936, top=20),
        dict(kind="logprobs", name="logprobs_prompt", dtype="fp32", rows=600, vocab=151936, top=5),
        # a short text and a long one, scored from their hidden rows
        dict(kind="score", name="score_short", dtype="bf16", rows=333, width=2048, vocab=32768),
        dict(kind="score", name="score_prompt", dtype="bf16", rows=2048, width=2560, vocab=151936),
    ]


def _spread(rng, low, high):
    """A whole number from ``low`` to ``high``, spread over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "tree", "accept", "copy", "logprobs", "logprobs", "score"))
    if kind == "tree":
        kv_heads, group = rng.choice(((8, 4), (4, 4), (4, 8), (2, 3), (8, 1), (4, 2)))
        fp32 = rng.random() < 0.2
        return dict(kind=kind, dtype="fp32" if fp32 else "bf16", seqs=_spread(rng, 1, 4 if fp32 else 16),
                    nodes=_spread(rng, 1, 16 if fp32 else 64), branch=rng.choice((1, 3, 8)), past=_spread(rng, 1, 600 if fp32 else 4096),
                    heads=kv_heads * group, kv_heads=kv_heads, dim=rng.choice((64, 128)), window=rng.choice((0, 0, 0, 700)))
    if kind == "accept":
        nodes = _spread(rng, 1, 64)
        return dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp32")), seqs=_spread(rng, 1, 16), nodes=nodes,
                    branch=rng.choice((1, 3, 8)), past=_spread(rng, 1, 300), taken=rng.randint(1, min(nodes, 12)), layers=rng.randint(1, 36),
                    kv_heads=rng.choice((2, 4)), dim=rng.choice((64, 128)))
    if kind == "copy":
        return dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp32")), pages=_spread(rng, 1, 32), layers=rng.randint(1, 36),
                    kv_heads=rng.choice((1, 2, 4)), dim=rng.choice((64, 128)))
    if kind == "logprobs":
        return dict(kind=kind, dtype=rng.choice(("fp32", "fp32", "bf16")), rows=_spread(rng, 1, 600),
                    vocab=rng.choice((151936, 32768, _spread(rng, 1000, 150000))), top=rng.choice((0, 1, 5, 20, 32)))
    return dict(kind=kind, dtype="bf16", rows=_spread(rng, 129, 2048), width=8 * rng.randint(128, 320),
                vocab=rng.choice((32768, _spread(rng, 8000, 151936))))


def _row_bytes(case):
    """Bytes of one token's keys and values in one layer."""
    return 2 * case["kv_heads"] * case["dim"] * DTYPES[case["dtype"]].itemsize


def _lengths(case):
    """Each sequence's number of nodes and of cached tokens in front of them: unequal, the longest as the case says."""
    n, p = case["nodes"], case["past"]
    nodes = [max(1, n - (3 * s * n) // (7 * case["seqs"])) for s in range(case["seqs"])]
    past = [max(1, p - (5 * s * p) // (8 * case["seqs"])) for s in range(case["seqs"])]
    return nodes, past


def work(case):
    kind, item = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "tree":
        nodes, past = _lengths(case)
        window = case["window"] or 1 << 30
        seen = [min(p, window + n) + n for n, p in zip(nodes, past)]
        return {"bytes": sum(seen) * _row_bytes(case) + 2 * sum(nodes) * case["heads"] * case["dim"] * item,
                "flops": sum(4 * n * (min(p, window) + n / 2) * case["heads"] * case["dim"] for n, p in zip(nodes, past))}
    if kind == "accept":
        nodes, _ = _lengths(case)
        moved = sum(min(case["taken"], n) - 1 for n in nodes)
        return {"bytes": 2 * moved * case["layers"] * _row_bytes(case) + 12 * sum(nodes) + 8 * sum(nodes), "flops": 0}
    if kind == "copy":
        return {"bytes": 2 * case["pages"] * PAGE * case["layers"] * _row_bytes(case), "flops": 0}
    if kind == "logprobs":
        return {"bytes": case["rows"] * (case["vocab"] * item + 12 + 8 * case["top"]), "flops": 5 * case["rows"] * case["vocab"]}
    return {"bytes": (case["rows"] + case["vocab"]) * case["width"] * item + 12 * case["rows"],
            "flops": 2 * case["rows"] * case["vocab"] * case["width"]}


# ------------------------------------------------------------------------------------------ the inputs

def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _trees(case, rng):
    """Parents of every sequence's nodes (the first is the root), a chain of ``taken`` of them in each for ``accept``."""
    nodes, _ = _lengths(case)
    parents, chains = [], []
    for n in nodes:
        taken = min(case.get("taken", 1), n)
        chain = [0] + sorted(rng.choice(np.arange(1, n), taken - 1, replace=False).tolist()) if n > 1 else [0]
        p = [-1] + [int(rng.integers(max(0, i - case["branch"]), i)) for i in range(1, n)]
        for a, b in zip(chain, chain[1:]):
            p[b] = a
        parents.append(p)
        chains.append(chain)
    return parents, chains


def _ancestors(parents, longest):
    """Which nodes of its sequence each node may look at: itself and those above it, ``[seqs, longest, longest]``."""
    seen = np.zeros((len(parents), longest, longest), dtype=bool)
    for s, p in enumerate(parents):
        for i, above in enumerate(p):
            if above >= 0:
                seen[s, i] = seen[s, above]
            seen[s, i, i] = True
    return seen


def _batch(case, rng):
    """What a step's plan holds: the sequences' slots, places and lengths, a page table with scattered pages, the trees."""
    nodes, past = _lengths(case)
    seqs, longest = len(nodes), max(nodes)
    held = [-(-(p + n) // PAGE) for p, n in zip(past, nodes)]
    order = rng.permutation(sum(held) + 3)
    table = np.zeros((seqs + 1, max(held)), dtype=np.int32)
    slots, at = rng.permutation(seqs + 1)[:seqs], 0
    for slot, h in zip(slots, held):
        table[slot, :h] = order[at:at + h]
        at += h
    parents, chains = _trees(case, rng)
    seen = _ancestors(parents, longest)
    depth = seen.sum(2) - 1
    words = -(-longest // 32)
    bits = np.zeros((seqs, longest, words * 32), dtype=np.uint8)
    bits[:, :, :longest] = seen
    masks = np.packbits(bits, axis=2, bitorder="little").view(np.int32)
    starts = np.concatenate([[0], np.cumsum(nodes)])[:-1]
    return dict(
        nodes=nodes, past=past, longest=longest, pages=int(sum(held) + 3), chains=chains, starts=starts, parents_host=parents,
        table=torch.from_numpy(table).to(DEVICE), slot=_ints(slots.tolist()), start=_ints(starts.tolist()), length=_ints(nodes),
        kv_len=_ints([p + n for p, n in zip(past, nodes)]),
        pos=_ints(np.concatenate([past[s] + depth[s, :n] for s, n in enumerate(nodes)]).tolist()),
        mask=torch.from_numpy(np.concatenate([masks[s, :n] for s, n in enumerate(nodes)])).to(DEVICE),
        parents=_ints(sum(parents, [])), seen=torch.from_numpy(seen).to(DEVICE))


def _stores(case, pages, g, layers):
    shape = (layers, pages, case["kv_heads"], PAGE, case["dim"])
    return [torch.randn(shape, generator=g, device=DEVICE, dtype=DTYPES[case["dtype"]]) for _ in range(2)]


def prepare(case, seed):
    kind, g, rng = case["kind"], _generator(seed), np.random.default_rng(seed)
    state = dict(case)
    if kind == "tree":
        b = _batch(case, rng)
        keys, values = _stores(case, b["pages"], g, 1)
        q = torch.randn((sum(b["nodes"]), case["heads"] * case["dim"]), generator=g, device=DEVICE, dtype=DTYPES[case["dtype"]])
        state.update(b=b, keys=keys[0], values=values[0], q=q, scale=case["dim"] ** -0.5)
    elif kind == "accept":
        b = _batch(case, rng)
        keys, values = _stores(case, b["pages"], g, case["layers"])
        # draws that lead down each chain; every other draw, and that of the chain's end, is no token of the tree
        tokens, drawn = rng.permutation(50000)[:sum(b["nodes"])], 50000 + rng.permutation(50000)[:sum(b["nodes"])]
        for first, chain in zip(b["starts"], b["chains"]):
            for a, c in zip(chain, chain[1:]):
                drawn[first + a] = tokens[first + c]
        state.update(b=b, keys=keys, values=values, tokens=_ints(tokens.tolist()), drawn=_ints(drawn.tolist()))
    elif kind == "copy":
        total = 2 * case["pages"] + 3
        keys, values = _stores(case, total, g, case["layers"])
        order = rng.permutation(total).tolist()
        state.update(keys=keys, values=values, source=order[:case["pages"]], target=order[case["pages"]:2 * case["pages"]])
    elif kind == "logprobs":
        # logits of a trained model: most of the weight on few entries
        x = torch.randn((case["rows"], case["vocab"]), generator=g, device=DEVICE).mul_(2.0)
        x.scatter_add_(1, torch.randint(0, case["vocab"], (case["rows"], 16), generator=g, device=DEVICE),
                       torch.rand((case["rows"], 16), generator=g, device=DEVICE).mul_(8.0))
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEVICE, dtype=torch.int32)
        state.update(logits=x.to(DTYPES[case["dtype"]]), tokens=tokens)
    else:
        h = torch.randn((case["rows"], case["width"]), generator=g, device=DEVICE, dtype=torch.bfloat16)
        head = torch.randn((case["vocab"], case["width"]), generator=g, device=DEVICE, dtype=torch.bfloat16).mul_(1.5 * case["width"] ** -0.5)
        tokens = torch.randint(0, case["vocab"], (case["rows"],), generator=g, device=DEVICE, dtype=torch.int32)
        state.update(h=h, head=head, tokens=tokens)
    return state


# ------------------------------------------------------------------------------------------ the calls

def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "accept": _plain_accept, "copy": _plain_copy, "logprobs": _plain_logprobs, "score": _plain_score}[state["kind"]](state)


def _own(state):
    from starter_b200 import ops

    kind = state["kind"]
    if kind == "tree":
        b = state["b"]
        return ops.attention_tree(state["q"], state["keys"], state["values"], b["table"], b["slot"], b["start"], b["length"], b["kv_len"],
                                  b["pos"], b["mask"], state["heads"], state["kv_heads"], state["dim"], state["scale"],
                                  window=state["window"] or None, max_q_len=b["longest"], kv_hint=max(b["past"]) + b["longest"])
    if kind == "accept":
        b = state["b"]
        count, path, taken = ops.cache_accept([(state["keys"], state["values"])], b["table"], b["slot"], b["start"], b["length"], b["kv_len"],
                                              state["tokens"], b["parents"], state["drawn"], max_q_len=b["longest"])
        return count, path, taken, state["keys"], state["values"]
    if kind == "copy":
        ops.cache_copy_pages([state["keys"], state["values"]], state["source"], state["target"])
        return state["keys"], state["values"]
    if kind == "logprobs":
        return ops.token_logprobs(state["logits"], state["tokens"], top=state["top"])
    return ops.linear_logprobs(state["h"], state["head"], state["tokens"])


def _padded(b):
    """Row of every (sequence, node) in the packing, and whether there is one."""
    node = torch.arange(b["longest"], device=DEVICE)
    return (b["start"].long()[:, None] + node).clamp_(max=sum(b["nodes"]) - 1), node < b["length"][:, None]


def _plain_tree(state):
    b, dim, kvh = state["b"], state["dim"], state["kv_heads"]
    group, n = state["heads"] // kvh, b["longest"]
    rows, real = _padded(b)
    q = state["q"].float().view(-1, kvh, group, dim)[rows].permute(0, 2, 3, 1, 4).flatten(2, 3)         # [seqs, kvh, group * n, dim]
    table = b["table"][b["slot"].long()].long()
    k, v = (t[table].permute(0, 2, 1, 3, 4).flatten(2, 3).float() for t in (state["keys"], state["values"]))   # [seqs, kvh, keys, dim]
    scores = (q @ k.transpose(2, 3)).view(len(b["nodes"]), kvh, group, n, -1) * state["scale"]
    j = torch.arange(k.shape[2], device=DEVICE)[None, :]
    past = (b["kv_len"] - b["length"]).long()[:, None]
    pos = b["pos"][rows].long()
    at = (j - past).clamp(0, n - 1)                                                                      # the node a key belongs to
    in_tree = (j >= past) & (j < b["kv_len"][:, None])
    seen = torch.gather(b["seen"], 2, at[:, None, :].expand(-1, n, -1)) & in_tree[:, None, :] | (j < past)[:, None, :]
    if state["window"]:
        key_pos = torch.where(in_tree, torch.gather(pos, 1, at), j)
        seen = seen & (key_pos[:, None, :] > pos[:, :, None] - state["window"])
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    o = (p.flatten(2, 3) @ v).view(len(b["nodes"]), kvh, group, n, dim) / p.sum(-1, keepdim=True).clamp(min=1e-38)
    return o.permute(0, 3, 1, 2, 4)[real].flatten(1).to(state["q"].dtype)


def _plain_accept(state):
    b, n = state["b"], state["b"]["longest"]
    rows, real = _padded(b)
    tokens, drawn = state["tokens"][rows], state["drawn"][rows]
    parent = b["parents"][rows].long()
    node = torch.arange(n, device=DEVICE)
    fits = real & (parent >= 0) & (tokens == torch.gather(drawn, 1, parent.clamp(min=0)))
    rival = (parent[:, :, None] == parent[:, None, :]) & fits[:, None, :] & (node[None, :] < node[:, None])  # a lower child that fits too
    fits = (fits & ~rival.any(2)) | (node == 0)
    taken = real & (~b["seen"] | fits[:, None, :]).all(2)
    count = taken.sum(1)
    path = torch.sort((~taken).to(torch.int8), dim=1, stable=True).indices
    inside = node < count[:, None]
    past = (b["kv_len"] - b["length"]).long()[:, None]
    table = b["table"][b["slot"].long()].long()
    # rows behind the accepted ones are copied onto themselves, what lies behind a sequence's last node is that node's row
    to = past + torch.minimum(node, b["length"].long()[:, None] - 1)
    source = torch.where(inside, past + path, to)
    to_page, from_page = torch.gather(table, 1, to // PAGE), torch.gather(table, 1, source // PAGE)
    to_off, from_off = to % PAGE, source % PAGE
    for store in (state["keys"], state["values"]):
        store[:, to_page, :, to_off] = store[:, from_page, :, from_off]
    return (count.int(), torch.where(inside, path, -1).int(), torch.where(inside, torch.gather(drawn, 1, path), -1).int(),
            state["keys"], state["values"])


def _plain_copy(state):
    source, target = (torch.tensor(t, device=DEVICE) for t in (state["source"], state["target"]))
    for store in (state["keys"], state["values"]):
        store[:, target] = store[:, source]
    return state["keys"], state["values"]


def _plain_logprobs(state):
    x = state["logits"].float()
    top = x.amax(1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    given = torch.gather(x, 1, state["tokens"].long()[:, None]) - lse
    entropy = lse - (e * x).sum(1, keepdim=True) / total
    # the largest first, the lowest index first among equals: one whole number says both
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -2 ** 31 - bits - 1, bits) * 2 ** 32 + (2 ** 31 - torch.arange(x.shape[1], device=DEVICE))
    ids = torch.topk(order, state["top"], dim=1).indices
    return given[:, 0], entropy[:, 0], torch.gather(x, 1, ids) - lse, ids.int()


def _plain_score(state):
    x = state["h"].float() @ state["head"].float().t()
    top = x.amax(1, keepdim=True)
    given = torch.gather(x, 1, state["tokens"].long()[:, None])
    e = (x - top).exp()
    total = e.sum(1, keepdim=True)
    lse = top + total.log()
    return (given - lse)[:, 0], (lse - (e * x).sum(1, keepdim=True) / total)[:, 0]


# ------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    return {"tree": _exact_tree, "accept": _exact_accept, "copy": _exact_copy, "logprobs": _exact_logprobs, "score": _exact_score}[state["kind"]](state)


def _place(b, s, j):
    """Page and offset of token ``j`` of sequence ``s``."""
    return int(b["table"][int(b["slot"][s]), j // PAGE]), j % PAGE


def _exact_tree(state):
    b, dim, kvh = state["b"], state["dim"], state["kv_heads"]
    group, out = state["heads"] // kvh, []
    for s, (n, past) in enumerate(zip(b["nodes"], b["past"])):
        first = int(b["starts"][s])
        pages = b["table"][int(b["slot"][s])].long()[:-(-(past + n) // PAGE)]
        k, v = (t[pages].transpose(0, 1).flatten(1, 2)[:, :past + n].double() for t in (state["keys"], state["values"]))
        pos = b["pos"][first:first + n].long()
        seen = torch.ones((n, past + n), dtype=torch.bool, device=DEVICE)
        for i in range(n):
            above, i_sees = i, set()
            while above >= 0:
                i_sees.add(above)
                above = b["parents_host"][s][above]
            seen[i, past:] = torch.tensor([m in i_sees for m in range(n)], device=DEVICE)
        if state["window"]:
            key_pos = torch.cat([torch.arange(past, device=DEVICE), pos])
            seen &= pos[:, None] - key_pos[None, :] < state["window"]
        q = state["q"][first:first + n].double().view(n, kvh, group, dim)
        w = torch.einsum("nhgd,hjd->hgnj", q, k) * state["scale"]
        w = torch.softmax(w.masked_fill(~seen, -math.inf), -1)
        out.append(torch.einsum("hgnj,hjd->nhgd", w, v).flatten(1))
    return torch.cat(out)


def _exact_accept(state):
    b = state["b"]
    seqs, longest = len(b["nodes"]), b["longest"]
    tokens, drawn = state["tokens"].tolist(), state["drawn"].tolist()
    count, path, taken = [], [[-1] * longest for _ in range(seqs)], [[-1] * longest for _ in range(seqs)]
    keys, values = state["keys"].clone(), state["values"].clone()
    for s, n in enumerate(b["nodes"]):
        first, at, walked = int(b["starts"][s]), 0, []
        while at is not None:
            walked.append(at)
            below = [c for c in range(n) if b["parents_host"][s][c] == at and tokens[first + c] == drawn[first + at]]
            at = below[0] if below else None
        count.append(len(walked))
        for i, node in enumerate(walked):
            path[s][i], taken[s][i] = node, drawn[first + node]
            (page, off), (to_page, to_off) = _place(b, s, b["past"][s] + node), _place(b, s, b["past"][s] + i)
            keys[:, to_page, :, to_off] = state["keys"][:, page, :, off]
            values[:, to_page, :, to_off] = state["values"][:, page, :, off]
    return _ints(count), _ints(path), _ints(taken), keys, values


def _exact_copy(state):
    keys, values = state["keys"].clone(), state["values"].clone()
    for a, c in zip(state["source"], state["target"]):
        keys[:, c], values[:, c] = state["keys"][:, a], state["values"][:, a]
    return keys, values


def _exact_rows(x, tokens, top):
    p = torch.log_softmax(x.double(), 1)
    order = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :top]
    given = p[torch.arange(len(x), device=DEVICE), tokens.long()]
    return given, -(p.exp() * p).sum(1), p.gather(1, order), order.int()


def _exact_logprobs(state):
    parts = [_exact_rows(x, t, state["top"]) for x, t in zip(state["logits"].split(64), state["tokens"].split(64))]
    return tuple(torch.cat(c) for c in zip(*parts))


def _exact_score(state):
    head = state["head"].double()
    parts = [_exact_rows(h.double() @ head.t(), t, 0)[:2] for h, t in zip(state["h"].split(256), state["tokens"].split(256))]
    return tuple(torch.cat(c) for c in zip(*parts))
