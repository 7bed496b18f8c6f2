"""Accepted drafts' cache rows and copied pages: exact moves, compared bit by bit with the same done one row at a time."""

import numpy as np
import pytest
import torch

from starter_b200 import ops
from starter_b200.cache import KVNeed, SequenceCache, StateNeed
from starter_b200.ops import KernelError

pytestmark = pytest.mark.gpu

PAGE = 64


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Step:
    """Trees of ``nodes`` behind ``past`` tokens in scattered pages; tokens from a small vocabulary, so that siblings collide."""

    def __init__(self, nodes, past, entries=3, kv_heads=2, dims=(32, 32), dtype=torch.bfloat16, vocab=4, seed=0, flat=False):
        rng = np.random.default_rng(seed)
        self.nodes, self.past = nodes, past
        held = [-(-(p + n) // PAGE) for p, n in zip(past, nodes)]
        self.pages = sum(held) + 1
        order, at = rng.permutation(self.pages), 0
        self.table = np.zeros((len(nodes) + 1, max(held + [1])), dtype=np.int32)
        self.slots = rng.permutation(len(nodes) + 1)[:len(nodes)].tolist()
        for slot, h in zip(self.slots, held):
            self.table[slot, :h] = order[at:at + h]
            at += h
        self.parents = [[-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)] if n else [] for n in nodes]
        self.tokens = [rng.integers(0, vocab, n).tolist() for n in nodes]
        self.drawn = [rng.integers(0, vocab, n).tolist() for n in nodes]
        self.starts = np.concatenate([[0], np.cumsum(nodes)]).astype(int).tolist()
        g = torch.Generator().manual_seed(seed)
        shape = ((entries,) if not flat else ()) + (self.pages, kv_heads, PAGE)
        self.keys, self.values = (torch.randint(-99, 99, shape + (d,), generator=g).to(dtype) for d in dims)

    def run(self, more=()):
        stores = [(self.keys.cuda(), self.values.cuda())] + [(k.cuda(), v.cuda()) for k, v in more]
        flat = lambda lists: ints([x for part in lists for x in part])  # noqa: E731
        out = ops.cache_accept(stores, torch.from_numpy(self.table).cuda(), ints(self.slots), ints(self.starts[:-1]), ints(self.nodes),
                               ints([p + n for p, n in zip(self.past, self.nodes)]), flat(self.tokens), flat(self.parents), flat(self.drawn),
                               max_q_len=max(self.nodes + [1]))
        return [t.cpu() for t in out], [(k.cpu(), v.cpu()) for k, v in stores]

    def ways(self):
        for n, parents, tokens, drawn in zip(self.nodes, self.parents, self.tokens, self.drawn):
            way, at = [], 0 if n else None
            while at is not None:
                way.append(at)
                at = next((c for c in range(at + 1, n) if parents[c] == at and tokens[c] == drawn[at]), None)
            yield way

    def moved(self, t):
        """The rows of ``t`` moved one by one, from a copy."""
        out = t.clone()
        for s, way in enumerate(self.ways()):
            for i, node in enumerate(way):
                src, dst = self.past[s] + node, self.past[s] + i
                a, b = int(self.table[self.slots[s], src // PAGE]), int(self.table[self.slots[s], dst // PAGE])
                out[..., b, :, dst % PAGE, :] = t[..., a, :, src % PAGE, :]
        return out

    def check(self, more=()):
        (count, path, taken), stores = self.run(more)
        width = max(self.nodes + [1])
        for s, way in enumerate(self.ways()):
            drawn = [self.drawn[s][i] for i in way]
            assert count[s] == len(way)
            assert path[s].tolist() == way + [-1] * (width - len(way)) and taken[s].tolist() == drawn + [-1] * (width - len(way))
        for (k, v), (k0, v0) in zip(stores, [(self.keys, self.values)] + list(more)):
            assert torch.equal(k, self.moved(k0)) and torch.equal(v, self.moved(v0))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("vocab", [1, 2, 4])
def test_walks_and_moves(seed, vocab):
    Step([1, 30, 64, 7, 0, 100], [0, 63, 10, 64, 5, 200], vocab=vocab, seed=seed).check()


@pytest.mark.parametrize("nodes", [1, 2, 127, 128, 129, 256])
def test_chains_that_are_taken_whole_or_cut(nodes):
    s = Step([nodes, nodes], [61, 640], seed=nodes)
    s.parents = [[-1] + list(range(nodes - 1))] * 2
    s.tokens = [list(range(nodes))] * 2
    s.drawn = [list(range(1, nodes)) + [5], [7] * nodes]
    s.check()


@pytest.mark.parametrize("dtype, dims", [(torch.float32, (16, 48)), (torch.bfloat16, (128, 64)), (torch.bfloat16, (6, 2)), (torch.float32, (1, 3)),
                                         (torch.bfloat16, (256, 256)), (torch.float32, (256, 200))])
def test_sizes_of_rows(dtype, dims):
    Step([40, 17], [100, 30], dims=dims, dtype=dtype, vocab=2, seed=3).check()


def test_one_entry_and_several_groups():
    Step([40, 17], [100, 30], flat=True, vocab=2, seed=4).check()
    s = Step([40, 17], [100, 30], vocab=2, seed=4)
    t = Step([40, 17], [100, 30], entries=1, kv_heads=5, dims=(16, 24), dtype=torch.float32, seed=4)
    s.check(more=[(t.keys, t.values)])


def test_many_entries_and_sequences():
    Step([12] * 33, [3 * i for i in range(33)], entries=20, kv_heads=4, vocab=2, seed=5).check()


def test_nodes_that_hang_on_nothing_are_nobodys_children():
    s = Step([8], [50], vocab=1, seed=6)
    s.parents = [[-1, -1, 5, 0, 4, 99, -7, 3]]         # 1, 2, 4, 5 and 6 name no node in front of themselves
    s.tokens = s.drawn = [[0] * 8]
    (count, path, _), _ = s.run()
    assert count.tolist() == [3] and path[0].tolist() == [0, 3, 7, -1, -1, -1, -1, -1]


def test_accept_captured_and_replayed():
    s = Step([20, 33], [100, 7], vocab=2, seed=7)
    keys, values = s.keys.cuda(), s.values.cuda()
    flat = lambda lists: ints([x for part in lists for x in part])  # noqa: E731
    args = ([(keys, values)], torch.from_numpy(s.table).cuda(), ints(s.slots), ints(s.starts[:-1]), ints(s.nodes),
            ints([p + n for p, n in zip(s.past, s.nodes)]), flat(s.tokens), flat(s.parents), flat(s.drawn))
    ops.cache_accept(*args, max_q_len=33)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        count, path, taken = ops.cache_accept(*args, max_q_len=33)
    other = Step([20, 33], [100, 7], vocab=2, seed=70)
    keys.copy_(s.keys), values.copy_(s.values)
    args[8].copy_(flat(other.drawn))
    s.drawn = other.drawn
    graph.replay()
    assert torch.equal(keys.cpu(), s.moved(s.keys)) and torch.equal(values.cpu(), s.moved(s.values))
    assert count.tolist() == [len(w) for w in s.ways()]


def test_accepted_rows_past_two_to_the_31_entries():
    """Pages and entries of a store whose offsets pass 2^31 entries."""
    s = Step([20, 9], [100, 30], entries=2, kv_heads=8, dims=(128, 128), vocab=2, seed=8)
    shift = 2 ** 30 // (8 * PAGE * 128) + 5
    wide = [torch.empty((2, shift + s.pages, 8, PAGE, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for w, t in zip(wide, (s.keys, s.values)):
        w[:, shift:] = t.cuda()
    flat = lambda lists: ints([x for part in lists for x in part])  # noqa: E731
    ops.cache_accept([tuple(wide)], torch.from_numpy(s.table).cuda() + shift, ints(s.slots), ints(s.starts[:-1]), ints(s.nodes),
                     ints([p + n for p, n in zip(s.past, s.nodes)]), flat(s.tokens), flat(s.parents), flat(s.drawn), max_q_len=20)
    for w, t in zip(wide, (s.keys, s.values)):
        assert torch.equal(w[:, shift:].cpu(), s.moved(t))
    before = wide[0][:, shift + 1].clone()
    ops.cache_copy_pages([wide[0]], [shift + 1], [shift])
    assert torch.equal(wide[0][:, shift], before) and torch.equal(wide[0][:, shift + 1], before)


def test_accept_where_new_memory_has_to_be_filled():
    """Deterministic algorithms fill what is allocated: the results are separate tensors then, with the same contents."""
    was = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        Step([20, 33], [100, 7], vocab=2, seed=7).check()
    finally:
        torch.use_deterministic_algorithms(was)


def test_accept_refusals():
    s = Step([8], [50])
    k, v = s.keys.cuda(), s.values.cuda()
    i = ints([0] * 8)
    one = ints([0])
    good = dict(stores=[(k, v)], block_table=one[None], seq_slot=one, seq_q_start=one, seq_q_len=ints([8]), seq_kv_len=ints([58]), tokens=i,
                parents=i, drawn=i, max_q_len=8)
    for change in (dict(max_q_len=0), dict(max_q_len=257), dict(stores=[]), dict(stores=[(k, v[:, :1])]), dict(stores=[(k, v[:2])]),
                   dict(stores=[(k[0, 0], v[0, 0])]), dict(parents=i[:-1]), dict(drawn=i.long()), dict(seq_q_len=ints([8, 8])),
                   dict(stores=[(k[..., :31].contiguous(), v)]), dict(stores=[(k.cpu(), v.cpu())])):
        with pytest.raises(KernelError):
            ops.cache_accept(**{**good, **change})


# ------------------------------------------------------------------------------------------ copies

@pytest.mark.parametrize("dtype, tail", [(torch.bfloat16, (2, 64, 128)), (torch.float32, (1, 64, 24)), (torch.uint8, (7,)), (torch.int32, (3, 5)),
                                         (torch.bfloat16, (3,)), (torch.float32, (64, 4096))])
@pytest.mark.parametrize("dim", [0, 1])
def test_copies_are_exact_and_touch_nothing_else(dtype, tail, dim):
    g = torch.Generator().manual_seed(1)
    a = torch.randint(0, 200, ((3, 20) if dim else (20,)) + tail, generator=g).to(dtype)
    b = torch.randint(0, 200, ((5, 23) if dim else (23,)) + (9,), generator=g).to(dtype)
    source, target = [4, 4, 0, 19], [7, 1, 18, 5]
    da, db = a.cuda(), b.cuda()
    ops.cache_copy_pages([da, db], source, target, dim=dim)
    for t in (a, b):
        for s, d in zip(source, target):
            if dim:
                t[:, d] = t[:, s]
            else:
                t[d] = t[s]
    assert torch.equal(da.cpu(), a) and torch.equal(db.cpu(), b)


def test_more_pairs_and_tensors_than_a_launch_takes():
    tensors = [torch.randn((2, 700, 1 + n % 3), device="cuda") for n in range(19)]
    want = [t.clone() for t in tensors]
    order = np.random.default_rng(0).permutation(700).tolist()
    source, target = order[:350], order[350:]
    ops.cache_copy_pages(tensors, source, target)
    for t, w in zip(tensors, want):
        w[:, target] = w[:, source]
        assert torch.equal(t, w)


def test_copy_refusals():
    t = torch.zeros((2, 5, 4), device="cuda")
    for stores, source, target in (([t], [0], [5]), ([t], [-1], [1]), ([t[:, :, :3]], [0], [1]), ([t, t[:, :3].contiguous()], [0], [4]), ([t[0, 0]], [0], [1])):
        with pytest.raises(KernelError):
            ops.cache_copy_pages(stores, source, target)
    ops.cache_copy_pages([t], [], [])


def test_a_forked_cache_on_the_device():
    kv = {0: KVNeed(2, 16), 1: KVNeed(2, 16), 2: KVNeed(1, 8, value_dim=24)}
    c = SequenceCache(kv, {0: StateNeed((3,)), 1: StateNeed((2, 5), "bfloat16")}, 64 * 12, 6, torch.bfloat16, "cuda")
    slot = c.open_sequence()
    c.reserve(slot, 100)
    c.advance(slot, 100)
    for t in c.keys + c.values + list(c.state.values()):
        t.copy_(torch.randn(t.shape))
    new = c.fork(slot, 3)
    c.sync_table()
    for s in new:
        assert c.block_table[s, :2].tolist() == c.owned_pages(s)
        for t in c.keys + c.values:
            assert torch.equal(t[:, c.owned_pages(s)], t[:, c.owned_pages(slot)])
        for t in c.state.values():
            assert torch.equal(t[s], t[slot])
    c.check()
