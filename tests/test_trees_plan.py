"""Drafted trees, forks and what the operators around them refuse, as far as no GPU is needed."""

import numpy as np
import pytest
import torch

from starter_b200 import ops
from starter_b200.cache import CacheFull, KVNeed, SequenceCache, StateNeed
from starter_b200.engine.batch import TREE_MAX_NODES, TreeEntry, plan_step, plan_trees
from starter_b200.ops import KernelError


def test_a_tree_becomes_positions_places_and_masks():
    parents = [-1, 0, 0, 1, 3, 2]
    a = plan_trees([TreeEntry(3, [9, 8, 7, 6, 5, 4], parents), TreeEntry(1, [2], [-1])], [100, 7])
    assert a["tok_pos"].tolist() == [100, 101, 101, 102, 103, 102, 7]
    assert a["tok_place"].tolist() == [100, 101, 102, 103, 104, 105, 7]
    assert a["tree_mask"].tolist() == [1, 0b11, 0b101, 0b1011, 0b11011, 0b100101, 1]
    assert a["parents"].tolist() == parents + [-1] and a["want_rows"].tolist() == list(range(7))
    assert a["seq_kv_len"].tolist() == [106, 8] and a["seq_q_len"].tolist() == [6, 1]


def test_masks_of_many_nodes_take_several_words():
    n = 70
    a = plan_trees([TreeEntry(0, list(range(n)), [-1] + list(range(n - 1)))], [0])
    masks = a["tree_mask"].reshape(n, 3).view(np.uint32)
    for i in range(n):
        bits = sum(int(w) << (32 * k) for k, w in enumerate(masks[i]))
        assert bits == (1 << (i + 1)) - 1


@pytest.mark.parametrize("tokens, parents", [
    ([1, 2], [-1]), ([1, 2], [0, 0]), ([1, 2], [-1, 1]), ([1, 2, 3], [-1, 2, 0]), ([1, 2], [-1, -1]), ([], []),
    ([0] * (TREE_MAX_NODES + 1), [-1] + [0] * TREE_MAX_NODES)])
def test_what_is_no_tree_is_refused(tokens, parents):
    with pytest.raises(ValueError):
        plan_trees([TreeEntry(0, tokens, parents)], [5])


def test_a_tree_outside_the_vocabulary_or_given_twice_is_refused():
    with pytest.raises(ValueError):
        plan_trees([TreeEntry(0, [99], [-1])], [5], vocab_size=50)
    with pytest.raises(ValueError):
        plan_trees([TreeEntry(0, [9], [-1]), TreeEntry(0, [9], [-1])], [5, 5])


def test_plan_step_is_what_it_was():
    a = plan_step([TreeEntry(2, [4, 5], [-1, 0])], [10])
    assert "tree_mask" not in a and a["tok_pos"].tolist() == [10, 11]


def test_the_limits_of_the_plan_and_of_the_kernels_agree():
    assert TREE_MAX_NODES == ops.TREE_MAX_NODES


# ------------------------------------------------------------------------------------------ forks

def make_cache(state=False, tokens=64 * 12, seqs=6):
    kv = {0: KVNeed(2, 16), 1: KVNeed(2, 16), 2: KVNeed(1, 8, value_dim=24)}
    return SequenceCache(kv, {0: StateNeed((3,)) if state else None}, tokens, seqs, torch.float32, "cpu")


def grown(cache, tokens):
    slot = cache.open_sequence()
    cache.reserve(slot, tokens)
    cache.advance(slot, tokens)
    for t in cache.keys + cache.values:
        t[:, cache.owned_pages(slot)] = torch.randn(t[:, cache.owned_pages(slot)].shape)
    return slot


@pytest.mark.parametrize("tokens", [1, 63, 64, 65, 128, 150])
def test_a_fork_shares_full_pages_and_copies_the_last(tokens):
    c = make_cache()
    slot = grown(c, tokens)
    free = c.pages.free_count
    new = c.fork(slot, 2)
    assert free - c.pages.free_count == (2 if tokens % 64 else 0)
    whole = tokens // 64
    for s in new:
        assert c.lengths[s] == tokens and c.owned_pages(s)[:whole] == c.owned_pages(slot)[:whole]
        for t in c.keys + c.values:
            assert torch.equal(t[:, c.owned_pages(s)], t[:, c.owned_pages(slot)])
    if tokens % 64:
        last = {c.owned_pages(s)[whole] for s in [slot] + new}
        assert len(last) == 3
    c.check()
    c.sync_table()
    for s in new:
        assert c.block_table[s, :len(c.owned_pages(s))].tolist() == c.owned_pages(s)
    # in any order of closing, every page goes back once and the others stay
    c.close_sequence(slot)
    c.check()
    c.reserve(new[0], tokens + 64)
    c.advance(new[0], 64)
    again = c.fork(new[0], 1)[0]
    c.check()
    for s in (new[1], again, new[0]):
        c.close_sequence(s)
        c.check()
    assert c.pages.held_count == 0 and c.slots.held_count == 0 and not c._holders


def test_a_fork_of_a_beginning():
    c = make_cache()
    slot = grown(c, 150)
    new = c.fork(slot, 1, length=70)[0]
    assert c.lengths[new] == 70 and len(c.owned_pages(new)) == 2 and c.owned_pages(new)[0] == c.owned_pages(slot)[0]
    empty = c.fork(slot, 1, length=0)[0]
    assert c.lengths[empty] == 0 and c.owned_pages(empty) == []
    c.check()
    with pytest.raises(ValueError):
        c.shorten(slot, 10)                    # its first page is shared
    c.shorten(slot, 64)
    c.shorten(new, 65)
    assert c.lengths[slot] == 64 and c.lengths[new] == 65


def test_forks_that_cannot_be():
    c = make_cache()
    slot = grown(c, 100)
    for bad in (dict(slot=5), dict(slot=slot, count=0), dict(slot=slot, length=101), dict(slot=slot, length=-1)):
        with pytest.raises(ValueError):
            c.fork(**bad)
    with pytest.raises(CacheFull):
        c.fork(slot, 6)                        # five slots are left
    grown(c, 64 * 8)                           # two pages are left
    free = (c.slots.free_count, c.pages.free_count)
    with pytest.raises(CacheFull):
        c.fork(slot, 3)
    assert (c.slots.free_count, c.pages.free_count) == free and not c._holders
    c.check()
    with pytest.raises(ValueError):
        c.shorten(slot, 101)
    with pytest.raises(ValueError):
        c.shorten(5, 0)


def test_a_fork_whose_copy_fails_changes_nothing(monkeypatch):
    c = make_cache(state=True)
    slot = grown(c, 70)
    free = (c.slots.free_count, c.pages.free_count)

    def broken(tensors, source, target, dim):
        raise RuntimeError("no")

    monkeypatch.setattr(c, "_copy_items", broken)
    with pytest.raises(RuntimeError):
        c.fork(slot, 2)
    assert (c.slots.free_count, c.pages.free_count) == free and not c._holders and c.lengths[slot] == 70
    c.check()


def test_a_state_is_copied_and_does_not_go_back():
    c = make_cache(state=True)
    slot = grown(c, 70)
    c.state[0][slot] = torch.tensor([1.0, 2.0, 3.0])
    new = c.fork(slot, 2)
    for s in new:
        assert c.state[0][s].tolist() == [1.0, 2.0, 3.0]
    with pytest.raises(ValueError):
        c.fork(slot, 1, length=64)
    with pytest.raises(ValueError):
        c.shorten(slot, 64)
    c.shorten(slot, 70)


# ------------------------------------------------------------------------------------------ refusals

def test_operands_on_the_host_are_refused():
    i = torch.zeros(1, dtype=torch.int32)
    store = torch.zeros((2, 1, 64, 16))
    with pytest.raises(KernelError, match="no CPU implementation"):
        ops.attention_tree(torch.zeros((1, 16)), store, store, i[None], i, i, i, i, i, i[None], 1, 1, 16, 0.25)
    with pytest.raises(KernelError, match="no CPU implementation"):
        ops.cache_accept([(store, store)], i[None], i, i, i, i, i, i, i, max_q_len=1)
    with pytest.raises(KernelError, match="no CPU implementation"):
        ops.cache_copy_pages([store], [0], [1], dim=0)
    with pytest.raises(KernelError, match="no CPU implementation"):
        ops.token_logprobs(torch.zeros((1, 5)), i)
    with pytest.raises(KernelError, match="no CPU implementation"):
        ops.linear_logprobs(torch.zeros((1, 8)), torch.zeros((5, 8)), i)


@pytest.mark.parametrize("source, target", [([0], [1, 2]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3])])
def test_copies_whose_order_would_matter_are_refused(source, target):
    with pytest.raises(KernelError):
        ops.cache_copy_pages([], source, target)


def test_copies_count_pages_by_the_first_or_second_dimension():
    with pytest.raises(KernelError):
        ops.cache_copy_pages([], [0], [1], dim=2)
