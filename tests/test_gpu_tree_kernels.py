"""Tree attention on each of its kernels by name, with keys whole and in parts: the cases that a step's size alone would send to one of them only."""

import math
import threading

import pytest
import torch

from starter_b200 import ops
from test_gpu_tree_attention import PAGE, Case, bush, chain, check, depth_of, sees_of, trees

pytestmark = pytest.mark.gpu

#: kernel, type, head size, parts
FORMS = [("plain", "fp32", 64, 1), ("plain", "fp32", 128, 4), ("plain", "bf16", 80, 3), ("plain", "bf16", 7, 1),
         ("mma", "bf16", 32, (1, 1)), ("mma", "bf16", 64, (2, 4)), ("mma", "bf16", 128, (2, 1)), ("mma", "bf16", 128, (1, 8)),
         ("tcgen05", "bf16", 64, 1), ("tcgen05", "bf16", 64, 4), ("tcgen05", "bf16", 128, 1), ("tcgen05", "bf16", 128, 2), ("tcgen05", "bf16", 128, 8)]
every_kernel = pytest.mark.parametrize("kernel, dtype, dim, parts", FORMS, ids=lambda v: str(v).replace(" ", ""))


def run(case, kernel, parts, **more):
    return ops.attention_tree(**{**case.on_device(), "kernel": kernel, "parts": parts, **more})


def spoil(case, seq, place, what, column=2, kv_head=0, which="v"):
    """Put what is no number at a place of a sequence's values (or keys)."""
    getattr(case, which)[int(case.table[case.slots[seq], place // PAGE]), kv_head, place % PAGE, column] = what


def check_finite(case, got):
    """Numbers within the bound, and none where a row sees a value that is none."""
    want, tol = case.want()
    got = got.double().cpu()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), f"first at {(torch.isfinite(got) != fine).nonzero()[0].tolist()}"
    assert ((got - want).abs()[fine] <= tol[fine]).all()


@every_kernel
@pytest.mark.parametrize("words", [2, 8, 9, 11])
def test_masks_wider_than_a_tree(kernel, dtype, dim, parts, words):
    """Words behind those that the nodes need, whatever their bits say."""
    sees, depth = trees([13, 40], seed=words)
    case = Case(dtype, 4, 2, dim, sees, [70, 131], depth, seed=words, words=words)
    case.mask[:, 2:] = -1
    check(case, run(case, kernel, parts))


@every_kernel
@pytest.mark.parametrize("nodes", [9, 40, 64])
def test_values_that_are_no_numbers(kernel, dtype, dim, parts, nodes):
    """In what is cached (every row sees them), at the root, and at leaves that one row each sees: with 40 nodes of 4 heads the last of them lie in
    the second tile of 128 rows alone."""
    parents = [-1] + [0] * (nodes - 1)
    for what, places in ((math.nan, [100 + 5]), (math.inf, [100 + nodes - 1]), (math.nan, [100 + 5, 100 + nodes - 2]), (-math.inf, [100, 100 + 7]),
                         (math.nan, [99]), (math.inf, [3, 100 + nodes - 1])):
        case = Case(dtype, 4, 1, dim, [sees_of(parents)], [100], [depth_of(parents)], seed=nodes)
        for n, place in enumerate(places):
            spoil(case, 0, place, what, column=(2 + 3 * n) % dim)
        check_finite(case, run(case, kernel, parts))


@every_kernel
def test_values_that_are_no_numbers_behind_weights_that_round_to_zero(kernel, dtype, dim, parts):
    """A weight is never zero in the formula: a row sees such a value however far its score lies below the row's largest."""
    for what, place in ((math.nan, 70 + 20), (math.inf, 70), (math.nan, 66), (-math.inf, 5)):
        parents = [-1] + [0] * 39
        case = Case(dtype, 4, 1, dim, [sees_of(parents)], [70], [depth_of(parents)], seed=place, spread=60.0)
        spoil(case, 0, place, what, column=3 % dim)
        check_finite(case, run(case, kernel, parts))


@pytest.mark.parametrize("dim, parts", [(64, 1), (128, 1), (128, 4)])
def test_both_tiles_know_of_values_that_are_no_numbers_in_every_run(dim, parts):
    """Both tiles' warps take the same values out of the shared tile; whoever comes second finds zeros."""
    parents = [-1] + [0] * 63
    case = Case("bf16", 8, 2, dim, [sees_of(parents)] * 5, [100, 61, 1, 400, 127], [depth_of(parents)] * 5, seed=dim)
    for seq, past in enumerate(case.past):
        for place in range(past, past + 64, 3):
            spoil(case, seq, place, math.nan, column=place % dim, kv_head=seq % 2)
    args = case.on_device()
    first = ops.attention_tree(**args, kernel="tcgen05", parts=parts)
    check_finite(case, first)
    for _ in range(200):
        assert torch.equal(ops.attention_tree(**args, kernel="tcgen05", parts=parts).isnan(), first.isnan())


def test_stores_of_unequal_page_counts_are_refused():
    """One table numbers the pages of both: a store with fewer would be read behind its end."""
    sees, depth = trees([5])
    good = Case("bf16", 4, 2, 64, sees, [100], depth).on_device()
    for which in ("k_store", "v_store"):
        for other in (good[which][:-1].contiguous(), torch.cat([good[which], good[which][:1]])):
            with pytest.raises(ops.KernelError, match="pages of keys"):
                ops.attention_tree(**{**good, which: other})
