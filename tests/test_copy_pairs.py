"""Which pairs of pages a copy refuses, whatever holds the numbers (no GPU needed: nothing is copied)."""

import numpy as np
import pytest
import torch

from starter_b200 import ops
from starter_b200.ops import KernelError

HOLDERS = [list, tuple, np.array, torch.tensor]


@pytest.mark.parametrize("held", HOLDERS, ids=lambda h: h.__name__)
@pytest.mark.parametrize("source, target", [([0, 1], [5, 5]), ([3, 4], [7, 3]), ([2], [2]), ([1, 2, 3], [4, 5, 4]), ([0, 1], [2]), ([0], [2, 3])])
def test_pairs_that_meet_are_refused(held, source, target):
    with pytest.raises(KernelError):
        ops.cache_copy_pages([], held(source), held(target))


@pytest.mark.parametrize("held", HOLDERS, ids=lambda h: h.__name__)
def test_pairs_that_do_not_meet_are_taken(held):
    ops.cache_copy_pages([], held([0, 0, 1, 9]), held([5, 6, 7, 8]))
    ops.cache_copy_pages([], held([]), held([]))


@pytest.mark.parametrize("source, target", [([0.5], [1]), ([0], [1.0]), (["0"], [1]), ([0], [1 << 40]), (None, [1]), ([0], None), (0, 1)])
def test_what_are_no_pages_is_refused(source, target):
    with pytest.raises(KernelError):
        ops.cache_copy_pages([], source, target)
