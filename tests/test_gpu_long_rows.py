"""Log probabilities of rows whose length is at an edge of what a block, a cluster or the alternatives take."""

import pytest
import torch

from starter_b200 import ops
from test_gpu_logprobs import expected, logits, near

pytestmark = pytest.mark.gpu


def check_rows(x, t, top, step=50):
    """Against 64 bits, some rows at a time; a thread adds up to a block's share of a row, with half a step of 2^-24 each (``expected`` counts 2,600)."""
    given, entropy, values, ids = ops.token_logprobs(x, t, top=top)
    more = x.shape[1] / 256 * 2.0 ** -24
    for at in range(0, x.shape[0], step):
        rows = slice(at, at + step)
        w_given, w_entropy, w_values, w_ids, rel, tol_h = expected(x[rows], t[rows], top)
        rel = rel + more
        near(given[rows], w_given, rel)
        near(entropy[rows], w_entropy, tol_h + more * (1 + 2 * w_entropy.abs()))
        near(values[rows], w_values, rel[:, None].expand_as(w_values))
        assert torch.equal(ids[rows], w_ids)


@pytest.mark.parametrize("dtype, rows, vocab", [(torch.float32, 300, 655_360), (torch.float32, 300, 655_354), (torch.float32, 150, 1_310_720),
                                                (torch.float32, 75, 2_621_440), (torch.bfloat16, 300, 1_310_720), (torch.float32, 2, 5_242_848)])
def test_alternatives_where_a_block_has_as_many_tiles_as_it_holds(dtype, rows, vocab):
    x, t = logits(rows, vocab, vocab, dtype)
    check_rows(x, t, 3)


@pytest.mark.parametrize("dtype, rows, vocab", [(torch.float32, 2, 5_300_000), (torch.float32, 40, 5_242_900), (torch.bfloat16, 2, 10_600_001)])
def test_rows_longer_than_alternatives_take(dtype, rows, vocab):
    check_rows(*logits(rows, vocab, vocab, dtype), 0)
