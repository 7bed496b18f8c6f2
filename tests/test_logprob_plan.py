"""How rows of logits are dealt to blocks, against what the launcher behind it takes (no GPU needed)."""

import pytest

from starter_b200 import ops

TILE = 16384
MOST_TILES = 160      # whose groups a block's shared memory holds
MOST_PARTS = 8        # blocks of a cluster


def launched_tiles(vocab, item, parts):
    """Tiles of the block with the most of them, for a row that may begin anywhere between two 32-byte boundaries (csrc/token_logprobs.cu, lp_slots)."""
    entries = TILE // item
    tiles = (vocab + 31 // item + entries - 1) // entries
    return -(-tiles // parts)


def lengths(item):
    longest = 4 * ops.LOGPROBS_MAX_VOCAB // item
    full = MOST_TILES * TILE // item
    for parts in (1, 2, 4, 8):
        for less in (0, 1, 31 // item - 1, 31 // item, 31 // item + 1, 32 // item, 33, 4096):
            for vocab in (parts * full - less, parts * full + less):
                if vocab <= longest:
                    yield vocab
    yield from (longest, longest - 1, 151936, 1)


@pytest.mark.parametrize("item", [2, 4])
@pytest.mark.parametrize("rows", [1, 2, 37, 74, 75, 148, 150, 296, 300, 592, 593, 600, 889, 1184])
def test_rows_with_alternatives_fit_what_a_block_holds(item, rows):
    for vocab in lengths(item):
        whole, parts = ops._logprob_plan(rows, vocab * item)
        assert parts in (1, 2, 4, 8) and 0 <= whole <= rows
        if whole < rows:
            assert launched_tiles(vocab, item, parts) <= MOST_TILES, (rows, vocab, parts)
        if whole:
            assert launched_tiles(vocab, item, 1) <= MOST_TILES, (rows, vocab)


@pytest.mark.parametrize("item", [2, 4])
@pytest.mark.parametrize("rows", [1, 2, 75, 300, 592, 600])
def test_rows_of_any_length_without_alternatives_have_a_plan(item, rows):
    for vocab in (5_242_848, 5_242_881, 10_485_761, 20_000_000, 2 ** 30):
        whole, parts = ops._logprob_plan(rows, vocab * item, False)
        assert parts in (1, 2, 4, 8) and parts <= MOST_PARTS and 0 <= whole <= rows
