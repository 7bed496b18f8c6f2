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


# ------------------------------------------------------------------------------------------ what the tests of the chosen kernel ask, of every kernel

@every_kernel
def test_masks_of_any_kind(kernel, dtype, dim, parts):
    """Rows that see nothing, rows that see what comes later, sequences of which nobody sees anything; 45 nodes of 4 heads are two tiles of 128 rows."""
    g = torch.Generator().manual_seed(5)
    n = 45
    any_mask = torch.rand((n, n), generator=g) < 0.3
    any_mask[[7, 40, 44]] = False
    any_mask[8] = True
    for past in (0, 77):
        check(case := Case(dtype, 4, 1, dim, [any_mask, torch.zeros((3, 3), dtype=torch.bool)], [past, 0], [[0] * n, [0, 1, 2]], seed=past),
              run(case, kernel, parts))


@every_kernel
def test_nobody_sees_anything(kernel, dtype, dim, parts):
    case = Case(dtype, 4, 1, dim, [torch.zeros((n, n), dtype=torch.bool) for n in (40, 1)], [0, 0], [[0] * 40, [0]], seed=1)
    assert not run(case, kernel, parts).any()


@every_kernel
@pytest.mark.parametrize("window", [1, 3, 64, 100, 10000])
def test_windows(kernel, dtype, dim, parts, window):
    sees, depth = trees([40, 64, 1], seed=window)
    check(case := Case(dtype, 4, 1, dim, sees, [150, 0, 300], depth, window=window, seed=window), run(case, kernel, parts))
    parents = chain(50)
    check(case := Case(dtype, 8, 2, dim, [sees_of(parents)], [130], [depth_of(parents)], window=window, seed=window), run(case, kernel, parts))


@every_kernel
def test_sequences_without_nodes(kernel, dtype, dim, parts):
    sees, depth = trees([0, 9, 0, 70, 0], seed=1)
    check(case := Case(dtype, 4, 2, dim, sees, [0, 100, 64, 5, 10], depth, seed=1), run(case, kernel, parts))


@every_kernel
@pytest.mark.parametrize("nodes", [6, 70])
def test_sharp_scores(kernel, dtype, dim, parts, nodes):
    """Maxima that grow along the keys: what has been added up is scaled down many times."""
    sees, depth = trees([nodes], seed=3)
    case = Case(dtype, 8, 2, dim, sees, [333], depth, seed=3, spread=30.0)
    grow = torch.linspace(0.05, 1.5, 333 + nodes)
    for j in range(333 + nodes):
        case.k[int(case.table[case.slots[0], j // PAGE]), :, j % PAGE] *= grow[j]
    check(case, run(case, kernel, parts))


@every_kernel
@pytest.mark.parametrize("nodes", [9, 40])
def test_keys_that_are_no_numbers(kernel, dtype, dim, parts, nodes):
    """A score that is no number makes its row none, and no other row."""
    parents = [-1] + [0] * (nodes - 1)
    for spoiled in (3, nodes - 1):
        case = Case(dtype, 4, 1, dim, [sees_of(parents)], [100], [depth_of(parents)], seed=nodes)
        spoil(case, 0, 100 + spoiled, math.nan, which="k")
        got = run(case, kernel, parts).cpu().double()
        want, tol = case.want()
        others = [i for i in range(nodes) if i != spoiled]
        assert got[spoiled].isnan().all() and ((got - want).abs() <= tol)[others].all()


@every_kernel
def test_captured_and_replayed_in_turn(kernel, dtype, dim, parts):
    """Two graphs of one step, replayed on another stream behind one another, and a call outside of them."""
    sees, depth = trees([40, 13], seed=8)
    case = Case(dtype, 8, 2, dim, sees, [300, 900], depth, seed=8)
    args = {**case.on_device(), "kernel": kernel, "parts": parts}
    ops.attention_tree(**args)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attention_tree(**args)
        graphs.append((graph, out))
    other = Case(dtype, 8, 2, dim, sees, [300, 900], depth, seed=9)
    args["q"].copy_(other.q)
    case.q = other.q
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for graph, _ in graphs * 2:
            graph.replay()
        alone = ops.attention_tree(**args)
    side.synchronize()
    check(case, alone)
    for _, out in graphs:
        assert torch.equal(out, alone)


def test_every_kernel_from_several_threads():
    jobs = []
    for n, (kernel, dtype, dim, parts) in enumerate(FORMS):
        sees, depth = trees([64, 20], seed=n)
        case = Case(dtype, 8, 2, dim, sees, [500, 90], depth, seed=n)
        jobs.append({**case.on_device(), "kernel": kernel, "parts": parts})
    alone = [ops.attention_tree(**args) for args in jobs]
    torch.cuda.synchronize()
    groups = [list(zip(jobs, alone))[first::4] for first in range(4)]
    start, wrong = threading.Barrier(len(groups)), []

    def work(pairs):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for _ in range(30):
                    got = [ops.attention_tree(**args) for args, _ in pairs]
                    torch.cuda.current_stream().synchronize()
                    wrong.extend("a result differs from that of one thread alone" for g, (_, w) in zip(got, pairs) if not torch.equal(g, w))
        except Exception as e:  # noqa: BLE001 - told below
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(pairs,)) for pairs in groups]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[0]


@every_kernel
def test_many_nodes_of_many_heads(kernel, dtype, dim, parts):
    """As many nodes as a tree has, and 16 heads on one: 1,024 and 640 rows behind a few keys."""
    parents = bush(256, 3)
    check(case := Case(dtype, 4, 1, dim, [sees_of(parents), sees_of(chain(1))], [30, 7], [depth_of(parents), [0]], seed=6), run(case, kernel, parts))
    parents = bush(40, 4)
    check(case := Case(dtype, 16, 1, dim, [sees_of(parents)], [66], [depth_of(parents)], seed=7), run(case, kernel, parts))
