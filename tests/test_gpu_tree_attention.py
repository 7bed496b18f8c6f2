"""Attention of drafted trees against a statement of it in 64 bits: types, head layouts, lengths, masks, what lies beside the keys."""

import math

import numpy as np
import pytest
import torch

from starter_b200 import ops
from starter_b200.ops import KernelError

pytestmark = pytest.mark.gpu

PAGE = 64
DT = {"bf16": torch.bfloat16, "fp32": torch.float32}


def chain(n):
    return [-1] + list(range(n - 1))


def bush(n, seed, reach=8):
    rng = np.random.default_rng(seed)
    return [-1] + [int(rng.integers(max(0, i - reach), i)) for i in range(1, n)]


def sees_of(parents):
    n = len(parents)
    seen = torch.zeros((n, n), dtype=torch.bool)
    for i, p in enumerate(parents):
        if p >= 0:
            seen[i] = seen[p]
        seen[i, i] = True
    return seen


def depth_of(parents):
    d = []
    for p in parents:
        d.append(d[p] + 1 if p >= 0 else 0)
    return d


class Case:
    """A step: ``sees`` is a list of [n, n] truth values per sequence, ``past`` the cached tokens in front of each."""

    def __init__(self, dtype, heads, kv_heads, dim, sees, past, depth, window=None, seed=0, spread=1.0, words=None, fill=float("nan")):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.window = DT[dtype], heads, kv_heads, dim, window
        self.sees, self.past, self.n = sees, past, [s.shape[0] for s in sees]
        held = [-(-(p + n) // PAGE) for p, n in zip(past, self.n)]
        self.pages = sum(held) + 2
        order = torch.randperm(self.pages, generator=g).tolist()
        seqs = len(past)
        self.table = torch.zeros((seqs + 2, max(held + [1])), dtype=torch.int32)
        self.slots = torch.randperm(seqs + 2, generator=g)[:seqs].tolist()
        shape = (self.pages, kv_heads, PAGE, dim)
        # what belongs to no sequence is no number: nobody may look at it
        self.k, self.v = (torch.full(shape, fill) for _ in range(2))
        at = 0
        for s, h in enumerate(held):
            self.table[self.slots[s], :h] = torch.tensor(order[at:at + h], dtype=torch.int32)
            for j in range(past[s] + self.n[s]):
                page = order[at + j // PAGE]
                self.k[page, :, j % PAGE] = torch.randn((kv_heads, dim), generator=g)
                self.v[page, :, j % PAGE] = torch.randn((kv_heads, dim), generator=g)
            at += h
        self.k, self.v = self.k.to(self.dtype), self.v.to(self.dtype)
        self.start = np.concatenate([[0], np.cumsum(self.n)]).astype(int)
        self.rows = int(self.start[-1])
        self.q = (torch.randn((self.rows, heads * dim), generator=g) * spread).to(self.dtype)
        self.scale = dim ** -0.5
        self.longest = max(self.n + [1])
        self.words = words or -(-self.longest // 32)
        mask = np.zeros((self.rows, self.words * 32), dtype=np.uint8)
        self.pos = []
        for s, seen in enumerate(sees):
            mask[self.start[s]:self.start[s + 1], :self.n[s]] = seen.numpy()
            self.pos += [past[s] + d for d in depth[s]]
        self.mask = torch.from_numpy(np.packbits(mask, axis=1, bitorder="little").view(np.int32).copy())

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def on_device(self):
        return dict(q=self.q.cuda(), k_store=self.k.cuda(), v_store=self.v.cuda(), block_table=self.table.cuda(),
                    seq_slot=self.ints(self.slots), seq_q_start=self.ints(self.start[:-1].tolist()), seq_q_len=self.ints(self.n),
                    seq_kv_len=self.ints([p + n for p, n in zip(self.past, self.n)]), tok_pos=self.ints(self.pos),
                    tree_mask=self.mask.cuda(), heads=self.heads, kv_heads=self.kv_heads, head_dim=self.dim, scale=self.scale,
                    window=self.window, max_q_len=self.longest, kv_hint=max(p + n for p, n in zip(self.past, self.n)))

    def want(self):
        """The result in 64 bits and how far a kernel may be off it.

        A product of D rounded terms is off by at most (D + 2) 2^-24 sum |q_d k_d| (scale and log2(e) round once more), so a weight by
        the factor exp of twice the largest of those, and by 2^-21 for the power of two; the sums over n keys, joined from parts, add
        (n + 8) 2^-24.  In bfloat16 weights are rounded to 8 bits (half a step 2^-8 of each) before the second product.  The result
        is rounded once."""
        out, tol = torch.zeros((self.rows, self.heads * self.dim), dtype=torch.float64), torch.zeros((self.rows, self.heads * self.dim), dtype=torch.float64)
        group = self.heads // self.kv_heads
        low = self.dtype == torch.bfloat16
        for s, (n, past) in enumerate(zip(self.n, self.past)):
            first = int(self.start[s])
            if n == 0:
                continue
            places = [(int(self.table[self.slots[s], j // PAGE]), j % PAGE) for j in range(past + n)]
            page, off = torch.tensor([p for p, _ in places]), torch.tensor([o for _, o in places])
            k, v = self.k[page, :, off].double(), self.v[page, :, off].double()       # [keys, kv_heads, dim]
            seen = torch.cat([torch.ones((n, past), dtype=torch.bool), self.sees[s]], 1)
            pos = torch.tensor(self.pos[first:first + n])
            if self.window:
                seen = seen & (torch.cat([torch.arange(past), pos])[None] > pos[:, None] - self.window)
            q = self.q[first:first + n].double().view(n, self.heads, self.dim)
            for h in range(self.heads):
                kh, vh = k[:, h // group], v[:, h // group]
                score, size = q[:, h] @ kh.nan_to_num().T * self.scale, q[:, h].abs() @ kh.nan_to_num().abs().T * self.scale
                score = score.masked_fill(~seen, -math.inf)
                top = score.amax(1, keepdim=True)
                p = torch.where(seen, (score - torch.where(top == -math.inf, 0.0, top)).exp(), 0.0)
                total = p.sum(1, keepdim=True)
                p = p / torch.where(total == 0, 1.0, total)
                for i in range(n):
                    use = seen[i].nonzero()[:, 0]
                    o, mean = p[i, use] @ vh[use], p[i, use] @ vh[use].abs()
                    off_by = 2 * float((size[i, use].max() if len(use) else 0.0) * (self.dim + 4) * 2.0 ** -24) + 2.0 ** -21 + (len(use) + 8) * 2.0 ** -24
                    if low:
                        off_by += 2.0 ** -8
                    at = slice(h * self.dim, (h + 1) * self.dim)
                    out[first + i, at] = o
                    tol[first + i, at] = mean * off_by * (1 + 2.0 ** -8) + o.abs() * torch.finfo(self.dtype).eps / 2 + 1e-37
        return out, tol


def check(case, got=None):
    if got is None:
        got = ops.attention_tree(**case.on_device())
    want, tol = case.want()
    got = got.double().cpu()
    assert got.shape == want.shape
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got)), "numbers where there are none, or the other way round"
    bad = ((got - want).abs() > tol) & ~nan
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                           f"{got[bad][0].item()} for {want[bad][0].item()}, within {tol[bad][0].item()}")


def trees(nodes, seed=0):
    parents = [bush(n, seed + i) if n else [] for i, n in enumerate(nodes)]
    return [sees_of(p) for p in parents], [depth_of(p) for p in parents]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("heads, kv_heads, dim", [(1, 1, 16), (4, 2, 32), (6, 2, 48), (4, 4, 64), (8, 2, 64), (3, 1, 128), (16, 4, 128),
                                                  (8, 1, 128), (5, 1, 80), (2, 1, 256), (2, 2, 6), (1, 1, 1), (32, 1, 64), (7, 1, 128)])
def test_heads_and_sizes(dtype, heads, kv_heads, dim):
    sees, depth = trees([1, 13, 5])
    check(Case(dtype, heads, kv_heads, dim, sees, [70, 131, 0], depth, seed=dim))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("past", [0, 1, 31, 32, 62, 63, 64, 65, 127, 128, 191, 700])
def test_cached_tokens_around_the_ends_of_pages(dtype, past):
    sees, depth = trees([1, 2, 66], seed=past)
    check(Case(dtype, 4, 2, 64, sees, [past] * 3, depth, seed=past))


@pytest.mark.parametrize("dtype, dim", [("fp32", 64), ("bf16", 64), ("bf16", 128), ("bf16", 32)])
@pytest.mark.parametrize("nodes", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 256])
def test_numbers_of_nodes(dtype, dim, nodes):
    sees, depth = trees([nodes, 1, nodes // 2], seed=nodes)
    check(Case(dtype, 4, 1, dim, sees, [90, 3, 64], depth, seed=nodes))


@pytest.mark.parametrize("dtype, dim", [("fp32", 128), ("bf16", 128), ("bf16", 64)])
@pytest.mark.parametrize("past, nodes", [(5000, 7), (9000, 40), (2100, 64)])
def test_long_sequences(dtype, dim, past, nodes):
    sees, depth = trees([nodes, 3], seed=past)
    check(Case(dtype, 8, 2, dim, sees, [past, past // 3], depth, seed=past))


@pytest.mark.parametrize("dtype, dim", [("fp32", 48), ("bf16", 16), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("window", [1, 2, 5, 64, 100, 10000])
def test_windows_go_by_positions(dtype, dim, window):
    sees, depth = trees([30, 64, 1], seed=window)
    check(Case(dtype, 4, 2, dim, sees, [150, 0, 300], depth, window=window, seed=window))
    parents = chain(40)
    check(Case(dtype, 8, 1, dim, [sees_of(parents)], [130], [depth_of(parents)], window=window, seed=window))


@pytest.mark.parametrize("dtype, dim", [("fp32", 32), ("bf16", 64), ("bf16", 128), ("bf16", 32)])
def test_masks_of_any_kind(dtype, dim):
    g = torch.Generator().manual_seed(5)
    n = 45
    any_mask = torch.rand((n, n), generator=g) < 0.3
    any_mask[7] = False                      # with nothing cached in front a row that sees nothing
    any_mask[8] = True                       # what comes later, too
    for past in (0, 77):
        check(Case(dtype, 4, 1, dim, [any_mask, torch.zeros((3, 3), dtype=torch.bool)], [past, 0], [[0] * n, [0, 1, 2]], seed=past))


@pytest.mark.parametrize("dtype, dim", [("fp32", 64), ("bf16", 64), ("bf16", 128), ("bf16", 32)])
def test_sequences_without_nodes(dtype, dim):
    sees, depth = trees([0, 9, 0, 21, 0], seed=1)
    check(Case(dtype, 4, 2, dim, sees, [0, 100, 64, 5, 10], depth, seed=1))


@pytest.mark.parametrize("dtype, dim", [("fp32", 64), ("bf16", 64), ("bf16", 128), ("bf16", 32)])
@pytest.mark.parametrize("nodes", [9, 40, 130])
def test_what_is_no_number_reaches_only_those_that_see_it(dtype, dim, nodes):
    parents = [-1] + [0] * (nodes - 1)       # leaves of one root: each sees itself, the root and what is cached
    for what in (math.nan, math.inf):
        c = Case(dtype, 4, 1, dim, [sees_of(parents)], [100], [depth_of(parents)], seed=nodes)
        for j, which in ((100 + 3, "k"), (100 + 5, "v"), (100 + nodes - 1, "v")):
            page = int(c.table[c.slots[0], j // PAGE])
            getattr(c, which)[page, 0, j % PAGE, 2] = what
        got = ops.attention_tree(**c.on_device()).cpu()
        for i in range(nodes):
            row = got[i].view(4, dim)
            if i == 3:
                assert not torch.isfinite(row.float()).all() or what == math.inf    # (a score of -inf weighs nothing)
            elif i in (5, nodes - 1):
                assert not torch.isfinite(row[:, 2].float()).any() and torch.isfinite(row[:, :2].float()).all()
            else:
                assert torch.isfinite(row.float()).all(), i


@pytest.mark.parametrize("dtype, dim", [("fp32", 64), ("bf16", 64), ("bf16", 128)])
@pytest.mark.parametrize("nodes", [6, 70])
def test_sharp_scores(dtype, dim, nodes):
    sees, depth = trees([nodes], seed=3)
    check(Case(dtype, 8, 2, dim, sees, [333], depth, seed=3, spread=30.0))


@pytest.mark.parametrize("dtype, dim", [("fp32", 64), ("bf16", 128)])
def test_more_words_than_needed_and_a_hint_that_is_wrong(dtype, dim):
    sees, depth = trees([20, 40], seed=4)
    c = Case(dtype, 8, 2, dim, sees, [400, 100], depth, seed=4, words=5)
    want, tol = c.want()
    for hint in (0, 1, 70, 100000):
        for longest in (40, 41, 64, 160):
            args = c.on_device()
            args.update(kv_hint=hint, max_q_len=longest)
            assert ((ops.attention_tree(**args).double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype, dim, nodes", [("fp32", 64, 10), ("bf16", 64, 6), ("bf16", 128, 64), ("bf16", 128, 20)])
def test_captured_on_another_stream_and_replayed(dtype, dim, nodes):
    sees, depth = trees([nodes, nodes // 2 + 1], seed=8)
    c = Case(dtype, 8, 2, dim, sees, [300, 900], depth, seed=8)
    args = c.on_device()
    first = ops.attention_tree(**args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.attention_tree(**args)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, again)
    graphs = []
    for _ in range(2):                       # two graphs, replayed in turn
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.attention_tree(**args)
        graphs.append((graph, out))
    other = Case(dtype, 8, 2, dim, sees, [300, 900], depth, seed=9)
    args["q"].copy_(other.q)
    for graph, out in graphs:
        graph.replay()
    c.q = other.q
    for _, out in graphs:
        check(c, out)


@pytest.mark.parametrize("dim, group, nodes", [(128, 4, 64), (64, 8, 20), (128, 3, 100), (128, 1, 256), (64, 7, 40), (128, 16, 9)])
@pytest.mark.parametrize("parts", [1, 2, 4, 8])
def test_keys_in_parts_on_tensor_memory(dim, group, nodes, parts):
    sees, depth = trees([nodes, 1, nodes // 2], seed=nodes)
    for past, window in (([700, 64, 0], None), ([1500, 300, 1023], 200)):
        c = Case("bf16", 2 * group, 2, dim, sees, past, depth, window=window, seed=nodes)
        check(c, ops.attention_tree(**c.on_device(), kernel="tcgen05", parts=parts))


@pytest.mark.parametrize("dim", [16, 32, 64, 128])
@pytest.mark.parametrize("parts", [(1, 1), (1, 5), (2, 3), (2, 8), (1, 2), (2, 7), (1, 8)])
def test_keys_in_parts_on_warps(dim, parts):
    sees, depth = trees([21, 1, 0, 40], seed=dim)
    c = Case("bf16", 6, 2, dim, sees, [800, 64, 0, 129], depth, window=300 if parts[1] % 2 else None, seed=dim)
    check(c, ops.attention_tree(**c.on_device(), kernel="mma", parts=parts))


@pytest.mark.parametrize("dtype, dim", [("fp32", 128), ("fp32", 200), ("bf16", 96), ("bf16", 7), ("fp32", 18)])
@pytest.mark.parametrize("parts", [1, 2, 5, 8])
def test_keys_in_parts_on_the_plain_kernel(dtype, dim, parts):
    sees, depth = trees([21, 1, 0, 40], seed=dim)
    c = Case(dtype, 6, 2, dim, sees, [800, 64, 0, 129], depth, window=300 if parts % 2 else None, seed=dim)
    check(c, ops.attention_tree(**c.on_device(), kernel="plain", parts=parts))


@pytest.mark.parametrize("kernel", ["plain", "mma", "tcgen05"])
def test_pages_past_two_to_the_31_entries(kernel):
    """The step's pages lie behind 2^31 entries of the stores (of each, 4.3 GB)."""
    sees, depth = trees([20, 3], seed=4)
    c = Case("bf16", 16, 8, 128, sees, [300, 70], depth, seed=4)
    args, shift = c.on_device(), 2 ** 31 // (8 * PAGE * 128) + 3
    for name in ("k_store", "v_store"):
        wide = torch.empty((shift + c.pages, 8, PAGE, 128), dtype=torch.bfloat16, device="cuda")
        wide[shift:] = args[name]
        args[name] = wide
    args["block_table"] = args["block_table"] + shift
    check(c, ops.attention_tree(**args, kernel=kernel))


@pytest.mark.parametrize("parts", [1, 2])
def test_a_wait_of_the_tree_attention_that_runs_out_is_reported(parts):
    """Half of a step's values are not copied: the wait gives up, the status says so, and the next call is right."""
    sees, depth = trees([64], seed=2)
    c = Case("bf16", 8, 2, 128, sees, [500], depth, seed=2)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    ops.attention_tree(**c.on_device(), kernel="tcgen05", parts=parts, status=status, withhold=(1, 2_000_000))
    torch.cuda.synchronize()
    assert status.item() == 16
    status.zero_()
    check(c, ops.attention_tree(**c.on_device(), kernel="tcgen05", parts=parts, status=status))
    assert status.item() == 0


def test_refusals():
    sees, depth = trees([5])
    c = Case("bf16", 4, 2, 64, sees, [10], depth)
    good = c.on_device()
    half = {k: good[k].half() for k in ("q", "k_store", "v_store")}
    for change in (dict(q=good["q"][:, :-64].contiguous()), dict(q=good["q"].float()), half, dict(heads=3), dict(kv_heads=0),
                   dict(head_dim=257), dict(window=0), dict(window=-3), dict(max_q_len=0), dict(max_q_len=257), dict(max_q_len=33),
                   dict(tok_pos=good["tok_pos"][:-1]), dict(tree_mask=good["tree_mask"][:-1]), dict(tree_mask=good["tree_mask"][:, 0]),
                   dict(seq_q_len=good["seq_q_len"].long()), dict(seq_slot=good["seq_slot"][:0]), dict(k_store=good["k_store"][:, :1].contiguous()),
                   dict(q=good["q"].t().contiguous().t()), dict(block_table=good["block_table"][0])):
        with pytest.raises(KernelError):
            ops.attention_tree(**{**good, **change})


def test_nothing_to_do():
    c = Case("bf16", 4, 2, 64, [torch.zeros((0, 0), dtype=torch.bool)], [10], [[]])
    args = c.on_device()
    assert ops.attention_tree(**args).shape == (0, 256)
