"""Log probabilities of given tokens, entropies and alternatives against 64 bits, from logits and from hidden rows."""

import math

import pytest
import torch

from starter_b200 import ops
from starter_b200.ops import KernelError

pytestmark = pytest.mark.gpu


def expected(x, tokens, top):
    """In 64 bits: log probabilities, entropies, alternatives and how far the float sums may be off.

    A weight exp(d), d = x - m, is off by 2^-21 and |d| 2^-22 of itself; sums of V weights in any order by V 2^-24 at most, of what one
    thread adds: 2,500 entries at most here; log and differences round to 2^-23 of what they are of."""
    x = x.double()
    m = x.amax(1, keepdim=True)
    d = x - torch.where(m == -math.inf, 0.0, m)
    p = d.exp()
    total = p.sum(1, keepdim=True)
    logp = d - total.log()
    w = p / total
    far = torch.where(w > 0, w * d.abs(), 0.0)
    entropy = -torch.where((w == 0), 0.0, w * logp).sum(1)               # (a row of nothing but minus infinity has none: 0 / 0)
    rel = 2.0 ** -20 + 2600 * 2.0 ** -24 + far.sum(1) * 2.0 ** -21
    # the weighted distances' sum has the weights' error, and that of its own terms
    second = (w * d.nan_to_num(neginf=0.0) ** 2).sum(1) * 2.0 ** -21
    tol_h = rel * (1 + 2 * far.sum(1)) + second
    order = torch.sort(torch.where(torch.isnan(x), -math.inf, x), dim=1, descending=True, stable=True).indices[:, :top]
    given = logp.gather(1, tokens.long().clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    return torch.where(tokens < 0, 0.0, given), entropy, logp.gather(1, order), order.int(), rel, tol_h


def near(got, want, tol):
    got, want = got.double().cpu(), want.cpu()
    inf = torch.isinf(want.float())                                      # (beyond what 32 bits hold)
    assert torch.equal(got[inf], want.float().double()[inf])
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    off = (got - want).abs() - (tol.cpu() + want.abs() * 2.0 ** -22)
    fine = inf | torch.isnan(want)
    assert (off[~fine] <= 0).all(), (off[~fine].max(), got[~fine][off[~fine].argmax()], want[~fine][off[~fine].argmax()])


def check(x, tokens, top):
    given, entropy, values, ids = ops.token_logprobs(x, tokens, top=top)
    w_given, w_entropy, w_values, w_ids, rel, tol_h = expected(x, tokens, top)
    near(given, w_given, rel)
    near(entropy, w_entropy, tol_h)
    near(values, w_values, rel[:, None].expand_as(w_values))
    assert torch.equal(ids, w_ids)
    assert given.dtype == entropy.dtype == values.dtype == torch.float32 and ids.dtype == torch.int32


def logits(rows, vocab, seed=0, dtype=torch.float32, size=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn((rows, vocab), generator=g, device="cuda") * size).to(dtype), torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 3, 31, 33, 255, 1000, 4095, 4096, 4097, 8191, 50001, 151936])
def test_sizes_of_vocabularies(dtype, vocab):
    for rows in (1, 3, 50):
        x, t = logits(rows, vocab, vocab + rows, dtype)
        for top in (0, 1, 5, 32):
            if top <= vocab:
                check(x, t, top)


@pytest.mark.parametrize("rows", [1, 2, 18, 19, 37, 38, 74, 75, 148, 149, 296, 297, 592, 593, 600, 666, 700, 889, 1184, 1186])
def test_numbers_of_rows(rows):
    x, t = logits(rows, 33333, rows)
    check(x, t, 20)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gap, shift", [(1, 0), (3, 1), (8, 3), (64, 0), (7, 5)])
def test_rows_further_apart_than_they_are_long(dtype, gap, shift):
    x, t = logits(9, 10007, gap, dtype)
    wide = torch.full((9, 10007 + gap + shift), 1e9, device="cuda", dtype=dtype)
    wide[:, shift:shift + 10007] = x
    check(wide[:, shift:shift + 10007], t, 7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_entries_are_listed_by_index(dtype):
    x = torch.zeros((3, 20000), device="cuda", dtype=dtype)
    x[1] = torch.arange(20000, device="cuda") % 7
    x[2, 12345:] = -5
    check(x, torch.tensor([0, 6, 19999], dtype=torch.int32, device="cuda"), 32)
    x, t = logits(6, 151936, 3, dtype)
    check((x * 2).round(), t, 32)


def test_the_order_of_entries():
    for direction in (1, -1):
        x = torch.arange(30000, device="cuda", dtype=torch.float32)[None] * direction * 1e-3
        check(x, torch.tensor([17], dtype=torch.int32, device="cuda"), 32)


def test_sharp_and_flat_rows():
    for size in (1e-3, 40.0, 1e4):
        x, t = logits(4, 20011, 5, size=size)
        check(x, t, 10)
    x = torch.full((2, 5000), -3.4e38, device="cuda")
    x[1, 77] = 3.4e38
    check(x, torch.tensor([3, 77], dtype=torch.int32, device="cuda"), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entries_of_minus_infinity(dtype):
    x, t = logits(5, 9001, 6, dtype)
    x[:, ::2] = -math.inf
    x[1] = -math.inf
    x[1, [5, 8000]] = torch.tensor([1.0, 2.0], device="cuda", dtype=dtype)
    x[2, :9000] = -math.inf
    t = torch.tensor([0, 8000, 9000, 1, 3], dtype=torch.int32, device="cuda")
    check(x, t, 6)
    given, entropy, _, _ = ops.token_logprobs(x, t, top=2)
    assert given[0] == -math.inf and torch.isnan(entropy[2])
    x[2, 7777] = 3
    t[2] = 7777
    check(x, t, 6)
    given, entropy, _, _ = ops.token_logprobs(x, t, top=2)
    assert given[2] == 0 and entropy[2] == 0


def test_rows_that_say_nothing():
    x, t = logits(5, 9001, 7)
    x[0] = -math.inf
    x[1, 300] = math.nan
    x[2, 300] = math.inf
    x[3] = math.nan
    given, entropy, values, ids = ops.token_logprobs(x, t, top=4)
    for row in range(4):
        assert torch.isnan(given[row]) and torch.isnan(entropy[row]) and torch.isnan(values[row]).all()
    assert ids[0].tolist() == [0, 1, 2, 3] and 300 not in ids[1].tolist() and ids[2, 0] == 300 and ids[3].tolist() == [-1] * 4
    order = torch.sort(x[1].nan_to_num(nan=-math.inf), descending=True, stable=True).indices[:4]
    assert ids[1].tolist() == order.tolist()
    check(x[4:], t[4:], 4)


def test_tokens_that_are_none():
    x, _ = logits(4, 777, 8)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    t = torch.tensor([-1, 776, 5, -99], dtype=torch.int32, device="cuda")
    given, _, _, _ = ops.token_logprobs(x, t, status=status)
    assert given[0] == 0 and given[3] == 0 and status.item() == 0
    given, entropy, _, _ = ops.token_logprobs(x, torch.tensor([0, 777, 1 << 30, 3], dtype=torch.int32, device="cuda"), status=status)
    assert torch.isnan(given).tolist() == [False, True, True, False] and torch.isfinite(entropy).all() and status.item() == 1


def test_more_rows_than_a_grid_dimension_counts():
    x, t = logits(66000, 40, 9)
    check(x, t, 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_alternatives_of_very_long_rows(dtype):
    for vocab in (700_001, 2_000_003, 5_242_000):
        x, t = logits(2, vocab, vocab, dtype)
        _, _, values, ids = ops.token_logprobs(x, t, top=32)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :32]
        assert torch.equal(ids, order.int())
    with pytest.raises(KernelError):
        ops.token_logprobs(logits(1, 11_000_000, 1, dtype)[0], t[:1], top=1)


def test_groups_that_hold_more_than_their_share():
    """The best entries in a few threads' pieces of every tile, and in ascending order: what the bar lets through overruns the buffer."""
    for dtype, piece in ((torch.float32, 16), (torch.bfloat16, 32)):
        x, t = logits(3, 151936, 12, dtype)
        place = torch.arange(151936, device="cuda")
        x = torch.where((place // piece) % 256 < 140, x + 100, x)
        check(x, t, 32)
        check(torch.sort(x, dim=1).values, t, 32)
        check(torch.sort(x, dim=1, descending=True).values, t, 32)


@pytest.mark.parametrize("rows", [12, 600, 1300])
def test_captured_and_replayed_on_a_stream(rows):
    x, t = logits(rows, 40000, 10)
    graph = torch.cuda.CUDAGraph()
    ops.token_logprobs(x, t, top=5)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = ops.token_logprobs(x, t, top=5)
    y, u = logits(rows, 40000, 11)
    x.copy_(y), t.copy_(u)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
        again = ops.token_logprobs(x, t, top=5)
    side.synchronize()
    for a, b in zip(out, again):
        assert torch.equal(a, b)
    w = expected(x, t, 5)
    assert torch.equal(out[3], w[3])


def test_rows_past_two_to_the_31_entries():
    """The last rows of 8.6 GB of logits."""
    rows = 2 ** 31 // 150001 + 3
    wide = torch.empty((rows, 150001), device="cuda")
    x, t = logits(2, 150001, 9)
    wide[:-2] = 0
    wide[-2:] = x
    got = ops.token_logprobs(wide, torch.cat([torch.zeros(rows - 2, dtype=torch.int32, device="cuda"), t]), top=4)
    want = expected(x, t, 4)
    near(got[0][-2:], want[0], want[4])
    near(got[1][-2:], want[1], want[5])
    assert torch.equal(got[3][-2:], want[3])


def test_logprob_refusals():
    x, t = logits(4, 100)
    for args, kw in (((x.half(), t), {}), ((x, t.long()), {}), ((x, t[:-1]), {}), ((x.t(), t), {}), ((x[0], t), {}), ((x[:, :0], t), {}),
                     ((x, t), dict(top=33)), ((x, t), dict(top=-1)), ((x[:, :5], t), dict(top=6))):
        with pytest.raises(KernelError):
            ops.token_logprobs(*args, **kw)
    out = ops.token_logprobs(x[:0], t[:0], top=3)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0, 3), (0, 3)]


# ------------------------------------------------------------------------------------------ from hidden rows

def score_case(rows, width, vocab, dtype, seed, size=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.randn((rows, width), generator=g, device="cuda").to(dtype)
    w = (torch.randn((vocab, width), generator=g, device="cuda") * size * width ** -0.5).to(dtype)
    return h, w, torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)


def check_score(h, w, t, softcap=None):
    given, entropy = ops.linear_logprobs(h, w, t, cap=softcap)
    x = h.double() @ w.double().T
    # a logit of K products summed in 32 bits is off by K 2^-24 of their sizes (tensor cores cut what a sum drops: a whole step,
    # 2^-23); the cap (slope at most 1) adds three roundings of its result
    size = h.double().abs() @ w.double().abs().T
    if softcap is not None:
        x = softcap * torch.tanh(x / softcap)
    off = size.amax(1) * (h.shape[1] + 2) * 2.0 ** -23 + x.abs().amax(1) * 2.0 ** -21
    w_given, w_entropy, _, _, rel, tol_h = expected(x, t, 0)
    near(given, w_given, rel + 2 * off)
    # the entropy's slope: the deviation of a logit's distance times its weight, twice, as every logit may be off
    near(entropy, w_entropy, tol_h + 2 * off * (1 + w_entropy.abs()) * 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [1, 17, 128, 129, 255, 256, 257, 300, 513])
def test_score_rows(dtype, rows):
    check_score(*score_case(rows, 256, 5003, dtype, rows))


@pytest.mark.parametrize("vocab", [1, 7, 8, 127, 128, 129, 255, 256, 257, 1000, 32768])
@pytest.mark.parametrize("width", [8, 64, 72, 1000])
def test_score_sizes(vocab, width):
    check_score(*score_case(200, width, vocab, torch.bfloat16, vocab + width))


@pytest.mark.parametrize("rows, width, vocab", [(1500, 512, 20000), (4100, 128, 9001), (200, 2560, 151936), (140, 130, 700), (260, 17, 300), (16385, 64, 300), (33000, 16, 200)])
def test_score_many(rows, width, vocab):
    check_score(*score_case(rows, width, vocab, torch.bfloat16, rows))


@pytest.mark.parametrize("rows", [3, 200])
def test_score_with_capped_logits(rows):
    check_score(*score_case(rows, 256, 3001, torch.bfloat16, rows, size=20.0), softcap=15.0)
    check_score(*score_case(rows, 256, 3001, torch.float32, rows, size=20.0), softcap=15.0)


def test_score_sharp_rows():
    check_score(*score_case(300, 512, 4001, torch.bfloat16, 1, size=30.0))


def test_score_tokens_that_are_none_and_rows_that_are_no_numbers():
    h, w, t = score_case(200, 64, 900, torch.bfloat16, 2)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    t[5], t[6] = -1, 900
    h[7, 3] = math.nan
    given, entropy = ops.linear_logprobs(h, w, t, status=status)
    assert given[5] == 0 and torch.isnan(given[6]) and torch.isnan(given[7]) and torch.isnan(entropy[7]) and status.item() == 1
    keep = [i for i in range(200) if i not in (5, 6, 7)]
    assert torch.isfinite(given[keep]).all() and torch.isfinite(entropy).sum() == 199


def test_score_captured_and_replayed():
    h, w, t = score_case(300, 128, 2000, torch.bfloat16, 3)
    ops.linear_logprobs(h, w, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.linear_logprobs(h, w, t)
    h2, _, t2 = score_case(300, 128, 2000, torch.bfloat16, 4)
    h.copy_(h2), t.copy_(t2)
    graph.replay()
    again = ops.linear_logprobs(h, w, t)
    assert torch.equal(out[0], again[0]) and torch.equal(out[1], again[1])


def test_a_wait_of_the_score_that_runs_out_is_reported():
    h, w, t = score_case(300, 256, 3000, torch.bfloat16, 5)
    status = torch.zeros((1,), dtype=torch.int32, device="cuda")
    ops.linear_logprobs(h, w, t, status=status, withhold=(1, 2_000_000))
    torch.cuda.synchronize()
    assert status.item() == 4
    status.zero_()
    ops.linear_logprobs(h, w, t, status=status)
    check_score(h, w, t)
    assert status.item() == 0


def test_score_refusals():
    h, w, t = score_case(5, 64, 900, torch.bfloat16, 2)
    for args in ((h.float(), w, t), (h, w[:, :32].contiguous(), t), (h, w, t[:-1]), (h, w, t.long()), (h[0], w, t), (h, w[:0], t), (h.half(), w.half(), t),
                 (h[:, ::2], w, t)):
        with pytest.raises(KernelError):
            ops.linear_logprobs(*args)
    out = ops.linear_logprobs(h[:0], w, t[:0])
    assert out[0].shape == (0,) and out[1].shape == (0,)
