"""The drafting and scoring operators called from several threads at once, each on a stream of its own: every result is what one thread gets alone."""

import threading

import pytest
import torch

from starter_b200 import ops

pytestmark = pytest.mark.gpu

PAGE = 64


def tree_call(dim, dtype, nodes, past, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = -(-(past + nodes) // PAGE)
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dtype)  # noqa: E731
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")  # noqa: E731
    words = -(-nodes // 32)
    mask = torch.full((nodes, words), -1, dtype=torch.int32, device="cuda")
    args = dict(q=make(nodes, 8 * dim), k_store=make(pages, 2, PAGE, dim), v_store=make(pages, 2, PAGE, dim), block_table=ints([list(range(pages))]),
                seq_slot=ints([0]), seq_q_start=ints([0]), seq_q_len=ints([nodes]), seq_kv_len=ints([past + nodes]),
                tok_pos=ints([past + i for i in range(nodes)]), tree_mask=mask, heads=8, kv_heads=2, head_dim=dim, scale=dim ** -0.5,
                max_q_len=nodes, kv_hint=past + nodes)
    return lambda: [ops.attention_tree(**args)]


def logprob_call(rows, vocab, top, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, vocab), generator=g, device="cuda")
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return lambda: list(ops.token_logprobs(x, t, top=top))


def score_call(rows, vocab, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h, w = (torch.randn(shape, generator=g, device="cuda").to(torch.bfloat16) for shape in ((rows, 256), (vocab, 256)))
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return lambda: list(ops.linear_logprobs(h, w, t))


def test_calls_from_several_threads():
    # sizes whose kernels want different amounts of shared memory each
    jobs = [[tree_call(dim, torch.float32, 20, 100 + dim, dim) for dim in (200, 96, 256, 128)],
            [tree_call(dim, torch.float32, 20, 100 + dim, dim) for dim in (104, 248, 160, 224)],
            [tree_call(dim, torch.bfloat16, 64, 900, dim) for dim in (128, 64, 16, 32)],
            [logprob_call(4, vocab, 9, vocab) for vocab in (150000, 300000, 3000, 600000)],
            [logprob_call(5, vocab, 3, vocab) for vocab in (500000, 40000, 800000, 200000)],
            [score_call(rows, vocab, rows) for rows, vocab in ((300, 5000), (129, 40000), (700, 900), (512, 33000))]]
    alone = [[call() for call in calls] for calls in jobs]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(jobs)), []

    def work(calls, wants):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                start.wait()
                for turn in range(20):
                    got = [call() for call in calls]
                    torch.cuda.current_stream().synchronize()
                    for g, w in zip(got, wants):
                        for a, b in zip(g, w):
                            if not torch.equal(a, b):
                                wrong.append(f"turn {turn}: a result differs from the one of a thread alone")
        except Exception as e:  # noqa: BLE001 - told below
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=pair) for pair in zip(jobs, alone)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[0]
