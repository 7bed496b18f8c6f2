"""Log probabilities directly behind the kernels that make the logits, which let the next kernel start before they end: eager, captured, over and over
into the same memory.  600 rows are a launch of whole rows and one of the rest, which reads the logits in front of its own wait."""

import pytest
import torch

from starter_b200 import ops
from test_gpu_logprobs import expected, near

pytestmark = pytest.mark.gpu


def made(capped, rows, vocab=33000, width=64):
    g = torch.Generator(device="cuda").manual_seed(rows)
    h = torch.randn((rows, width), generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn((vocab, width), generator=g, device="cuda").to(torch.bfloat16)
    t = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)

    def step(wait=False):
        logits = ops.linear(h, w, out_float=True)
        if capped:
            ops.softcap(logits, 20.0)
        if wait:
            torch.cuda.synchronize()
        return ops.token_logprobs(logits, t, top=5), logits

    return h, t, step


@pytest.mark.parametrize("capped", [True, False])
@pytest.mark.parametrize("rows", [8, 600, 1300])
def test_behind_the_kernels_that_make_the_logits(capped, rows):
    h, t, step = made(capped, rows)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured, _ = step()
    seen = []
    for turn in range(12):
        # (the logits of the turn before lie in the same memory: what is read too early is theirs)
        h.copy_(torch.randn_like(h))
        graph.replay()
        eager, _ = step()
        want, logits = step(wait=True)
        for a, b, c in zip(captured, eager, want):
            assert torch.equal(a, c) and torch.equal(b, c), turn
        seen.append(want[0].clone())
    assert not any(torch.equal(seen[0], s) for s in seen[1:])
    w_given, w_entropy, w_values, w_ids, rel, tol_h = expected(logits, t, 5)
    near(want[0], w_given, rel), near(want[1], w_entropy, tol_h), near(want[2], w_values, rel[:, None].expand_as(w_values))
    assert torch.equal(want[3], w_ids)

