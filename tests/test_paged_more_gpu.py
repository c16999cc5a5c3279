"""More calls of the paged-cache operators: every wait's last phase, and what the
descriptions of the entry points say about odd calls."""
import random

import pytest
import torch

import arcllm_b200 as A
import gpu_util as G
import paged_util as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,tile", [(128, 80), (64, 96)])
@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 6, 11])
def test_attention_ends_after_any_number_of_tiles(dim, tile, tiles):
    """About one item per SM: its tiles fill the ring in part, just, or several times, and every copy is waited for
    (a wait for a phase that never comes would set the timeout bit)."""
    b = P.Batch([(tile * tiles - 20, 17)] * 148, 1, 1, dim, 16, "bf16")
    b.call()
    b.check()
    assert P.device_error() == 0


# ---- logits -----------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 3, 17])
def test_choice_among_the_parts_of_a_row(rows):
    """The largest value lies in another CTA's part of the row from call to call, with nothing between the calls."""
    vocab, calls = 70001, 150
    r = random.Random(rows)
    at = [[r.randrange(vocab) for _ in range(rows)] for _ in range(calls)]
    x = [torch.randn((rows, vocab), generator=torch.Generator().manual_seed(i)).to(G.dev()) for i in range(3)]
    logits = [x[i % 3].clone() for i in range(calls)]
    for y, places in zip(logits, at):
        y[torch.arange(rows), torch.tensor(places)] = 50.0
    best = torch.full((calls, rows), -7, dtype=torch.int32, device=G.dev())
    out = torch.empty_like(x[0])
    for i, y in enumerate(logits):
        A.call("arcllm_cuda_logits_process", A.GGML_F32, G.ptr(y), vocab, rows, vocab, None, 0, None, None, None, None,
               None, None, None, None, None, 0, G.ptr(out), vocab, G.ptr(best[i]), G.stream())
    assert best.tolist() == at
    assert P.device_error() == 0
