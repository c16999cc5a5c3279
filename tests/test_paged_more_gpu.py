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


# ---- attention: values that are no numbers -----------------------------------
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("lens,at", [([(100, 600), (40, 1)], 350), ([(0, 130), (900, 40)], 60), ([(700, 90)], 3)])
def test_attention_of_a_key_that_is_no_number_in_many_rows(dim, bad, lens, at):
    """One element of one key of a request with many rows, in the first tile or a later one: rows before its position
    are as they were; of the others those whose score is NaN or +inf have no softmax, and to those with a score of
    -inf the position has no weight."""
    b = P.Batch(lens, 1, 4, dim, 16, "f16")
    kv, n = b.lens[0]
    b.cache.k[int(b.table[0, at // 16]), at % 16, 0, 7] = bad
    b.call()
    got = b.out.float().cpu().double()[:n, :4 * dim].view(n, 4, dim)
    q, k, v, pos = b.q[:n], b.k[0], b.v[0], torch.arange(kv, kv + n)
    want, tol = P.attention_plain(q, k, v, pos, b.scale, 0, 0, "f16")
    without = torch.arange(kv + n) != at
    want2, tol2 = P.attention_plain(q, k[without], v[without], pos - 1, b.scale, 0, 0, "f16")
    score = torch.where(q[..., 7] == 0, float("nan"), q[..., 7].double() * bad)  # its one term that is not finite
    after, unseen = pos >= at, score == -float("inf")
    off = (got - want).abs() <= tol
    assert off[~after].all()
    assert ((got - want2).abs() <= tol2)[after[:, None] & unseen].all()
    assert torch.isnan(got[after[:, None] & ~unseen]).all()
    first = b.out[:n].clone()
    b.cache.k[int(b.table[0, at // 16]), at % 16, 0, 7] = P.dev(k[at, 0, 7])
    b.call()
    b.check()  # all of it, and the other requests, without the bad value
    assert torch.equal(b.out[:n][~after.to(b.out.device)], first[~after.to(b.out.device)])
    assert P.device_error() == 0


# ---- launch overlap -----------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128])
def test_steps_with_launch_overlap_give_the_same_bits(dim):
    """Plan, two layers of rotary store and attention (the second takes the first one's output), constrained choice:
    one after another with every kernel allowed to start early, each call behind the one it needs; two sets of inputs
    in turn with nothing between the steps, and captured."""
    heads, gq, page, name, steps = 2, 4, 16, "bf16", 8
    kv, new = [300, 90, 0, 1500, 17], [1, 200, 77, 1, 2]
    n, qh, d = len(kv), heads * gq, G.dev()
    qn, kn, rows = qh * dim, heads * dim, sum(new) + 5
    used, need = sum(-(-a // page) for a in kv), sum(-(-(a + b) // page) for a, b in zip(kv, new))
    pages = list(range(need + 3))
    random.Random(1).shuffle(pages)
    width = max(-(-(a + b) // page) for a, b in zip(kv, new)) + 1
    table, at = [], 0
    for a in kv:
        k = -(-a // page)
        table.append(pages[at:at + k] + [-1] * (width - k))
        at += k
    table = torch.tensor(table, dtype=torch.int32, device=d)
    kv_len, new_len, free, n_free = P.i32(kv), P.i32(new), P.i32(pages[used:]), P.i32([len(pages) - used])
    row_start, total, n_out = P.i32([0] * (n + 1)), P.i32([0] * n), P.i32([0])
    positions, slots = P.i32([0] * rows), P.i32([0] * rows)
    caches = [P.Cache(len(pages), page, heads, dim, name, i == 1, 0.0) for i in range(2)]
    for i, c in enumerate(caches):
        c.k.copy_(P.normal(c.k.shape, 2 * i, name))
        c.v.copy_(P.normal(c.v.shape, 2 * i + 1, name))
    x = [P.dev(P.normal((rows, qn + 2 * kn), 10 + i, name)) for i in range(2)]
    f, s = P.frequencies(dim)
    fd = P.dev(f)
    q = torch.zeros((rows, qn), dtype=P.DT[name], device=d)
    mid = torch.zeros_like(q)
    size = A.C.c_uint64()
    A.call("arcllm_cuda_attention_paged_workspace", qh, heads, dim, A.C.byref(size))
    ws = torch.empty(size.value, dtype=torch.uint8, device=d)
    history = P.dev(torch.randint(0, qn, (rows, 33), generator=torch.Generator().manual_seed(3), dtype=torch.int32))
    said, rep = P.i32([33] * rows), torch.full((rows,), 1.3, device=d)

    def step(x, out, best, st):
        A.call("arcllm_cuda_paged_plan", G.ptr(kv_len), G.ptr(new_len), n, page, len(pages), G.ptr(free), G.ptr(n_free),
               G.ptr(table), width, rows, G.ptr(row_start), G.ptr(total), G.ptr(positions), G.ptr(slots), G.ptr(n_out),
               st)
        for c, src, dst in zip(caches, (x, mid), (mid, out)):
            A.call("arcllm_cuda_rope_kv_paged", A.GGML_BF16, G.ptr(src), src.stride(0), G.ptr(x[:, qn:]), x.stride(0),
                   G.ptr(x[:, qn + kn:]), x.stride(0), None, None, None, G.ptr(fd), dim, A.ROPE_HALVES, s,
                   G.ptr(positions), G.ptr(slots), rows, qh, c.ref(), G.ptr(q), qn, st)
            A.call("arcllm_cuda_attention_paged", G.ptr(q), qn, c.ref(), G.ptr(table), width, G.ptr(row_start),
                   G.ptr(total), n, rows, rows, qh, dim ** -0.5, 0, 0, G.ptr(dst), qn, G.ptr(ws), ws.numel(), st)
        A.call("arcllm_cuda_logits_process", A.GGML_BF16, G.ptr(out), qn, rows, qn, G.ptr(history), 33, None,
               G.ptr(said), G.ptr(rep), None, None, None, None, None, None, 0, G.ptr(out), qn, G.ptr(best), st)

    def results():
        return (torch.zeros((rows, qn), dtype=P.DT[name], device=d), torch.full((rows,), -7, dtype=torch.int32, device=d))

    def same(got, want):
        return all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(got, want))

    plain = [results() for _ in x]
    for y, r in zip(x, plain):
        step(y, *r, G.stream())
    torch.cuda.synchronize()
    assert not same(*plain) and torch.isfinite(plain[0][0][:sum(new)].float()).all()
    q.zero_(), mid.zero_()
    got = [results() for _ in range(2 * steps)]
    replayed = [results() for _ in x]
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    A.call("arcllm_cuda_set_launch_overlap", 1)
    try:
        for i, r in enumerate(got):
            step(x[i % 2], *r, G.stream())
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            for y, r in zip(x, replayed):
                step(y, *r, A.C.c_void_p(stream.cuda_stream))
    finally:
        A.call("arcllm_cuda_set_launch_overlap", 0)
    for i, r in enumerate(got):
        assert same(r, plain[i % 2]), i
    for _ in range(5):
        for r in replayed:
            r[0].zero_(), r[1].fill_(-7)
        g.replay()
        torch.cuda.synchronize()
        assert all(same(r, w) for r, w in zip(replayed, plain))
    assert P.device_error() == 0
