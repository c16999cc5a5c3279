"""Penalties, biases, masks and the greedy choice on batches of logits.  Every
step is one fp32 operation per logit, so the plain form (numpy, the same steps)
has to give the same bits."""
import ctypes as C

import numpy as np
import pytest
import torch

import arcllm_b200 as A
import gpu_util as G
import paged_util as P

pytestmark = pytest.mark.gpu


def plain(x, history, prompt, total, rep, freq, pres, biases, mask, name):
    """x [rows, vocab] float32 (holding values of the type); biases: a list of (id, value) per row."""
    x = x.copy()
    f32 = np.float32
    rows, vocab = x.shape
    with np.errstate(all="ignore"):
        for r in range(rows):
            if history is not None:
                h = history[r][:max(0, min(total[r], history.shape[1]))]
                p = 0 if prompt is None else max(0, prompt[r])
                ok = lambda t: t[(t >= 0) & (t < vocab)]  # noqa: E731
                seen = np.unique(ok(h))
                ids, count = np.unique(ok(h[p:]), return_counts=True)
                if rep is not None:
                    y = x[r, seen]
                    x[r, seen] = np.where(y > 0, y / f32(rep[r]), y * f32(rep[r]))
                if freq is not None:
                    x[r, ids] = x[r, ids] - f32(freq[r]) * count.astype(f32)
                if pres is not None:
                    x[r, ids] = x[r, ids] - f32(pres[r])
            if biases is not None:
                for t, b in dict(biases[r]).items():
                    if 0 <= t < vocab:
                        x[r, t] = x[r, t] + f32(b)
            if mask is not None:
                bits = (mask[r][:, None] >> np.arange(32, dtype=np.uint32)) & 1
                x[r][bits.reshape(-1)[:vocab] == 0] = -np.inf
    y = torch.from_numpy(x).to(P.DT[name])
    z = y.float().numpy()
    z = np.where(np.isfinite(z), z, -np.inf)
    best = [int(v.argmax()) if v.max() > -np.inf else -1 for v in z]
    return y, best


def run(x, history=None, prompt=None, total=None, rep=None, freq=None, pres=None, biases=None, mask=None, name="f32",
        pad=0, off=0, in_place=False, want_best=True, out_off=None):
    rows, vocab = x.shape
    t = torch.from_numpy(x).to(P.DT[name])
    buf = torch.full((rows, vocab + pad + off), 7.0, dtype=P.DT[name], device=G.dev())
    xd = buf[:, off:off + vocab]
    xd.copy_(t)
    o = off if out_off is None else out_off
    obuf = torch.full((rows, vocab + pad + o), 7.0, dtype=P.DT[name], device=G.dev())
    out = xd if in_place else obuf[:, o:o + vocab]
    up = lambda v, ty: None if v is None else torch.from_numpy(np.ascontiguousarray(v, dtype=ty)).to(G.dev())  # noqa: E731
    hd, pd, td = up(history, np.int32), up(prompt, np.int32), up(total, np.int32)
    rd, fd, sd = up(rep, np.float32), up(freq, np.float32), up(pres, np.float32)
    bs = bi = bv = None
    if biases is not None:
        bs = up(np.cumsum([0] + [len(b) for b in biases]), np.int32)
        flat = [e for b in biases for e in b] + [(0, 0.0)]
        bi, bv = up([e[0] for e in flat], np.int32), up([e[1] for e in flat], np.float32)
    md = up(mask.view(np.int32), np.int32) if mask is not None else None
    best = torch.full((rows,), -7, dtype=torch.int32, device=G.dev())
    A.call("arcllm_cuda_logits_process", P.GGML[name], G.ptr(xd), xd.stride(0), rows, vocab, G.ptr(hd),
           0 if history is None else history.shape[1], G.ptr(pd), G.ptr(td), G.ptr(rd), G.ptr(fd), G.ptr(sd), G.ptr(bs),
           G.ptr(bi), G.ptr(bv), G.ptr(md), 0 if mask is None else mask.shape[1], G.ptr(out), out.stride(0),
           G.ptr(best) if want_best else None, G.stream())
    torch.cuda.synchronize()
    want, pick = plain(t.float().numpy(), history, prompt, total, rep, freq, pres, biases, mask, name)
    got = out.cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    assert same.all(), (~same).nonzero()[:4]
    assert best.tolist() == (pick if want_best else [-7] * rows)
    assert (buf[:, off + vocab:] == 7.0).all() and (buf[:, :off] == 7.0).all()
    if not in_place:
        assert (obuf[:, o + vocab:] == 7.0).all() and (obuf[:, :o] == 7.0).all()
    return best.tolist()


def inputs(rows, vocab, hist, seed=0, words=None):
    r = np.random.default_rng(seed)
    x = r.normal(0, 3, (rows, vocab)).astype(np.float32)
    history = (r.random((rows, hist)) ** 4 * vocab).astype(np.int32)
    total = r.integers(0, hist + 1, rows)
    prompt = r.integers(0, hist + 1, rows)
    par = [r.uniform(a, b, rows).astype(np.float32) for a, b in ((0.8, 1.6), (-0.2, 0.7), (-0.2, 0.7))]
    biases = [[(int(t), float(np.float32(v))) for t, v in zip(r.integers(-2, vocab + 2, n), r.normal(0, 4, n))]
              for n in r.integers(0, 40, rows)]
    mask = r.integers(0, 2 ** 32, (rows, words or (vocab + 31) // 32), dtype=np.uint32)
    return x, history, prompt, total, par, biases, mask


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,hist", [(1, 152064, 300), (3, 1000, 50), (9, 32000, 4000), (2, 1, 3), (5, 37, 5),
                                             (4, 4096, 1), (2, 200003, 100)])
def test_all_constraints(name, rows, vocab, hist):
    x, h, p, t, (rep, freq, pres), b, m = inputs(rows, vocab, hist, vocab)
    run(x, h, p, t, rep, freq, pres, b, m, name)


@pytest.mark.parametrize("name,pad,off", [("f32", 3, 0), ("f32", 4, 4), ("f16", 1, 1), ("bf16", 8, 8), ("bf16", 3, 0)])
def test_strides_and_in_place(name, pad, off):
    x, h, p, t, (rep, freq, pres), b, m = inputs(6, 5003, 64, 3, words=160)
    run(x, h, p, t, rep, freq, pres, b, m, name, pad, off)
    run(x, h, p, t, rep, freq, pres, b, m, name, pad, off, in_place=True)


@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 8, 9, 31, 33, 1025, 70001])
def test_rows_that_start_anywhere(name, vocab):
    x, h, p, t, (rep, freq, pres), b, m = inputs(5, vocab, 40, vocab)
    for off in range(1, 8):
        run(x, h, p, t, rep, freq, pres, b, m, name, off % 3, off)
        run(x, h, p, t, rep, freq, pres, b, m, name, 1, off, in_place=True)
    run(x, h, p, t, rep, freq, pres, b, m, name, 1, 3, out_off=4)
    run(x, h, p, t, rep, freq, pres, b, m, name, 0, 1, out_off=0)


def test_each_constraint_alone():
    x, h, p, t, (rep, freq, pres), b, m = inputs(4, 9000, 200, 5)
    run(x)
    run(x, want_best=False)
    run(x, h, p, t)
    run(x, h, p, t, rep=rep)
    run(x, h, None, t, freq=freq)
    run(x, h, p, t, pres=pres)
    run(x, biases=b)
    run(x, mask=m)


def test_choice_of_ties_and_rows_with_nothing_left():
    x = np.zeros((6, 70000), np.float32)
    x[0, [69000, 17, 40000]] = 5.0
    x[1] = -np.inf
    x[2] = np.nan
    x[3, [3, 9]] = [np.inf, 2.0]
    x[4, 0] = -0.0  # equal to the zeros behind it
    x[5, :] = -3.0e38
    m = np.full((6, 2188), 0xffffffff, np.uint32)
    m[5] = 0
    assert run(x, mask=m) == [17, -1, -1, 9, 0, -1]
    m[5, 2187] = 1 << 15
    assert run(x, mask=m)[5] == 69999


def test_histories_with_padding_and_lengths_out_of_range():
    x, h, _, _, (rep, freq, pres), _, _ = inputs(4, 300, 20, 6)
    h[0, 5:] = -1
    h[1, ::2] = 300
    h[2, 3], h[2, 4] = -2 ** 31, 2 ** 31 - 1
    run(x, h, np.array([3, -5, 100, 0]), np.array([20, 25, 20, -4]), rep, freq, pres)


def test_the_last_of_several_biases_counts_every_time():
    x = np.zeros((2, 50), np.float32)
    b = [[(7, float(i)) for i in range(2000)] + [(3, 1.0), (3, -1.0)], []]
    for _ in range(5):
        run(x, biases=b)


def test_more_rows_than_a_grid_dimension():
    r = np.random.default_rng(1)
    x = r.normal(0, 1, (65537, 8)).astype(np.float32)
    h = r.integers(0, 8, (65537, 2)).astype(np.int32)
    run(x, h, None, np.full(65537, 2), rep=np.full(65537, 1.5, np.float32))


def test_matches_argmax_of_the_library():
    x = np.random.default_rng(2).normal(0, 1, (3, 152064)).astype(np.float32)
    xd = G.to_dev(x)
    scratch = G.empty_u8(16)
    best = run(x)
    for r in range(3):
        i, ok = C.c_uint32(), C.c_int()
        A.call("arcllm_cuda_argmax", G.ptr(xd[r]), 152064, G.ptr(scratch), C.byref(i), C.byref(ok), G.stream())
        assert i.value == best[r] and ok.value == 1


@pytest.mark.parametrize("name", ["f32", "bf16"])
@pytest.mark.parametrize("rows,vocab,hist", [(200, 30000, 20000), (1, 70001, 40000), (3, 9000, 9000)])
def test_histories_that_name_most_of_the_vocabulary(name, rows, vocab, hist):
    """More named tokens, and more history entries, than a CTA holds at a time."""
    x, h, p, t, (rep, freq, pres), b, m = inputs(rows, vocab, hist, 17)
    r = np.random.default_rng(5)
    for i in range(min(rows, 3)):
        h[i] = r.permutation(vocab)[:hist]
    t[:3] = hist
    for i in range(3, rows):  # the others are short, for the plain form's sake
        t[i] = min(t[i], 30)
    run(x, h, p, t, rep, freq, pres, b, m, name)
    run(x, h, p, t, rep, freq, pres, b, m, name, 1, 3, in_place=True)


def test_rows_of_more_than_one_chunk():
    x, h, p, t, (rep, freq, pres), b, m = inputs(296, 140003, 50, 23)
    h[:, ::3] = 131000 + h[:, ::3] % 9003
    run(x, h, p, t, rep, freq, pres, b, m, "f32")
    run(x, h, p, t, rep, freq, pres, b, m, "f16", 0, 1)


def test_captured_and_on_two_streams():
    rows, vocab, hist = 7, 70001, 500
    x, h, p, t, (rep, freq, pres), b, m = inputs(rows, vocab, hist, 11)
    want, pick = plain(x, h, p, t, rep, freq, pres, None, m, "f32")
    hd, pd, td, rd, fd, sd = (G.to_dev(np.ascontiguousarray(v)) for v in (
        h.astype(np.int32), np.asarray(p, np.int32), np.asarray(t, np.int32), np.asarray(rep, np.float32),
        np.asarray(freq, np.float32), np.asarray(pres, np.float32)))
    md = G.to_dev(m.view(np.int32))
    sets = [(G.to_dev(x), torch.zeros((rows, vocab), device=G.dev()), torch.zeros(rows, dtype=torch.int32, device=G.dev()))
            for _ in range(3)]

    def go(stream, xd, out, best):
        A.call("arcllm_cuda_logits_process", A.GGML_F32, G.ptr(xd), vocab, rows, vocab, G.ptr(hd), hist, G.ptr(pd),
               G.ptr(td), G.ptr(rd), G.ptr(fd), G.ptr(sd), None, None, None, G.ptr(md), m.shape[1], G.ptr(out), vocab,
               G.ptr(best), C.c_void_p(stream.cuda_stream))

    streams = [torch.cuda.Stream() for _ in range(2)]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=streams[0]):
        go(streams[0], *sets[2])
    for _ in range(5):
        for st, v in zip(streams, sets):
            go(st, *v)
        g.replay()
    torch.cuda.synchronize()
    for _, out, best in sets:
        assert (out.cpu() == want).all() and best.tolist() == pick
