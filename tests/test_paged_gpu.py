"""The operators of a batch over a paged cache against plain forms in 64 bits:
the step plan, the rotary store, the attention of new rows, and all of them
together in a captured step."""
import ctypes as C
import random

import pytest
import torch

import arcllm_b200 as A
import gpu_util as G
import paged_util as P

pytestmark = pytest.mark.gpu


# ---- plan -------------------------------------------------------------------
@pytest.mark.parametrize("n,page,most_kv,most_new,spare", [(1, 16, 0, 1, 0), (1, 16, 40, 1, 5), (7, 16, 300, 40, 3),
                                                           (64, 48, 900, 1, 0), (300, 128, 500, 9, 1000),
                                                           (4097, 16, 50, 3, 1), (8192, 1, 5, 2, 0)])
def test_plan(n, page, most_kv, most_new, spare):
    r = random.Random(n)
    kv = [r.choice([0, page, r.randint(0, most_kv)]) for _ in range(n)]
    new = [r.choice([0, 1, r.randint(0, most_new)]) for _ in range(n)]
    width = max(-(-(a + b) // page) for a, b in zip(kv, new)) + 1
    used = sum(-(-a // page) for a in kv)
    need = sum(-(-(a + b) // page) for a, b in zip(kv, new)) - used
    pages = list(range(used + need + 2))
    r.shuffle(pages)
    table, at = [], 0
    for a in kv:
        k = -(-a // page)
        table.append(pages[at:at + k] + [-9] * (width - k))
        at += k
    rows = max(1, sum(new) + spare)
    td = torch.tensor(table, dtype=torch.int32, device=G.dev())
    got = P.plan(kv, new, page, len(pages), pages[used:], td, rows)
    assert got == P.plan_plain(kv, new, page, pages[used:], table, rows)
    assert G.host(td).tolist() == table
    assert P.device_error() == 0


@pytest.mark.parametrize("kv,new,rows,free,width,n_free",
                         [([5, 20], [4, 60], 63, 8, 8, None), ([5, 20], [4, 60], 64, 2, 8, None),
                          ([5, 20], [4, 60], 64, 8, 4, None), ([5, -1], [4, 60], 64, 8, 8, None),
                          ([5, 20], [4, -60], 64, 8, 8, None), ([5, 2 ** 31 - 1], [4, 1], 64, 8, 8, None),
                          ([5, 20], [4, 60], 64, 8, 8, -1)])
def test_plan_of_a_step_that_does_not_fit_is_empty(kv, new, rows, free, width, n_free):
    td = torch.full((2, width), 3, dtype=torch.int32, device=G.dev())
    got = P.plan(kv, new, 16, 40, list(range(10, 10 + free)), td, rows, n_free)
    assert got == dict(row_start=[0, 0, 0], kv_total=kv, positions=[0] * rows, slots=[-1] * rows,
                       n_free_out=[free if n_free is None else n_free])
    assert (G.host(td) == 3).all()
    assert P.device_error() == P.BOUNDS and P.device_error() == 0


def test_plan_with_page_numbers_outside_the_cache():
    table = [[99, -9], [3, -9]]
    td = torch.tensor(table, dtype=torch.int32, device=G.dev())
    got = P.plan([5, 16], [2, 2], 16, 40, [1, 40], td, 4)
    assert got["slots"] == [-1] * 4 and got["row_start"] == [0, 2, 4]  # an old page, then a free one
    assert P.device_error() == P.BOUNDS
    got = P.plan([5, 16], [2, 2], 16, 100, [1, 40], td, 4)
    assert got["slots"] == [99 * 16 + 5, 99 * 16 + 6, 640, 641] and P.device_error() == 0


# ---- rotary store -----------------------------------------------------------
def rope_case(act, name, q_heads, heads, dim, rot, half, page, heads_first, bias, rows, scaling=A.ROPE_NONE, off=0,
              pad=0, far=20000, in_place=False):
    qn, kn = q_heads * dim, heads * dim
    x = P.normal((rows, qn + 2 * kn), 3, act, 2.0)
    wide = torch.full((rows, qn + 2 * kn + off + pad), 9.0, dtype=P.DT[act])
    wide[:, off:off + x.shape[1]] = x
    xd = P.dev(wide)[:, off:off + x.shape[1]]
    b = [P.normal((n,), 5, "f32") if bias else None for n in (qn, kn, kn)]
    bd = [None if t is None else P.dev(t) for t in b]
    n_pages = -(-rows // page) + 3
    cache = P.Cache(n_pages, page, heads, dim, name, heads_first, 5.0)
    r = random.Random(rows)
    slots = r.sample(range(n_pages * page), rows)
    pos = [r.randint(0, far) for _ in range(rows)]
    gone = [i for i in range(rows) if i % 5 == 4]  # rows without a request
    for i in gone:
        slots[i] = -1
    f, s = P.frequencies(rot, scaling)
    fd, sd, pd = P.dev(f), P.i32(slots), P.i32(pos)
    q, k, v = xd[:, :qn], xd[:, qn:qn + kn], xd[:, qn + kn:]
    out = q if in_place else torch.full((rows, qn + 8), 5.0, dtype=P.DT[name], device=G.dev())[:, :qn]
    before = out.float().cpu().clone()
    A.call("arcllm_cuda_rope_kv_paged", P.GGML[act], G.ptr(q), q.stride(0), G.ptr(k), k.stride(0), G.ptr(v),
           v.stride(0), G.ptr(bd[0]), G.ptr(bd[1]), G.ptr(bd[2]), G.ptr(fd), rot, int(half), s, G.ptr(pd), G.ptr(sd),
           rows, q_heads, cache.ref(), G.ptr(out), out.stride(0), G.stream())
    torch.cuda.synchronize()
    y = [t.double() for t in x.split([qn, kn, kn], 1)]
    y = [(t + (0 if u is None else u.double())).view(rows, -1, dim) for t, u in zip(y, b)]
    size = [t.abs() for t in y]
    p = torch.tensor(pos)
    want = [P.rotate(y[0], p, f, s, half), P.rotate(y[1], p, f, s, half), y[2]]
    # half a step of the result; before it fp32: the sum with the bias, cos and sin (2^-22 each), two products, a sum
    h = P.half_step(name)
    tol = []
    for t, m in zip(want, size):
        pair = m.amax(-1, keepdim=True) * 2 * s
        tol.append(h * t.abs() + 2.0 ** -20 * pair + (2.0 ** -24 if name == "f16" else 0))
    got_q = out.float().cpu().double().view(rows, q_heads, dim)
    live = [i for i in range(rows) if i not in gone]
    assert ((got_q - want[0])[live].abs() <= tol[0][live]).all()
    assert (out.float().cpu()[gone] == before[gone]).all()
    for pages, t, e in ((cache.k, want[1], tol[1]), (cache.v, want[2], tol[2])):
        flat = pages.float().cpu().double().reshape(n_pages * page, heads, dim)
        idx = [slots[i] for i in live]
        assert ((flat[idx] - t[live]).abs() <= e[live]).all()
        rest = [i for i in range(n_pages * page) if i not in set(idx)]
        assert (flat[rest] == 5.0).all()
    assert P.device_error() == 0


@pytest.mark.parametrize("act,name", [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "bf16"),
                                      ("bf16", "bf16"), ("bf16", "f16")])
@pytest.mark.parametrize("half", [False, True])
def test_rope_store_types(act, name, half):
    rope_case(act, name, 7, 1, 128, 128, half, 16, False, True, 11)


@pytest.mark.parametrize("q_heads,heads,dim,rot,page,heads_first,rows,scaling",
                         [(28, 4, 128, 128, 16, False, 1, A.ROPE_NONE), (28, 4, 128, 32, 48, True, 37, A.ROPE_LINEAR),
                          (4, 4, 64, 16, 128, True, 130, A.ROPE_NTK), (3, 1, 64, 64, 16, False, 700, A.ROPE_YARN),
                          (32, 8, 128, 64, 64, True, 600, A.ROPE_YARN), (1, 1, 16, 16, 1, False, 5, A.ROPE_NONE)])
@pytest.mark.parametrize("half", [False, True])
def test_rope_store_shapes(q_heads, heads, dim, rot, page, heads_first, rows, scaling, half):
    rope_case("bf16", "bf16", q_heads, heads, dim, rot, half, page, heads_first, rows % 2 == 1, rows, scaling)


@pytest.mark.parametrize("dim,rot,off,pad", [(128, 128, 1, 0), (128, 128, 0, 3), (96, 24, 0, 0), (10, 6, 0, 0),
                                             (2, 2, 1, 1), (64, 2, 0, 0)])
@pytest.mark.parametrize("half", [False, True])
def test_rope_store_element_by_element(dim, rot, off, pad, half):
    """Rows, heads or rotated parts that do not fall on 16 bytes."""
    rope_case("f32", "f16", 5, 2, dim, rot, half, 7, False, True, 9, off=off, pad=pad)


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_rope_in_place_and_far_positions(name):
    rope_case(name, name, 8, 2, 128, 128, True, 16, True, False, 21, in_place=True)
    rope_case("f32", name, 8, 2, 128, 64, False, 16, True, False, 21, far=2 ** 31 - 1)


def test_rope_of_one_projection_in_place_captured_and_on_two_streams():
    """q, k, v as parts of the same rows, q rotated where it stands; every way of calling gives the same bits."""
    rows, qh, heads, dim, name = 70, 6, 2, 128, "bf16"
    qn, kn = qh * dim, heads * dim
    x = P.normal((rows, qn + 2 * kn), 31, name)
    pos = torch.arange(rows) * 1000
    f, s = P.frequencies(dim)
    fd, pd, sd = P.dev(f), P.i32(pos.tolist()), P.i32(range(rows))
    want = P.rotate(x[:, :qn].double().view(rows, qh, dim), pos, f, s, True)

    def go(stream, xd, cache):
        A.call("arcllm_cuda_rope_kv_paged", P.GGML[name], G.ptr(xd), xd.stride(0), G.ptr(xd[:, qn:]), xd.stride(0),
               G.ptr(xd[:, qn + kn:]), xd.stride(0), None, None, None, G.ptr(fd), dim, A.ROPE_HALVES, s, G.ptr(pd),
               G.ptr(sd), rows, qh, cache.ref(), G.ptr(xd), xd.stride(0), C.c_void_p(stream.cuda_stream))

    sets = [(P.dev(x), P.Cache(5, 16, heads, dim, name, i == 1)) for i in range(3)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=streams[0]):
        go(streams[0], *sets[2])
    assert (sets[2][0].cpu() == x).all()
    for st, v in zip(streams, sets):
        go(st, *v)
    g.replay()
    torch.cuda.synchronize()
    first = sets[0][0].cpu()
    # one product each and their sum in fp32, angles and their sines to 2^-22, then the type's half step
    size = x[:, :qn].double().view(rows, qh, dim).abs()
    tol = P.half_step(name) * want.abs() + (size + size.roll(dim // 2, -1)) * 2.0 ** -20
    assert ((first[:, :qn].double().view(rows, qh, dim) - want).abs() <= tol).all()
    assert (first[:, qn:] == x[:, qn:]).all()
    for xd, cache in sets:
        assert (xd.cpu() == first).all()
        assert (cache.v.reshape(-1, heads, dim)[:rows].cpu().flatten(1) == x[:, qn + kn:]).all()
        assert (cache.k.reshape(-1, heads, dim)[:rows] == sets[0][1].k.reshape(-1, heads, dim)[:rows]).all()
    assert P.device_error() == 0


def test_rope_slots_outside_the_cache_are_skipped():
    cache = P.Cache(2, 16, 1, 64, "f16", False, 5.0)
    x = torch.zeros((4, 64), dtype=torch.float16, device=G.dev())
    out = torch.full((4, 64), 5.0, dtype=torch.float16, device=G.dev())
    f, s = P.frequencies(64)
    fd = P.dev(f)
    for slots, pos in (([32, 1, 2 ** 31 - 1, 3], [0, 1, 2, 3]), ([0, 1, 2, 3], [-1, 1, -2 ** 31, 3])):
        out.fill_(5.0)
        cache.k.fill_(5.0)
        sd, pd = P.i32(slots), P.i32(pos)
        A.call("arcllm_cuda_rope_kv_paged", A.GGML_F16, G.ptr(x), 64, G.ptr(x), 64, G.ptr(x), 64, None, None, None,
               G.ptr(fd), 64, 1, s, G.ptr(pd), G.ptr(sd), 4, 1, cache.ref(), G.ptr(out), 64, G.stream())
        assert G.host(out)[:, 0].tolist() == [5, 0, 5, 0]
        assert (G.host(cache.k.float()).reshape(32, 64)[[1, 3]] == 0).all()
        assert (G.host(cache.k.float()).reshape(32, 64)[[0, 2] + list(range(4, 32))] == 5).all()
        assert P.device_error() == P.BOUNDS


# ---- attention --------------------------------------------------------------
FEW = [(0, 1), (1, 1), (14, 1), (15, 1), (16, 1), (500, 1), (127, 1), (63, 2), (0, 2), (3, 0), (0, 0), (1000, 1)]
MANY = [(0, 17), (0, 128), (1, 129), (130, 33), (255, 300), (0, 0), (1000, 40), (77, 600)]


@pytest.mark.parametrize("name", ["f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads,gq,page,heads_first", [(2, 2, 16, False), (4, 7, 16, True), (1, 1, 48, False),
                                                       (1, 8, 64, True), (3, 5, 128, False)])
def test_attention_few_rows(name, dim, heads, gq, page, heads_first):
    lens = [(a, b if b * gq <= 16 else 1) for a, b in FEW]
    b = P.Batch(lens, heads, gq, dim, page, name, heads_first)
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("name,dim", [("f16", 128), ("bf16", 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (16, 0), (100, 4), (100, 130), (5000, 4),
                                          (2 ** 32 - 1, 2 ** 32 - 1)])
def test_attention_few_rows_window(name, dim, window, sinks):
    b = P.Batch(FEW, 2, 4, dim, 16, name, window=window, sinks=sinks)
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("lens", [[(0, 1)], [(4000, 1)], [(20000, 1)], [(70, 1)] * 600, [(0, 1)] * 300 + [(9000, 1)],
                                  [(3, 0)] * 50 + [(700, 1)] + [(3, 0)] * 50])
def test_attention_few_rows_lengths(lens):
    b = P.Batch(lens, 1, 7, 128, 16, "bf16")
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("heads,gq,page,heads_first,name,dim",
                         [(2, 2, 16, False, "f16", 128), (1, 7, 16, True, "bf16", 128), (1, 1, 48, False, "bf16", 64),
                          (2, 1, 64, True, "f16", 64), (1, 16, 128, False, "f16", 128), (1, 5, 256, True, "bf16", 64),
                          (1, 24, 16, False, "bf16", 128), (1, 128, 32, False, "f16", 64)])
def test_attention_many_rows(heads, gq, page, heads_first, name, dim):
    lens = [(a, n) for a, n in MANY if n * gq <= 2600] + [(200, 1), (5, 2)]
    b = P.Batch(lens, heads, gq, dim, page, name, heads_first)
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("window,sinks,page", [(1, 0, 16), (64, 0, 48), (64, 1, 16), (129, 4, 16), (200, 130, 64),
                                               (128, 257, 32), (4096, 4, 16),
                                               (2 ** 32 - 1, 0, 16), (100, 2 ** 32 - 1, 16)])
@pytest.mark.parametrize("name,dim", [("bf16", 128), ("f16", 64)])
def test_attention_many_rows_window(window, sinks, page, name, dim):
    b = P.Batch(MANY + [(900, 1), (2000, 30)], 1, 3, dim, page, name, window=window, sinks=sinks)
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("lens", [[(0, 1500)], [(6000, 20)], [(3, 5), (0, 1), (9000, 64)], [(0, 40)] * 60])
def test_attention_many_rows_lengths(lens):
    b = P.Batch(lens, 1, 4, 128, 16, "bf16")
    b.call()
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("lens", [[(300, 1), (40, 2)], [(300, 50), (40, 1)]])
def test_attention_sharp_scores(lens):
    """Scores of several hundred: the running maximum moves far and often."""
    b = P.Batch(lens, 2, 4, 128, 16, "f16", sigma=6.0)
    b.call()
    b.check()


def test_attention_of_requests_that_do_not_fit():
    b = P.Batch([(40, 2), (3, 4), (50, 30), (9, 1)], 1, 4)
    b.kv_total[1] = 3  # fewer positions than rows
    b.call()
    b.check(skip=(1,))
    assert P.device_error() == P.BOUNDS
    b.kv_total[1], b.kv_total[2] = 7, b.page * b.width + 1  # a table row too short
    b.out.fill_(5.0)
    b.call()
    b.check(skip=(2,))
    assert P.device_error() == P.BOUNDS
    b.kv_total[2] = 80
    b.out.fill_(5.0)
    b.call(max_new=29)
    b.check(skip=(2,))
    assert P.device_error() == P.BOUNDS


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, -2 ** 31])
def test_attention_page_outside_the_cache_reads_zeros(new, bad):
    b = P.Batch([(40, new), (33, 1)], 1, 4)
    b.k[0][16:32], b.v[0][16:32] = 0, 0
    b.table[0, 1] = bad
    b.call()
    b.check()
    assert P.device_error() == P.BOUNDS


def test_attention_offsets_past_32_bits():
    """Pages 2^31 elements apart."""
    page, heads, dim = 16, 1, 128
    stride = 2 ** 31 + 64
    raw = torch.empty(2 * stride + 9 * page * dim, dtype=torch.float16, device=G.dev())
    for lens in ([(40, 1)], [(20, 28)]):
        b = P.Batch(lens, heads, 4, dim, page, "f16")
        k, v = (raw.as_strided((3, page, heads, dim), (stride, dim, dim, 1), at) for at in (0, 8 * dim * page))
        kv = [(b.k[0], k), (b.v[0], v)]
        table = [2, 0, 1]
        for host, pages in kv:
            pages.fill_(float("nan"))
            for i, p in enumerate(table):
                part = host[16 * i:16 * i + 16]
                pages[p, :len(part)] = P.dev(part)
        b.cache.k, b.cache.v = k, v
        b.table[0, :3] = P.i32(table)
        b.call()
        b.check()
        assert P.device_error() == 0


def test_attention_other_stream_and_replay():
    """A captured call replays with other lengths; two streams with a workspace each."""
    b = P.Batch([(700, 1), (30, 40), (90, 1)], 2, 4, name="bf16")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        b.call(C.c_void_p(s.cuda_stream))
    g.replay()
    b.check()
    c = P.Batch([(11, 40), (500, 1), (260, 1)], 2, 4, name="bf16", seed=2)
    b.cache.k[:c.cache.n_pages], b.cache.v[:c.cache.n_pages] = c.cache.k[:b.cache.n_pages], c.cache.v[:b.cache.n_pages]
    b.table.fill_(-1)
    w = min(b.width, c.width)
    b.table[:, :w] = c.table[:, :w]
    for name in ("row_start", "kv_total", "qd"):
        getattr(b, name).copy_(getattr(c, name))
    b.out.fill_(5.0)
    g.replay()
    c.out.copy_(b.out)
    c.check()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [P.Batch([(900, 1), (5, 70)], 1, 8, seed=3 + i) for i in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, x in zip(streams, both):
            x.call(C.c_void_p(st.cuda_stream))
    torch.cuda.synchronize()
    for x in both:
        x.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("lens", [[(5, 1)] * 4096, [(2, 17)] * 400 + [(0, 0)] * 3000 + [(40, 1)]])
def test_attention_many_requests(lens):
    b = P.Batch(lens, 1, 1, 64, 16, "f16")
    b.call(max_new=2 ** 32 - 1)
    b.check()
    assert P.device_error() == 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,gq", [([(0, 17)], 1), ([(9, 1)], 20), ([(0, 6)], 3)])
def test_attention_fewer_rows_than_a_tile_takes(dim, lens, gq):
    b = P.Batch(lens, 1, gq, dim, 16, "bf16", spare_rows=0)
    b.call()
    b.check()
    assert P.device_error() == 0


def test_attention_beside_q_in_one_array():
    """q and out as parts of the same rows."""
    b = P.Batch([(30, 40), (90, 1)], 2, 4, dim=64)
    n = b.qh * 64
    both = torch.full((b.rows + 3, 2 * n + 8), 5.0, dtype=torch.float16, device=G.dev())
    both[:b.rows, :n] = P.dev(b.q.flatten(1))
    b.qd, b.out = both[:, :n], both[:, n:2 * n]
    b.call()
    b.out = torch.cat([b.out, torch.full_like(b.out, 5.0)], 1)
    b.check()


@pytest.mark.parametrize("lens", [[(100, 1), (40, 1)], [(100, 50), (40, 1)]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_attention_of_scores_that_are_no_numbers(lens, bad):
    """A query, or a visible key, that is not finite: the rows whose scores are NaN or +inf for it have no softmax (a
    score of -inf, where q is negative, only has no weight), the others are as they were."""
    b = P.Batch(lens, 1, 4)
    b.qd[0, 3] = bad  # row 0, head 0
    page = int(b.table[1, 1])
    b.cache.k[page, 2, 0, 7] = bad  # position 18 of request 1
    b.q[0, 0] = 0  # the plain form's place for it
    b.call()
    got = b.out.float().cpu()
    rows = b.rows - 1
    assert not torch.isfinite(got[0, :128]).any()
    for h in range(4):
        none = bad != bad or b.q[rows, h, 7] > 0
        assert torch.isfinite(got[rows, 128 * h:128 * h + 128]).any() != none
    want, tol = P.attention_plain(b.q[:rows], b.k[0], b.v[0], torch.arange(100, 100 + rows), b.scale, 0, 0, "f16")
    off = (got[:rows, :512].double().view(rows, 4, 128) - want).abs() <= tol
    off[0, 0] = True
    assert off.all()


def test_attention_repeats_bit_for_bit():
    b = P.Batch([(3000, 1), (30, 400), (90, 1)], 2, 7, name="bf16")
    b.call()
    first = G.host(b.out.view(torch.int16)).copy()
    for _ in range(3):
        b.call()
        assert (G.host(b.out.view(torch.int16)) == first).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1024, 4)])
def test_attention_long_work_repeats_bit_for_bit(dim, window, sinks):
    """Enough tiles per SM for its warps to drift apart."""
    b = P.Batch([(2500, 700), (100, 900)], 8, 2, dim, 32, "bf16", window=window, sinks=sinks)
    b.call()
    b.check()
    first = b.out.view(torch.int16).clone()
    for _ in range(200):
        b.out.fill_(5.0)
        b.call()
        assert torch.equal(b.out.view(torch.int16), first)
    assert P.device_error() == 0


# ---- all of them together ---------------------------------------------------
def test_steps_of_a_batch():
    """Prompts, then tokens, through plan, rotary store, attention and the
    constrained choice, in one captured step replayed with new lengths; K and V
    of every request are kept apart, in 64 bits, beside it."""
    qh, heads, dim, page, name, vocab, n = 8, 2, 64, 16, "bf16", 500, 3
    d = G.dev()
    n_pages, width, cap = 24, 8, 40
    free = P.i32(reversed(range(n_pages)))
    kv_len, new_len, n_free = P.i32([0] * n), P.i32([0] * n), P.i32([n_pages])
    table = torch.full((n, width), -1, dtype=torch.int32, device=d)
    row_start, kv_total, n_out = P.i32([0] * (n + 1)), P.i32([0] * n), P.i32([0])
    positions, slots = P.i32([0] * cap), P.i32([0] * cap)
    cache = P.Cache(n_pages, page, heads, dim, name, True)
    qn, kn = qh * dim, heads * dim
    x = torch.zeros((cap, qn + 2 * kn), device=d)
    q = torch.zeros((cap, qn), dtype=P.DT[name], device=d)
    out = torch.zeros((cap, qn), dtype=P.DT[name], device=d)
    f, s = P.frequencies(dim)
    fd = P.dev(f)
    size = C.c_uint64()
    A.call("arcllm_cuda_attention_paged_workspace", qh, heads, dim, C.byref(size))
    ws = torch.empty(size.value, dtype=torch.uint8, device=d)
    logits = torch.zeros((n, vocab), device=d)
    history = torch.zeros((n, 64), dtype=torch.int32, device=d)
    said = P.i32([0] * n)
    rep = torch.full((n,), 1.7, device=d)
    best = P.i32([0] * n)
    done = torch.zeros_like(logits)

    def step(st):
        A.call("arcllm_cuda_paged_plan", G.ptr(kv_len), G.ptr(new_len), n, page, n_pages, G.ptr(free), G.ptr(n_free),
               G.ptr(table), width, cap, G.ptr(row_start), G.ptr(kv_total), G.ptr(positions), G.ptr(slots),
               G.ptr(n_out), st)
        A.call("arcllm_cuda_rope_kv_paged", A.GGML_F32, G.ptr(x), x.stride(0), G.ptr(x[:, qn:]), x.stride(0),
               G.ptr(x[:, qn + kn:]), x.stride(0), None, None, None, G.ptr(fd), dim, A.ROPE_HALVES, s,
               G.ptr(positions), G.ptr(slots), cap, qh, cache.ref(), G.ptr(q), qn, st)
        A.call("arcllm_cuda_attention_paged", G.ptr(q), qn, cache.ref(), G.ptr(table), width, G.ptr(row_start),
               G.ptr(kv_total), n, cap, cap, qh, dim ** -0.5, 0, 0, G.ptr(out), qn, G.ptr(ws), ws.numel(), st)
        A.call("arcllm_cuda_logits_process", A.GGML_F32, G.ptr(logits), vocab, n, vocab, G.ptr(history), 64, None,
               G.ptr(said), G.ptr(rep), None, None, None, None, None, None, 0, G.ptr(done), vocab, G.ptr(best), st)

    stream = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        step(C.c_void_p(stream.cuda_stream))
    ks, vs = [[torch.zeros((0, heads, dim), dtype=torch.float64)] * n for _ in range(2)]
    lens = [0] * n
    tokens = [[] for _ in range(n)]
    rnd = torch.Generator().manual_seed(4)
    for new in ([17, 1, 9], [1, 1, 1], [1, 0, 20], [1, 30, 1], [0, 1, 0], [1, 1, 1]):
        rows = sum(new)
        kv_len.copy_(P.i32(lens))
        new_len.copy_(P.i32(new))
        xh = torch.randn((cap, qn + 2 * kn), generator=rnd)
        x.copy_(xh)
        lh = torch.randn((n, vocab), generator=rnd)
        logits.copy_(lh)
        out.fill_(5.0)
        g.replay()
        n_free.copy_(n_out)
        torch.cuda.synchronize()
        got, at = out.float().cpu().double(), 0
        for r, m in enumerate(new):
            pos = torch.arange(lens[r], lens[r] + m)
            part = xh[at:at + m].double()
            qr = P.rotate(part[:, :qn].view(m, qh, dim), pos, f, s, True).to(P.DT[name])
            kr = P.rotate(part[:, qn:qn + kn].view(m, heads, dim), pos, f, s, True).to(P.DT[name])
            ks[r] = torch.cat([ks[r], kr.double()])
            vs[r] = torch.cat([vs[r], part[:, qn + kn:].view(m, heads, dim).to(P.DT[name]).double()])
            if m:
                want, tol = P.attention_plain(qr, ks[r], vs[r], pos, dim ** -0.5, 0, 0, name)
                # a q or k element near the middle of two values may round the other way: one step, 2h of itself, in
                # one of the factors of a score, which moves the weights by no more than as many of the score
                tol = tol + 4 * P.half_step(name) * want.abs().amax() * 4
                assert ((got[at:at + m].view(m, qh, dim) - want).abs() <= tol).all()
            lens[r] += m
            at += m
        assert (got[rows:] == 5.0).all()
        for r in range(n):
            y = lh[r].clone()
            for t in set(tokens[r]):
                y[t] = y[t] / 1.7 if y[t] > 0 else y[t] * 1.7
            assert int(best[r]) == int(y.argmax())
            tokens[r].append(int(best[r]))
            history[r, len(tokens[r]) - 1] = tokens[r][-1]
        said.copy_(P.i32(len(t) for t in tokens))
    assert int(n_free) == n_pages - sum(-(-a // page) for a in lens)
    assert P.device_error() == 0
