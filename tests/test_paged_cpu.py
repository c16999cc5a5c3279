"""Host side of the paged-cache operators: refusals (before any device work),
rotary frequencies, workspace sizes."""
import ctypes as C
import math

import pytest

import arcllm_b200 as A

P = C.c_void_p
INVALID, ALIGN, SHAPE = b"ARC_E_INVALID_ARGUMENT", b"ARC_E_ALIGNMENT", b"ARC_E_UNSUPPORTED_SHAPE"


def status(name, args):
    L = A.lib()
    return L.arcllm_cuda_status_string(getattr(L, name)(*args))


def changed(good, at, value):
    bad = list(good)
    bad[at] = value
    return bad


def test_plan_refusals():
    f = "arcllm_cuda_paged_plan"
    # kv_len, new_len, n, page, n_pages, free, n_free, table, stride, max_rows, row_start, total, positions, slots, n_out
    good = [P(1 << 20), P(2 << 20), 8, 16, 100, P(3 << 20), P(4 << 20), P(5 << 20), 10, 64, P(6 << 20), P(7 << 20),
            P(8 << 20), P(9 << 20), P(10 << 20), None]
    for i in (0, 1, 5, 6, 7, 10, 11, 12, 13, 14):
        assert status(f, changed(good, i, None)) == INVALID, i
    for i in (2, 3, 4, 8, 9):
        assert status(f, changed(good, i, 0)) == INVALID, i
    assert status(f, changed(good, 9, 2 ** 31)) == INVALID
    assert status(f, changed(good, 4, 2 ** 27)) == SHAPE  # 2^31 slots
    assert status(f, changed(good, 2, 8193)) == SHAPE
    assert status(f, changed(good, 14, good[6])) == INVALID  # n_free in place
    assert status(f, changed(good, 11, P((1 << 20) + 28))) == INVALID  # over the last kv_len
    assert status(f, changed(good, 12, P((2 << 20) - 252))) == INVALID  # 64 positions reach into new_len


def kv(**k):
    d = dict(k_pages=1 << 20, v_pages=2 << 20, page_stride=16 * 128, token_stride=128, head_stride=128, n_pages=8,
             page_size=16, kv_heads=1, head_dim=128, type=A.GGML_F16)
    d.update(k)
    return C.byref(A.PagedKV(**d))


BAD_CACHE = [(dict(k_pages=None), INVALID), (dict(v_pages=None), INVALID), (dict(type=A.GGML_F32), INVALID),
             (dict(n_pages=0), INVALID), (dict(page_size=0), INVALID), (dict(kv_heads=0), INVALID),
             (dict(head_dim=0), INVALID), (dict(n_pages=2 ** 27), SHAPE), (dict(token_stride=127), INVALID),
             (dict(head_stride=100), INVALID), (dict(page_stride=64), INVALID)]


def test_rope_refusals():
    f = "arcllm_cuda_rope_kv_paged"
    a = [P(i << 20) for i in range(3, 12)]
    # act, q, stride, k, stride, v, stride, bq, bk, bv, freqs, rot, layout, scale, positions, slots, rows, q_heads, kv,
    # q_out, stride
    good = [A.GGML_F32, a[0], 512, a[1], 128, a[2], 128, None, None, None, a[3], 128, 0, 1.0, a[4], a[5], 3, 4, kv(),
            a[6], 512, None]
    for i in (1, 3, 5, 10, 14, 15, 18, 19):
        assert status(f, changed(good, i, None)) == INVALID, i
    for i, v in ((0, 12), (2, 511), (4, 127), (6, 127), (20, 511), (11, 0), (11, 127), (11, 130), (12, 2), (17, 0)):
        assert status(f, changed(good, i, v)) == INVALID, (i, v)
    for k, want in BAD_CACHE:
        assert status(f, changed(good, 18, kv(**k))) == want, k
    assert status(f, changed(good, 18, kv(head_dim=5, token_stride=5, head_stride=5))) == INVALID
    assert status(f, changed(good, 16, 0)) == b"ARC_OK"
    same = changed(good, 19, a[0])  # in place, but fp32 q into fp16
    assert status(f, same) == INVALID
    half = changed(same, 0, A.GGML_F16)
    assert status(f, changed(half, 20, 520)) == INVALID  # other rows
    assert status(f, changed(changed(good, 0, A.GGML_F16), 19, P((3 << 20) + 1000))) == INVALID  # half a row on
    assert status(f, changed(good, 19, P((3 << 20) + 2048))) == INVALID  # row 1 of q
    for i in (1, 2):  # k, v: rows of 512 bytes, 3 of them
        assert status(f, changed(good, 19, a[i])) == INVALID
        assert status(f, changed(good, 19, P(((3 + i) << 20) + 1520))) == INVALID
    # q, k, v in one projection's rows (4 + 1 + 1 heads of 128 halves), q in place: not refused, over k refused
    fused = changed(changed(changed(changed(half, 2, 768), 4, 768), 6, 768), 20, 768)
    fused = changed(changed(fused, 3, P((3 << 20) + 1024)), 5, P((3 << 20) + 1280))
    assert status(f, fused) != INVALID
    assert status(f, changed(fused, 19, P((3 << 20) + 16))) == INVALID
    assert status(f, changed(fused, 3, P((3 << 20) + 1008))) == INVALID
    assert status(f, changed(fused, 5, P((3 << 20) + 1536 + 1008))) == INVALID  # the next row's q


def test_attention_refusals():
    f = "arcllm_cuda_attention_paged"
    a = [P(i << 20) for i in range(3, 12)]
    n = C.c_uint64()
    A.call("arcllm_cuda_attention_paged_workspace", 4, 1, 128, C.byref(n))
    # q, stride, kv, table, stride, row_start, total, n, rows, max_new, q_heads, scale, window, sinks, out, stride, ws, bytes
    good = [a[0], 512, kv(), a[1], 9, a[2], a[3], 5, 20, 3, 4, 0.1, 0, 0, a[4], 512, a[5], n.value, None]
    for i in (0, 2, 3, 5, 6, 14, 16):
        assert status(f, changed(good, i, None)) == INVALID, i
    for i, v, want in ((1, 504, INVALID), (15, 504, INVALID), (1, 516, ALIGN), (15, 516, ALIGN), (4, 0, INVALID),
                       (7, 4097, SHAPE), (8, 2 ** 31, INVALID), (10, 0, SHAPE), (11, 0.0, INVALID),
                       (11, -1.0, INVALID), (11, math.inf, INVALID), (11, math.nan, INVALID),
                       (17, n.value - 1, INVALID), (0, P(8), ALIGN), (14, P(8), ALIGN), (16, P(8), ALIGN)):
        assert status(f, changed(good, i, v)) == want, (i, v)
    for k, want in BAD_CACHE + [(dict(head_dim=96), SHAPE), (dict(page_size=24), SHAPE), (dict(k_pages=8), ALIGN),
                                (dict(token_stride=132), ALIGN), (dict(page_stride=2 ** 39), SHAPE),
                                (dict(kv_heads=3), SHAPE)]:
        assert status(f, changed(good, 2, kv(**k))) == want, k
    assert status(f, changed(changed(changed(good, 10, 129), 1, 129 * 128), 15, 129 * 128)) == SHAPE  # heads a group
    for i in (7, 8, 9):
        assert status(f, changed(good, i, 0)) == b"ARC_OK", i  # nothing to do
    assert status(f, changed(good, 14, a[0])) == INVALID  # out is q
    assert status(f, changed(good, 14, P((3 << 20) + 1024 + 512))) == INVALID  # between its rows
    assert status(f, changed(changed(good, 14, P((3 << 20) + 1024)), 15, 520)) == INVALID


def test_attention_workspace():
    n = C.c_uint64()
    w = "arcllm_cuda_attention_paged_workspace"
    A.call(w, 28, 4, 128, C.byref(n))
    assert 0 < n.value <= 64 << 20
    assert status(w, [28, 4, 96, C.byref(n)]) == SHAPE and status(w, [28, 3, 128, C.byref(n)]) == SHAPE
    assert status(w, [28, 0, 128, C.byref(n)]) == SHAPE and status(w, [28, 4, 128, None]) == INVALID


def test_logits_refusals():
    f = "arcllm_cuda_logits_process"
    a = [P(i << 20) for i in range(1, 16)]
    # type, logits, stride, rows, vocab, history, stride, prompt, total, rep, freq, pres, b_start, b_ids, b_values, mask,
    # stride, out, stride, best
    good = [A.GGML_F32, a[0], 100, 2, 100, a[1], 7, a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], 4, a[11],
            100, a[12], None]
    for i in (1, 5, 8, 13, 14, 17):
        assert status(f, changed(good, i, None)) == INVALID, i
    for i, v in ((0, 12), (2, 99), (18, 99), (4, 0), (16, 3), (6, 2 ** 30)):
        assert status(f, changed(good, i, v)) == INVALID, (i, v)
    assert status(f, changed(good, 1, P((1 << 20) + 2))) == ALIGN
    assert status(f, changed(good, 17, P((1 << 20) + 400))) == INVALID  # row 1 of the logits
    assert status(f, changed(changed(good, 17, a[0]), 18, 104)) == INVALID  # the same start, other rows
    assert status(f, changed(good, 3, 0)) == b"ARC_OK"


@pytest.mark.parametrize("rot", [2, 16, 64, 128])
def test_rope_frequencies(rot):
    def freqs(*args):
        f, s = (C.c_double * (rot // 2))(), C.c_float()
        A.call("arcllm_cuda_rope_freqs", *args, f, C.byref(s))
        return list(f), s.value

    def near(got, want):
        assert all(abs(g - w) <= 1e-14 * w for g, w in zip(got, want))

    plain = [1e6 ** (-2 * i / rot) for i in range(rot // 2)]
    got, s = freqs(A.ROPE_NONE, rot, 1e6, 0.0, 0.0)
    near(got, plain)
    assert s == 1.0
    near(freqs(A.ROPE_LINEAR, rot, 1e6, 4.0, 0.0)[0], [x / 4 for x in plain])
    base = 1e6 * 4.0 ** (rot / (rot - 2)) if rot > 2 else 1e6
    near(freqs(A.ROPE_NTK, rot, 1e6, 4.0, 0.0)[0], [base ** (-2 * i / rot) for i in range(rot // 2)])
    got, s = freqs(A.ROPE_YARN, rot, 1e6, 4.0, 4096.0)
    assert abs(s - (0.1 * math.log(4) + 1)) < 1e-7
    turns = [4096 * x / (2 * math.pi) for x in plain]
    for g, x, t in zip(got, plain, turns):  # fast pairs as they are, slow ones / 4, between them in order
        assert x / 4 * (1 - 1e-14) <= g <= x * (1 + 1e-14)
        if t > 60:
            assert abs(g - x) <= 1e-14 * x
        if t < 0.5 and rot >= 16:
            assert abs(g - x / 4) <= 1e-14 * x


def test_rope_frequency_refusals():
    f, s = (C.c_double * 64)(), C.c_float()
    w = "arcllm_cuda_rope_freqs"
    for args in ([4, 128, 1e6, 4.0, 1.0], [-1, 128, 1e6, 4.0, 1.0], [0, 127, 1e6, 1.0, 1.0], [0, 0, 1e6, 1.0, 1.0],
                 [0, 128, 0.0, 1.0, 1.0], [0, 128, math.inf, 1.0, 1.0], [1, 128, 1e6, 0.5, 1.0],
                 [1, 128, 1e6, math.nan, 1.0], [3, 128, 1e6, 4.0, 0.0], [3, 128, 1.0, 4.0, 4096.0]):
        assert status(w, args + [f, C.byref(s)]) == INVALID, args
    assert status(w, [0, 128, 1e6, 1.0, 1.0, None, C.byref(s)]) == INVALID
    assert status(w, [0, 128, 1e6, 1.0, 1.0, f, None]) == INVALID
