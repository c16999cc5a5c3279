"""Calls of the paged-cache operators that would write one place twice, leave the
arrays or read words that are not aligned: refused before any device work."""
import itertools
import random

import arcllm_b200 as A
from test_paged_cpu import ALIGN, INVALID, P, SHAPE, changed, kv, status

a = [P(i << 20) for i in range(3, 16)]
ROPE = [A.GGML_F32, a[0], 512, a[1], 512, a[2], 512, None, None, None, a[3], 128, 0, 1.0, a[4], a[5], 3, 4, kv(), a[6],
        512, None]


def rope(**k):
    return status("arcllm_cuda_rope_kv_paged", changed(ROPE, 18, kv(**k)))


def test_store_into_a_cache_whose_places_overlap():
    for k in (dict(kv_heads=4),  # heads and tokens one stride
              dict(kv_heads=4, token_stride=511), dict(page_stride=16 * 128 - 8),
              dict(kv_heads=2, head_stride=16 * 128, page_stride=16 * 128),
              dict(kv_heads=2, head_stride=15 * 128, page_stride=32 * 128),
              dict(page_stride=128, token_stride=7 * 128),  # pages within a token, one too many
              dict(v_pages=1 << 20), dict(v_pages=(1 << 20) + 254), dict(v_pages=(1 << 20) - 7 * 16 * 256)):
        assert rope(**k) == INVALID, k
    for k in (dict(kv_heads=4, token_stride=512, page_stride=16 * 512),
              dict(kv_heads=4, head_stride=16 * 128, page_stride=4 * 16 * 128),
              dict(page_stride=128, token_stride=8 * 128),
              dict(n_pages=1, page_stride=128), dict(page_size=1, token_stride=9999), dict(head_stride=129),
              dict(page_stride=2 * 16 * 128, v_pages=(1 << 20) + 16 * 256),  # K and V of a page in turn
              dict(token_stride=256, page_stride=16 * 256, v_pages=(1 << 20) + 256),  # of a token
              dict(v_pages=(1 << 20) + 8 * 16 * 256), dict(v_pages=(1 << 20) - 8 * 16 * 256)):
        assert rope(**k) not in (INVALID, SHAPE, ALIGN), k


def test_store_into_small_caches_of_every_kind():
    """Refused exactly where two places are one, for strides in any order; layouts that fit without nesting may be
    refused, too."""
    r = random.Random(1)
    seen = set()
    for _ in range(3000):
        pages, page, heads, dim = r.randint(1, 3), r.randint(1, 3), r.randint(1, 3), 2
        strides = [r.choice([2, 2, 4, 6, 8, 12, 18, 24, 36, 54, 3, 5, 7]) for _ in range(3)]
        off = r.choice([0, 1, 2, 3, 4, 6, 8, 12, 24, 54, 60, 108, 200])
        k = [sum(i * s for i, s in zip(at, strides)) + d
             for at in itertools.product(range(pages), range(page), range(heads)) for d in range(dim)]
        twice = len(set(k)) < len(k) or bool(set(k) & {x + off for x in k})
        args = changed(ROPE, 11, 2)
        args[18] = kv(n_pages=pages, page_size=page, kv_heads=heads, head_dim=dim, page_stride=strides[0],
                      token_stride=strides[1], head_stride=strides[2], v_pages=(1 << 20) + 2 * off)
        refused = status("arcllm_cuda_rope_kv_paged", args) == INVALID
        steps = sorted((s, n) for s, n in zip(strides, (pages, page, heads)) if n > 1)
        span, nested = dim, True
        for s, n in steps:
            nested &= s >= span
            span += s * (n - 1)
        assert refused == (twice or not nested), (pages, page, heads, strides, off)
        seen.add((twice, nested))
    assert len(seen) == 4


def test_arrays_that_are_not_aligned_to_their_type():
    """(entry point, a call that passes, {argument: size of a word})"""
    plan = [a[0], a[1], 8, 16, 100, a[2], a[3], a[4], 10, 64, a[5], a[6], a[7], a[8], a[9], None]
    attn = [a[0], 512, kv(), a[1], 9, a[2], a[3], 5, 20, 3, 4, 0.1, 0, 0, a[4], 512, a[5], 1 << 30, None]
    logits = [A.GGML_F16, a[0], 100, 2, 100, a[1], 7, a[2], a[3], a[4], a[5], a[6], a[7], a[8], a[9], a[10], 4, a[11],
              100, a[12], None]
    biased = changed(changed(changed(ROPE, 7, a[7]), 8, a[8]), 9, a[9])
    half = changed(ROPE, 0, A.GGML_BF16)
    for f, good, words in (("paged_plan", plan, dict.fromkeys((0, 1, 5, 6, 7, 10, 11, 12, 13, 14), 4)),
                           ("rope_kv_paged", biased, {1: 4, 3: 4, 5: 4, 7: 4, 8: 4, 9: 4, 10: 8, 14: 4, 15: 4, 19: 2}),
                           ("rope_kv_paged", half, {1: 2, 3: 2, 5: 2}),
                           ("attention_paged", attn, {0: 16, 3: 4, 5: 4, 6: 4, 14: 16, 16: 16}),
                           ("logits_process", logits, {1: 2, 17: 2, **dict.fromkeys((5, 7, 8, 9, 10, 11, 12, 13, 14,
                                                                                     15, 19), 4)})):
        for i, n in words.items():
            for off in range(1, n):
                got = status("arcllm_cuda_" + f, changed(good, i, P(good[i].value + off)))
                assert got == ALIGN, (f, i, off, got)
            got = status("arcllm_cuda_" + f, changed(good, i, P(good[i].value + n)))
            assert got not in (ALIGN, INVALID), (f, i, got)
    for k in (dict(k_pages=(1 << 20) + 1), dict(v_pages=(2 << 20) + 1)):
        assert rope(**k) == ALIGN


def test_attention_strides_and_scales_past_what_its_arithmetic_holds():
    """No tensor map steps 2^40 bytes; a scale whose multiple of log2 e is infinite has no scores."""
    f = "arcllm_cuda_attention_paged"
    good = [a[0], 512, kv(), a[1], 9, a[2], a[3], 5, 20, 30, 4, 0.1, 0, 0, a[4], 512, a[5], 1 << 30, None]
    for i in (1, 15):
        assert status(f, changed(good, i, 2 ** 39)) == SHAPE
        assert status(f, changed(good, i, 2 ** 62)) == SHAPE
    assert status(f, changed(good, 11, 2.5e38)) == INVALID
    assert status(f, changed(good, 11, 2.3e38)) not in (INVALID, SHAPE)


def test_plan_into_arrays_that_overlap():
    """Outputs one over another, the table over an input or an output."""
    f = "arcllm_cuda_paged_plan"
    good = [a[0], a[1], 8, 16, 100, a[2], a[3], a[4], 10, 64, a[5], a[6], a[7], a[8], a[9], None]
    size = {0: 32, 1: 32, 6: 4, 7: 320, 10: 36, 11: 32, 12: 256, 13: 256, 14: 4}
    for i in (7, 10, 11, 12, 13, 14):
        for j in size:
            if i == j:
                continue
            for at in (good[j].value, good[j].value + size[j] - 4, good[j].value + 4 - size[i]):
                assert status(f, changed(good, i, P(at))) == INVALID, (i, j, at)
            for at in (good[j].value + size[j], good[j].value - size[i]):
                assert status(f, changed(good, i, P(at))) != INVALID, (i, j, at)
