"""Plain forms in 64 bits of the paged-cache operators, and the inputs of their
GPU tests.  Everything here is computed on the CPU."""
import ctypes as C
import math

import numpy as np
import torch

import arcllm_b200 as A
import gpu_util as G

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": A.GGML_F32, "f16": A.GGML_F16, "bf16": A.GGML_BF16}
BOUNDS = 2  # device error word


def half_step(name):
    """Largest relative rounding error of a type."""
    return torch.finfo(DT[name]).eps / 2


def normal(shape, seed, name, sigma=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * sigma).to(DT[name])


def dev(t):
    return t.to(G.dev())


def i32(v):
    return torch.tensor(list(v), dtype=torch.int32, device=G.dev())


def device_error():
    bits = C.c_uint32(0)
    A.call("arcllm_cuda_device_error", G.stream(), C.byref(bits))
    return bits.value


class Cache:
    """Pages of K and V in either order, and their descriptor."""

    def __init__(self, n_pages, page, heads, dim, name, heads_first, fill=float("nan")):
        shape = (n_pages, heads, page, dim) if heads_first else (n_pages, page, heads, dim)
        self.k, self.v = (torch.full(shape, fill, dtype=DT[name], device=G.dev()) for _ in range(2))
        if heads_first:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.page, self.dim, self.heads, self.name, self.n_pages = page, dim, heads, name, n_pages

    def ref(self):
        return paged_kv(self.k, self.v, self.name)


def paged_kv(k, v, name):
    """Descriptor of (pages, tokens, heads, dim) tensors."""
    n, page, heads, dim = k.shape
    return C.byref(A.PagedKV(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), n, page, heads, dim,
                             GGML[name]))


# ---- plan -------------------------------------------------------------------
def plan(kv, new, page, n_pages, free, table, max_rows, n_free=None):
    """One call; table is written.  Returns the outputs on the host."""
    n = len(kv)
    out = dict(row_start=torch.full((n + 1,), 77, dtype=torch.int32, device=G.dev()),
               kv_total=torch.full((n,), 77, dtype=torch.int32, device=G.dev()),
               positions=torch.full((max_rows,), 77, dtype=torch.int32, device=G.dev()),
               slots=torch.full((max_rows,), 77, dtype=torch.int32, device=G.dev()),
               n_free_out=torch.full((1,), 77, dtype=torch.int32, device=G.dev()))
    kvd, nwd = i32(kv), i32(new)
    fr, nf = i32(free if len(free) else [0]), i32([len(free) if n_free is None else n_free])
    A.call("arcllm_cuda_paged_plan", G.ptr(kvd), G.ptr(nwd), n, page, n_pages, G.ptr(fr), G.ptr(nf), G.ptr(table),
           table.shape[1], max_rows, G.ptr(out["row_start"]), G.ptr(out["kv_total"]), G.ptr(out["positions"]),
           G.ptr(out["slots"]), G.ptr(out["n_free_out"]), G.stream())
    return {k: G.host(v).tolist() for k, v in out.items()}


def plan_plain(kv, new, page, free, table, max_rows):
    """The same with lists; table: a list of rows, changed in place."""
    free = list(free)
    start, pos, slot = [0], [], []
    for r, (a, b) in enumerate(zip(kv, new)):
        for i in range(-(-a // page), -(-(a + b) // page)):
            table[r][i] = free.pop()
        for p in range(a, a + b):
            pos.append(p)
            slot.append(table[r][p // page] * page + p % page)
        start.append(start[-1] + b)
    pad = max_rows - len(pos)
    return dict(row_start=start, kv_total=[a + b for a, b in zip(kv, new)], positions=pos + [0] * pad,
                slots=slot + [-1] * pad, n_free_out=[len(free)])


# ---- rotary store -----------------------------------------------------------
def frequencies(rot, scaling=A.ROPE_NONE, theta=1e6, factor=4.0, trained=4096.0):
    f = (C.c_double * (rot // 2))()
    s = C.c_float()
    A.call("arcllm_cuda_rope_freqs", scaling, rot, theta, factor, trained, f, C.byref(s))
    return torch.tensor(list(f), dtype=torch.float64), s.value


def rotate(x, pos, freqs, scale, half):
    """x [rows, heads, dim] in 64 bits, pos [rows]."""
    n = 2 * len(freqs)
    ang = pos.double()[:, None, None] * freqs
    c, s = torch.cos(ang) * scale, torch.sin(ang) * scale
    y = x.clone()
    ia = torch.arange(n // 2) if half else 2 * torch.arange(n // 2)
    ib = ia + n // 2 if half else ia + 1
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y


# ---- attention --------------------------------------------------------------
def visible(pos, n, window, sinks):
    j = torch.arange(n)
    see = j[None] <= pos[:, None]
    if window:
        see &= (j[None] > pos[:, None] - window) | (j[None] < sinks)
    return see


def attention_plain(q, k, v, pos, scale, window, sinks, name):
    """q [rows, q_heads, dim], k and v [positions, heads, dim].  Returns the
    output and how far each element of a kernel's may be from it.

    With w the exact weights: rounding each weight to the type moves an element
    by at most h * sum w|v|, rounding the result by h |o| <= h sum w|v| (1 + h).
    A score is a sum of dim products in fp32, scaled, in units of log 2: off by
    at most (dim + 8) 2^-24 times its sum of absolute products, in any order,
    and so is the running maximum that cancels; a weight, and the sum it is
    divided by, by twice that.  The fp32 sums of weights and of products add
    (positions + 16) 2^-24.  The hardware's exponential is off by at most 2^-21,
    in a weight and in the sum."""
    q, k, v = q.double(), k.double(), v.double()
    g = q.shape[1] // k.shape[1]
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    see = visible(pos, k.shape[0], window, sinks)
    s = torch.einsum("rhd,jhd->hrj", q, kk) * scale
    s = torch.where(see[None], s, -math.inf)
    w = torch.softmax(s, -1)
    out = torch.einsum("hrj,jhd->rhd", w, vv)
    mass = torch.einsum("hrj,jhd->rhd", w, vv.abs())
    big = torch.where(see[None], torch.einsum("rhd,jhd->hrj", q.abs(), kk.abs()) * scale, 0.0).amax(-1).T[..., None]
    h = half_step(name)
    d, n = q.shape[2], k.shape[0]
    rel = 2 * h + h * h + 4 * (d + 8) * 2.0 ** -24 * big + 2 * (n + 16) * 2.0 ** -24
    rel = rel + 2 * 2.0 ** -21
    return out, rel * mass + 1e-30 + (2.0 ** -24 if name == "f16" else 0.0)  # fp16: half of its smallest number, rounded up


class Batch:
    """Requests with (cached, new) lengths over a cache of their own: every
    place that no row may see holds NaN, in the cache, in unused pages and, with
    a window, in pages that have slid out of it (whose table entries are -1)."""

    def __init__(self, lens, heads=2, gq=2, dim=128, page=16, name="f16", heads_first=False, window=0, sinks=0,
                 seed=1, spare_rows=3, evict=True, sigma=1.0):
        self.lens, self.heads, self.gq, self.dim, self.page, self.name = lens, heads, gq, dim, page, name
        self.window, self.sinks = window, sinks
        self.rows = sum(n for _, n in lens)
        rng = np.random.default_rng(seed)
        blocks = [-(-(a + b) // page) for a, b in lens]
        self.width = max(max(blocks), 1) + 2
        self.cache = Cache(sum(blocks) + 4, page, heads, dim, name, heads_first)
        order = rng.permutation(self.cache.n_pages).tolist()
        table = np.full((len(lens), self.width), -1, np.int32)
        self.k, self.v = [], []
        at = 0
        for r, (a, b) in enumerate(lens):
            n = a + b
            k, v = (normal((n, heads, dim), 100 * seed + 10 * r + i, name, sigma if i == 0 else 1.0) for i in (0, 1))
            self.k.append(k)
            self.v.append(v)
            first = max(0, a + 1 - window) if window and b else 0  # the first position that slides in
            for i in range(blocks[r]):
                lo, hi = i * page, min((i + 1) * page, n)
                seen = [j for j in range(lo, hi) if j >= first or j < sinks] if evict else list(range(lo, hi))
                if not seen:
                    continue
                p = order[at]
                at += 1
                table[r, i] = p
                self.cache.k[p, [j - lo for j in seen]] = dev(k[seen])
                self.cache.v[p, [j - lo for j in seen]] = dev(v[seen])
        self.table = torch.from_numpy(table).to(G.dev())
        starts = np.cumsum([0] + [b for _, b in lens])
        self.row_start, self.kv_total = i32(starts), i32(a + b for a, b in lens)
        self.qh = heads * gq
        self.q = normal((self.rows, self.qh, dim), 7777 + seed, name, sigma)
        wide = self.qh * dim + 24  # rows wider than the heads: strides are taken
        self.qd = torch.full((self.rows + spare_rows, wide), float("nan"), dtype=DT[name], device=G.dev())
        self.qd[:self.rows, :self.qh * dim] = dev(self.q.flatten(1))
        self.out = torch.full((self.rows + spare_rows, wide + 8), 5.0, dtype=DT[name], device=G.dev())
        n = C.c_uint64()
        A.call("arcllm_cuda_attention_paged_workspace", self.qh, heads, dim, C.byref(n))
        self.workspace = torch.full((n.value,), 0xA5, dtype=torch.uint8, device=G.dev())
        self.scale = dim ** -0.5
        self.max_new = max(max(b for _, b in lens), 1)

    def call(self, stream=None, max_new=None):
        A.call("arcllm_cuda_attention_paged", G.ptr(self.qd), self.qd.stride(0), self.cache.ref(), G.ptr(self.table),
               self.width, G.ptr(self.row_start), G.ptr(self.kv_total), len(self.lens), self.qd.shape[0],
               max_new or self.max_new, self.qh, self.scale, self.window, self.sinks, G.ptr(self.out),
               self.out.stride(0), G.ptr(self.workspace), self.workspace.numel(), stream or G.stream())

    def check(self, skip=()):
        got = G.host(self.out.float())
        at = 0
        worst = 0.0
        for r, (a, b) in enumerate(self.lens):
            if b and r not in skip:
                pos = torch.arange(a, a + b)
                want, tol = attention_plain(self.q[at:at + b], self.k[r], self.v[r], pos, self.scale, self.window,
                                            self.sinks, self.name)
                have = torch.from_numpy(got[at:at + b, :self.qh * self.dim]).double().view(b, self.qh, self.dim)
                off = (have - want).abs() / tol
                assert torch.isfinite(have).all(), "request %d" % r
                assert off.max() <= 1.0, "request %d: %.2f of the bound" % (r, off.max())
                worst = max(worst, float(off.max()))
            elif r in skip:
                assert (got[at:at + b, :self.qh * self.dim] == 5.0).all()
            at += b
        assert (got[self.rows:] == 5.0).all() and (got[:, self.qh * self.dim:] == 5.0).all()
        return worst
