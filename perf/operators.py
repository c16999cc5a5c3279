"""Cases, plain forms and calls of the serving operators over a paged KV cache.

One step of a batch of requests: the plan (row offsets, block tables, slots), the rotary embedding with the store
into the pages, the attention of the new rows over them, and the sampling constraints on the logits that come out.
``own`` selects between the plain torch forms and the calls of ``libarcllm_cuda.so``.
"""
import ctypes as C
import random

import torch

own = False

DTYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
SCALING = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}
THETA = 1.0e6


# ---- cases ------------------------------------------------------------------
def listed():
    return [
        # a decode step of a large batch: a request in sixteen needs a new page
        dict(name="plan_decode", op="plan", requests=256, chunks=0, chunk=0, context=8192, page=16, spare=0, lens=1),
        # a step that mixes decodes with chunks of prompts, into buffers of a captured graph's capacity
        dict(name="plan_prompts", op="plan", requests=96, chunks=48, chunk=1024, context=4096, page=16, spare=777,
             lens=2),
        # the decode step of the repository's 28/4-head model: fp32 projections, fp16 cache, 48 requests
        dict(name="rope_decode", op="rope", rows=48, act="f32", type="f16", q_heads=28, kv_heads=4, head_dim=128,
             rot_dim=128, half=False, scaling="none", bias=True, page=16, heads_first=False),
        # a long prompt with a context beyond the trained one, pages by head
        dict(name="rope_prompt", op="rope", rows=8192, act="bf16", type="bf16", q_heads=32, kv_heads=8, head_dim=128,
             rot_dim=128, half=True, scaling="yarn", bias=False, page=64, heads_first=True),
        # an odd number of rows, half of each head rotated
        dict(name="rope_partial", op="rope", rows=777, act="f16", type="f16", q_heads=16, kv_heads=16, head_dim=64,
             rot_dim=32, half=True, scaling="linear", bias=True, page=32, heads_first=False),
        # one user, one token: latency
        dict(name="attention_one", op="attention", requests=1, chunks=0, chunk=0, context=1027, type="f16", q_heads=28,
             kv_heads=4, head_dim=128, page=16, heads_first=False, window=0, sinks=0, lens=3),
        # decode of a batch with ragged contexts: bandwidth
        dict(name="attention_decode", op="attention", requests=64, chunks=0, chunk=0, context=8192, type="bf16",
             q_heads=32, kv_heads=8, head_dim=128, page=64, heads_first=True, window=0, sinks=0, lens=4),
        # decodes and chunks of prompts in one step
        dict(name="attention_mixed", op="attention", requests=33, chunks=8, chunk=509, context=4096, type="f16",
             q_heads=28, kv_heads=4, head_dim=128, page=16, heads_first=False, window=0, sinks=0, lens=5),
        # two long prompts: tensor cores
        dict(name="attention_prompt", op="attention", requests=2, chunks=2, chunk=6000, context=2048, type="bf16",
             q_heads=28, kv_heads=4, head_dim=128, page=16, heads_first=False, window=0, sinks=0, lens=6),
        # a sliding window with the first tokens kept, one KV head per query head
        dict(name="attention_window", op="attention", requests=12, chunks=6, chunk=1500, context=8192, type="bf16",
             q_heads=16, kv_heads=16, head_dim=64, page=32, heads_first=False, window=1024, sinks=4, lens=7),
        # one user's logits (the repository's vocabulary): latency
        dict(name="logits_one", op="logits", rows=1, vocab=152064, type="f32", history=301, biases=0, mask=False,
             lens=8),
        # a batch under a grammar, with biases and long histories
        dict(name="logits_batch", op="logits", rows=128, vocab=152064, type="f32", history=4096, biases=64, mask=True,
             lens=9),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["plan", "rope", "attention", "attention", "logits"])
    seed = rng.randrange(1, 1 << 20)
    if op == "plan":
        n = _log(rng, 1, 512)
        chunks = rng.randint(0, n)
        return dict(op=op, requests=n, chunks=chunks, chunk=_log(rng, 1, max(2, 49152 // max(1, chunks))),
                    context=_log(rng, 1, 8192), page=rng.choice([16, 32, 48, 64, 128]),
                    spare=rng.choice([0, rng.randint(1, 999)]), lens=seed)
    if op == "rope":
        d = rng.choice([64, 128])
        kvh = rng.choice([1, 2, 4, 8])
        return dict(op=op, rows=_log(rng, 1, 8192), act=rng.choice(["f32", "f16", "bf16"]),
                    type=rng.choice(["f16", "bf16"]), q_heads=kvh * rng.choice([1, 3, 4, 7]), kv_heads=kvh, head_dim=d,
                    rot_dim=rng.choice([d, d // 2, d // 4]), half=rng.random() < 0.5,
                    scaling=rng.choice(sorted(SCALING)), bias=rng.random() < 0.5,
                    page=rng.choice([16, 32, 48, 64, 128]), heads_first=rng.random() < 0.5)
    if op == "attention":
        kvh, gq = rng.choice([(1, 8), (1, 5), (2, 2), (4, 7), (4, 1), (8, 4), (2, 16), (8, 1), (4, 6)])
        chunks = rng.choice([0, 0, 1, rng.randint(1, 12)])
        n = chunks + _log(rng, 1, 48) if chunks == 0 or rng.random() < 0.6 else chunks
        context = _log(rng, 1, 8192)
        # the plain form's scores (requests x rows x heads x positions) stay within 6 GB
        most = int(1.5e9 / (n * kvh * gq * (context + 64)))
        chunk = max(2, min(_log(rng, 2, 2048), most // 2)) if chunks else 0
        window = rng.choice([0, 0, _log(rng, 1, 4096)])
        return dict(op=op, requests=n, chunks=chunks, chunk=chunk, context=context,
                    type=rng.choice(["f16", "bf16"]), q_heads=kvh * gq, kv_heads=kvh, head_dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 48, 64, 128]), heads_first=rng.random() < 0.5, window=window,
                    sinks=rng.choice([0, 1, 4, 130]) if window else 0, lens=seed)
    vocab = rng.choice([152064, 4096, 32000, rng.randint(1000, 160000)])
    return dict(op=op, rows=max(1, min(_log(rng, 1, 160), 19000000 // vocab)), vocab=vocab,
                type=rng.choice(["f32", "f16", "bf16"]), history=_log(rng, 1, 4096),
                biases=rng.choice([0, _log(rng, 1, 300)]), mask=rng.random() < 0.5, lens=seed)


def _lengths(c):
    """(cached, new) tokens of each request; they belong to the case, so that its work does."""
    r = random.Random(c["lens"])
    n, new, kv = c["requests"], [], []
    for i in range(n):
        if i < c["chunks"]:
            new.append(max(1, c["chunk"] - (r.randint(0, c["chunk"] // 4) if i else 0)))
            kv.append(r.choice([0, r.randint(0, c["context"])]))
        else:
            new.append(1)
            kv.append(c["context"] - 1 if n == 1 else r.randint(0, c["context"] - 1))
    order = list(range(n))
    r.shuffle(order)
    return [kv[i] for i in order], [new[i] for i in order]


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _normal(shape, g, dtype, sigma=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * sigma).to(dtype)


def _pages(n_pages, c, g, fill=True):
    """(pages, tokens, heads, dim), in memory as the case says."""
    h, p, d = c["kv_heads"], c["page"], c["head_dim"]
    shape = (n_pages, h, p, d) if c["heads_first"] else (n_pages, p, h, d)
    t = _normal(shape, g, DTYPE[c["type"]]) if fill else torch.zeros(shape, dtype=DTYPE[c["type"]], device="cuda")
    return t.transpose(1, 2) if c["heads_first"] else t


# ---- inputs -----------------------------------------------------------------
def prepare(c, seed):
    return {"plan": _prepare_plan, "rope": _prepare_rope, "attention": _prepare_attention,
            "logits": _prepare_logits}[c["op"]](c, seed)


def _tables(kv, page, order, width):
    """block tables of requests with `kv` tokens, pages taken from `order` in turn; and how many were taken"""
    rows, at = [], 0
    for n in kv:
        k = -(-n // page)
        rows.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return _ints(rows), at


def _prepare_plan(c, seed):
    kv, new = _lengths(c)
    p, n = c["page"], c["requests"]
    width = max(-(-(a + b) // p) for a, b in zip(kv, new)) + 3
    n_pages = sum(-(-(a + b) // p) for a, b in zip(kv, new)) + 19
    order = torch.randperm(n_pages, generator=_gen(seed), device="cuda").tolist()
    table, used = _tables(kv, p, order, width)
    rows = sum(new) + c["spare"]
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(c=c, kv_len=_ints(kv), new_len=_ints(new), table=table, free=_ints(order[used:]),
                n_free=_ints([n_pages - used]), n_pages=n_pages, rows=rows, row_start=torch.zeros(n + 1, **i32),
                kv_total=torch.zeros(n, **i32), positions=torch.zeros(rows, **i32), slots=torch.zeros(rows, **i32),
                n_free_out=torch.zeros(1, **i32))


def _frequencies(c):
    """Angle per position of each rotated pair (64 bits) and the factor on cos and sin."""
    import math
    d, kind, factor, trained = c["rot_dim"], c["scaling"], 4.0, 4096.0
    theta = THETA * factor ** (d / (d - 2.0)) if kind == "ntk" and d > 2 else THETA
    f = [theta ** (-2.0 * i / d) for i in range(d // 2)]
    if kind == "linear":
        f = [x / factor for x in f]
    if kind != "yarn":
        return f, 1.0

    def turns_at(turns):  # the pair that turns so often over the trained context
        return d * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(THETA))

    low, high = max(0.0, math.floor(turns_at(32.0))), min(d - 1.0, math.ceil(turns_at(1.0)))
    keep = [1.0 - min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(d // 2)]
    return [x / factor * (1.0 - k) + x * k for x, k in zip(f, keep)], 0.1 * math.log(factor) + 1.0


def _prepare_rope(c, seed):
    g = _gen(seed)
    t, d, act = c["rows"], c["head_dim"], DTYPE[c["act"]]
    qn, kn = c["q_heads"] * d, c["kv_heads"] * d
    qkv = _normal((t, qn + 2 * kn), g, act)  # one projection's output: rows are wider than q, k or v
    n_pages = -(-t // c["page"]) + 7
    slots = torch.randperm(n_pages * c["page"], generator=g, device="cuda")[:t].to(torch.int32)
    positions = torch.randint(0, 16384, (t,), generator=g, device="cuda", dtype=torch.int32)
    bias = [_normal((n,), g, torch.float32, 0.3) if c["bias"] else None for n in (qn, kn, kn)]
    freqs, scale = _frequencies(c)
    return dict(c=c, q=qkv[:, :qn], k=qkv[:, qn:qn + kn], v=qkv[:, qn + kn:], bias=bias, slots=slots,
                positions=positions, freqs=torch.tensor(freqs, dtype=torch.float64, device="cuda"), scale=scale,
                k_pages=_pages(n_pages, c, g, False), v_pages=_pages(n_pages, c, g, False),
                out=torch.zeros((t, qn), dtype=DTYPE[c["type"]], device="cuda"))


def _prepare_attention(c, seed):
    g = _gen(seed)
    kv, new = _lengths(c)
    total = [a + b for a, b in zip(kv, new)]
    p, d, t = c["page"], c["head_dim"], sum(new)
    width = max(-(-n // p) for n in total)
    n_pages = sum(-(-n // p) for n in total) + 5
    table, _ = _tables(total, p, torch.randperm(n_pages, generator=g, device="cuda").tolist(), width)
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(c=c, q=_normal((t, c["q_heads"] * d), g, DTYPE[c["type"]], 1.5), k_pages=_pages(n_pages, c, g),
                v_pages=_pages(n_pages, c, g), table=table, row_start=_ints(start), kv_total=_ints(total), rows=t,
                max_new=max(new), max_kv=max(total), n_pages=n_pages,
                out=torch.zeros((t, c["q_heads"] * d), dtype=DTYPE[c["type"]], device="cuda"),
                workspace=torch.empty(96 << 20, dtype=torch.uint8, device="cuda"))


def _prepare_logits(c, seed):
    g, r = _gen(seed), random.Random(c["lens"])
    n, v, h = c["rows"], c["vocab"], c["history"]
    total = [h if i == 0 else r.randint(0, h) for i in range(n)]
    prompt = [r.randint(0, x) for x in total]
    # tokens of a text repeat: a power law over the vocabulary
    u = torch.rand((n, h), generator=g, device="cuda", dtype=torch.float64)
    history = (u.pow(6) * v).to(torch.int32).clamp_(max=v - 1)
    param = lambda lo, hi: torch.rand(n, generator=g, device="cuda") * (hi - lo) + lo  # noqa: E731
    count = [r.randint(0, c["biases"]) if c["biases"] else 0 for _ in range(n)]
    start = [0]
    for x in count:
        start.append(start[-1] + x)
    s = dict(c=c, logits=_normal((n, v), g, DTYPE[c["type"]], 3.0), history=history, prompt_len=_ints(prompt),
             total_len=_ints(total), repetition=param(1.0, 1.5), frequency=param(0.0, 0.5), presence=param(0.0, 0.5),
             bias_start=None, bias_ids=None, bias_values=None, bias_row=None, mask=None,
             out=torch.zeros((n, v), dtype=DTYPE[c["type"]], device="cuda"),
             best=torch.zeros(n, dtype=torch.int32, device="cuda"))
    if c["biases"]:
        m = start[-1]
        s["bias_start"] = _ints(start)
        s["bias_ids"] = torch.randint(0, v, (m,), generator=g, device="cuda", dtype=torch.int32)
        s["bias_values"] = _normal((m,), g, torch.float32, 4.0)
    if c["mask"]:
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (n, (v + 31) // 32), generator=g, device="cuda",
                                  dtype=torch.int64).to(torch.int32)
    return s


# ---- one pass ---------------------------------------------------------------
def run(s):
    op = s["c"]["op"]
    if own:
        return {"plan": _call_plan, "rope": _call_rope, "attention": _call_attention,
                "logits": _call_logits}[op](s)
    return {"plan": _plain_plan, "rope": _plain_rope, "attention": _plain_attention, "logits": _plain_logits}[op](s)


def _call(name, *args):
    import arcllm_b200
    arcllm_b200.call(name, *args, torch.cuda.current_stream().cuda_stream)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _paged_kv(s):
    import arcllm_b200
    c, k = s["c"], s["k_pages"]
    return C.byref(arcllm_b200.PagedKV(k.data_ptr(), s["v_pages"].data_ptr(), k.stride(0), k.stride(1), k.stride(2),
                                       k.shape[0], c["page"], c["kv_heads"], c["head_dim"], GGML[c["type"]]))


def _call_plan(s):
    c, t = s["c"], s["table"]
    _call("arcllm_cuda_paged_plan", _ptr(s["kv_len"]), _ptr(s["new_len"]), c["requests"], c["page"], s["n_pages"],
          _ptr(s["free"]), _ptr(s["n_free"]), _ptr(t), t.shape[1], s["rows"], _ptr(s["row_start"]),
          _ptr(s["kv_total"]), _ptr(s["positions"]), _ptr(s["slots"]), _ptr(s["n_free_out"]))
    return {k: s[k] for k in ("row_start", "kv_total", "table", "positions", "slots", "n_free_out")}


def _plain_plan(s):
    p, kv, new = s["c"]["page"], s["kv_len"].long(), s["new_len"].long()
    total = kv + new
    end = new.cumsum(0)
    had, need = (kv + p - 1) // p, (total + p - 1) // p
    need = need - had
    first = s["n_free"].long() - 1 - (need.cumsum(0) - need)  # free pages are taken from the end, request by request
    j = torch.arange(s["table"].shape[1], device="cuda")[None] - had[:, None]
    taken = s["free"][(first[:, None] - j).clamp(0, s["free"].numel() - 1)]
    table = torch.where((j >= 0) & (j < need[:, None]), taken, s["table"])
    row = torch.arange(s["rows"], device="cuda")
    used = row < end[-1]
    req = torch.searchsorted(end, row, right=True).clamp(max=kv.numel() - 1)
    pos = kv[req] + row - (end - new)[req]
    slot = table[req, (pos // p).clamp(0, table.shape[1] - 1)].long() * p + pos % p
    i32 = torch.int32
    return dict(row_start=torch.cat([end.new_zeros(1), end]).to(i32), kv_total=total.to(i32), table=table,
                positions=torch.where(used, pos, 0).to(i32), slots=torch.where(used, slot, -1).to(i32),
                n_free_out=(s["n_free"].long() - need.sum()).to(i32))


def _call_rope(s):
    c, b = s["c"], s["bias"]
    _call("arcllm_cuda_rope_kv_paged", GGML[c["act"]], _ptr(s["q"]), s["q"].stride(0), _ptr(s["k"]), s["k"].stride(0),
          _ptr(s["v"]), s["v"].stride(0), _ptr(b[0]), _ptr(b[1]), _ptr(b[2]), _ptr(s["freqs"]), c["rot_dim"],
          int(c["half"]), s["scale"], _ptr(s["positions"]), _ptr(s["slots"]), c["rows"], c["q_heads"], _paged_kv(s),
          _ptr(s["out"]), s["out"].stride(0))
    return s["out"], s["k_pages"], s["v_pages"]


def _rotated(x, heads, s):
    c, n = s["c"], s["c"]["rot_dim"]
    x = x.view(x.shape[0], heads, c["head_dim"])
    angle = s["positions"].double()[:, None] * s["freqs"][None]
    cos, sin = ((f(angle) * s["scale"]).float()[:, None] for f in (torch.cos, torch.sin))
    a, b = (x[..., :n // 2], x[..., n // 2:n]) if c["half"] else (x[..., 0:n:2], x[..., 1:n:2])
    ra, rb = a * cos - b * sin, a * sin + b * cos
    r = torch.cat([ra, rb], -1) if c["half"] else torch.stack([ra, rb], -1).flatten(-2)
    return torch.cat([r, x[..., n:]], -1)


def _plain_rope(s):
    c, (bq, bk, bv) = s["c"], s["bias"]
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    if bq is not None:
        q, k, v = q + bq, k + bk, v + bv
    t = DTYPE[c["type"]]
    page, at = (s["slots"] // c["page"]).long(), (s["slots"] % c["page"]).long()
    s["k_pages"][page, at] = _rotated(k, c["kv_heads"], s).to(t)
    s["v_pages"][page, at] = v.view(-1, c["kv_heads"], c["head_dim"]).to(t)
    return _rotated(q, c["q_heads"], s).flatten(1).to(t), s["k_pages"], s["v_pages"]


def _call_attention(s):
    c, t, w = s["c"], s["table"], s["workspace"]
    _call("arcllm_cuda_attention_paged", _ptr(s["q"]), s["q"].stride(0), _paged_kv(s), _ptr(t), t.shape[1],
          _ptr(s["row_start"]), _ptr(s["kv_total"]), c["requests"], s["rows"], s["max_new"], c["q_heads"],
          c["head_dim"] ** -0.5, c["window"], c["sinks"], _ptr(s["out"]), s["out"].stride(0), _ptr(w), w.numel())
    return s["out"]


def _plain_attention(s):
    c = s["c"]
    n, h, d, hq = c["requests"], c["kv_heads"], c["head_dim"], c["q_heads"]
    g, m, start, total = hq // h, s["max_new"], s["row_start"].long(), s["kv_total"].long()
    new = start[1:] - start[:-1]
    row = (start[:-1, None] + torch.arange(m, device="cuda")).clamp(max=s["rows"] - 1)
    q = s["q"].float().view(-1, h, g, d)[row].permute(0, 2, 3, 1, 4).reshape(n, h, g * m, d)
    blocks = s["table"].clamp(min=0).long()
    k = s["k_pages"][blocks].flatten(1, 2)[:, :s["max_kv"]].float()
    v = s["v_pages"][blocks].flatten(1, 2)[:, :s["max_kv"]].float()
    at = torch.arange(k.shape[1], device="cuda")
    v = torch.where((at < total[:, None])[..., None, None], v, 0.0)
    pos = (total - new)[:, None] + torch.arange(m, device="cuda")  # position of each new row
    see = (at <= pos[..., None]) & (at < total[:, None, None])
    if c["window"]:
        see &= (at > pos[..., None] - c["window"]) | (at < c["sinks"])
    x = torch.matmul(q * d ** -0.5, k.permute(0, 2, 3, 1)).view(n, h, g, m, -1)
    x = torch.where(see[:, None, None], x, -torch.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    o = torch.matmul(x.view(n, h, g * m, -1), v.permute(0, 2, 1, 3)).view(n, h, g, m, d)
    o = o / x.sum(-1, keepdim=True).clamp(min=1e-30)
    t = torch.arange(s["rows"], device="cuda")
    req = torch.searchsorted(start[1:], t, right=True)
    return o.permute(0, 3, 1, 2, 4)[req, t - start[req]].reshape(s["rows"], hq * d).to(DTYPE[c["type"]])


def _call_logits(s):
    c, m = s["c"], s["mask"]
    b = [s[k] for k in ("bias_start", "bias_ids", "bias_values")]
    if b[0] is not None and b[1].numel() == 0:  # no row has an entry: nothing to point at
        b = [None] * 3
    _call("arcllm_cuda_logits_process", GGML[c["type"]], _ptr(s["logits"]), s["logits"].stride(0), c["rows"],
          c["vocab"], _ptr(s["history"]), s["history"].shape[1], _ptr(s["prompt_len"]), _ptr(s["total_len"]),
          _ptr(s["repetition"]), _ptr(s["frequency"]), _ptr(s["presence"]), _ptr(b[0]), _ptr(b[1]), _ptr(b[2]),
          _ptr(m), 0 if m is None else m.shape[1], _ptr(s["out"]), s["out"].stride(0), _ptr(s["best"]))
    return s["out"], s["best"]


def _plain_logits(s):
    c, h = s["c"], s["history"].long()
    x = s["logits"].float()
    at = torch.arange(h.shape[1], device="cuda")[None]
    said, told = at < s["total_len"][:, None], at < s["prompt_len"][:, None]
    count = torch.zeros_like(x).scatter_add_(1, h, (said & ~told).float())
    seen = torch.zeros_like(x).scatter_add_(1, h, said.float()) > 0
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count
    x = torch.where(count > 0, x - s["presence"][:, None], x)
    if s["bias_ids"] is not None:  # of several entries for one token the last one counts
        m = s["bias_ids"].numel()
        i = torch.arange(m, device="cuda")
        row = torch.searchsorted(s["bias_start"][1:], i, right=True)
        last = torch.full((x.numel(),), -1, dtype=torch.long, device="cuda")
        last.scatter_reduce_(0, row * c["vocab"] + s["bias_ids"], i, "amax")
        last = last.view_as(x)
        x = torch.where(last >= 0, x + s["bias_values"][last.clamp(min=0)] if m else x, x)
    if s["mask"] is not None:
        v = torch.arange(c["vocab"], device="cuda")
        x = torch.where((s["mask"][:, v // 32] >> (v % 32)) & 1 == 1, x, -torch.inf)
    x = x.to(DTYPE[c["type"]])
    y = torch.where(torch.isfinite(x), x, -torch.inf)
    top = y.amax(1, keepdim=True)
    first = torch.where(y == top, torch.arange(c["vocab"], device="cuda"), c["vocab"]).amin(1)
    return x, torch.where(top[:, 0] > -torch.inf, first, -1).to(torch.int32)


# ---- the definition in 64 bits ----------------------------------------------
def exact(c, seed):
    if c["op"] == "plan":
        return None  # whole numbers
    s = prepare(c, seed)
    return {"rope": _exact_rope, "attention": _exact_attention, "logits": _exact_logits}[c["op"]](s)


def _exact_rope(s):
    c = s["c"]
    t, d, n = c["rows"], c["head_dim"], c["rot_dim"]
    x = [y.double() + (0.0 if b is None else b.double()) for y, b in zip((s["q"], s["k"], s["v"]), s["bias"])]
    x = [y.reshape(t, -1, d) for y in x]
    turn = s["scale"] * torch.exp(1j * s["positions"].double()[:, None, None] * s["freqs"])
    done = []
    for y in x[:2]:
        pair = torch.stack([y[..., :n // 2], y[..., n // 2:n]], -1) if c["half"] else y[..., :n].unflatten(-1, (-1, 2))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = torch.cat([z[..., 0], z[..., 1]], -1) if c["half"] else z.flatten(-2)
        done.append(torch.cat([z, y[..., n:]], -1))
    pages = []
    for y in (done[1], x[2]):
        whole = torch.zeros((s["k_pages"].shape[0] * c["page"], c["kv_heads"], d), dtype=torch.float64, device="cuda")
        whole[s["slots"].long()] = y
        pages.append(whole.view(s["k_pages"].shape))
    return done[0].flatten(1), pages[0], pages[1]


def _exact_attention(s):
    c, d = s["c"], s["c"]["head_dim"]
    g = c["q_heads"] // c["kv_heads"]
    start, total, table = s["row_start"].tolist(), s["kv_total"].tolist(), s["table"].tolist()
    out = torch.zeros((s["rows"], c["q_heads"], d), dtype=torch.float64, device="cuda")
    for r, n in enumerate(total):
        lo, hi = start[r], start[r + 1]
        used = table[r][:-(-n // c["page"])]
        k, v = (x[used].reshape(-1, c["kv_heads"], d)[:n].double() for x in (s["k_pages"], s["v_pages"]))
        j = torch.arange(n, device="cuda")
        for at in range(lo, hi, 2048):
            rows = slice(at, min(hi, at + 2048))
            i = torch.arange(rows.start, rows.stop, device="cuda")[:, None] - hi + n
            hidden = j > i
            if c["window"]:
                hidden = hidden | ((j <= i - c["window"]) & (j >= c["sinks"]))
            for h in range(c["q_heads"]):
                q = s["q"][rows, h * d:(h + 1) * d].double()
                w = (q @ k[:, h // g].T / d ** 0.5).masked_fill(hidden, float("-inf"))
                out[rows, h] = torch.softmax(w, -1) @ v[:, h // g]
    return out.flatten(1)


def _exact_logits(s):
    c = s["c"]
    x = s["logits"].double()
    total, prompt = s["total_len"].tolist(), s["prompt_len"].tolist()
    for r in range(c["rows"]):
        ids, count = s["history"][r, prompt[r]:total[r]].long().unique(return_counts=True)
        seen = s["history"][r, :total[r]].long().unique()
        y = x[r, seen]
        rep = s["repetition"][r].double()
        x[r, seen] = torch.where(y > 0, y / rep, y * rep)
        x[r, ids] -= s["frequency"][r].double() * count + s["presence"][r].double()
        if s["bias_ids"] is not None:
            lo, hi = s["bias_start"][r].item(), s["bias_start"][r + 1].item()
            for i, b in dict(zip(s["bias_ids"][lo:hi].tolist(), s["bias_values"][lo:hi].tolist())).items():
                x[r, i] += b
    if s["mask"] is not None:
        bits = (s["mask"][:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
        x[bits.flatten(1)[:, :c["vocab"]] == 0] = float("-inf")
    return x, None


# ---- what a pass cannot do without ------------------------------------------
def _visible(kv, new, window, sinks):
    """(query, position) pairs that a request's new rows see, and the positions that any of them sees"""
    pairs = 0
    if not window:
        return new * kv + new * (new + 1) // 2, kv + new
    for i in range(kv, kv + new):
        pairs += min(window, i + 1) + min(sinks, max(0, i + 1 - window))
    first = max(0, kv + 1 - window)
    return pairs, kv + new - first + min(sinks, first)


def work(c):
    if c["op"] == "plan":
        kv, new = _lengths(c)
        n, p, t = c["requests"], c["page"], sum(new)
        pages = sum(-(-(a + b) // p) + (-a // p) for a, b in zip(kv, new))
        # lengths in and out, one old table entry each, the pages taken and written, two numbers a row
        return dict(bytes=4 * (5 * n + 2 * pages + 2 * (t + c["spare"])), flops=0)
    if c["op"] == "rope":
        q, k = c["rows"] * c["q_heads"] * c["head_dim"], c["rows"] * c["kv_heads"] * c["head_dim"]
        return dict(bytes=(q + 2 * k) * (SIZE[c["act"]] + SIZE[c["type"]]) + 8 * c["rows"], flops=3 * (q + k))
    if c["op"] == "attention":
        kv, new = _lengths(c)
        seen = [_visible(a, b, c["window"], c["sinks"]) for a, b in zip(kv, new)]
        pairs, read = (sum(x) for x in zip(*seen))
        d = c["head_dim"]
        return dict(bytes=2 * d * (2 * sum(new) * c["q_heads"] + 2 * read * c["kv_heads"]),
                    flops=4 * d * c["q_heads"] * pairs)
    n, v = c["rows"], c["vocab"]
    r = random.Random(c["lens"])
    history = sum(c["history"] if i == 0 else r.randint(0, c["history"]) for i in range(n))
    return dict(bytes=2 * n * v * SIZE[c["type"]] + 4 * history + 4 * c["biases"] * n + (n * v // 8 if c["mask"] else 0),
                flops=4 * n * v)
