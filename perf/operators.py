"""Workloads of the serving operators: appending to a paged 4-bit key/value cache, attention over it, sampling.

Each case can run in plain torch operations (`own` false) or through liblancius_b200 (`own` true) on the same
inputs; `exact` restates the operators in 64 bits. The cache holds 4-bit codes -7 .. 7 (plus 8), two per byte, with
one e4m3 scale per 16 channels: [page][kv head][slot][D / 2] code bytes and [page][kv head][slot][D / 16] scale bytes.
"""
import math
import random

import torch

own = False

GROUP = 16
BASE = 10000.0


def listed():
    return [
        # one user's next token: latency of the smallest call
        {"name": "append_one_token", "op": "append", "seqs": 1, "ctx": 1000, "new": 1, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # a serving batch's next tokens, every sequence at its own length
        {"name": "append_batch_step", "op": "append", "seqs": 128, "ctx": 4000, "new": 1, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # prompts of odd lengths entering the cache, small heads
        {"name": "append_prompts", "op": "append", "seqs": 5, "ctx": 1999, "new": 1999, "hq": 16, "hkv": 16, "dim": 64, "page": 32},
        # one user, short context
        {"name": "attend_one_short", "op": "attention", "seqs": 1, "ctx": 777, "new": 1, "hq": 32, "hkv": 8, "dim": 128, "page": 16},
        # one user, a long document
        {"name": "attend_one_long", "op": "attention", "seqs": 1, "ctx": 131072, "new": 1, "hq": 32, "hkv": 8, "dim": 128, "page": 64},
        # the benchmark's decode shape (32 sequences, 8 heads of 128, here up to 8192 keys each), one key head per query head
        {"name": "attend_batch_heads", "op": "attention", "seqs": 32, "ctx": 8192, "new": 1, "hq": 8, "hkv": 8, "dim": 128, "page": 16},
        # the largest: a full serving batch with eight query heads per key head
        {"name": "attend_batch_grouped", "op": "attention", "seqs": 64, "ctx": 8000, "new": 1, "hq": 64, "hkv": 8, "dim": 128, "page": 32},
        # several drafted tokens per sequence checked at once, small heads
        {"name": "attend_drafts", "op": "attention", "seqs": 24, "ctx": 3001, "new": 5, "hq": 16, "hkv": 4, "dim": 64, "page": 16},
        # one wide key head for all query heads
        {"name": "attend_wide_head", "op": "attention", "seqs": 16, "ctx": 5000, "new": 1, "hq": 8, "hkv": 1, "dim": 256, "page": 16},
        # one user's token, every filter on
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 32000, "filters": "all", "bits": 32},
        # a batch drawn from the whole distribution
        {"name": "sample_batch_open", "op": "sample", "rows": 64, "vocab": 131072, "filters": "none", "bits": 32},
        # a large batch in which each row has its own filters; logits that came out of 16 bits, so with many ties
        {"name": "sample_batch_mixed", "op": "sample", "rows": 200, "vocab": 50021, "filters": "mixed", "bits": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("append", "attention", "attention", "sample"))
    if op == "sample":
        vocab = _log(rng, 1000, 140000)
        rows = _log(rng, 1, min(256, 1 + 10000000 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "filters": rng.choice(("none", "all", "mixed")), "bits": rng.choice((16, 32))}
    dim = rng.choice((64, 128, 256))
    hkv = rng.choice((1, 2, 4, 8)) if dim > 64 else rng.choice((2, 4, 8, 12))
    hq = hkv * rng.choice((1, 2, 4, 8))
    page = rng.choice((8, 16, 32, 64))
    if op == "append":
        if rng.random() < 0.5:
            new, seqs = 1, _log(rng, 1, 200)
            ctx = _log(rng, 1, 8000)
        else:
            new = _log(rng, 2, 2000)
            seqs = _log(rng, 1, max(1, min(16, 40000000 // (new * (hq + 2 * hkv) * dim))))
            ctx = new + rng.randrange(1000)
    else:
        new = rng.choice((1, 1, 1, 2, 3, 6))
        ctx = new + _log(rng, 30, 120000)
        seqs = _log(rng, 1, max(1, min(96, 400000000 // (ctx * hkv * dim))))
    return {"op": op, "seqs": seqs, "ctx": ctx, "new": new, "hq": hq, "hkv": hkv, "dim": dim, "page": page}


def _lengths(case):
    """New tokens and keys of each sequence: a batch's lengths lie between half of `ctx` and `ctx`, one sequence has all of it."""
    rng = random.Random(case["seqs"] * 1000003 + case["ctx"])
    n, ctx = case["new"], case["ctx"]
    new = [n if n < 16 or i == 0 else rng.randint((n + 1) // 2, n) for i in range(case["seqs"])]
    return new, [max(k, ctx if i == 0 else rng.randint((ctx + 1) // 2, ctx)) for i, k in enumerate(new)]


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 24 * case["rows"], "flops": 3 * n}
    hq, hkv, d = case["hq"], case["hkv"], case["dim"]
    new, keys = _lengths(case)
    row = 2 * hkv * (d // 2 + d // GROUP)   # one token's keys and values in the cache
    if case["op"] == "append":   # q, k, v in; q, the cache's rows and the rows read back out
        t = sum(new)
        return {"bytes": t * (4 * d * (hq + 2 * hkv) + 4 * d * hq + 2 * row + 8 * d * hkv), "flops": t * d * (3 * hq + 3 * hkv + 6 * hkv)}
    seen = sum(n * k - n * (n - 1) // 2 for n, k in zip(new, keys))
    return {"bytes": sum(keys) * row + 8 * d * hq * sum(new), "flops": 4 * d * hq * seen}


# ---- inputs -----------------------------------------------------------------------------------------------

def _quantise(x):
    """[..., D] -> code bytes [..., D / 2] and scale bytes [..., D / 16]."""
    g = x.unflatten(-1, (-1, GROUP))
    a = g.abs().amax(-1)
    s = (a / torch.full_like(a, 7.0)).clamp(max=448.0).to(torch.float8_e4m3fn)   # by a number, torch multiplies with 1/7
    f = s.float().unsqueeze(-1)
    y = torch.where(f > 0, g / torch.where(f > 0, f, torch.ones_like(f)), torch.zeros_like(g))
    c = (y.round().clamp(-7, 7) + 8).to(torch.uint8).flatten(-2)
    return c[..., 0::2] + 16 * c[..., 1::2], s.view(torch.uint8)


def _values(codes, scales):
    """The inverse of _quantise, in FP32."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float() - 8.0
    return (c.unflatten(-1, (-1, GROUP)) * scales.view(torch.float8_e4m3fn).float().unsqueeze(-1)).flatten(-2)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    if case["op"] == "sample":
        rows, v = case["rows"], case["vocab"]
        x = randn(rows, v) * (1.0 + 2.5 * rand(rows, 1))
        if case["bits"] == 16:
            x = x.bfloat16().float()
        x = torch.where(rand(rows, v) < 0.01, torch.full_like(x, -math.inf), x)   # tokens that the program forbids
        s = {"case": case, "logits": x, "u": rand(rows), "temperature": None, "top_k": None, "top_p": None, "min_p": None}
        if case["filters"] != "none":
            s["temperature"] = 0.5 + rand(rows)
            s["top_k"] = (1 + 199 * rand(rows)).int()
            s["top_p"] = 0.8 + 0.19 * rand(rows)
            s["min_p"] = 0.1 * rand(rows)
        if case["filters"] == "mixed":   # each filter off in half of the rows; one row in eight takes the largest logit
            s["temperature"] = torch.where(rand(rows) < 0.125, 0.0, s["temperature"])
            s["top_k"] = torch.where(rand(rows) < 0.5, 0, s["top_k"]).int()
            s["top_p"] = torch.where(rand(rows) < 0.5, 1.0, s["top_p"])
            s["min_p"] = torch.where(rand(rows) < 0.5, 0.0, s["min_p"])
        return s
    new, keys = _lengths(case)
    hq, hkv, d, ps = case["hq"], case["hkv"], case["dim"], case["page"]
    pages = [-(-k // ps) for k in keys]
    width, total = max(pages), sum(pages) + 1
    order = torch.randperm(total, device="cuda", generator=gen).int()
    table = torch.zeros(len(keys), width, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    i32 = {"dtype": torch.int32, "device": "cuda"}
    s = {"case": case, "table": table, "seq_len": torch.tensor(keys, **i32), "start": torch.tensor(starts, **i32),
         "tokens": starts[-1], "max_len": max(keys), "max_new": max(new)}
    if case["op"] == "append":
        for name in ("k", "v"):
            s[name + "_codes"] = torch.zeros(total, hkv, ps, d // 2, dtype=torch.uint8, device="cuda")
            s[name + "_scales"] = torch.zeros(total, hkv, ps, d // GROUP, dtype=torch.uint8, device="cuda")
        s["qkv"] = randn(starts[-1], (hq + 2 * hkv) * d) * (0.5 + 1.5 * rand((hq + 2 * hkv) * d))   # one projection's output
        return s
    for name in ("k", "v"):
        spread = 0.5 + 1.5 * rand(hkv, 1, d)   # channels differ in size
        s[name + "_codes"] = torch.empty(total, hkv, ps, d // 2, dtype=torch.uint8, device="cuda")
        s[name + "_scales"] = torch.empty(total, hkv, ps, d // GROUP, dtype=torch.uint8, device="cuda")
        step = max(1, 32000000 // (hkv * ps * d))
        for p in range(0, total, step):
            n = min(step, total - p)
            s[name + "_codes"][p:p + n], s[name + "_scales"][p:p + n] = _quantise(randn(n, hkv, ps, d) * spread)
    s["q"] = randn(starts[-1], hq * d) * 1.2
    return s


# ---- the plain forms --------------------------------------------------------------------------------------

def _place(s):
    """Sequence, position, page and slot of every new token."""
    t = torch.arange(s["tokens"], dtype=torch.int32, device="cuda")
    seq = torch.searchsorted(s["start"], t, right=True) - 1
    pos = (s["seq_len"][seq] - s["start"][seq + 1] + t).long()
    ps = s["case"]["page"]
    return seq, pos, s["table"][seq, pos // ps].long(), pos % ps


def _rotate(x, pos):
    """[T, H, D] by the position's angles, pairs (2c, 2c + 1): in 64 bits, as positions go far; rounded once."""
    d = x.shape[-1]
    a = pos.double()[:, None, None] * BASE ** (-torch.arange(0, d, 2, dtype=torch.float64, device=x.device) / d)
    c, n, x0, x1 = a.cos(), a.sin(), x[..., 0::2].double(), x[..., 1::2].double()
    return torch.stack((x0 * c - x1 * n, x0 * n + x1 * c), -1).flatten(-2).float()


def _append(s):
    c = s["case"]
    hq, hkv, d = c["hq"], c["hkv"], c["dim"]
    q, k, v = s["qkv"].split((hq * d, hkv * d, hkv * d), 1)
    _, pos, page, slot = _place(s)
    q = _rotate(q.unflatten(1, (hq, d)), pos).flatten(1)
    k = _rotate(k.unflatten(1, (hkv, d)), pos)
    s["k_codes"][page, :, slot], s["k_scales"][page, :, slot] = _quantise(k)
    s["v_codes"][page, :, slot], s["v_scales"][page, :, slot] = _quantise(v.unflatten(1, (hkv, d)))
    return (q, _values(s["k_codes"][page, :, slot], s["k_scales"][page, :, slot]),
            _values(s["v_codes"][page, :, slot], s["v_scales"][page, :, slot]))


def _attend(s):
    c = s["case"]
    hq, hkv, d, b, n = c["hq"], c["hkv"], c["dim"], c["seqs"], s["max_new"]
    seq, pos, _, _ = _place(s)
    at = torch.arange(s["tokens"], device="cuda") - s["start"][seq]
    q = torch.zeros(b, n, hq * d, device="cuda")
    q[seq, at] = s["q"]
    q = q.view(b, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    limit = torch.full((b, n), -1, device="cuda")
    limit[seq, at] = pos
    table = s["table"].long()
    k = _values(s["k_codes"][table], s["k_scales"][table]).permute(0, 2, 4, 1, 3).reshape(b, hkv, d, -1)
    x = (q @ k).view(b, hkv, hq // hkv, n, -1) / math.sqrt(d)
    del k
    key = torch.arange(x.shape[-1], device="cuda")
    x = torch.where(key <= limit[:, None, None, :, None], x, torch.full_like(x, -math.inf))
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    v = _values(s["v_codes"][table], s["v_scales"][table])
    v = torch.where(key.view(1, -1, 1, c["page"], 1) < s["seq_len"].view(-1, 1, 1, 1, 1), v, torch.zeros_like(v))
    v = v.permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)
    o = (p.view(b, hkv, -1, x.shape[-1]) @ v).view(b, hkv, hq // hkv, n, d)
    return o.permute(0, 3, 1, 2, 4).reshape(b, n, hq * d)[seq, at]


def _sample(s):
    """In 64 bits: one token more or less before a border changes the answer."""
    x = s["logits"].double()
    rows, v = x.shape

    def per_row(name, off):
        return torch.full((rows, 1), off, dtype=torch.float64, device="cuda") if s[name] is None else s[name].double()[:, None]

    t, k, p, mp = per_row("temperature", 1.0), per_row("top_k", 0), per_row("top_p", 1.0), per_row("min_p", 0.0)
    m = x.amax(1, keepdim=True)
    w = torch.exp((x - m) / torch.where(t > 0, t, 1.0))
    ranked, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(v, device="cuda")
    keep = ((rank < torch.where(k > 0, k, v)) & (ws >= mp)) | (rank == 0)
    mass = (ws * keep).cumsum(1)
    before = torch.cat((torch.zeros_like(m), mass[:, :-1]), 1)
    keep &= (p >= 1) | (before < p * mass[:, -1:]) | (rank == 0)
    kept = torch.zeros_like(keep).scatter(1, order, keep)
    run_ = (w * kept).cumsum(1)
    token = (run_ <= s["u"].double()[:, None] * run_[:, -1:]).sum(1)
    last = torch.where(kept, rank, torch.zeros_like(rank)).amax(1)
    first = torch.where(x == m, rank, torch.full_like(rank, v)).amin(1)
    return torch.where(t[:, 0] > 0, torch.minimum(token, last), first).int()


# ---- the framework's calls --------------------------------------------------------------------------------

def _handle(s):
    """The library and the two descriptions of the cache, which a program keeps as long as its buffers."""
    if "handle" not in s:
        import lancius_b200 as L
        lib = L.load()
        if s["case"]["op"] == "sample":
            s["handle"] = (lib,)
            return s["handle"]
        c = s["case"]
        pages = L.KvPages(s["k_codes"].data_ptr(), s["v_codes"].data_ptr(), s["k_scales"].data_ptr(), s["v_scales"].data_ptr(),
                          s["k_codes"].shape[0], c["page"], c["hkv"], c["dim"], 1.0, 1.0)
        batch = L.KvBatch(s["table"].data_ptr(), s["table"].shape[1], s["seq_len"].data_ptr(), s["start"].data_ptr(),
                          c["seqs"], s["tokens"], s["max_len"], s["max_new"])
        bytes_ = lib.lcu_attention_paged_workspace(pages, batch, c["hq"])
        s["handle"] = (lib, pages, batch, torch.empty(max(bytes_, 16), dtype=torch.uint8, device="cuda"), bytes_)
    return s["handle"]


def _ok(status):
    if status != 0:
        raise RuntimeError("lancius error %d" % status)


def _own_append(s):
    lib, pages, batch, _, _ = _handle(s)
    c, t, qkv, stream = s["case"], s["tokens"], s["qkv"], torch.cuda.current_stream().cuda_stream
    hq, hkv, d = c["hq"], c["hkv"], c["dim"]
    q = torch.empty(t, hq * d, device="cuda")
    k = torch.empty(t, hkv, d, device="cuda")
    v = torch.empty(t, hkv, d, device="cuda")
    at, ld = qkv.data_ptr(), qkv.stride(0)
    _ok(lib.lcu_kv_append_paged(pages, batch, q.data_ptr(), at, ld, hq, at + 4 * hq * d, ld, at + 4 * (hq + hkv) * d, ld, BASE, stream))
    _ok(lib.lcu_kv_read_paged(k.data_ptr(), v.data_ptr(), pages, batch, stream))
    return q, k, v


def _own_attend(s):
    lib, pages, batch, space, bytes_ = _handle(s)
    q, hq = s["q"], s["case"]["hq"]
    out = torch.empty_like(q)
    _ok(lib.lcu_attention_paged(out.data_ptr(), q.data_ptr(), q.stride(0), hq, pages, batch, space.data_ptr(), bytes_,
                                torch.cuda.current_stream().cuda_stream))
    return out


def _own_sample(s):
    lib, = _handle(s)
    x = s["logits"]
    token = torch.empty(x.shape[0], dtype=torch.int32, device="cuda")
    t, k, p, mp = (None if s[n] is None else s[n].data_ptr() for n in ("temperature", "top_k", "top_p", "min_p"))
    _ok(lib.lcu_sample(token.data_ptr(), x.data_ptr(), x.stride(0), x.shape[0], x.shape[1], t, k, p, mp, s["u"].data_ptr(),
                       torch.cuda.current_stream().cuda_stream))
    return token


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "attention": _own_attend, "sample": _own_sample}[op](state)
    return {"append": _append, "attention": _attend, "sample": _sample}[op](state)


# ---- 64 bits ----------------------------------------------------------------------------------------------

def _grid8():
    """The non-negative e4m3 numbers, by their bits."""
    return [(b & 7) * 2.0 ** -9 if b < 8 else (1 + (b & 7) / 8) * 2.0 ** ((b >> 3) - 7) for b in range(127)]


def _nearest(y, grid):
    """Index of the grid point nearest to each y >= 0; halfway between two, the even index."""
    g = torch.tensor(grid, dtype=torch.float64, device=y.device)
    hi = torch.searchsorted(g, y.contiguous()).clamp(1, len(grid) - 1)
    lo = hi - 1
    a, b = y - g[lo], g[hi] - y
    return torch.where((b < a) | ((b == a) & (hi % 2 == 0)), hi, lo)


def _held(x):
    """What the cache holds of [T, H, D] numbers: FP32 values in, 64 bits out."""
    t, h, d = x.shape
    g = x.float().double().view(t, h, d // GROUP, GROUP)
    grid = torch.tensor(_grid8(), dtype=torch.float64, device=x.device)
    a = g.abs().max(3).values
    s = grid[_nearest(a / torch.full_like(a, 7), _grid8())].unsqueeze(3)
    y = g.abs() / s.clamp(min=1e-300)
    e = _nearest(y, [float(i) for i in range(8)]).double()
    return (torch.copysign(e, g) * s).view(t, h, d)


def exact(case, seed):
    if case["op"] == "sample":   # whole numbers
        return None
    s = prepare(case, seed)
    new, keys = _lengths(case)
    hq, hkv, d, ps = case["hq"], case["hkv"], case["dim"], case["page"]
    if case["op"] == "append":
        pos = torch.cat([torch.arange(k - n, k, dtype=torch.float64) for n, k in zip(new, keys)]).cuda()
        freq = torch.exp(-math.log(BASE) * 2 / d * torch.arange(d // 2, dtype=torch.float64)).cuda()
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), torch.outer(pos, freq))[:, None]
        x = s["qkv"].double().view(len(pos), hq + 2 * hkv, d)
        z = torch.view_as_real(torch.view_as_complex(x[:, :hq + hkv].reshape(len(pos), hq + hkv, d // 2, 2)) * turn).flatten(2)
        return z[:, :hq].flatten(1), _held(z[:, hq:]), _held(x[:, hq + hkv:])
    out, at, q = [], 0, s["q"].double().view(-1, hkv, hq // hkv, d)
    grid = torch.tensor(_grid8(), dtype=torch.float64, device="cuda")
    for b, (n, k) in enumerate(zip(new, keys)):
        ids = s["table"][b, :-(-k // ps)].long()
        both = []
        for name in ("k", "v"):
            code = s[name + "_codes"][ids].transpose(1, 2).reshape(-1, hkv, d // 2)[:k].long()
            scale = s[name + "_scales"][ids].transpose(1, 2).reshape(-1, hkv, d // GROUP)[:k].long()
            x = torch.empty(k, hkv, d, dtype=torch.float64, device="cuda")
            x[..., 0::2], x[..., 1::2] = code % 16 - 8, code // 16 - 8
            both.append(x * grid[scale].repeat_interleave(GROUP, 2))
        x = torch.einsum("nhgd,khd->nhgk", q[at:at + n], both[0]) * d ** -0.5
        hidden = torch.arange(k, device="cuda") > torch.arange(k - n, k, device="cuda")[:, None]
        p = torch.softmax(x.masked_fill(hidden[:, None, None], -math.inf), 3)
        out.append(torch.einsum("nhgk,khd->nhgd", p, both[1]).reshape(n, hq * d))
        at += n
    return torch.cat(out)
