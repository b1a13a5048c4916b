"""Operators of one serving step over a paged key/value cache: cases, inputs, plain forms and exact values.

A step takes the rows of a ragged batch of new tokens, rotates queries and keys by each token's own position, writes keys
and values into the pages of a cache, attends over that cache, and draws the next ids.  Each case below is one of those
operators at one set of sizes; `run` computes it with elementary torch operations, or, where `own` is true, makes the calls
of the framework's entry points.
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
SIZES = {"bf16": 2, "f32": 4}
WORKSPACE_BYTES = 96 << 20


# ---- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # rotary positions: eight sequences of a decode batch, each far into its own text; the smallest call
        dict(name="rope_step", op="rope", tokens=8, qh=16, kvh=4, hd=128, rd=128, layout="half", scaling="yarn", far=100000, backward=False, dtype="bf16"),
        # gradients of queries and keys of a training batch of 8 x 2048 tokens
        dict(name="rope_train_backward", op="rope", tokens=16384, qh=16, kvh=4, hd=128, rd=128, layout="interleaved", scaling="plain", far=2048, backward=True, dtype="bf16"),
        # part of an odd head rotated, in 32 bits
        dict(name="rope_part_of_head_f32", op="rope", tokens=4097, qh=12, kvh=3, hd=80, rd=24, layout="half", scaling="bands", far=40000, backward=False, dtype="f32"),
        # one new token for each of 64 sequences: rotate, write the pages
        dict(name="append_step", op="append", n_seq=64, q_lo=1, q_hi=1, kv_lo=50, kv_hi=4000, qh=16, kvh=4, hd=128, page=16, layout="interleaved", dtype="bf16", lens=1),
        # a long prompt's chunk enters the cache
        dict(name="append_chunk", op="append", n_seq=2, q_lo=3500, q_hi=4500, kv_lo=4500, kv_hi=9000, qh=32, kvh=8, hd=128, page=64, layout="half", dtype="bf16", lens=2),
        # attention: four short conversations, where latency counts
        dict(name="attn_step_short", op="attn", n_seq=4, q_lo=1, q_hi=1, kv_lo=200, kv_hi=700, qh=16, kvh=4, hd=128, page=16, dtype="bf16", lens=3),
        # a full decode batch of very different lengths
        dict(name="attn_step_ragged", op="attn", n_seq=64, q_lo=1, q_hi=1, kv_lo=100, kv_hi=12000, qh=32, kvh=8, hd=128, page=32, dtype="bf16", lens=4),
        # a chunk of a long prompt over what came before it
        dict(name="attn_chunk", op="attn", n_seq=1, q_lo=1024, q_hi=1024, kv_lo=30011, kv_hi=30011, qh=32, kvh=8, hd=128, page=64, dtype="bf16", lens=5),
        # chunks and single tokens in one batch
        dict(name="attn_mixed", op="attn", n_seq=40, q_lo=1, q_hi=500, kv_lo=300, kv_hi=4000, qh=16, kvh=4, hd=128, page=16, dtype="bf16", lens=6),
        # small heads in 32 bits, a few tokens each (a draft checked by the model)
        dict(name="attn_draft_f32", op="attn", n_seq=7, q_lo=1, q_hi=9, kv_lo=60, kv_hi=1500, qh=8, kvh=2, hd=64, page=16, dtype="f32", lens=7),
        # sampling: a decode batch with every filter
        dict(name="sample_filters", op="sample", batch=64, vocab=32000, top_k=50, top_p=0.9, min_p=0.05, spread=3.0, dtype="bf16"),
        # a large vocabulary, nucleus only
        dict(name="sample_nucleus_large", op="sample", batch=32, vocab=100256, top_k=0, top_p=0.95, min_p=0.0, spread=3.0, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "sample"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "rope":
        hd = rng.choice([64, 72, 80, 96, 128, 256])
        rd = hd if rng.random() < 0.5 else 2 * rng.randint(1, hd // 2)
        kvh = rng.choice([1, 2, 3, 4, 8])
        qh = kvh * rng.choice([1, 2, 3, 4])
        most = max(2, (16384 * 20 * 128 // 2) // ((qh + kvh) * hd))
        return dict(op=op, tokens=_log(rng, 1, min(16384, most)), qh=qh, kvh=kvh, hd=hd, rd=rd, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["plain", "linear", "ntk", "yarn", "bands"]), far=_log(rng, 100, 1000000), backward=rng.random() < 0.4, dtype=dtype)
    if op == "append":
        kvh = rng.choice([1, 2, 4, 8])
        step = rng.random() < 0.5
        q_hi = 1 if step else _log(rng, 2, 2000)
        n = rng.randint(1, 200) if step else rng.randint(1, 4)
        return dict(op=op, n_seq=n, q_lo=1, q_hi=q_hi, kv_lo=q_hi, kv_hi=q_hi + _log(rng, 1, 5000), qh=kvh * rng.choice([1, 2, 4]), kvh=kvh,
                    hd=rng.choice([64, 80, 128]), page=rng.choice([8, 16, 32, 64, 128]), layout=rng.choice(["half", "interleaved"]), dtype=dtype, lens=rng.randrange(1 << 30))
    if op == "attn":
        kvh, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 4, 5, 8])
        kind = rng.choice(["step", "draft", "chunk", "mixed"])
        if kind == "step":
            n, q_lo, q_hi, kv = rng.randint(1, 64), 1, 1, _log(rng, 50, 6000)
        elif kind == "draft":
            n, q_lo, q_hi, kv = rng.randint(1, 16), 1, rng.randint(2, 16), _log(rng, 100, 4000)
        elif kind == "chunk":
            q_lo = _log(rng, 17, 1000)
            n, q_hi, kv = rng.randint(1, 3), q_lo + rng.randint(0, 24), q_lo + 24 + _log(rng, 1, 7000)
        else:
            n, q_lo, q_hi, kv = rng.randint(3, 24), 1, _log(rng, 20, 400), _log(rng, 400, 3000)
        if dtype == "f32":
            n, q_hi, kv = min(n, 4), min(q_hi, 64), min(kv, 1000)
            q_lo = min(q_lo, q_hi)
        return dict(op=op, n_seq=n, q_lo=q_lo, q_hi=q_hi, kv_lo=min(kv, q_hi), kv_hi=kv, qh=kvh * group, kvh=kvh, hd=rng.choice([64, 128, 128] if dtype == "bf16" else [64, 80, 128]),
                    page=rng.choice([8, 16, 32, 64, 128]), dtype=dtype, lens=rng.randrange(1 << 30))
    vocab = _log(rng, 200, 131072)
    return dict(op=op, batch=_log(rng, 1, max(2, min(64, (32 * 100256) // vocab))), vocab=vocab, top_k=rng.choice([0, 1, 20, 50, 1000]), top_p=rng.choice([1.0, 0.95, 0.8, 0.3]),
                min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), spread=rng.choice([1.0, 3.0, 6.0]), dtype=dtype)


def _lengths(c):
    """(new tokens, cached positions with them) of each sequence: the same for every seed."""
    r = random.Random(c["lens"])
    q = [_log(r, c["q_lo"], c["q_hi"]) for _ in range(c["n_seq"])]
    return q, [max(n, _log(r, max(1, c["kv_lo"]), c["kv_hi"])) for n in q]


def work(c):
    es = SIZES[c["dtype"]]
    if c["op"] == "rope":
        return {"bytes": 2 * c["tokens"] * (c["qh"] + c["kvh"]) * c["hd"] * es + 4 * c["tokens"], "flops": 3 * c["tokens"] * (c["qh"] + c["kvh"]) * c["rd"]}
    if c["op"] == "append":
        t = sum(_lengths(c)[0])
        return {"bytes": 2 * t * (c["qh"] + 2 * c["kvh"]) * c["hd"] * es, "flops": 3 * t * (c["qh"] + c["kvh"]) * c["hd"]}
    if c["op"] == "attn":
        q, kv = _lengths(c)
        seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(q, kv))
        return {"bytes": 2 * sum(kv) * c["kvh"] * c["hd"] * es + 2 * sum(q) * c["qh"] * c["hd"] * es + 4 * sum(q) * c["qh"], "flops": 4 * c["hd"] * c["qh"] * seen}
    return {"bytes": c["batch"] * c["vocab"] * es + 32 * c["batch"], "flops": 3 * c["batch"] * c["vocab"]}


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _frequencies(hd, rd, scaling, base=10000.0, factor=8.0, original=4096.0, beta_fast=32.0, beta_slow=1.0, low=1.0, high=4.0):
    """(radians per position of each pair, amplitude), in 64 bits."""
    i = torch.arange(rd // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / rd)
    amplitude = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "ntk" and rd > 2:
        f = (base * factor ** (rd / (rd - 2.0))) ** (-2.0 * i / rd)
    elif scaling == "yarn":
        at = lambda turns: rd * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(at(beta_fast))), min(rd - 1, math.ceil(at(beta_slow)))
        ramp = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        amplitude = 0.1 * math.log(factor) + 1.0
    elif scaling == "bands":
        share = ((original * f / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        f = (1 - share) * f / factor + share * f
    return f, amplitude


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(c, seed):
    g = _generator(seed)
    dt = DTYPES[c["dtype"]]
    randn = lambda *shape, t=dt: torch.randn(*shape, generator=g, device="cuda", dtype=t)  # noqa: E731
    s = {"case": c}
    if c["op"] == "rope":
        f, s["amplitude"] = _frequencies(c["hd"], c["rd"], c["scaling"])
        s["freqs"] = f.cuda()
        s["positions"] = torch.randint(0, c["far"], (c["tokens"],), generator=g, device="cuda", dtype=torch.int32)
        s["q"], s["k"] = randn(c["tokens"], c["qh"], c["hd"]), randn(c["tokens"], c["kvh"], c["hd"])
        s["q_out"], s["k_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"])
        return s
    if c["op"] in ("append", "attn"):
        q, kv = _lengths(c)
        P = c["page"]
        pages = [-(-m // P) for m in kv]
        n_pages, wide = sum(pages) + 3, max(pages)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
        table = torch.full((c["n_seq"], wide), -1, dtype=torch.int32, device="cuda")
        n = torch.tensor(pages, device="cuda")
        table[torch.arange(wide, device="cuda")[None, :] < n[:, None]] = order[:sum(pages)]
        s["table"], s["kv_len"] = table, torch.tensor(kv, dtype=torch.int32, device="cuda")
        s["q_start"] = torch.tensor([0] + torch.tensor(q).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        s["rows"], s["max_q"] = sum(q), max(q)
        s["k_pages"], s["v_pages"] = randn(n_pages, P, c["kvh"], c["hd"]), randn(n_pages, P, c["kvh"], c["hd"])
        s["q"] = randn(s["rows"], c["qh"], c["hd"])
        s["out"] = torch.zeros_like(s["q"])
        if c["op"] == "append":
            f, s["amplitude"] = _frequencies(c["hd"], c["hd"], "plain")
            s["freqs"] = f.cuda()
            s["k"], s["v"] = randn(s["rows"], c["kvh"], c["hd"]), randn(s["rows"], c["kvh"], c["hd"])
        else:
            # what lies behind a sequence's last position in its last page was never written
            where = torch.arange(wide * P, device="cuda")[None, :]
            past = (where >= s["kv_len"][:, None]) & (where < n[:, None] * P)
            seq, at = past.nonzero(as_tuple=True)
            for pages in (s["k_pages"], s["v_pages"]):
                pages[table[seq, at // P].long(), at % P] = float("nan")
            s["q"] *= 1.5
            s["lse"] = torch.zeros(s["rows"], c["qh"], dtype=torch.float32, device="cuda")
            s["workspace"] = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
        return s
    B, V = c["batch"], c["vocab"]
    s["logits"] = (randn(B, V, t=torch.float32) * c["spread"]).to(dt)
    s["logits"][torch.rand(B, V, generator=g, device="cuda") < 0.03] = float("-inf")  # ids that a grammar forbids
    s["logits"][:, 0] = 0.0
    s["uniform"] = torch.rand(B, generator=g, device="cuda")
    s["temperature"] = 0.5 + torch.rand(B, generator=g, device="cuda")
    s["temperature"][B // 2] = 0.0 if B > 4 else 1.0
    s["top_k"] = torch.full((B,), c["top_k"], dtype=torch.int32, device="cuda")
    s["top_p"], s["min_p"] = torch.full((B,), c["top_p"], device="cuda"), torch.full((B,), c["min_p"], device="cuda")
    s["tokens"], s["kept"], s["prob"] = (torch.empty(B, dtype=t, device="cuda") for t in (torch.int32, torch.int32, torch.float32))
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------
def _rotate(x, angle, amplitude, layout, rd):
    """x [tokens, heads, hd] in 32 bits, angle [tokens, rd/2] in 64 bits."""
    cos, sin = (amplitude * angle.cos()).float()[:, None, :], (amplitude * angle.sin()).float()[:, None, :]
    a, b = (x[..., 0:rd:2], x[..., 1:rd:2]) if layout == "interleaved" else (x[..., :rd // 2], x[..., rd // 2:rd])
    u, v = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((u, v), -1).flatten(-2) if layout == "interleaved" else torch.cat((u, v), -1)
    return torch.cat((turned, x[..., rd:]), -1)


def _rope(s):
    c = s["case"]
    angle = s["positions"].double()[:, None] * s["freqs"][None, :] * (-1.0 if c["backward"] else 1.0)
    return [_rotate(s[n].float(), angle, s["amplitude"], c["layout"], c["rd"]).to(s[n].dtype) for n in ("q", "k")]


def _slots(s):
    """(sequence, position) of every row of new tokens."""
    row = torch.arange(s["rows"], device="cuda")
    seq = torch.searchsorted(s["q_start"].long(), row, right=True) - 1
    return seq, (s["kv_len"].long()[seq] - s["q_start"].long()[seq + 1] + row)


def _append(s):
    c = s["case"]
    seq, pos = _slots(s)
    angle = pos.double()[:, None] * s["freqs"][None, :]
    page, at = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    s["k_pages"][page, at] = _rotate(s["k"].float(), angle, s["amplitude"], c["layout"], c["hd"]).to(s["k"].dtype)
    s["v_pages"][page, at] = s["v"]
    s["out"].copy_(_rotate(s["q"].float(), angle, s["amplitude"], c["layout"], c["hd"]))
    return [s["out"], s["k_pages"], s["v_pages"]]


def _attn(s):
    c = s["case"]
    n, P, G, hd = c["n_seq"], c["page"], c["qh"] // c["kvh"], c["hd"]
    q_start, kv_len = s["q_start"].long(), s["kv_len"].long()
    wide = s["table"].shape[1] * P
    at = torch.arange(wide, device="cuda")
    page = s["table"].long().clamp(min=0)[:, at // P]
    there = (at[None, :] < kv_len[:, None])[..., None, None]
    k, v = (torch.where(there, p[page, at % P].float(), 0.0).permute(0, 2, 1, 3) for p in (s["k_pages"], s["v_pages"]))   # [n, kvh, wide, hd]
    row = q_start[:-1, None] + torch.arange(s["max_q"], device="cuda")[None, :]
    real = row < q_start[1:, None]
    row = row.clamp(max=s["rows"] - 1)
    q = s["q"].float()[row].view(n, s["max_q"], c["kvh"], G, hd).permute(0, 2, 3, 1, 4).reshape(n, c["kvh"], G * s["max_q"], hd)
    score = (q @ k.transpose(-1, -2)).view(n, c["kvh"], G, s["max_q"], wide) * (1.0 / math.sqrt(hd))
    pos = (kv_len - q_start[1:])[:, None] + row
    score.masked_fill_((at[None, None, :] > pos[..., None])[:, None, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (score - top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(n, c["kvh"], G * s["max_q"], wide) @ v).view(n, c["kvh"], G, s["max_q"], hd) / total
    o = o.permute(0, 3, 1, 2, 4).reshape(n, s["max_q"], c["qh"], hd)
    lse = (total.log() + top)[..., 0].permute(0, 3, 1, 2).reshape(n, s["max_q"], c["qh"])
    s["out"][row[real]] = o[real].to(s["out"].dtype)
    s["lse"][row[real]] = lse[real]
    return [s["out"], s["lse"]]


def _sample(s):
    x = s["logits"].double()
    T, k = s["temperature"].double()[:, None], s["top_k"].long()[:, None]
    top_p, min_p, u = s["top_p"].double()[:, None], s["min_p"].double()[:, None], s["uniform"].double()[:, None]
    V = x.shape[1]
    greedy = T <= 0
    w = ((x - x.amax(-1, keepdim=True)) / torch.where(greedy, 1.0, T)).exp()
    order = x.sort(dim=-1, descending=True, stable=True).indices
    ranked = w.gather(-1, order)
    rank = torch.arange(V, device="cuda")[None, :]
    keep = (ranked > 0) & ((k <= 0) | (rank < k))
    mass = torch.where(keep, ranked, 0.0)
    before = mass.cumsum(-1) - mass
    keep &= (top_p >= 1) | (before < top_p * mass.sum(-1, keepdim=True))
    keep &= ranked >= min_p
    keep = torch.where(greedy, rank == 0, keep)
    kept = torch.zeros_like(keep).scatter_(-1, order, keep)
    mass = torch.where(kept, w, 0.0)
    run_ = mass.cumsum(-1)
    total = run_[:, -1:]
    token = ((run_ > u * total) & kept).to(torch.uint8).argmax(-1, keepdim=True)
    return [token[:, 0].to(torch.int32), kept.sum(-1).to(torch.int32), (mass.gather(-1, token) / total)[:, 0].float()]


# ---- the framework's calls ----------------------------------------------------------------------------------------------
_context = []


def _ctx():
    """The program's context, on torch's current stream."""
    if not _context:
        _context.append(importlib.import_module("large-language-model_b200.bridge"))
        _context.append(_context[0].Context(0))
    _context[1].use_stream(torch.cuda.current_stream().cuda_stream)
    return _context


def _handles(s):
    """The descriptors that a program makes once of the arrays it works on."""
    if "handles" not in s:
        bridge, ctx = _ctx()
        names = {torch.bfloat16: "bf16", torch.float32: "f32", torch.float64: "f64", torch.int32: "i32"}
        h = {n: ctx.wrap(t.data_ptr(), tuple(t.shape), names[t.dtype]) for n, t in s.items() if isinstance(t, torch.Tensor) and t.dtype in names}
        c = s["case"]
        if "freqs" in s:
            h["rope"] = bridge.RopeConfig.make(c["hd"], c.get("rd", c["hd"]), layout=c["layout"], amplitude=s["amplitude"])
        if "table" in s:
            h["cache"] = bridge.PagedCache(h["k_pages"], h["v_pages"])
            h["batch"] = bridge.PagedBatch(h["q_start"], h["kv_len"], h["table"], s["rows"], s["max_q"])
        if "workspace" in s:
            h["workspace"] = ctx.wrap(s["workspace"].data_ptr(), (WORKSPACE_BYTES // 4,), "f32")
        s["handles"] = h
    return s["handles"]


def _own(s):
    _, ctx = _ctx()
    h, c = _handles(s), s["case"]
    if c["op"] == "rope":
        (ctx.rope_positions_backward if c["backward"] else ctx.rope_positions_forward)(h["rope"], h["freqs"], h["positions"], h["q"], h["k"], out=(h["q_out"], h["k_out"]))
        return [s["q_out"], s["k_out"]]
    if c["op"] == "append":
        ctx.paged_append(h["cache"], h["batch"], h["k"], h["v"], rope=h["rope"], freqs=h["freqs"], q=h["q"], q_out=h["out"])
        return [s["out"], s["k_pages"], s["v_pages"]]
    if c["op"] == "attn":
        ctx.paged_attn(h["cache"], h["batch"], h["q"], out=h["out"], lse=h["lse"], workspace=h["workspace"])
        return [s["out"], s["lse"]]
    ctx.sample_given(h["logits"], h["uniform"], h["temperature"], h["top_k"], h["top_p"], h["min_p"], out=(h["tokens"], h["kept"], h["prob"]))
    return [s["tokens"], s["kept"], s["prob"]]


PLAIN = {"rope": _rope, "append": _append, "attn": _attn, "sample": _sample}


def run(s):
    return _own(s) if own else PLAIN[s["case"]["op"]](s)


# ---- exact values -------------------------------------------------------------------------------------------------------
def _turned(x, pos, freqs, amplitude, layout, rd, sign=1.0):
    """The rotation as a product with e^(i theta) of numbers in 64 bits."""
    x = x.double()
    z = torch.polar(torch.full((), float(amplitude), dtype=torch.float64, device=x.device), sign * pos.double()[:, None] * freqs)[:, None, :]
    y = x.clone()
    if layout == "interleaved":
        y[..., :rd] = torch.view_as_real(torch.view_as_complex(x[..., :rd].unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    else:
        r = torch.complex(x[..., :rd // 2], x[..., rd // 2:rd]) * z
        y[..., :rd // 2], y[..., rd // 2:rd] = r.real, r.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "rope":
        return [_turned(s[n], s["positions"], s["freqs"], s["amplitude"], c["layout"], c["rd"], -1.0 if c["backward"] else 1.0) for n in ("q", "k")]
    if c["op"] == "sample":
        x, u = s["logits"].double().cpu(), s["uniform"].double().tolist()
        tokens, kept, prob = [], [], []
        for b in range(c["batch"]):
            T = float(s["temperature"][b])
            if T <= 0:
                tokens.append(int((x[b] == x[b].max()).nonzero()[0])); kept.append(1); prob.append(1.0)
                continue
            ids = torch.argsort(-x[b], stable=True)
            ids = ids[x[b][ids] > -math.inf]
            ids = ids[:c["top_k"]] if c["top_k"] > 0 else ids
            w = ((x[b][ids] - x[b].max()) / T).exp()
            run_ = w.cumsum(0)
            top_p, min_p = float(s["top_p"][b]), float(s["min_p"][b])
            n = len(ids) if top_p >= 1 else 1 + int((run_[:-1] < top_p * run_[-1]).sum())
            n = min(n, int((w >= min_p).sum()))
            ids, at = ids[:n].sort()
            w = w[:n][at]
            run_ = w.cumsum(0)
            t = int((run_ <= u[b] * run_[-1]).sum())
            tokens.append(int(ids[t])); kept.append(n); prob.append(float(w[t] / run_[-1]))
        return [torch.tensor(tokens, dtype=torch.int32), torch.tensor(kept, dtype=torch.int32), torch.tensor(prob, dtype=torch.float64)]
    q, kv = _lengths(c)
    P, first, out = c["page"], 0, s["q"].double().clone()
    k_pages, v_pages = s["k_pages"], s["v_pages"]
    if c["op"] == "append":
        k_pages, v_pages = k_pages.double(), v_pages.double()
    lse = torch.zeros(s["rows"], c["qh"], dtype=torch.float64, device="cuda")
    for i, (n, m) in enumerate(zip(q, kv)):
        rows, pos = slice(first, first + n), torch.arange(m - n, m, device="cuda")
        first += n
        ids = s["table"][i].long()
        if c["op"] == "append":
            out[rows] = _turned(s["q"][rows], pos, s["freqs"], s["amplitude"], c["layout"], c["hd"])
            k_pages[ids[pos // P], pos % P] = _turned(s["k"][rows], pos, s["freqs"], s["amplitude"], c["layout"], c["hd"])
            v_pages[ids[pos // P], pos % P] = s["v"][rows].double()
            continue
        used = ids[:-(-m // P)]
        k, v = (p[used].flatten(0, 1)[:m].double() for p in (k_pages, v_pages))
        hide = torch.arange(m, device="cuda")[None, :] > pos[:, None]
        for h in range(c["qh"]):
            g = h // (c["qh"] // c["kvh"])
            score = (s["q"][rows, h].double() @ k[:, g].T / math.sqrt(c["hd"])).masked_fill_(hide, -math.inf)
            lse[rows, h] = score.logsumexp(-1)
            out[rows, h] = score.softmax(-1) @ v[:, g]
    return [out, k_pages, v_pages] if c["op"] == "append" else [out, lse]
