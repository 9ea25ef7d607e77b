"""Cases of the serving operators: the page plan, the append to a paged KV cache, attention of a
chunk of new tokens over that cache, and sampling of the next tokens.

A step of a server that keeps many sequences of unequal lengths on the GPU runs them in this order:
the plan gives every new token its place in the cache (block tables and slots from the sequences'
lengths), the append normalises, rotates and stores the new keys and values, attention reads each
sequence's pages, and the sampler picks the tokens from the logits and given random numbers.

`own = False` computes the operators in elementary torch operations; `own = True` calls
trixium_b200.ops.
"""

import math
import random

import torch

own = False

_F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# Cases ----------------------------------------------------------------------------------------------

def listed():
    qwen8b = dict(n_head=32, n_kv=8, head_dim=128, rope_dims=128, gated=False)
    qwen17 = dict(n_head=16, n_kv=8, head_dim=128, rope_dims=128, gated=False)
    hybrid27 = dict(n_head=24, n_kv=4, head_dim=256, rope_dims=64, gated=True)
    return [
        # One token for each of 32 running sequences: the plan of every decode step.
        dict(name="plan_decode", op="plan", nseq=32, single=100, idle=0, new_lo=1, new_hi=1, ctx_lo=500, ctx_hi=2000,
             mix=1, page=16, max_pages=256),
        # A busy server: most sequences decode, some bring a prompt chunk, some wait.
        dict(name="plan_mixed", op="plan", nseq=256, single=75, idle=5, new_lo=2, new_hi=1024, ctx_lo=0, ctx_hi=8192,
             mix=2, page=16, max_pages=1024),
        # The append of a decode step at batch 16.
        dict(name="append_decode", op="append", nseq=16, single=100, idle=0, new_lo=1, new_hi=1, ctx_lo=700,
             ctx_hi=1100, mix=3, page=16, cache="f16", q="f16", **qwen8b),
        # The append of several prompts' chunks, gated heads of 256 with a partial rotation.
        dict(name="append_chunk", op="append", nseq=5, single=0, idle=0, new_lo=300, new_hi=1001, ctx_lo=0, ctx_hi=4000,
             mix=4, page=64, cache="bf16", q="bf16", **hybrid27),
        # Decode at batch 16 and about 1,000 tokens of context.
        dict(name="attn_decode", op="attn", nseq=16, single=100, idle=0, new_lo=1, new_hi=1, ctx_lo=700, ctx_hi=1100,
             mix=5, page=16, cache="f16", q="f16", window=0, sinks=0, **qwen8b),
        # Decode of a few long sequences, the queries kept in 32 bits.
        dict(name="attn_decode_long", op="attn", nseq=3, single=100, idle=0, new_lo=1, new_hi=1, ctx_lo=28000,
             ctx_hi=32000, mix=6, page=32, cache="f16", q="f32", window=0, sinks=0, **qwen17),
        # One prompt chunk behind a cached prefix: the arithmetic-bound end.
        dict(name="attn_chunk", op="attn", nseq=1, single=0, idle=0, new_lo=2048, new_hi=2048, ctx_lo=6001, ctx_hi=6001,
             mix=7, page=64, cache="f16", q="f16", window=0, sinks=0, **qwen8b),
        # Prompt chunks and decoding sequences in one call, gated heads of 256.
        dict(name="attn_mixed", op="attn", nseq=9, single=60, idle=0, new_lo=100, new_hi=700, ctx_lo=0, ctx_hi=4096,
             mix=8, page=16, cache="bf16", q="bf16", window=0, sinks=0, **hybrid27),
        # A long chunk with a sliding window and the first tokens kept visible, queries in 32 bits.
        dict(name="attn_window", op="attn", nseq=1, single=0, idle=0, new_lo=4096, new_hi=4096, ctx_lo=4000,
             ctx_hi=4000, mix=9, page=16, cache="f16", q="f32", window=1024, sinks=4, **qwen17),
        # The token of one interactive sequence, every filter on.
        dict(name="sample_one", op="sample", rows=1, vocab=151936, logits="f32", modes="all"),
        # The tokens of a batch of 32 with each request's own settings.
        dict(name="sample_batch", op="sample", rows=32, vocab=151936, logits="f32", modes="mixed"),
        # Many sequences over a smaller, odd vocabulary, logits of 16 bits with many ties.
        dict(name="sample_many", op="sample", rows=333, vocab=32003, logits="bf16", modes="mixed"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_once(rng):
    op = rng.choice(["plan", "append", "attn", "attn", "attn", "sample", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log_int(rng, 1, 333), vocab=_log_int(rng, 1000, 151936),
                    logits=rng.choice(["f32", "f32", "f16", "bf16"]), modes=rng.choice(["all", "mixed", "mixed"]))
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        return dict(op=op, nseq=_log_int(rng, 1, 256), single=rng.choice([0, 50, 75, 100]), idle=rng.choice([0, 5, 20]),
                    new_lo=1, new_hi=_log_int(rng, 1, 1024), ctx_lo=0, ctx_hi=_log_int(rng, 16, 8192),
                    mix=rng.randrange(1 << 30), page=page, max_pages=9216 // page)
    hd = rng.choice([64, 128, 128, 256])
    n_kv = rng.choice([1, 2, 4, 8])
    gated = rng.random() < 0.3
    cache = rng.choice(["f16", "f16", "bf16"])
    c = dict(op=op, single=rng.choice([0, 50, 100, 100]), idle=rng.choice([0, 0, 10]), new_lo=1,
             mix=rng.randrange(1 << 30), page=page, cache=cache,
             q=rng.choice(["f16", "f32"]) if cache == "f16" else "bf16", n_head=n_kv * rng.choice([1, 2, 3, 4, 6, 8]),
             n_kv=n_kv, head_dim=hd, rope_dims=hd if rng.random() < 0.6 else hd // 4, gated=gated, ctx_lo=0)
    c["nseq"] = _log_int(rng, 1, 32)
    c["new_hi"] = _log_int(rng, 1, 4096)
    c["ctx_hi"] = _log_int(rng, 1, 32000)
    if op == "attn":
        c["window"] = _log_int(rng, 1, 4096) if rng.random() < 0.3 else 0
        c["sinks"] = rng.choice([0, 1, 4, 130]) if c["window"] else 0
    return c


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        t = top.setdefault(c["op"], [0, 0])
        t[0], t[1] = max(t[0], w["bytes"]), max(t[1], w["flops"])
    while True:
        c = _draw_once(rng)
        w = work(c)
        if w["bytes"] > top[c["op"]][0] or w["flops"] > top[c["op"]][1]:
            continue
        if c["op"] == "append" and sum(_lens(c)[0]) > 4000:
            continue
        if c["op"] != "sample" and sum(_lens(c)[0]) == 0:
            continue
        return c


def _lens(case):
    """New and cached tokens of every sequence, from the case alone."""
    r = random.Random(case["mix"])
    new, cached = [], []
    for _ in range(case["nseq"]):
        p = r.random() * 100
        if p < case["idle"]:
            n = 0
        elif p < case["idle"] + case["single"]:
            n = 1
        else:
            n = r.randint(case["new_lo"], case["new_hi"])
        new.append(n)
        cached.append(r.randint(case["ctx_lo"], case["ctx_hi"]))
    return new, cached


# What a pass cannot do without ------------------------------------------------------------------------

_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _visible(pos, window, sinks):
    """Positions a query at `pos` sees."""
    if not window or pos + 1 <= window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        return {"bytes": n * v * _SIZE[case["logits"]] + 24 * n, "flops": 4 * n * v}
    new, cached = _lens(case)
    rows, p = sum(new), case["page"]
    if case["op"] == "plan":
        taken = sum(-(-(n + c) // p) - -(-c // p) for n, c in zip(new, cached))
        return {"bytes": 4 * (2 * case["nseq"] + 2 * taken + 2 * rows + 3 * case["nseq"] + 3), "flops": rows}
    h, kv, hd = case["n_head"], case["n_kv"], case["head_dim"]
    if case["op"] == "append":
        read = rows * (h + 2 * kv) * hd * 4
        write = rows * hd * (h * _SIZE[case["q"]] + 2 * kv * _SIZE[case["cache"]])
        return {"bytes": read + write + 8 * rows, "flops": rows * (h + kv) * hd * 6}
    pairs = kvread = 0
    for n, c in zip(new, cached):
        if n == 0:
            continue
        w, s = case["window"], case["sinks"]
        if w:
            pairs += sum(_visible(c + i, w, s) for i in range(n))
            lo = max(0, c + 1 - w)
            kvread += c + n - lo + min(s, lo)
        else:
            pairs += n * c + n * (n + 1) // 2
            kvread += c + n
    byts = 2 * rows * h * hd * _SIZE[case["q"]] + 2 * kvread * kv * hd * 2
    byts += rows * h * hd * 4 if case["gated"] else 0
    byts += 4 * sum(-(-(n + c) // p) for n, c in zip(new, cached) if n)
    return {"bytes": byts, "flops": 4 * pairs * h * hd}


# Inputs -----------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _inputs(case, seed):
    g = _gen(seed)
    dev = "cuda"
    randn = lambda *s, dt=torch.float32: torch.randn(*s, generator=g, device=dev).to(dt)
    if case["op"] == "sample":
        n, v = case["rows"], case["vocab"]
        r = random.Random(seed)
        # Logits as a language model gives them: a broad bulk and a few tokens far above it.
        x = randn(n, v) * 2.2
        hot = torch.randint(0, v, (n, 24), generator=g, device=dev)
        x.scatter_add_(1, hot, 6.0 + 3.0 * randn(n, 24).abs())
        temp, k, p, m = [], [], [], []
        for i in range(n):
            mode = 5 if case["modes"] == "all" else r.randrange(6)
            temp.append(0.0 if mode == 0 else r.uniform(0.5, 1.3))
            k.append(r.randint(5, 200) if mode in (2, 5) else 0)
            p.append(r.uniform(0.7, 0.98) if mode in (3, 5) else 1.0)
            m.append(r.uniform(0.01, 0.1) if mode in (4, 5) else 0.0)
        f = lambda a: torch.tensor(a, dtype=torch.float32, device=dev)
        return dict(logits=x.to(_F[case["logits"]]), u=torch.rand(n, generator=g, device=dev), temperature=f(temp),
                    top_k=torch.tensor(k, dtype=torch.int32, device=dev), top_p=f(p), min_p=f(m))
    new, cached = _lens(case)
    b, page, rows = case["nseq"], case["page"], sum(new)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
    have = [-(-c // page) for c in cached]
    need = [-(-(n + c) // page) if n else h for n, c, h in zip(new, cached, have)]
    max_pages = case.get("max_pages") or max(1, max(need))
    n_pages = sum(need) + 37
    perm = torch.randperm(n_pages, generator=g, device=dev).to(torch.int32)
    used = sum(have)
    tables = torch.full((b, max_pages), -1, dtype=torch.int32, device=dev)
    ph = perm.cpu()
    host = torch.full((b, max_pages), -1, dtype=torch.int32)
    at = 0
    for i, h in enumerate(have):
        host[i, :h] = ph[at:at + h]
        at += h
    tables.copy_(host)
    st = dict(cached=i32(cached), new=i32(new), free=perm[used:].clone(), n_free=i32([n_pages - used]), tables=tables,
              n_pages=n_pages)
    if case["op"] == "plan":
        return st
    # The plan's outputs: the tables with the new pages, row offsets, positions and slots.
    take = n_pages - used
    for i in range(b):
        for j in range(have[i], need[i]):
            take -= 1
            host[i, j] = ph[used + take]
    tables.copy_(host)
    cu, pos, slots = [0], [], []
    for i in range(b):
        p0 = torch.arange(cached[i], cached[i] + new[i])
        pos.append(p0)
        slots.append(host[i].long()[p0 // page] * page + p0 % page)
        cu.append(cu[-1] + new[i])
    st.update(lens=i32([n + c for n, c in zip(new, cached)]), cu=i32(cu), pos=torch.cat(pos).to(torch.int32).to(dev),
              slots=torch.cat(slots).to(torch.int32).to(dev), rows=rows, max_pages=max_pages, max_new=max(new))
    h, kv, hd = case["n_head"], case["n_kv"], case["head_dim"]
    pool = lambda: randn(n_pages, page, kv, hd, dt=_F[case["cache"]])
    st["kpages"], st["vpages"] = pool(), pool()
    if case["op"] == "append":
        st["q"] = randn(rows, h * hd * (2 if case["gated"] else 1)) * 1.7
        st["k"], st["v"] = randn(rows, kv * hd) * 1.3, randn(rows, kv * hd)
        st["q_norm"], st["k_norm"] = 1 + 0.1 * randn(hd), 1 + 0.1 * randn(hd)
        n = case["rope_dims"]
        st["rope_freq"] = (1e6 ** (-2.0 * torch.arange(n // 2, dtype=torch.float64) / n)).to(torch.float32).to(dev)
        st["q_out"] = torch.zeros(rows, h, hd, dtype=_F[case["q"]], device=dev)
    else:
        st["q"] = randn(rows, h, hd, dt=_F[case["q"]])
        st["gate"] = randn(rows, h * 2 * hd) if case["gated"] else None
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    st["case"] = case
    if not own or case["op"] == "sample":
        if own:
            from trixium_b200 import ops
            st["ctx"] = ops.default_context()
        elif case["op"] == "plan":
            st["rows_cap"] = sum(_lens(case)[0])
        return st
    from trixium_b200 import ops
    st["ctx"] = ops.default_context()
    rows = sum(_lens(case)[0])
    plan = st["plan"] = ops.PagedPlan(case["nseq"], rows, st["tables"].shape[1], case["page"], st["n_pages"])
    plan.tables.copy_(st["tables"])
    if case["op"] != "plan":
        plan.lens.copy_(st["lens"])
        plan.cu.copy_(st["cu"])
        plan.pos.copy_(st["pos"])
        plan.slots.copy_(st["slots"])
        st["shape"] = ops.paged_shape(case["n_head"], case["n_kv"], case["head_dim"], rope_dims=case["rope_dims"],
                                      gated=case["gated"], eps=1e-6, window=case.get("window", 0),
                                      sinks=case.get("sinks", 0))
    return st


# One pass ---------------------------------------------------------------------------------------------

def run(st):
    op = st["case"]["op"]
    if own:
        from trixium_b200 import ops
        ctx = st["ctx"]
        if op == "plan":
            plan = ops.paged_plan(ctx, st["plan"], st["cached"], st["new"], st["free"], st["n_free"])
            return [plan.tables, plan.lens, plan.cu, plan.slots, plan.pos, plan.n_free]
        if op == "append":
            q = ops.paged_append(ctx, st["shape"], st["plan"], st["q"], st["k"], st["v"], st["q_norm"], st["k_norm"],
                                 st["rope_freq"], st["kpages"], st["vpages"], q_out=st["q_out"])
            return [q, st["kpages"], st["vpages"]]
        if op == "attn":
            return ops.attn_paged(ctx, st["shape"], st["plan"], st["q"], st["kpages"], st["vpages"], gate=st["gate"],
                                  max_new=st["max_new"])
        return ops.sample_rows(ctx, st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])
    return {"plan": _plan, "append": _append, "attn": _attn, "sample": _sample}[op](st)


def _plan(st):
    page = st["case"]["page"]
    cached, new, free = st["cached"], st["new"], st["free"]
    dev = cached.device
    lens = cached + new
    have = (cached + page - 1) // page
    need = torch.where(new > 0, (lens + page - 1) // page, have)
    first = torch.cumsum(need - have, 0) - (need - have)
    col = torch.arange(st["tables"].shape[1], device=dev)[None, :]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    idx = st["n_free"] - 1 - (first[:, None] + col - have[:, None])
    tables = torch.where(fresh, free[idx.clamp(0, free.numel() - 1).long()], st["tables"])
    cu = torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), torch.cumsum(new, 0)])
    row = torch.arange(st["rows_cap"], device=dev)
    seq = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    pos = cached[seq] + row - cu[seq]
    slots = tables[seq, pos // page] * page + pos % page
    n_free = st["n_free"] - torch.sum(need - have)
    i32 = torch.int32
    return [tables, lens.to(i32), cu.to(i32), slots.to(i32), pos.to(i32), n_free.to(i32)]


def _rotate(x, pos, freq, w, eps):
    """RMSNorm over the head, then the rotation of pairs (d, d + half) by pos * freq rounded to 32 bits."""
    x = x * torch.rsqrt(torch.mean(x * x, -1, keepdim=True) + eps) * w
    half = freq.numel()
    ang = (pos.float()[:, None] * freq[None, :]).double()
    c, s = torch.cos(ang).float()[:, None, :], torch.sin(ang).float()[:, None, :]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def _append(st):
    c = st["case"]
    h, kv, hd, rows = c["n_head"], c["n_kv"], c["head_dim"], st["rows"]
    q = st["q"].view(rows, h, -1)[..., :hd]
    qr = _rotate(q, st["pos"], st["rope_freq"], st["q_norm"], 1e-6)
    kr = _rotate(st["k"].view(rows, kv, hd), st["pos"], st["rope_freq"], st["k_norm"], 1e-6)
    st["q_out"].copy_(qr)
    slots = st["slots"].long()
    st["kpages"].view(-1, kv, hd)[slots] = kr.to(st["kpages"].dtype)
    st["vpages"].view(-1, kv, hd)[slots] = st["v"].view(rows, kv, hd).to(st["vpages"].dtype)
    return [st["q_out"], st["kpages"], st["vpages"]]


def _attn(st):
    c = st["case"]
    h, kv, hd, page = c["n_head"], c["n_kv"], c["head_dim"], c["page"]
    rep = h // kv
    new, cached = _lens(c)
    out = torch.empty(st["rows"], h, hd, dtype=torch.float32, device="cuda")
    row = 0
    for i, (n, m) in enumerate(zip(new, cached)):
        if n == 0:
            continue
        length = n + m
        pages = st["tables"][i, :-(-length // page)].long()
        k = st["kpages"][pages].reshape(-1, kv, hd)[:length].float()
        v = st["vpages"][pages].reshape(-1, kv, hd)[:length].float()
        q = st["q"][row:row + n].float().view(n, kv, rep, hd)
        qp = torch.arange(m, length, device="cuda")[:, None]
        kp = torch.arange(length, device="cuda")[None, :]
        seen = kp <= qp
        if c["window"]:
            seen &= (kp > qp - c["window"]) | (kp < c["sinks"])
        for j in range(kv):
            s = torch.matmul(q[:, j].permute(1, 0, 2), k[:, j].t()) / math.sqrt(hd)
            s = s.masked_fill(~seen, -math.inf)
            e = torch.exp(s - s.amax(-1, keepdim=True))
            o = torch.matmul(e, v[:, j]) / e.sum(-1, keepdim=True)
            out[row:row + n, j * rep:(j + 1) * rep] = o.permute(1, 0, 2)
        row += n
    if st["gate"] is not None:
        g = st["gate"].view(st["rows"], h, 2 * hd)[..., hd:]
        out = out / (1 + torch.exp(-g))
    return out.to(_F[c["q"]])


def _sample(st):
    """Descending by logit, ties by index; the first top_k; of those the shortest prefix whose share
    reaches top_p; of those the tokens of at least min_p times the largest probability.  The token is
    the first in index order whose running weight passes u times the total."""
    x = st["logits"].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    n, v = x.shape
    t = st["temperature"].double()[:, None]
    vals, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = vals[:, :1]
    greedy = t <= 0
    w = torch.exp((vals - top) / torch.where(greedy, torch.ones_like(t), t))
    w = torch.where(vals == top, torch.ones_like(w), w)
    w = torch.where(torch.isneginf(vals), torch.zeros_like(w), w)
    rank = torch.arange(v, device=x.device)[None, :]
    k = st["top_k"][:, None].long()
    w = torch.where((k > 0) & (rank >= k), torch.zeros_like(w), w)
    before = torch.cumsum(w, 1) - w
    p = st["top_p"].double()[:, None]
    w = torch.where((p < 1) & (rank > 0) & (before >= p * w.sum(1, keepdim=True)), torch.zeros_like(w), w)
    w = torch.where(w >= st["min_p"].double()[:, None], w, torch.zeros_like(w))
    by_index = torch.zeros_like(w).scatter_(1, order, w)
    run_sum = torch.cumsum(by_index, 1)
    target = st["u"].double()[:, None] * run_sum[:, -1:]
    token = (run_sum <= target).sum(1)
    last = (by_index > 0).mul(rank + 1).amax(1) - 1
    token = torch.minimum(token, last)
    return torch.where(greedy[:, 0], torch.where(torch.isneginf(top[:, 0]), -1, order[:, 0]), token).to(torch.int32)


# The definitions in 64 bits ---------------------------------------------------------------------------

def exact(case, seed):
    if case["op"] in ("plan", "sample"):
        return None
    st = _inputs(case, seed)
    h, kv, hd, page = case["n_head"], case["n_kv"], case["head_dim"], case["page"]
    rows = st["rows"]
    f64 = torch.float64
    if case["op"] == "append":
        half = case["rope_dims"] // 2
        # The angle of a rotation is the 32-bit product of position and frequency, as in the cache's
        # other writers.
        ang = torch.outer(st["pos"].to(torch.float32), st["rope_freq"]).to(f64).view(rows, 1, half)
        spin = torch.polar(torch.ones_like(ang), ang)

        def head(x, w):
            x = x.to(f64)
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / hd + 1e-6) * w.to(f64)
            z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * spin
            return torch.cat((z.real, z.imag, x[..., 2 * half:]), dim=-1)

        kp, vp = st["kpages"].to(f64), st["vpages"].to(f64)
        at = st["slots"].long()
        kp.view(-1, kv, hd).index_copy_(0, at, head(st["k"].view(rows, kv, hd), st["k_norm"]))
        vp.view(-1, kv, hd).index_copy_(0, at, st["v"].view(rows, kv, hd).to(f64))
        return [head(st["q"].view(rows, h, -1)[:, :, :hd], st["q_norm"]), kp, vp]
    new, cached = _lens(case)
    out = torch.zeros(rows, h, hd, dtype=f64, device="cuda")
    start = 0
    for i in range(case["nseq"]):
        total = new[i] + cached[i]
        if new[i] == 0:
            continue
        at = torch.arange(total, device="cuda")
        slot = st["tables"][i].long()[at // page] * page + at % page
        for lo in range(0, new[i], 512):
            n = min(512, new[i] - lo)
            here = cached[i] + lo + torch.arange(n, device="cuda").view(n, 1)
            hidden = at.view(1, -1) > here
            if case["window"]:
                hidden |= (here - at >= case["window"]) & (at >= case["sinks"])
            for j in range(h):
                g = j // (h // kv)
                key = st["kpages"].view(-1, kv, hd)[slot, g].to(f64)
                val = st["vpages"].view(-1, kv, hd)[slot, g].to(f64)
                s = st["q"][start + lo:start + lo + n, j].to(f64) @ key.T * hd ** -0.5
                out[start + lo:start + lo + n, j] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ val
        start += new[i]
    if st["gate"] is not None:
        out *= torch.sigmoid(st["gate"].view(rows, h, 2, hd)[:, :, 1].to(f64))
    return out
