"""Plain 64-bit restatements of the paged-cache operators, and cases for their tests."""
import math

import torch


def pages_of(n, page):
    return -(-n // page)


def plan(cached, new, tables, free, n_free, page):
    """Host plan: (tables, lens, cu, slots, pos, last, n_free) as Python lists; free is a list."""
    tables = [list(t) for t in tables]
    cu, slots, pos, last, lens = [0], [], [], [], []
    for b, (c, n) in enumerate(zip(cached, new)):
        if n:
            for j in range(pages_of(c, page), pages_of(c + n, page)):
                n_free -= 1
                tables[b][j] = free[n_free]
        for p in range(c, c + n):
            slots.append(tables[b][p // page] * page + p % page)
            pos.append(p)
        cu.append(cu[-1] + n)
        last.append(cu[-1] - 1 if n else 0)
        lens.append(c + n)
    return tables, lens, cu, slots, pos, last, n_free


def rotate(x, pos, freq, w, eps):
    """RMSNorm and rotation of x [rows, heads, hd] in 64 bits (the angle is the fp32 product)."""
    hd, half = x.shape[-1], freq.numel()
    x = x.double()
    x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + eps) * w.double()
    if not half:
        return x
    ang = (pos.float()[:, None] * freq[None, :]).double()[:, None, :]
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., 2 * half:]], -1)


def visible(p0, n, length, window, sinks, device):
    q = torch.arange(p0, p0 + n, device=device)[:, None]
    k = torch.arange(length, device=device)[None, :]
    m = k <= q
    if window:
        m &= (q - k < window) | (k < sinks)
    return m


def attention(q, k, v, p0, window=0, sinks=0):
    """q [n, H, hd] at positions p0.., k, v [L, n_kv, hd]: (out, weighted |v|, largest sum |q||k|) in 64
    bits; the second is what a relative error of the weights is scaled by, the third bounds the scores'."""
    n, H, hd = q.shape
    kv = k.shape[1]
    rep = H // kv
    q, k, v = q.double(), k.double(), v.double()
    m = visible(p0, n, k.shape[0], window, sinks, q.device)
    out, mag = torch.empty_like(q), torch.empty_like(q)
    smax = 0.0
    for h in range(H):
        g = h // rep
        s = q[:, h] @ k[:, g].T / math.sqrt(hd)
        s = s.masked_fill(~m, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out[:, h] = p @ v[:, g]
        mag[:, h] = p @ v[:, g].abs()
        smax = max(smax, float((q[:, h].abs() @ k[:, g].abs().T).max()) / math.sqrt(hd))
    return out, mag, smax


class Cache:
    """Pools whose unused places hold NaN, tables in random order, for sequences of the given lengths
    (positions in the cache after the step)."""

    def __init__(self, ops, lens, new, kv, hd, page, dtype, seed, spare=5, max_rows=None, fill=float("nan")):
        g = torch.Generator().manual_seed(seed)
        need = [pages_of(n, page) for n in lens]
        n_pages = sum(need) + spare
        perm = torch.randperm(n_pages, generator=g).tolist()
        rows = sum(new)
        self.plan = ops.PagedPlan(len(lens), max_rows or max(rows, 1), max(max(need), 1), page, n_pages)
        dev = "cuda"
        kp = torch.full((n_pages, page, kv, hd), fill, dtype=dtype)
        vp = torch.full_like(kp, fill)
        self.k, self.v = [], []
        tab = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(lens):
            ids = perm[at:at + need[b]]
            at += need[b]
            tab[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
            k = torch.randn(n, kv, hd, generator=g).to(dtype)
            v = torch.randn(n, kv, hd, generator=g).to(dtype)
            for j, i in enumerate(ids):
                part = k[j * page:(j + 1) * page]
                kp[i, :len(part)] = part
                vp[i, :len(part)] = v[j * page:(j + 1) * page]
            self.k.append(k.to(dev))
            self.v.append(v.to(dev))
        self.kp, self.vp = kp.to(dev), vp.to(dev)
        self.plan.tables.copy_(tab)
        self.plan.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        self.plan.cu.copy_(torch.tensor(cu, dtype=torch.int32))
        self.cu, self.lens, self.new, self.rows = cu, lens, new, rows
        self.free = perm[at:]

    def check(self, q, out, gate=None, window=0, sinks=0):
        """Assert out against the 64-bit attention of every sequence's rows.  Tolerance, per element, of A =
        sum p |v|: a 16-bit type rounds each weight and the output by half a step h (h A + h |ref|); the
        scores' error moves the weights by 2 ds with ds <= (2^-22 + 16 * 2^-23) sum |q||k| for split
        queries (products exact to 2^-22, sixteen roundings on the way of a sum of at most 256 products of
        tensor-core depth 16) and 16 * 2^-23 for exact 16-bit products; ex2, the rescalings and the joining
        of pieces add 2^-19, the sum of L weights L * 2^-26."""
        f32 = q.dtype == torch.float32
        h = 0.0 if f32 else torch.finfo(q.dtype).eps / 2
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            r0, L = self.cu[b], self.lens[b]
            ref, mag, smax = attention(q[r0:r0 + n], self.k[b], self.v[b], L - n, window, sinks)
            ds = smax * (17 * 2.0 ** -23 + 2.0 ** -22)
            if gate is not None:
                H, hd = q.shape[1:]
                s = torch.sigmoid(gate[r0:r0 + n].view(n, H, 2, hd)[:, :, 1].double())
                ref, mag = ref * s, mag * s
            tol = h * ref.abs() + mag * (h + 2 * ds + 2.0 ** -19 + L * 2.0 ** -26) + 1e-30
            if not f32:
                tol = tol + torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps
            err = (out[r0:r0 + n].double() - ref).abs()
            assert bool(torch.isfinite(out[r0:r0 + n]).all()), (b, "not finite")
            worst = float((err / tol).max())
            assert worst <= 1.0, (b, n, L, worst)
