"""Sampling (trx_sample_rows) against a plain restatement of its definition in 64-bit floats: the sort,
the filters and the draw, row by row in numpy."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from trixium_b200 import ops as o
    return o


@pytest.fixture(scope="module")
def ctx(ops):
    c = ops.Context(0)
    yield c
    c.close()


def draw(x, u, t, k, p, m):
    """The definition for one row of float64 logits."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.argsort(-x, kind="stable")
    top = x[order[0]]
    if top == -np.inf:
        return -1
    if not t > 0:
        return int(order[0])
    v = x[order]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((v - top) / t)
    w[v == top] = 1.0
    w[v == -np.inf] = 0.0
    if k > 0:
        w[k:] = 0
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        cut = before >= p * w.sum()
        cut[0] = False
        w[cut] = 0
    w[~(w >= m)] = 0
    by = np.zeros_like(w)
    by[order] = w
    run = np.cumsum(by)
    if run[-1] == 0:
        return -1
    return int(min(np.searchsorted(run, u * run[-1], side="right"), np.flatnonzero(by)[-1]))


def check(ops, ctx, x, u, t, k, p, m):
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")
    got = ops.sample_rows(ctx, x, f(u), f(t), torch.tensor(k, dtype=torch.int32, device="cuda"), f(p), f(m)).tolist()
    xs = x.double().cpu().numpy()
    r = lambda a: np.asarray(a, dtype=np.float32).astype(np.float64)
    want = [draw(xs[i], r(u)[i], r(t)[i], k[i], r(p)[i], r(m)[i]) for i in range(len(u))]
    assert got == want
    assert ctx.errors() == 0


def settings(rng, n):
    t = rng.choice([0.0, 0.3, 0.8, 1.0, 1.7, 50.0], n)
    k = rng.choice([0, 0, 1, 2, 17, 50, 400, 3000, 10 ** 6], n)
    p = rng.choice([1.0, 1.0, 0.0, 0.1, 0.5, 0.9, 0.999], n)
    m = rng.choice([0.0, 0.0, 0.01, 0.2, 1.0], n)
    return t.tolist(), [int(i) for i in k], p.tolist(), m.tolist()


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4099, 32003, 151936])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n", [1, 24])
def test_sampling_matches_definition(ops, ctx, V, dtype, n):
    rng = np.random.default_rng(V + n)
    g = torch.Generator().manual_seed(V)
    x = torch.randn(n, V, generator=g) * 2.5
    x[:, :: max(1, V // 20)] += 5 * torch.rand(n, x[:, :: max(1, V // 20)].shape[1], generator=g)
    for rep in range(3):
        t, k, p, m = settings(rng, n)
        check(ops, ctx, x.to(getattr(torch, dtype)).cuda(), rng.random(n, dtype=np.float32).tolist(), t, k, p, m)


@pytest.mark.parametrize("kind", ["equal", "two_values", "one_high", "wide", "narrow", "minus_inf", "nan", "plus_inf",
                                  "zeros", "signed_zeros", "lowest"])
@pytest.mark.parametrize("V", [700, 60001])
def test_sampling_odd_rows(ops, ctx, kind, V):
    """Ties across every border, rows with masked, infinite and undefined logits."""
    n = 40
    rng = np.random.default_rng(len(kind) + V)
    g = torch.Generator().manual_seed(V)
    x = torch.randn(n, V, generator=g)
    if kind == "equal":
        x = torch.full((n, V), -3.25)
    elif kind == "two_values":
        x = (x > 0.5).float() * 2
    elif kind == "one_high":
        x[:, V // 3] = 1e4
    elif kind == "wide":
        x *= 1e30
    elif kind == "narrow":
        x = 5 + x * 1e-6
    elif kind == "minus_inf":
        x[x < 1.0] = -float("inf")
    elif kind == "nan":
        x[:, ::3] = float("nan")
    elif kind == "plus_inf":
        x[:, 5::97] = float("inf")
    elif kind == "zeros":
        x = torch.zeros(n, V)
        x[:, ::2] = -0.0
        x = x + 0.0
    elif kind == "signed_zeros":  # equal: ties by index
        x = torch.round(x * 0.6)
    else:
        x[x < 1.2] = torch.finfo(torch.float32).min
    t, k, p, m = settings(rng, n)
    check(ops, ctx, x.cuda(), rng.random(n, dtype=np.float32).tolist(), t, k, p, m)


@pytest.mark.parametrize("n", [2, 5])
@pytest.mark.parametrize("V", [163841, 262147, 1000003])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_sampling_rows_beyond_shared_memory(ops, ctx, n, V, dtype):
    """Rows too long to be kept on chip are read again in every pass (few rows: kept by larger clusters)."""
    rng = np.random.default_rng(V)
    x = torch.randn(n, V, generator=torch.Generator().manual_seed(V)) * 3
    for rep in range(3):
        t, k, p, m = settings(rng, n)
        check(ops, ctx, x.to(getattr(torch, dtype)).cuda(), rng.random(n, dtype=np.float32).tolist(), t, k, p, m)


def test_sampling_many_rows(ops, ctx):
    """More rows than clusters fit the device at once."""
    n, V = 1500, 2003
    rng = np.random.default_rng(2)
    t, k, p, m = settings(rng, n)
    check(ops, ctx, torch.randn(n, V, generator=torch.Generator().manual_seed(2)).cuda() * 3,
          rng.random(n, dtype=np.float32).tolist(), t, k, p, m)


def test_sampling_undefined_and_infinite_settings(ops, ctx):
    """Settings outside the definition's ranges end in a token of the row or -1."""
    x = torch.randn(6, 5003, generator=torch.Generator().manual_seed(4)).cuda()
    nan, inf = float("nan"), float("inf")
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")
    k = torch.tensor([0, 7, 0, 3000, -1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    for t, p, m, u in ((inf, 0.9, 0.0, 0.5), (nan, 0.9, 0.1, 0.5), (1e-40, 0.9, 0.0, 0.5), (0.8, nan, 0.0, 0.5),
                       (0.8, 0.9, nan, 0.5), (0.8, 0.9, 0.0, nan), (0.8, 0.9, 0.0, -3.0), (0.8, 0.9, 0.0, inf),
                       (0.8, -1.0, 0.0, 0.5), (0.8, 0.9, -1.0, 2.0), (-inf, inf, inf, 0.5), (0.8, 1e-30, 0.0, 0.5)):
        tok = ops.sample_rows(ctx, x, f([u] * 6), f([t] * 6), k, f([p] * 6), f([m] * 6))
        assert bool(((tok >= -1) & (tok < 5003)).all()), (t, p, m, u, tok)
    assert ctx.errors() == 0


def test_sampling_rows_without_a_token(ops, ctx):
    x = torch.full((3, 5000), -float("inf"), device="cuda")
    x[1] = float("nan")
    x[2, 4321] = -1e30
    check(ops, ctx, x, [0.5] * 3, [1.0, 0.0, 0.7], [0, 5, 3], [0.9, 1.0, 0.5], [0.0, 0.1, 0.1])
    check(ops, ctx, x, [0.5] * 3, [1.0] * 3, [0] * 3, [1.0] * 3, [1.5] * 3)  # min_p above 1 keeps nothing


@pytest.mark.parametrize("u", [0.0, 1.0 - 2.0 ** -24, 1.0])
def test_sampling_ends_of_the_draw(ops, ctx, u):
    x = torch.randn(8, 3001, generator=torch.Generator().manual_seed(1)).cuda()
    x[:, -7:] = -float("inf")
    x[:, :3] = -float("inf")
    check(ops, ctx, x, [u] * 8, [1.0] * 8, [0, 0, 5, 5, 0, 0, 2000, 2990], [1.0, 0.9, 1.0, 0.5, 1.0, 0.2, 1.0, 0.99],
          [0, 0, 0, 0, 0.3, 0, 0, 0.0])


def test_sampling_frequencies(ops, ctx):
    """Over an even grid of random numbers every token comes as often as its share, to one draw."""
    n, V = 4096, 11
    row = torch.tensor([0.0, 1.0, -2.0, 0.5, 1.0, -float("inf"), 2.0, 0.0, -1.0, 0.25, 1.5])
    x = row.expand(n, V).contiguous().cuda()
    u = ((torch.arange(n) + 0.5) / n).cuda()
    one = torch.ones(n, device="cuda")
    tok = ops.sample_rows(ctx, x, u, one, torch.zeros(n, dtype=torch.int32, device="cuda"), one, 0 * one)
    share = torch.bincount(tok.long(), minlength=V).cpu().double() / n
    want = torch.softmax(row.double(), 0)
    assert float((share - want).abs().max()) <= 1.0 / n


def test_sampling_strided_rows_graph_and_stream(ops, ctx):
    rng = np.random.default_rng(0)
    wide = torch.randn(6, 2 * 5003, generator=torch.Generator().manual_seed(3)).cuda()
    x = wide[:, 5003 // 2:5003 // 2 + 5003]
    t, k, p, m = settings(rng, 6)
    check(ops, ctx, x, rng.random(6, dtype=np.float32).tolist(), t, k, p, m)
    f = lambda a: torch.tensor(a, dtype=torch.float32, device="cuda")
    args = [torch.rand(6, device="cuda"), f([0.9] * 6), torch.full((6,), 40, dtype=torch.int32, device="cuda"),
            f([0.9] * 6), f([0.0] * 6)]
    tok = torch.zeros(6, dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.sample_rows(ctx, x, *args, tokens=tok)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_rows(ctx, x, *args, tokens=tok)
    for _ in range(3):
        wide.copy_(torch.randn_like(wide))
        args[0].copy_(torch.rand(6))
        tok.fill_(-9)
        graph.replay()
        torch.cuda.synchronize()
        want = ops.sample_rows(ctx, x, *args)
        assert tok.tolist() == want.tolist()
        check(ops, ctx, x, args[0].tolist(), [0.9] * 6, [40] * 6, [0.9] * 6, [0.0] * 6)


@pytest.mark.parametrize("V", [700, 60001])
@pytest.mark.parametrize("temperature", [1e-45, 1e-40, 4e-38, 1e-37, 7e-31, 1e-20])
def test_sampling_tiny_temperatures(ops, ctx, V, temperature):
    """The largest logits' ties alone have weight: the definition's token, cut by top-k and drawn by u."""
    n = 24
    rng = np.random.default_rng(V)
    x = torch.round(torch.randn(n, V, generator=torch.Generator().manual_seed(V)) * 4)
    x[::2] = torch.round(x[::2] / 8)  # many ties
    _, k, p, m = settings(rng, n)
    check(ops, ctx, x.cuda(), rng.random(n, dtype=np.float32).tolist(), [temperature] * n, k, p, m)


@pytest.mark.parametrize("V", [700, 60001])
@pytest.mark.parametrize("size", [1e-44, 1e-40, 1e-38, 1e-37, 1e-36, 1e-30])
def test_sampling_logits_next_to_zero(ops, ctx, V, size):
    """Equal weights in an order of their own, the logits' differences down to the smallest number."""
    n = 24
    rng = np.random.default_rng(V)
    x = torch.randn(n, V, generator=torch.Generator().manual_seed(V)) * size
    t, k, p, m = settings(rng, n)
    check(ops, ctx, x.cuda(), rng.random(n, dtype=np.float32).tolist(), t, k, p, m)
