"""The paged KV cache on the GPU: the plan (trx_paged_plan, trx_paged_release), the append
(trx_paged_append) and attention over the pages (trx_attn_paged), each against a plain restatement
(tests/paged_ref.py), and a run of them together against the batch decoder's arithmetic."""
import math
import random

import pytest
import torch

import paged_ref as R

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


def i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


# Plan -------------------------------------------------------------------------------------------------

def plan_case(nseq, page, new_hi, ctx_hi, seed, spare=7):
    r = random.Random(seed)
    cached = [r.choice([0, page - 1, page, page + 1, r.randint(0, ctx_hi)]) for _ in range(nseq)]
    new = [r.choice([0, 1, 1, r.randint(1, new_hi)]) for _ in range(nseq)]
    need = [R.pages_of(c + n, page) for c, n in zip(cached, new)]
    n_pages = sum(need) + spare
    perm = list(range(n_pages))
    r.shuffle(perm)
    max_pages = max(1, max(need)) + 2
    tables, at = [], 0
    for c in cached:
        h = R.pages_of(c, page)
        tables.append(perm[at:at + h] + [-1] * (max_pages - h))
        at += h
    return cached, new, tables, perm[at:], n_pages, max_pages


@pytest.mark.parametrize("nseq,page,new_hi,ctx_hi", [(1, 16, 1, 40), (1, 1024, 3000, 5000), (3, 16, 50, 70),
                                                     (32, 16, 1, 900), (33, 64, 300, 2000), (257, 16, 200, 500),
                                                     (1024, 32, 40, 100)])
@pytest.mark.parametrize("inplace", [False, True])
def test_plan_matches_host(ops, ctx, nseq, page, new_hi, ctx_hi, inplace):
    cached, new, tables, free, n_pages, max_pages = plan_case(nseq, page, new_hi, ctx_hi, seed=nseq + page)
    want = R.plan(cached, new, tables, free, len(free), page)
    rows = want[2][-1]
    plan = ops.PagedPlan(nseq, rows + 9, max_pages, page, n_pages)
    plan.tables.copy_(i32(tables))
    dfree = i32(free)
    if inplace:
        plan.lens.copy_(i32(cached))
        plan.n_free.fill_(len(free))
        ops.paged_plan(ctx, plan, plan.lens, i32(new), dfree, plan.n_free)
    else:
        dc, dn, df = i32(cached), i32(new), i32([len(free)])
        for _ in range(2):  # the same call again gives the same plan
            ops.paged_plan(ctx, plan, dc, dn, dfree, df)
        assert dc.tolist() == cached and df.tolist() == [len(free)]
    got = [t.tolist() for t in (plan.tables, plan.lens, plan.cu, plan.slots, plan.pos, plan.last, plan.n_free)]
    assert got[0] == want[0] and got[1] == want[1] and got[2] == want[2]
    assert got[3] == want[3] + [-1] * 9 and got[4] == want[4] + [-1] * 9  # rows behind the last as they were
    assert got[5] == want[5] and got[6] == [want[6]]
    assert dfree.tolist() == free
    assert ctx.errors() == 0


@pytest.mark.parametrize("bad", ["pages", "rows", "negative_new", "negative_cached", "too_long", "n_free"])
def test_plan_that_does_not_fit_does_nothing(ops, ctx, bad):
    from trixium_b200 import _lib
    cached, new, tables, free, n_pages, max_pages = plan_case(5, 16, 60, 90, seed=3)
    new[2] = 40
    cached[1], new[1] = 0, 1
    tables[1] = [-1] * max_pages
    need = sum(R.pages_of(c + n, 16) - R.pages_of(c, 16) for c, n in zip(cached, new) if n)
    rows, n_free = sum(new), len(free)
    if bad == "pages":
        n_free = need - 1
    elif bad == "rows":
        rows -= 1
    elif bad == "negative_new":
        new[3] = -1
    elif bad == "negative_cached":
        cached[3] = -5
    elif bad == "too_long":
        new[1] = max_pages * 16 + 1
        rows += new[1]
    else:
        n_free = n_pages + 1
    plan = ops.PagedPlan(5, rows, max_pages, 16, n_pages)
    plan.tables.copy_(i32(tables))
    plan.cu.fill_(77)
    ops.paged_plan(ctx, plan, i32(cached), i32(new), i32(free), i32([n_free]))
    assert ctx.errors() == (_lib.DEV_PAGES if bad == "pages" else _lib.DEV_RANGE)
    assert plan.cu.tolist() == [0] * 6 and plan.last.tolist() == [0] * 5
    assert plan.lens.tolist() == cached and plan.n_free.tolist() == [n_free]
    assert plan.tables.tolist() == tables and plan.slots.tolist() == [-1] * rows


def test_plan_free_stack_shorter_than_its_height(ops, ctx):
    """n_free beyond the stack's own tensor is refused; nothing behind it is read."""
    from trixium_b200 import _lib
    plan = ops.PagedPlan(1, 40, 4, 16, 6)
    ops.paged_plan(ctx, plan, i32([0]), i32([20]), i32([1, 2]), i32([3]))
    assert ctx.errors() == _lib.DEV_RANGE
    assert plan.cu.tolist() == [0, 0] and plan.tables.tolist() == [[-1] * 4]
    ops.paged_plan(ctx, plan, i32([0]), i32([20]), i32([1, 2]), i32([2]))
    assert ctx.errors() == 0 and plan.tables.tolist() == [[2, 1, -1, -1]]


def test_plan_bad_page_id(ops, ctx):
    from trixium_b200 import _lib
    plan = ops.PagedPlan(2, 40, 4, 16, 6)
    ops.paged_plan(ctx, plan, i32([0, 0]), i32([20, 5]), i32([1, 6, 3]), i32([3]))
    assert ctx.errors() == _lib.DEV_RANGE
    assert plan.slots.tolist()[:25] == [3 * 16 + i for i in range(16)] + [-1] * 4 + [16 + i for i in range(5)]


def test_release_returns_pages_in_order(ops, ctx):
    from trixium_b200 import _lib
    page, n_pages = 16, 12
    plan = ops.PagedPlan(4, 200, 6, page, n_pages)
    free = i32(list(range(n_pages)))
    plan.n_free.fill_(n_pages)
    ops.paged_plan(ctx, plan, plan.lens, i32([17, 0, 33, 64]), free, plan.n_free)
    assert plan.tables.tolist() == [[11, 10] + [-1] * 4, [-1] * 6, [9, 8, 7] + [-1] * 3, [6, 5, 4, 3] + [-1] * 2]
    ops.paged_release(ctx, plan, i32([1, 1, 0, 5]), plan.lens, free, plan.n_free)
    assert free.tolist()[:9] == [0, 1, 2, 11, 10, 6, 5, 4, 3] and plan.n_free.tolist() == [9]
    assert plan.lens.tolist() == [0, 0, 33, 0]
    assert plan.tables.tolist() == [[-1] * 6, [-1] * 6, [9, 8, 7] + [-1] * 3, [-1] * 6]
    assert ctx.errors() == 0
    # More pages than the stack holds, or an entry that is no page: nothing changes.
    plan.n_free.fill_(10)
    ops.paged_release(ctx, plan, i32([0, 0, 1, 0]), plan.lens, free, plan.n_free)
    assert ctx.errors() == _lib.DEV_RANGE and plan.lens.tolist() == [0, 0, 33, 0] and plan.n_free.tolist() == [10]
    plan.n_free.fill_(9)
    plan.tables[2, 1] = n_pages
    ops.paged_release(ctx, plan, i32([0, 0, 1, 0]), plan.lens, free, plan.n_free)
    assert ctx.errors() == _lib.DEV_RANGE and plan.lens.tolist() == [0, 0, 33, 0] and plan.n_free.tolist() == [9]


# Append -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("H,kv,hd,rope,gated", [(4, 2, 64, 64, False), (6, 2, 128, 128, False), (3, 1, 128, 32, True),
                                                (24, 4, 256, 64, True), (2, 2, 256, 256, False), (16, 1, 64, 0, False),
                                                (1, 1, 64, 8, False)])
@pytest.mark.parametrize("cache,qt", [("float16", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16"),
                                      ("bfloat16", "float32")])
def test_append_matches_definition(ops, ctx, H, kv, hd, rope, gated, cache, qt):
    ct, qd = getattr(torch, cache), getattr(torch, qt)
    g = torch.Generator(device="cuda").manual_seed(H + hd)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    new, lens, page = [1, 0, 7, 1, 30], [1, 9, 40, 70001, 30], 16
    rows = sum(new)
    shape = ops.paged_shape(H, kv, hd, rope_dims=rope, gated=gated, eps=1e-6)
    plan = ops.PagedPlan(5, rows + 4, 70016 // page, page, 60)
    plan.cu.copy_(i32([0, 1, 1, 8, 9, 39]))
    pos = [0] + list(range(33, 40)) + [70000] + list(range(30))
    slots = torch.randperm(60 * page, generator=torch.Generator().manual_seed(1))[:rows].tolist()
    plan.pos[:rows] = i32(pos)
    plan.slots[:rows] = i32(slots)
    # Rows of one wide projection buffer: strided inputs.
    qw, kw = H * hd * (2 if gated else 1), kv * hd
    wide = rnd(rows + 4, qw + 2 * kw + 8) * 3
    q, k, v = wide[:, :qw], wide[:, qw:qw + kw], wide[:, qw + kw:qw + 2 * kw]
    qn, kn = 1 + 0.1 * rnd(hd), 1 + 0.1 * rnd(hd)
    freq = (1e6 ** (-2.0 * torch.arange(rope // 2, dtype=torch.float64) / max(rope, 1))).float().cuda()
    kp = rnd(60, page, kv, hd).to(ct)
    vp = rnd(60, page, kv, hd).to(ct)
    k0, v0 = kp.clone(), vp.clone()
    q_out = torch.full((rows + 4, H, hd), 7.0, dtype=qd, device="cuda")
    ops.paged_append(ctx, shape, plan, q, k, v, qn, kn, freq if rope else None, kp, vp, q_out=q_out)
    assert ctx.errors() == 0
    dpos, ds = i32(pos), torch.tensor(slots, device="cuda")
    qr = R.rotate(q[:rows].reshape(rows, H, -1)[..., :hd], dpos, freq, qn, 1e-6)
    kr = R.rotate(k[:rows].reshape(rows, kv, hd), dpos, freq, kn, 1e-6)
    # fp32 work: a norm within 8 roundings (2^-21), the pair's products and sum against the pair's size,
    # cosines within 2 units in the last place; then half a step of the type.
    def close(got, ref, dt, ref_pair):
        h = torch.finfo(dt).eps / 2
        tol = ref.abs() * h + ref_pair * 2.0 ** -20 + (torch.finfo(dt).tiny * torch.finfo(dt).eps if dt != torch.float32 else 0)
        assert bool(((got.double() - ref).abs() <= tol).all())

    def pair(x):
        half = freq.numel()
        m = x.abs()
        if half:
            s = m[..., :half] + m[..., half:2 * half]
            m = torch.cat([s, s, m[..., 2 * half:]], -1)
        return m
    close(q_out[:rows], qr, qd, pair(qr))
    assert bool((q_out[rows:] == 7.0).all())  # rows behind the last as they were
    close(kp.view(-1, kv, hd)[ds], kr, ct, pair(kr))
    assert torch.equal(vp.view(-1, kv, hd)[ds], v[:rows].reshape(rows, kv, hd).to(ct))
    rest = torch.ones(60 * page, dtype=torch.bool, device="cuda")
    rest[ds] = False
    assert torch.equal(kp.view(-1, kv, hd)[rest], k0.view(-1, kv, hd)[rest])
    assert torch.equal(vp.view(-1, kv, hd)[rest], v0.view(-1, kv, hd)[rest])


def test_append_more_rows_than_blocks(ops, ctx):
    """70,000 rows: a block takes several."""
    n, hd = 70000, 64
    g = torch.Generator(device="cuda").manual_seed(9)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")
    plan = ops.PagedPlan(1, n, n // 16, 16, n // 16)
    ops.paged_plan(ctx, plan, i32([0]), i32([n]), torch.arange(n // 16, dtype=torch.int32, device="cuda"), i32([n // 16]))
    q, k, v = rnd(n, 2 * hd), rnd(n, hd), rnd(n, hd)
    qn, kn = 1 + 0.1 * rnd(hd), 1 + 0.1 * rnd(hd)
    freq = (1e4 ** (-torch.arange(hd // 2, dtype=torch.float64) / 32)).float().cuda()
    kp = torch.zeros(n // 16, 16, 1, hd, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    qo = ops.paged_append(ctx, ops.paged_shape(2, 1, hd), plan, q, k, v, qn, kn, freq, kp, vp, q_dtype=torch.float32)
    assert ctx.errors() == 0
    slots = plan.slots.long()
    qr = R.rotate(q.view(n, 2, hd), plan.pos, freq, qn, 1e-6)
    kr = R.rotate(k.view(n, 1, hd), plan.pos, freq, kn, 1e-6)
    size = lambda x: (x.abs()[..., :hd // 2] + x.abs()[..., hd // 2:]).repeat(1, 1, 2)  # of a rotated pair
    # As in test_append_matches_definition.
    assert bool(((qo.double() - qr).abs() <= size(qr) * 2.0 ** -20 + qr.abs() * 2.0 ** -24).all())
    kg = kp.view(n, 1, hd)[slots].double()
    assert bool(((kg - kr).abs() <= size(kr) * 2.0 ** -20 + kr.abs() * 2.0 ** -11 + 2.0 ** -24).all())
    assert torch.equal(vp.view(n, 1, hd)[slots], v.view(n, 1, hd).half())


def test_append_bad_slots_store_nothing(ops, ctx):
    from trixium_b200 import _lib
    shape = ops.paged_shape(2, 1, 64)
    plan = ops.PagedPlan(1, 4, 1, 16, 2)
    plan.cu.copy_(i32([0, 3]))
    plan.pos.copy_(i32([0, 1, 2, 3]))
    plan.slots.copy_(i32([-1, 32, 5, 6]))
    x = torch.ones(4, 128, device="cuda")
    w, f = torch.ones(64, device="cuda"), torch.ones(32, device="cuda")
    kp = torch.zeros(2, 16, 1, 64, dtype=torch.float16, device="cuda")
    vp = torch.zeros_like(kp)
    ops.paged_append(ctx, shape, plan, x, x[:, :64], x[:, 64:], w, w, f, kp, vp)
    assert ctx.errors() == _lib.DEV_RANGE
    assert vp.view(32, 64)[:, 0].nonzero().flatten().tolist() == [5]


# Attention --------------------------------------------------------------------------------------------

SHAPES = [(4, 4, 64), (8, 2, 64), (16, 1, 64), (4, 2, 128), (8, 2, 128), (3, 1, 128), (6, 1, 256), (2, 2, 256)]
TYPES = [("float16", "float16"), ("float16", "float32"), ("bfloat16", "bfloat16")]
LENGTHS = [
    ([1], [1]),                                       # the first token of all
    ([1, 1, 1], [1, 64, 65]),
    ([1] * 5, [16, 17, 700, 1, 129]),
    ([3, 0, 1, 5], [3, 77, 300, 200]),                # an idle sequence between
    ([130], [130]),
    ([1, 200, 1, 33], [500, 263, 128, 33]),
]


def run_case(ops, ctx, H, kv, hd, ct, qt, new, lens, page, window=0, sinks=0, gated=False, seed=0, max_new=None):
    C = R.Cache(ops, lens, new, kv, hd, page, ct, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    q = torch.randn(C.rows, H, hd, generator=g, device="cuda").to(qt)
    gate = torch.randn(C.rows, H * 2 * hd, generator=g, device="cuda") if gated else None
    shape = ops.paged_shape(H, kv, hd, rope_dims=0, gated=gated, window=window, sinks=sinks)
    out = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, gate=gate, max_new=max_new)
    assert ctx.errors() == 0
    C.check(q, out, gate, window, sinks)
    return C, q, out, shape


@pytest.mark.parametrize("new,lens", LENGTHS)
@pytest.mark.parametrize("H,kv,hd", SHAPES)
@pytest.mark.parametrize("cache,qt", TYPES)
def test_attention_matches_definition(ops, ctx, H, kv, hd, cache, qt, new, lens):
    run_case(ops, ctx, H, kv, hd, getattr(torch, cache), getattr(torch, qt), new, lens, 16, seed=hd + len(new),
             max_new=max(new))


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("new,lens", [([1, 1], [400, 1025]), ([150, 70], [260, 1300])])
def test_attention_page_sizes(ops, ctx, page, new, lens):
    run_case(ops, ctx, 8, 2, 128, torch.float16, torch.float16, new, lens, page, seed=page)


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (16, 4), (64, 64), (100, 130), (257, 3), (1000, 4), (5000, 9)])
@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 650, 1031]), ([300, 1, 2], [700, 400, 2])])
def test_attention_window_and_sinks(ops, ctx, window, sinks, cache, qt, new, lens):
    run_case(ops, ctx, 4, 2, 128, getattr(torch, cache), getattr(torch, qt), new, lens, 32, window, sinks, seed=window)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 1], [90, 700]), ([140, 1], [300, 90])])
def test_attention_gate(ops, ctx, hd, new, lens):
    run_case(ops, ctx, 12, 4, hd, torch.float16, torch.float32, new, lens, 16, gated=True, seed=hd)


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("H,kv,hd", [(2, 2, 256), (12, 4, 256), (6, 1, 256), (5, 1, 256), (12, 4, 128), (8, 2, 64)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 90, 2000]), ([700, 1, 45], [3000, 900, 45]),
                                      ([130, 0, 3], [130, 9, 1000]), ([40] * 9, [40 + 300 * b for b in range(9)])])
def test_attention_gate_of_every_type(ops, ctx, H, kv, hd, cache, qt, new, lens):
    """Gates from a slice of wider rows: whole and cut items, partial tiles, several pieces of a block, groups of
    heads that do not divide a tile; 16-bit heads of 256 take them through the ring in shared memory."""
    dt = getattr(torch, qt)
    C = R.Cache(ops, lens, new, kv, hd, 16, getattr(torch, cache), hd + H)
    g = torch.Generator(device="cuda").manual_seed(H)
    q = torch.randn(C.rows, H, hd, generator=g, device="cuda").to(dt)
    wide = torch.randn(C.rows, 2 * H * hd + 12, generator=g, device="cuda") * 3
    shape = ops.paged_shape(H, kv, hd, rope_dims=0, gated=True)
    call = lambda: ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, gate=wide[:, 8:-4], max_new=max(new))
    out = call()
    assert ctx.errors() == 0
    C.check(q, out, wide[:, 8:-4])
    assert torch.equal(out, call())
    wide[:, 8:-4] = 200.0  # sigmoid 1: the bits of the call without a gate
    plain = ops.attn_paged(ctx, ops.paged_shape(H, kv, hd, rope_dims=0), C.plan, q, C.kp, C.vp, max_new=max(new))
    assert torch.equal(call(), plain)
    wide[:, 8:-4] = -200.0  # sigmoid 0
    assert bool((call() == 0).all())


@pytest.mark.parametrize("new,lens", [([1], [40000]), ([1] * 40, [37 * i + 1 for i in range(40)]), ([5, 900], [9000, 2500])])
def test_attention_long_and_many(ops, ctx, new, lens):
    """One sequence cut among all blocks, many short ones, and long prompts."""
    C, q, out, shape = run_case(ops, ctx, 8, 2, 128, torch.float16, torch.float16, new, lens, 16, seed=7)
    again = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, max_new=max(new))
    third = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, max_new=max(new))
    assert torch.equal(again, third)  # the same bits again: nothing depends on the order of arrival


def test_attention_rows_outside_stay(ops, ctx):
    """Rows behind the last sequence, and of a sequence that does not fit, are left as they were."""
    from trixium_b200 import _lib
    C = R.Cache(ops, [50, 60, 70], [2, 20, 1], 2, 64, 16, torch.float16, 3, max_rows=30)
    q = torch.randn(30, 4, 64, device="cuda").half()
    shape = ops.paged_shape(4, 2, 64, rope_dims=0)
    out = torch.full_like(q, 9.0)
    ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out)
    assert ctx.errors() == 0
    C.check(q, out)
    assert bool((out[23:] == 9.0).all())
    out.fill_(9.0)
    ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out, max_new=4)  # sequence 1 brings 20
    assert ctx.errors() == _lib.DEV_RANGE
    assert bool((out[2:22] == 9.0).all())
    C.new[1] = 0
    C.check(q, out)
    C.plan.lens[0] = 1  # fewer positions than new rows
    out.fill_(9.0)
    ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out)
    assert ctx.errors() == _lib.DEV_RANGE
    assert bool((out[:2] == 9.0).all())
    # More rows in cu than the tensors have.
    C.plan.lens[0] = 50
    out.fill_(9.0)
    ops.attn_paged(ctx, shape, C.plan, q[:22], C.kp, C.vp, out=out)
    assert ctx.errors() == _lib.DEV_RANGE
    assert bool((out[22:] == 9.0).all())
    # No rows at all.
    C.plan.cu.zero_()
    out.fill_(9.0)
    ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out)
    assert ctx.errors() == 0 and bool((out == 9.0).all())


@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("new", [1, 90])
def test_attention_bad_page_reads_zeros(ops, ctx, bad, new):
    from trixium_b200 import _lib
    C = R.Cache(ops, [100], [new], 1, 128, 16, torch.float16, 5)
    q = torch.randn(new, 4, 128, device="cuda")
    C.plan.tables[0, 2] = bad
    out = ops.attn_paged(ctx, ops.paged_shape(4, 1, 128, rope_dims=0), C.plan, q, C.kp, C.vp)
    assert ctx.errors() == _lib.DEV_RANGE
    C.k[0][32:48] = 0
    C.v[0][32:48] = 0
    C.check(q, out)


@pytest.mark.parametrize("new", [1, 70])
def test_attention_on_another_stream_and_in_a_graph(ops, ctx, new):
    C = R.Cache(ops, [300, 40], [new, 1], 2, 128, 16, torch.float16, 6)
    q = torch.randn(C.rows, 8, 128, device="cuda").half()
    shape = ops.paged_shape(8, 2, 128, rope_dims=0)
    out = torch.zeros_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out)
    s.synchronize()
    C.check(q, out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, out=out)
    # New lengths, offsets and queries at the replay: sequence 1 brings its row and two more.
    for step in range(3):
        q.copy_(torch.randn_like(q))
        out.zero_()
        if step == 2:
            C.new, C.cu = [new - 1, 2], [0, new - 1, new + 1]
            C.plan.cu.copy_(i32(C.cu))
        graph.replay()
        torch.cuda.synchronize()
        C.check(q, out)
    assert ctx.errors() == 0


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("window,sinks", [(2 ** 30, 2 ** 30), (1, 2 ** 30), (2 ** 30, 0)])
def test_attention_largest_window_and_sinks(ops, ctx, cache, qt, window, sinks):
    run_case(ops, ctx, 4, 2, 64, getattr(torch, cache), getattr(torch, qt), [150, 1, 0], [400, 129, 5], 16, window, sinks)


@pytest.mark.parametrize("new", [1, 2, 40])
def test_attention_many_sequences(ops, ctx, new):
    """The most sequences a plan takes, every third one idle."""
    n = [0 if b % 3 == 2 else new for b in range(1024)]
    run_case(ops, ctx, 4, 1, 64, torch.float16, torch.float16, n, [c + b % 50 for b, c in enumerate(n)], 16, max_new=new)


@pytest.mark.parametrize("qt", ["float16", "float32"])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_of_two_contexts_at_once(ops, ctx, new, qt):
    """Two contexts on two streams, launches in turn: each the bits it gives alone."""
    other = ops.Context(0)
    made = []
    for c, seed in ((ctx, 1), (other, 2)):
        C = R.Cache(ops, [3000, 700, 64], [new, 1, 1], 2, 128, 16, torch.float16, seed)
        q = torch.randn(C.rows, 8, 128, device="cuda").to(getattr(torch, qt))
        shape = ops.paged_shape(8, 2, 128, rope_dims=0)
        made.append((c, C, shape, q, ops.attn_paged(c, shape, C.plan, q, C.kp, C.vp), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for c, C, shape, q, alone, s in made:
            with torch.cuda.stream(s):
                outs.append((ops.attn_paged(c, shape, C.plan, q, C.kp, C.vp), alone))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in outs)
    assert ctx.errors() == 0 and other.errors() == 0
    other.close()


@pytest.mark.parametrize("new", [1, 80])
def test_pages_behind_4_billion_bytes(ops, ctx, new):
    """A pool of more than 2^31 elements, the sequence's pages at both of its ends."""
    kv, hd, page, L = 8, 256, 16, 100
    n_pages = 2 ** 31 // (kv * hd * page) + 40
    kp = torch.empty(n_pages, page, kv, hd, dtype=torch.bfloat16, device="cuda")
    vp = torch.empty_like(kp)
    g = torch.Generator(device="cuda").manual_seed(0)
    k, v = [torch.randn(L, kv, hd, generator=g, device="cuda").bfloat16() for _ in range(2)]
    ids = [n_pages - 1, 0, n_pages - 2, n_pages - 30, 1, n_pages - 3, n_pages - 31]
    plan = ops.PagedPlan(1, new, len(ids), page, n_pages)
    free = i32(ids[::-1])
    old = L - new
    have = R.pages_of(old, page)
    plan.tables[0, :have] = i32(ids[:have])
    for p in range(old):
        kp[ids[p // page], p % page], vp[ids[p // page], p % page] = k[p], v[p]
    ops.paged_plan(ctx, plan, i32([old]), i32([new]), free, i32([len(ids) - have]))
    shape = ops.paged_shape(kv * 2, kv, hd, rope_dims=0, eps=0.0)
    one = torch.ones(hd, device="cuda")
    q = torch.randn(new, kv * 2 * hd, generator=g, device="cuda")
    raw = torch.randn(new, kv * hd, generator=g, device="cuda")
    qr = ops.paged_append(ctx, shape, plan, q, raw, v[old:].float().view(new, -1), one, one, None, kp, vp)
    assert ctx.errors() == 0
    for p in range(old, L):
        assert torch.equal(vp[ids[p // page], p % page], v[p])
        k[p] = kp[ids[p // page], p % page]
    ref = R.rotate(raw.view(new, kv, hd), plan.pos, one[:0], one, 0.0)
    assert bool(((k[old:].double() - ref).abs() <= ref.abs() * (2.0 ** -8 + 2.0 ** -20)).all())
    out = ops.attn_paged(ctx, shape, plan, qr, kp, vp)
    assert ctx.errors() == 0
    C = R.Cache.__new__(R.Cache)
    C.k, C.v, C.cu, C.lens, C.new = [k], [v], [0, new], [L], [new]
    C.check(qr, out)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_small_weights_beside_a_large_one(ops, ctx, hd, new):
    """fp32 queries: the largest weight meets zeros of V, so that the output is what the small weights (about
    1e-6 of it) give; they keep their precision."""
    L = 200
    C = R.Cache(ops, [L], [new], 1, hd, 16, torch.float16, 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randn(new, 4, hd, generator=g, device="cuda") * 3
    # One key along the mean query: its score is some 14 above the others'.
    k = torch.randn(L, 1, hd, generator=g, device="cuda") * 0.3
    base = torch.randn(hd, generator=g, device="cuda")
    q += base * 4
    k[70, 0] = base * (14.0 * hd ** 0.5 / (4 * float(base @ base)))
    k -= (k @ base)[..., None] / (base @ base) * base * (torch.arange(L, device="cuda")[:, None, None] != 70)
    k = k.half()
    v = torch.randn(L, 1, hd, generator=g, device="cuda").half()
    v[70] = 0
    for j in range(0, L, 16):
        page = int(C.plan.tables[0, j // 16])
        n = min(16, L - j)
        C.kp[page, :n], C.vp[page, :n] = k[j:j + n], v[j:j + n]
    C.k, C.v = [k], [v]
    out = ops.attn_paged(ctx, ops.paged_shape(4, 1, hd, rope_dims=0), C.plan, q, C.kp, C.vp, max_new=max(new, 1))
    assert ctx.errors() == 0
    C.check(q, out)


@pytest.mark.parametrize("cache,qt", TYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [1, 3000, 70]), ([3, 90, 1], [3, 2500, 70])])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_attention_undefined_queries_stay_undefined(ops, ctx, cache, qt, hd, new, lens, value):
    """A query that is not finite gives NaN, as the definition does (whole and cut items, one visible position
    and many), and every other row and head the bits it gives without it."""
    C = R.Cache(ops, lens, new, 2, hd, 16, getattr(torch, cache), 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(C.rows, 4, hd, generator=g, device="cuda").to(getattr(torch, qt))
    shape = ops.paged_shape(4, 2, hd, rope_dims=0)
    clean = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, max_new=max(new))
    bad = torch.zeros(C.rows, 4, dtype=torch.bool, device="cuda")
    for r, h in [(0, 0), (C.rows // 2, 3), (C.rows - 1, 1)]:
        bad[r, h] = True
        q[r, h, 5] = value
        b = next(b for b in range(3) if r < C.cu[b + 1])
        i, first = r - C.cu[b], lens[b] - new[b]
        ref = R.attention(q[r:r + 1], C.k[b][:first + i + 1], C.v[b][:first + i + 1], first + i)[0]
        assert bool(torch.isnan(ref[0, h]).all())
    out = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, max_new=max(new))
    assert ctx.errors() == 0
    assert bool(torch.isnan(out[bad]).all())
    assert torch.equal(out[~bad], clean[~bad])


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("field,value", [("lens", -2 ** 31), ("lens", -1), ("lens", 0), ("lens", 2 ** 31 - 1),
                                         ("cu", -2 ** 31), ("cu", 2 ** 31 - 1)])
def test_attention_lengths_and_offsets_far_out_of_range(ops, ctx, field, value, new):
    """The ends of 32 bits where a sequence's length or offset should be: its rows stay as they were (an offset's
    neighbour's too), the others are right."""
    from trixium_b200 import _lib
    C = R.Cache(ops, [300, 200, 150], [new, new, new], 2, 64, 16, torch.float16, 3)
    q = torch.randn(C.rows, 4, 64, device="cuda").half()
    getattr(C.plan, field)[1] = value
    out = torch.full_like(q, 9.0)
    ops.attn_paged(ctx, ops.paged_shape(4, 2, 64, rope_dims=0), C.plan, q, C.kp, C.vp, out=out, max_new=new)
    assert ctx.errors() == _lib.DEV_RANGE
    for b in (1,) if field == "lens" else (0, 1):
        assert bool((out[C.cu[b]:C.cu[b + 1]] == 9.0).all())
        C.new[b] = 0
    C.check(q, out)


@pytest.mark.parametrize("cache,qt,size", [(*t, s) for t in TYPES for s in (0.5, 4.0, 32.0, 256.0, 4096.0)] +
                         [("bfloat16", "bfloat16", 2.0 ** 40)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 3)])
def test_attention_large_scores(ops, ctx, cache, qt, size, hd, new, window, sinks):
    """Scores up to 2^30 (bf16: 2^58), far beyond what their rounding leaves of a weight's exponent: every next
    key scores higher by more than that rounding, so the softmax is the last visible key's alone (the keys of the
    bf16 case come in fours of equal keys with equal values) and the output its value."""
    L, dt = 400, getattr(torch, cache)
    C = R.Cache(ops, [L], [new], 1, hd, 16, dt, 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    sign = (torch.rand(hd, generator=g, device="cuda") < 0.5).float() * 2 - 1
    at = torch.arange(L, device="cuda")
    k = ((4096 + (8 * at if cache == "float16" else 32 * (at // 4)))[:, None, None].float() * sign).to(dt)  # exact
    v = torch.randn(L, 1, hd, generator=g, device="cuda").to(dt)
    if cache != "float16":
        v = v[at // 4 * 4]
    put_pages(C, k, v)
    # Scores of one row differ by at least 8 * size * hd (32 for bf16) / sqrt(hd) from key to key: 32 for the smallest,
    # a weight of 2^-46.  Rounded to 32 bits a score is off by 16 * 2^-23 of at most 2 * 7300 * size * sqrt(hd), less
    # than 1 / 250 of that difference.
    q = ((1 + torch.rand(new, 4, 1, generator=g, device="cuda")) * size * sign).to(getattr(torch, qt))
    shape = ops.paged_shape(4, 1, hd, rope_dims=0, window=window, sinks=sinks)
    out = ops.attn_paged(ctx, shape, C.plan, q, C.kp, C.vp, max_new=new)
    assert ctx.errors() == 0
    want = v[L - new:].expand(new, 4, hd).double()
    # The weight and the output are rounded to the type (fp32 queries: the weight to 2^-22), sums and quotient to 2^-20.
    h = torch.finfo(q.dtype).eps / 2
    tol = want.abs() * (2 * h + h * h + 2.0 ** -20) + 2.0 ** -40 * float(v.abs().max()) + \
        (torch.finfo(dt).tiny * torch.finfo(dt).eps if q.dtype == dt else 0)
    assert bool(((out.double() - want).abs() <= tol).all())


def put_pages(C, k, v):
    """The pools' positions of a cache of one sequence."""
    for j in range(0, len(k), 16):
        page, n = int(C.plan.tables[0, j // 16]), min(16, len(k) - j)
        C.kp[page, :n], C.vp[page, :n] = k[j:j + n], v[j:j + n]


@pytest.mark.parametrize("cache,qt", [("float16", "float16"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 60])
def test_attention_small_weights_of_16_bit_queries(ops, ctx, cache, qt, hd, new):
    """In every sixteen positions one of a large weight whose value is 0: the output is what the small weights
    (about 2^-23 of the large ones) give.  A weight is kept to half a step of the type, in fp16 or 2^-32 of the
    row's largest."""
    L, dt = 200, getattr(torch, cache)
    C = R.Cache(ops, [L], [new], 1, hd, 16, dt, 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(hd, generator=g, device="cuda")
    base /= base.norm()
    q = (base * 8 + torch.randn(new, 4, hd, generator=g, device="cuda") * 0.3).to(dt)
    k = torch.randn(L, 1, hd, generator=g, device="cuda") * 0.3
    k -= (k @ base)[..., None] * base
    k[6::16, 0] = base * (16 * hd ** 0.5 / 8)  # a score of some 16
    k = k.to(dt)
    v = (torch.randn(L, 1, hd, generator=g, device="cuda") * 512).to(dt)
    v[6::16] = 0
    put_pages(C, k, v)
    out = ops.attn_paged(ctx, ops.paged_shape(4, 1, hd, rope_dims=0), C.plan, q, C.kp, C.vp, max_new=new)
    assert ctx.errors() == 0
    ref, mag, smax = R.attention(q, k, v, L - new)
    # As in Cache.check; in fp16 besides 2^-32 of the row's largest weight for every position that it sees.
    h = torch.finfo(dt).eps / 2
    ds = smax * (17 * 2.0 ** -23 + 2.0 ** -22)
    tol = h * ref.abs() + mag * (h + 2 * ds + 2.0 ** -19 + L * 2.0 ** -26) + torch.finfo(dt).tiny * torch.finfo(dt).eps
    if dt == torch.float16:
        seen = R.visible(L - new, new, L, 0, 0, "cuda")[:, None]
        s = (q.double() @ k[:, 0].double().T / math.sqrt(hd)).masked_fill(~seen, -math.inf)
        tol = tol + 2.0 ** -32 * torch.softmax(s, -1).amax(-1, keepdim=True) * (seen.double() @ v[:, 0].double().abs())
    assert float(((out.double() - ref).abs() / tol).max()) <= 1.0


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 150])
def test_attention_smallest_weights_of_fp32_queries(ops, ctx, hd, new):
    """In every sixteen positions one of a large weight whose value is 0: the output is what the small weights give,
    2^-24 to 2^-34 of the large ones and equal, so that their errors add up: each is within the larger of 2^-22 of
    itself and 2^-39 of the row's largest."""
    L = 400
    C = R.Cache(ops, [L], [new], 1, hd, 16, torch.float16, 8)
    g = torch.Generator(device="cuda").manual_seed(3)
    base = torch.randn(hd, generator=g, device="cuda").half()
    k = (base.float() / 8).half().expand(L, 1, hd).clone()
    k[::16, 0] = base
    v = torch.full((L, 1, hd), 1024.0, dtype=torch.float16, device="cuda")
    v[::16] = 0
    put_pages(C, k, v)
    seen = torch.arange(L - new, L, device="cuda").double()[:, None, None] + 1
    large = torch.ceil(seen / 16)
    for rep in range(1 if new > 1 else 60):
        d = (24 + 10 * torch.rand(new, 4, 1, generator=g, device="cuda")) * 8 / 7  # 7/8 of it: log2 of large over small
        q = base.float() * (d * math.log(2) * math.sqrt(hd) / float(base.float() @ base.float()))
        out = ops.attn_paged(ctx, ops.paged_shape(4, 1, hd, rope_dims=0), C.plan, q, C.kp, C.vp, max_new=new)
        assert ctx.errors() == 0
        ref, mag, smax = R.attention(q, k, v, L - new)
        ds = smax * (17 * 2.0 ** -23 + 2.0 ** -22)
        tol = mag * (2.0 ** -22 + 2 * ds + 2.0 ** -19 + L * 2.0 ** -26) + 2.0 ** -39 / large * (seen - large) * 1024
        worst = float(((out.double() - ref).abs() / tol).max())
        assert worst <= 1.0, worst


# All together -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("ct,qt", [("float16", "float32"), ("bfloat16", "bfloat16")])
def test_steps_of_a_ragged_batch(ops, ctx, ct, qt):
    """Plan, append and attention over steps that mix prompts, chunks and decode, with a sequence that
    ends and another that takes its pages: every step against the 64-bit operators on the whole history."""
    ct, qt = getattr(torch, ct), getattr(torch, qt)
    H, kv, hd, page, n_pages = 6, 2, 128, 16, 30
    g = torch.Generator(device="cuda").manual_seed(0)
    shape = ops.paged_shape(H, kv, hd, rope_dims=64)
    plan = ops.PagedPlan(3, 96, 20, page, n_pages)
    free = i32(torch.randperm(n_pages, generator=torch.Generator().manual_seed(2)).tolist())
    plan.n_free.fill_(n_pages)
    kp = torch.full((n_pages, page, kv, hd), float("nan"), dtype=ct, device="cuda")
    vp = kp.clone()
    qn, kn = torch.ones(hd, device="cuda"), torch.ones(hd, device="cuda")
    freq = (1e4 ** (-2.0 * torch.arange(32, dtype=torch.float64) / 64)).float().cuda()
    hist = [[torch.zeros(0, kv, hd, dtype=ct, device="cuda")] * 2 for _ in range(3)]
    steps = [([40, 0, 7], None), ([33, 1, 1], None), ([1, 50, 1], None), ([1, 1, 1], 0), ([70, 1, 0], None), ([1, 1, 1], None)]
    lens = [0, 0, 0]
    for new, done in steps:
        rows = sum(new)
        qkv = torch.randn(96, (H + 2 * kv) * hd, generator=g, device="cuda")
        q, k, v = qkv[:, :H * hd], qkv[:, H * hd:(H + kv) * hd], qkv[:, (H + kv) * hd:]
        ops.paged_plan(ctx, plan, plan.lens, i32(new), free, plan.n_free)
        qr = ops.paged_append(ctx, shape, plan, q, k, v, qn, kn, freq, kp, vp, q_dtype=qt)
        out = ops.attn_paged(ctx, shape, plan, qr, kp, vp, max_new=max(new))
        assert ctx.errors() == 0
        C = R.Cache.__new__(R.Cache)
        C.new, C.cu = new, plan.cu.tolist()
        pos = plan.pos[:rows]
        kr = R.rotate(k[:rows].reshape(rows, kv, hd), pos, freq, kn, 1e-6)
        for b in range(3):
            lens[b] += new[b]
            at = plan.slots[C.cu[b]:C.cu[b + 1]].long()
            kb, vb = kp.view(-1, kv, hd)[at], vp.view(-1, kv, hd)[at]
            ref = kr[C.cu[b]:C.cu[b + 1]]
            assert bool(((kb.double() - ref).abs() <= ref.abs() * torch.finfo(ct).eps / 2 + 1e-5).all())
            hist[b] = [torch.cat([hist[b][0], kb]), torch.cat([hist[b][1], vb])]
        C.lens, C.k, C.v = list(lens), [h[0] for h in hist], [h[1] for h in hist]
        assert plan.lens.tolist() == lens
        C.check(qr, out)
        if done is not None:
            ops.paged_release(ctx, plan, i32([int(b == done) for b in range(3)]), plan.lens, free, plan.n_free)
            lens[done] = 0
            hist[done] = [torch.zeros(0, kv, hd, dtype=ct, device="cuda")] * 2
            assert ctx.errors() == 0
    used = sum(R.pages_of(n, page) for n in lens)
    assert plan.n_free.tolist() == [n_pages - used]
