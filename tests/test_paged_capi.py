"""Refusals of the paged-cache and sampling entry points: every one is a host check before any CUDA
call, so it is tested without a GPU (no pointer here is ever dereferenced)."""
import ctypes

import pytest
import torch

from trixium_b200 import _lib

ARG, UNSUPPORTED = -1, -6
P = ctypes.c_void_p(0x10000)   # aligned, never touched
ODD = ctypes.c_void_p(0x10008)
N = None


def pages(**kw):
    d = dict(nseq=4, max_rows=64, page=16, max_pages=8, n_pages=100, tables=0x10000, lens=0x10000, cu=0x10000,
             slots=0x10000, pos=0x10000, last=0x10000, n_free=0x10000)
    d.update(kw)
    return ctypes.byref(_lib.Pages(**d))


def shape(**kw):
    d = dict(n_head=8, n_kv=2, head_dim=128, rope_dims=128, gated=0, eps=1e-6, window=0, sinks=0)
    d.update(kw)
    return ctypes.byref(_lib.PagedShape(**d))


BAD_PAGES = [(dict(nseq=0), ARG), (dict(max_rows=0), ARG), (dict(max_pages=0), ARG), (dict(n_pages=0), ARG),
             (dict(page=8), UNSUPPORTED), (dict(page=24), UNSUPPORTED), (dict(page=2048), UNSUPPORTED),
             (dict(nseq=1025), UNSUPPORTED), (dict(max_rows=(1 << 22) + 1), UNSUPPORTED),
             (dict(max_pages=(1 << 20) + 1), UNSUPPORTED), (dict(page=1024, n_pages=1 << 21), UNSUPPORTED),
             (dict(page=1024, max_pages=1 << 20, n_pages=1 << 22), UNSUPPORTED), (dict(tables=None), ARG)]
BAD_SHAPES = [(dict(n_head=0), ARG), (dict(n_kv=0), ARG), (dict(n_head=7), ARG), (dict(head_dim=96), UNSUPPORTED),
              (dict(head_dim=512, rope_dims=0), UNSUPPORTED), (dict(rope_dims=136), ARG), (dict(rope_dims=12), UNSUPPORTED),
              (dict(n_head=34), UNSUPPORTED), (dict(eps=-1.0), ARG), (dict(eps=float("nan")), ARG),
              (dict(window=(1 << 30) + 1), UNSUPPORTED), (dict(sinks=(1 << 30) + 1), UNSUPPORTED)]


def call_plan(L, pg, ctx=P, args=(P, P, P, P)):
    return L.trx_paged_plan(ctx, pg, *args[:3], 10, args[3], N)


def call_append(L, sh, pg, q=P, qld=1024, k=P, kld=256, v=P, vld=256, qn=P, kn=P, f=P, kp=P, vp=P, ct=1, qo=P, qt=1):
    return L.trx_paged_append(P, sh, pg, q, qld, k, kld, v, vld, qn, kn, f, kp, vp, ct, qo, qt, N)


def call_attn(L, sh, pg, q=P, qt=1, gate=N, gld=0, kp=P, vp=P, ct=1, mx=4, out=P):
    return L.trx_attn_paged(P, sh, pg, q, qt, gate, gld, kp, vp, ct, mx, out, N)


@pytest.mark.parametrize("kw,status", BAD_PAGES)
def test_bad_pages_are_refused(kw, status):
    L = _lib.lib()
    assert call_plan(L, pages(**kw)) == status
    assert L.trx_paged_release(P, pages(**kw), P, P, P, P, N) == status
    assert call_append(L, shape(), pages(**kw)) == status
    assert call_attn(L, shape(), pages(**kw)) == status


@pytest.mark.parametrize("kw,status", BAD_SHAPES)
def test_bad_shapes_are_refused(kw, status):
    L = _lib.lib()
    assert call_append(L, shape(**kw), pages()) == status
    assert call_attn(L, shape(**kw), pages()) == status


def test_null_and_misaligned_pointers_are_refused():
    L = _lib.lib()
    assert call_plan(L, pages(), ctx=N) == ARG
    for i in range(4):
        args = [P] * 4
        args[i] = N
        assert call_plan(L, pages(), args=args) == ARG
        assert L.trx_paged_release(P, pages(), *args, N) == ARG
    for f in ("lens", "cu", "slots", "pos", "last", "n_free"):
        assert call_plan(L, pages(**{f: None})) == ARG
    for f in ("q", "k", "v", "qn", "kn", "kp", "vp", "qo"):
        assert call_append(L, shape(), pages(), **{f: N}) == ARG
        assert call_append(L, shape(), pages(), **{f: ODD}) == ARG
    assert call_append(L, shape(), pages(), f=N) == ARG
    for f in ("q", "kp", "vp", "out"):
        assert call_attn(L, shape(), pages(), **{f: N}) == ARG
        assert call_attn(L, shape(), pages(), **{f: ODD}) == ARG
    for f in ("cu", "lens"):
        assert call_attn(L, shape(), pages(**{f: None})) == ARG
    assert L.trx_paged_plan(P, None, P, P, P, 10, P, N) == ARG


def test_strides_and_types_are_refused():
    L = _lib.lib()
    assert call_append(L, shape(), pages(), qld=1023) == ARG      # not a multiple of 4
    assert call_append(L, shape(), pages(), qld=1020) == ARG      # shorter than a row
    assert call_append(L, shape(gated=1), pages(), qld=1024) == ARG
    assert call_append(L, shape(), pages(), kld=252) == ARG
    assert call_append(L, shape(), pages(), vld=258) == ARG
    assert call_append(L, shape(), pages(), ct=0) == ARG
    assert call_append(L, shape(), pages(), ct=1, qt=2) == ARG
    assert call_append(L, shape(), pages(), ct=3, qt=3) == ARG
    assert call_attn(L, shape(), pages(), ct=2, qt=1) == ARG
    assert call_attn(L, shape(), pages(), ct=2, qt=0) == UNSUPPORTED   # fp32 queries over a bf16 cache
    assert call_attn(L, shape(), pages(), mx=0) == ARG
    assert call_attn(L, shape(gated=1), pages()) == ARG                # gated without a gate
    assert call_attn(L, shape(), pages(), gate=P, gld=2048) == ARG     # a gate without gated
    assert call_attn(L, shape(gated=1), pages(), gate=P, gld=2044) == ARG
    assert call_attn(L, shape(gated=1), pages(), gate=ODD, gld=2048) == ARG


def test_sample_refusals():
    L = _lib.lib()

    def call(x=P, t=0, ld=100, V=100, n=3, u=P, rest=(P, P, P, P), tok=P, ctx=P):
        return L.trx_sample_rows(ctx, x, t, ld, V, n, u, *rest, tok, N)
    assert call(ctx=N) == ARG and call(x=N) == ARG and call(u=N) == ARG and call(tok=N) == ARG
    for i in range(4):
        rest = [P] * 4
        rest[i] = N
        assert call(rest=rest) == ARG
    assert call(t=3) == ARG and call(t=-1) == ARG
    assert call(V=0) == ARG and call(n=0) == ARG and call(ld=99) == ARG
    assert call(V=(1 << 22) + 1, ld=1 << 23) == UNSUPPORTED
    assert call(n=(1 << 20) + 1) == UNSUPPORTED


def test_python_checks_name_the_argument():
    from trixium_b200 import ops
    dev = torch.device("cpu")
    with pytest.raises(ValueError, match="cached"):
        ops._buf(torch.zeros(3, dtype=torch.int64), torch.int32, 3, "cached", dev)
    with pytest.raises(ValueError, match="cached"):
        ops._buf(torch.zeros(3, dtype=torch.int32), torch.int32, 4, "cached", dev)
    with pytest.raises(ValueError, match="cached"):
        ops._buf(torch.zeros(8, dtype=torch.int32)[::2], torch.int32, 4, "cached", dev)
    assert ops._mat(torch.zeros(4, 10)[:, 2:8], torch.float32, 6, "q", dev)[1] == 10
    with pytest.raises(ValueError, match="q"):
        ops._mat(torch.zeros(10, 4).t(), torch.float32, 10, "q", dev)
    with pytest.raises(ValueError, match="q"):
        ops._mat(torch.zeros(1, 6).expand(4, 6), torch.float32, 6, "q", dev)
    with pytest.raises(ValueError):
        ops.PagedPlan(2, 8, 2, 24, 10, device="cpu")


def test_plans_keep_their_buffers_and_device(monkeypatch):
    """A plan's buffers cannot be replaced (the library holds their addresses), and a plan on another device
    than the context's is refused before anything is launched."""
    from trixium_b200 import ops
    plan = ops.PagedPlan(2, 8, 2, 16, 10, device="cpu")
    for name in ("lens", "tables", "max_rows", "other"):
        with pytest.raises(AttributeError, match=name):
            setattr(plan, name, torch.zeros(2, dtype=torch.int32))
    plan.lens.fill_(3)

    class Ctx:
        device, h = torch.device("cuda", 0), None
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    monkeypatch.setattr(ops, "_raw_stream", lambda dev: 0)
    z = torch.zeros(10, dtype=torch.int32)
    with pytest.raises(ValueError, match="plan on cpu"):
        ops.paged_plan(Ctx, plan, z, z, z, z)
    with pytest.raises(ValueError, match="plan on cpu"):
        ops.paged_release(Ctx, plan, z, z, z, z)
    x, w = torch.zeros(8, 256), torch.zeros(64)
    pool = torch.zeros(10, 16, 2, 64, dtype=torch.float16)
    shape = ops.paged_shape(4, 2, 64)
    with pytest.raises(ValueError, match="plan on cpu"):
        ops.paged_append(Ctx, shape, plan, x, x[:, :128], x[:, 128:], w, w, w, pool, pool)
    with pytest.raises(ValueError, match="plan on cpu"):
        ops.attn_paged(Ctx, shape, plan, x.view(8, 4, 64), pool, pool)
    with pytest.raises(ValueError, match="plan on cuda:1"):
        ops._stream_of(Ctx, torch.device("cuda", 1))
    assert ops._stream_of(Ctx, torch.device("cuda", 0)) == 0
    with pytest.raises(ValueError):
        ops.PagedPlan(0, 8, 2, 16, 10, device="cpu")
    p = ops.PagedPlan(2, 8, 2, 16, 10, device="cpu")
    s = ops.paged_shape(8, 2, 128)
    with pytest.raises(ValueError, match="kpages"):
        ops._pools(s, p, torch.zeros(10, 16, 2, 128), torch.zeros(10, 16, 2, 128))
    with pytest.raises(ValueError, match="vpages"):
        ops._pools(s, p, torch.zeros(10, 16, 2, 128).half(), torch.zeros(10, 16, 2, 128))


def test_tensors_of_other_heads_are_refused(monkeypatch):
    """Queries, outputs and pools whose heads are not the shape's: enough elements, in other places."""
    from trixium_b200 import ops

    class Ctx:
        device, h = torch.device("cpu"), None
    called = []
    monkeypatch.setattr(ops, "_stream_of", lambda ctx, on=None: 0)
    monkeypatch.setattr(ops._lib, "check", lambda status, what: called.append(what))
    monkeypatch.setattr(ops._lib, "lib", lambda: type("L", (), {n: staticmethod(lambda *a: 0) for n in
                                                                ("trx_attn_paged", "trx_paged_append")}))
    plan = ops.PagedPlan(2, 8, 2, 16, 10, device="cpu")
    shape = ops.paged_shape(4, 2, 64)
    half = lambda *s: torch.zeros(*s, dtype=torch.float16)
    pool, q = half(10, 16, 2, 64), half(8, 4, 64)
    for bad in (half(8, 8, 64), half(8, 4, 128), half(8, 64, 4), half(32, 64), half(2048), half(8, 2, 4, 64)):
        with pytest.raises(ValueError, match="q: expected"):
            ops.attn_paged(Ctx, shape, plan, bad, pool, pool)
        with pytest.raises(ValueError, match="out: expected"):
            ops.attn_paged(Ctx, shape, plan, q, pool, pool, out=bad)
        with pytest.raises(ValueError, match="q_out: expected"):
            x, w = torch.zeros(8, 256), torch.zeros(64)
            ops.paged_append(Ctx, shape, plan, x, x[:, :128], x[:, 128:], w, w, w, pool, pool, q_out=bad)
    for bad in (half(10, 16, 4, 64), half(10, 16, 64, 2), half(10, 32, 2, 64), half(20, 16, 2, 128), half(10, 16, 128),
                half(20480)):
        with pytest.raises(ValueError, match="kpages: expected"):
            ops.attn_paged(Ctx, shape, plan, q, bad, pool)
        with pytest.raises(ValueError, match="vpages: expected"):
            ops.attn_paged(Ctx, shape, plan, q, pool, bad)
    assert not called
    for ok in (q, q.view(8, 256)):
        ops.attn_paged(Ctx, shape, plan, ok, pool, pool.view(160, 2, 64), out=q)
    assert called == ["trx_attn_paged"] * 2
