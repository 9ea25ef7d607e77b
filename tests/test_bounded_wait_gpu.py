"""Failure detection on the device without a fault: a matvec launch told to wait for a peer
exchange that no rank ever signals (trx_matvec_f_tp with a wait counter left at zero) gives up after
its bounded wait (200 ms of %globaltimer per CTA), records TRX_DEV_TIMEOUT in the context's error
word, finishes its work, and leaves the context usable: the next plain launch on the same context
is bit-exact and raises no error bit.  Nothing here faults, traps or hangs the GPU: the wait is a
plain bounded poll of a device counter."""
import ctypes
import time

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_unsignalled_exchange_times_out_and_context_survives():
    from oracle import build as cor
    from trixium_b200 import _lib, image, ops
    ctx = ops.Context(0)
    try:
        t, x = image.synthetic_matvec_case(512, 2048, seed=5, kind=5)
        w = ops.DeviceTensor(t)
        xd = torch.from_numpy(x).cuda()
        want, bad = cor.matvec_f(t.packed, t.rows, t.cols, 5, t.bias, t.rshift, x)
        assert bad == 0
        counter = torch.zeros(1, dtype=torch.int32, device="cuda")   # nothing ever adds to it
        step = torch.zeros(1, dtype=torch.int32, device="cuda")
        tp = _lib.TpXfer()
        tp.world, tp.rank = 2, 0                                     # waits for 2 arrivals
        tp.wait = ctypes.c_void_p(counter.data_ptr())
        tp.step = ctypes.c_void_p(step.data_ptr())
        torch.cuda.synchronize()
        t0 = time.perf_counter()
        y = ops.matvec_f(ctx, w, xd, tp=tp)
        torch.cuda.synchronize()
        waited = time.perf_counter() - t0
        assert ctx.errors() == _lib.TRX_DEV_TIMEOUT
        assert 0.15 < waited < 5.0, waited
        # The launch still computed its rows from its own input.
        assert np.array_equal(y.cpu().numpy().view(np.uint32), want.view(np.uint32))
        # The context works afterwards: a plain launch, bit-exact, no error bits.
        y2 = ops.matvec_f(ctx, w, xd)
        assert np.array_equal(y2.cpu().numpy().view(np.uint32), want.view(np.uint32))
        assert ctx.errors() == 0
    finally:
        ctx.close()


def test_counts_that_an_unfinished_launch_left_are_cleared_with_its_error():
    """A kernel that gives up after a bounded wait leaves the arrival counts of the items it shared with other
    blocks; reading the timeout clears them, so that the calls behind it join whole items again.  The counts are
    put in place from the host, where such a launch would have left them."""
    import paged_ref as R
    from trixium_b200 import _lib, image, ops
    cu = ctypes.CDLL("libcuda.so.1")
    ctx = ops.Context(0)
    try:
        C = R.Cache(ops, [3000, 700], [1, 1], 2, 128, 16, torch.float16, 1)
        D = R.Cache(ops, [3000, 700], [60, 90], 2, 128, 16, torch.float16, 2)
        shape = ops.paged_shape(8, 2, 128, rope_dims=0)
        calls = []
        for c in (C, D):  # the kernels of few and of many rows, with cut items
            q = torch.randn(c.rows, 8, 128, device="cuda").half()
            calls.append(lambda f=1, c=c, q=q: ops.attn_paged(ctx, shape, c.plan, f * q, c.kp, c.vp, max_new=max(c.new)))
        clean = [f() for f in calls]
        # The counts: the fifth word of the context, 4,096 of them, an allocation of their own, zero now.
        n = 4096
        at = (ctypes.c_uint64 * 5).from_address(ctx.h.value)[4]
        base, size = ctypes.c_uint64(0), ctypes.c_size_t(0)
        assert cu.cuMemGetAddressRange_v2(ctypes.byref(base), ctypes.byref(size), ctypes.c_uint64(at)) == 0
        assert base.value == at and 4 * n <= size.value < 1 << 20
        buf = (ctypes.c_uint32 * n)()
        torch.cuda.synchronize()
        assert cu.cuMemcpyDtoH_v2(buf, ctypes.c_uint64(at), ctypes.c_size_t(4 * n)) == 0
        assert not any(buf)
        # A wait that runs out, and what it may have left.
        t, x = image.synthetic_matvec_case(512, 2048, seed=5, kind=5)
        tp = _lib.TpXfer()
        counter, step = [torch.zeros(1, dtype=torch.int32, device="cuda") for _ in range(2)]
        tp.world, tp.rank = 2, 0
        tp.wait, tp.step = ctypes.c_void_p(counter.data_ptr()), ctypes.c_void_p(step.data_ptr())
        ops.matvec_f(ctx, ops.DeviceTensor(t), torch.from_numpy(x).cuda(), tp=tp)
        torch.cuda.synchronize()
        ctypes.memset(buf, 0, 4 * n)
        for i in range(n):
            buf[i] = 1 + i % 2
        assert cu.cuMemcpyHtoD_v2(ctypes.c_uint64(at), buf, ctypes.c_size_t(4 * n)) == 0
        assert ctx.errors() == _lib.TRX_DEV_TIMEOUT
        for f, want in zip(calls, clean):
            f(-3)  # other pieces in scratch than the ones that are looked for
            assert torch.equal(f(), want)
        assert ctx.errors() == 0
    finally:
        ctx.close()
