"""Bounded waits of the serving step's kernels that run out, without a GPU fault:
the next launch of a kernel is made to expect 16 bytes more than its copies
bring (minq_debug_inject_stall), so its waits end at their limit. The call comes
back, the status is reported once, and the next call is right."""
import time

import numpy as np
import pytest

from test_gpu_serving import _fill, dev, torch  # noqa: F401


def test_stall_refuses_other_kernels(mq):
    from minq_b200 import _lib
    L = _lib.lib()
    for kernel in (-1, 3, 1 << 20):
        assert L.minq_debug_inject_stall(kernel) == _lib.ERR_ARG
        assert b"kv4_attend" in L.minq_last_error()


def _stalled(mq, torch, kernel, call):
    """(output of the stalled call, output of the calls around it)."""
    from minq_b200 import _lib
    L = _lib.lib()
    want = call().clone()
    torch.cuda.synchronize()
    assert L.minq_device_status() == _lib.OK
    assert L.minq_debug_inject_stall(kernel) == _lib.OK
    t0 = time.perf_counter()
    got = call()
    torch.cuda.synchronize()
    took = time.perf_counter() - t0
    assert 0.9 < took < 30.0, took
    assert L.minq_device_status() == _lib.ERR_TIMEOUT
    assert L.minq_device_status() == _lib.OK  # once
    t0 = time.perf_counter()
    assert torch.equal(call(), want)
    torch.cuda.synchronize()
    assert time.perf_counter() - t0 < 0.5  # the stall was for one launch
    assert L.minq_device_status() == _lib.OK
    return got, want


def _attend(mq, torch, nh, nkv, hd, lens, new):
    kp, vp, table, kv, vv = _fill(mq, torch, 1, lens, nkv, hd, 16)
    start = [0] + np.cumsum(new).tolist()
    q = torch.randn(start[-1], nh, hd, device="cuda")
    args = (q, dev(torch, start), dev(torch, lens), table, kp, vp)
    return lambda: mq.kv4_attend(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd,new", [(8, 2, 128, 1), (14, 2, 64, 1), (32, 8, 128, 4)])
@pytest.mark.parametrize("lens", [[300, 5000], [20]])
def test_attend_wait_runs_out(mq, torch, nh, nkv, hd, new, lens):
    _stalled(mq, torch, 0, _attend(mq, torch, nh, nkv, hd, lens, [new] * len(lens)))


@pytest.mark.gpu
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 128), (14, 2, 64)])
@pytest.mark.parametrize("lens,new", [([64], [64]), ([900, 3000, 40], [200, 64, 1])])
def test_attend_chunk_wait_runs_out(mq, torch, nh, nkv, hd, lens, new):
    """Tensor memory and the copies in flight are let go: the next calls run."""
    _stalled(mq, torch, 1, _attend(mq, torch, nh, nkv, hd, lens, new))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 5000), (3, 151936), (40, 20000)])
@pytest.mark.parametrize("temperature", [0.0, 1.0])
def test_sample_rows_wait_runs_out(mq, torch, rows, n, temperature):
    """Every row of the stalled call gets token 0."""
    x, u = torch.randn(rows, n, device="cuda"), torch.rand(rows, device="cuda")
    x[:, 0] = -5.0
    t = torch.full((rows,), temperature, device="cuda")
    tp = torch.full((rows,), 0.9, device="cuda")
    got, _ = _stalled(mq, torch, 2, lambda: mq.sample_rows(x, u, temperature=t, top_p=tp))
    assert not got.any()
