"""Shared-prefix runs of several host threads on one stream: a run is two launches, which have to follow each other."""
import threading

import numpy as np
import pytest
import torch

from pie_b200 import ops
from tests.test_gpu_shared_prefix import Batch, _workspace
from tests.util import dev


@pytest.mark.gpu
@pytest.mark.parametrize("wrappers, lse", [(1, False), (1, True), (4, False)])
def test_threads_on_one_stream_and_workspace(wrappers, lse):
    b = Batch([(60, [9, 30, 2, 5] * 4)], 8, 2, seed=31)
    ws = _workspace()
    w = [b.plan(ops.BatchSharedPrefixDecodeWrapper(ws)) for _ in range(wrappers)]
    pool = b.pool.cuda()
    queries = [(b.q * (0.25 * (i + 1))).cuda() for i in range(4)]
    run = lambda i: w[i % wrappers].run(queries[i], pool, return_lse=lse)  # noqa: E731
    first = (lambda x: x[0]) if lse else (lambda x: x)
    want = [first(run(i)) for i in range(4)]
    torch.cuda.synchronize()
    start, wrong, failed = threading.Barrier(4), [0] * 4, []

    def work(i):
        try:
            start.wait(timeout=30)
            for _ in range(20):
                got = [first(run(i)) for _ in range(25)]
                wrong[i] += sum(not torch.equal(g, want[i]) for g in got)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and wrong == [0] * 4
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
def test_threads_of_different_wrappers_on_one_stream_and_workspace():
    b = Batch([(60, [9, 30, 2, 5] * 4)], 8, 2, seed=32)
    ws = _workspace()
    n = len(b.lens)
    tables = [dev(x) for x in (b.indptr, b.indices, b.last)]
    shared, plain, first = ops.BatchSharedPrefixDecodeWrapper(ws), *(ops.BatchDecodeWithPagedKVCacheWrapper(ws) for _ in range(2))
    b.plan(shared)
    plain.plan(*tables, 8, 2, 128, 16, q_data_type=torch.bfloat16)
    first.plan(*tables, 8, 2, 128, 16, q_data_type=torch.bfloat16, window_left=600, first_tokens=20)
    pool = b.pool.cuda()
    calls = [lambda q: shared.run(q, pool), lambda q: plain.run(q, pool), lambda q: first.run(q, pool),
             lambda q: plain.run_fused(q, *rows, pos, scratch)]
    rows = [torch.zeros((n, 2, 128), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    pos, scratch = dev(np.array(b.lens, dtype=np.int32) - 1), b.pool.cuda()
    queries = [(b.q * (0.25 * (i + 1))).cuda() for i in range(4)]
    want = [call(q) for call, q in zip(calls, queries)]
    torch.cuda.synchronize()
    start, wrong, failed = threading.Barrier(4), [0] * 4, []

    def work(i):
        try:
            start.wait(timeout=30)
            for _ in range(20):
                got = [calls[i](queries[i]) for _ in range(25)]
                wrong[i] += sum(not torch.equal(g, want[i]) for g in got)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed and wrong == [0] * 4
    assert ops.device_error("cuda") is None
