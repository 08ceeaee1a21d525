"""The first call that a host thread makes of the device, for every entry point whose kernels copy by tensor map."""
import threading

import numpy as np
import pytest
import torch

from pie_b200 import ops
from tests.util import dev, make_scenario


def _in_a_thread(fn):
    result = []

    def work():
        try:
            result.append(fn())
        except Exception as e:  # noqa: BLE001
            result.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    if isinstance(result[0], Exception):
        raise result[0]
    return result[0]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["decode", "first", "fused", "prefix", "prefill", "prefill_first"])
def test_the_first_call_of_a_thread(kind):
    prefill = kind.startswith("prefill")
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(3, 5), (200, 70), (0, 130)] if prefill else [(c, 1) for c in (3, 200, 77)])
    m, n = sc.meta, sc.q.shape[0]
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    tables = (dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), sc.hq, sc.hkv, sc.d, sc.page_size)
    extra = dict(window_left=60, first_tokens=3) if kind in ("first", "prefill_first") else {}
    if prefill:
        w = ops.BatchPrefillWithPagedKVCacheWrapper(ws)
        w.plan(dev(m.qo_indptr), *tables, causal=True, q_data_type=sc.dtype, **extra)
    else:
        w = (ops.BatchSharedPrefixDecodeWrapper if kind == "prefix" else ops.BatchDecodeWithPagedKVCacheWrapper)(ws)
        w.plan(*tables, q_data_type=sc.dtype, **extra)
    q, pool = sc.q.cuda(), sc.pool.cuda()
    if kind == "fused":
        k, v = (torch.zeros((n, 2, 128), dtype=sc.dtype, device="cuda") for _ in range(2))
        pos = dev(np.array([c for c in (3, 200, 77)], dtype=np.int32))
        call = lambda: w.run_fused(q, k, v, pos, pool)  # noqa: E731
    else:
        call = lambda: w.run(q, pool)  # noqa: E731
    want = call()
    torch.cuda.synchronize()
    got = _in_a_thread(call)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and ops.device_error("cuda") is None
