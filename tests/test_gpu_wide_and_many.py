"""Shapes at which the kernels change over: wide tokens in the multi-axis append, and batches of more than one slice."""
import numpy as np
import pytest
import torch

from pie_b200 import ops
from tests import plain64 as P
from tests.test_gpu_shared_prefix import Batch, _workspace
from tests.util import dev, make_scenario

THETA = 500000.0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype, hq, hkv, d, sections, interleave", [
    (torch.bfloat16, 64, 8, 128, (16, 24, 24), False),   # two stages of the ring
    (torch.float16, 64, 8, 128, (16, 24, 24), True),
    (torch.bfloat16, 32, 8, 256, (32, 48, 48), False),   # the widest token of which two fit
    (torch.bfloat16, 64, 8, 256, (32, 48, 48), False),   # one too wide for that: through registers, many tokens
    (torch.float32, 64, 8, 128, (16, 24, 24), True),
    (torch.bfloat16, 64, 8, 128, (8, 12, 12), False),    # half of a head rotated: element-wise, many tokens
])
def test_wide_tokens(dtype, hq, hkv, d, sections, interleave):
    n, page_size = 1301, 16
    g = torch.Generator().manual_seed(hq + d)
    q, k, v = (torch.randn((n, h, d), generator=g).to(dtype) for h in (hq, hkv, hkv))
    pos = torch.randint(0, 50000, (3, n), generator=g, dtype=torch.int32)
    pages = -(-n // page_size)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    pool = torch.full((pages, 2, page_size, hkv, d), 3.0, dtype=dtype, device="cuda")
    rope = ops.AxisRopeConfig(mode="plain", theta=THETA, scale=1.0, sections=sections, interleave=interleave)
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = ops.rope_axes_append_paged_kv_cache(q.cuda(), k.cuda(), v.cuda(), pos.cuda(), torch.zeros_like(slots), slots, pool,
                                              order.cuda(), i32(0, pages), i32((n - 1) % page_size + 1), rope)
    assert ops.device_error("cuda") is None
    by_token = pool[order.cuda().long()].transpose(1, 2).reshape(-1, 2, hkv, d).cpu()
    for have, src in ((got.cpu(), q), (by_token[:n, 0], k)):
        ref, size = P.rotate_axes(src, pos, sections, False, THETA, interleave)
        assert ((have.double() - ref).abs() <= P.rotation_tolerance(dtype, ref, size)).all()
    assert torch.equal(by_token[:n, 1], v) and bool((by_token[n:] == 3).all())  # rows behind the last token stay


@pytest.mark.gpu
@pytest.mark.parametrize("hq, hkv", [(8, 2), (3, 1)])
def test_more_requests_than_a_slice_with_tails_that_are_split(hq, hkv):
    tails = [(37 * i) % 90 for i in range(560)]
    tails[3], tails[555], tails[559] = 4000, 5000, 3001  # the last two in the second slice
    b = Batch([(24, tails), (40, [2500, 7])], hq, hkv, seed=41)
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()))
    q, pool = b.q.cuda(), b.pool.cuda()
    got = w.run(q, pool, return_lse=True)
    assert ops.device_error("cuda") is None
    b.check(got)
    again = w.run(q, pool)
    assert torch.equal(again, got[0]) and not w.workspace_buffer[: ops.COUNTER_BYTES].any()


@pytest.mark.gpu
def test_a_group_with_an_outlier_is_right_and_one_apart_shares():
    tails = [9, 30, 2, 50]
    b = Batch([(60, tails), (0, [0]), (60, tails)], 16, 4, seed=42)
    for ends in ([0, 9], [0, 5, 9], [0, 4, 5, 9]):
        w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()), groups=dev(torch.tensor(ends, dtype=torch.int32).numpy()))
        b.check(w.run(b.q.cuda(), b.pool.cuda(), return_lse=True))
    assert ops.device_error("cuda") is None


@pytest.fixture(scope="module")
def far_pool():
    """A cache of more than 2^31 elements (4.6 GB), of which the tests use the last pages."""
    return torch.empty((70000, 2, 16, 8, 128), dtype=torch.bfloat16, device="cuda")


def _far(pool, far):
    """(`far` with the pages of `pool` at its end, what to add to a page id)"""
    n = pool.shape[0]
    far[-n:] = pool
    return far, far.shape[0] - n


@pytest.mark.gpu
def test_shared_prefix_in_a_long_cache(far_pool):
    b = Batch([(60, [9, 30, 2, 300]), (8, [1, 2])], 32, 8, seed=43)
    near = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace())).run(b.q.cuda(), b.pool.cuda())
    far, shift = _far(b.pool.cuda(), far_pool)
    b.indices = b.indices + shift
    got = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace())).run(b.q.cuda(), far)
    assert torch.equal(got, near) and ops.device_error("cuda") is None


@pytest.mark.gpu
@pytest.mark.parametrize("prefill", [False, True])
def test_first_tokens_in_a_long_cache(far_pool, prefill):
    sc = make_scenario(32, 8, 128, torch.bfloat16, [(200, 70), (0, 130)] if prefill else [(c, 1) for c in (3, 700, 77)])
    m, outs = sc.meta, []
    far, shift = _far(sc.pool.cuda(), far_pool)
    for pool, add in ((sc.pool.cuda(), 0), (far, shift)):
        tables = (dev(m.kv_indptr), dev(m.kv_indices + np.int32(add)), dev(m.kv_last_page_len), 32, 8, 128, 16)
        extra = dict(window_left=60, first_tokens=3, q_data_type=torch.bfloat16)
        if prefill:
            w = ops.BatchPrefillWithPagedKVCacheWrapper(_workspace())
            w.plan(dev(m.qo_indptr), *tables, causal=True, **extra)
        else:
            w = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
            w.plan(*tables, **extra)
        outs.append(w.run(sc.q.cuda(), pool))
    assert torch.equal(*outs) and ops.device_error("cuda") is None


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 1300])
def test_axes_in_a_long_cache(far_pool, n):
    pages = -(-n // 16)
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn((n, h, 128), generator=g).to(torch.bfloat16).cuda() for h in (32, 8, 8))
    pos = torch.randint(0, 50000, (3, n), generator=g, dtype=torch.int32).cuda()
    slots = torch.arange(n, dtype=torch.int32, device="cuda")
    rope = ops.AxisRopeConfig(mode="plain", theta=THETA, scale=1.0, sections=(16, 24, 24))
    near = torch.zeros((pages, 2, 16, 8, 128), dtype=torch.bfloat16, device="cuda")
    far, shift = _far(near, far_pool)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    outs = [ops.rope_axes_append_paged_kv_cache(q, k, v, pos, torch.zeros_like(slots), slots, pool,
                                                torch.arange(pages, dtype=torch.int32, device="cuda") + add, i32(0, pages),
                                                i32((n - 1) % 16 + 1), rope) for pool, add in ((near, 0), (far, shift))]
    assert torch.equal(*outs) and torch.equal(near, far[shift:]) and ops.device_error("cuda") is None
