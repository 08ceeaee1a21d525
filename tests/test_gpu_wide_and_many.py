"""Shapes at which the kernels change over: wide tokens in the multi-axis append, and batches of more than one slice."""
import pytest
import torch

from pie_b200 import ops
from tests import plain64 as P
from tests.test_gpu_shared_prefix import Batch, _workspace
from tests.util import dev

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
