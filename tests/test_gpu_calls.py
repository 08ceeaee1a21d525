"""The native way from Python into the short calls: the same results, bit for bit, as the functions' own checks lead to,
and the same refusals."""
import copy
import ctypes as C

import numpy as np
import pytest
import torch

from pie_b200 import _calls, _lib, ops
from tests.util import dev, make_scenario


# ---- on the CPU
def test_what_is_not_a_cuda_tensor_is_declined():
    table = _axes().prepared()
    t = torch.zeros(2, 2, 8)
    i = torch.zeros(2, dtype=torch.int32)
    args = (t, t, t, i.view(1, 2), i, i, torch.zeros(1, 2, 16, 2, 8), i, i, None)
    assert _calls.rope_axes_append(C.addressof(table), *args) is False
    assert _calls.rope_axes_append(C.addressof(table), None, 3, "x", *args[3:]) is False
    plan = _calls.plan(0, _lib.SharedPrefixArgs(), None)
    assert _calls.decode_run(plan, t, t, None) is False
    assert _calls.decode_run(plan, None, 1, None) is False
    assert _calls.prefill_run(plan, None, t, t, None) is False and _calls.prefill_run(plan, (2, 1), t, t, None) is False


def test_wrong_counts_sizes_and_capsules_raise():
    with pytest.raises(ValueError, match="sizes"):
        _calls.plan(0, _lib.AttnOptions(), None)
    with pytest.raises(ValueError, match="sizes"):
        _calls.plan(0, _lib.SharedPrefixArgs(), _lib.SharedPrefixArgs())
    with pytest.raises(TypeError):
        _calls.decode_run(None)
    with pytest.raises(ValueError):
        _calls.decode_run(object(), None, None, None)
    with pytest.raises(TypeError):
        _calls.rope_axes_append(1, 2)
    with pytest.raises(TypeError):
        _calls.prefill_run(_calls.plan(0, _lib.SharedPrefixArgs(), _lib.AttnOptions()), (1,), None, None, None)


def test_a_copied_config_lays_out_its_own_table():
    rope = _axes(sections=[4, 2, 2])
    first = rope.prepared()
    for other in (copy.copy(rope), copy.deepcopy(rope)):
        assert other.__dict__["_table"] is None and other.sections == (4, 2, 2)
        assert list(other.prepared().turn) == list(first.turn) and other.prepared() is not first
    assert rope.prepared() is first


# ---- on the GPU
def _axes(sections=(16, 24, 24), **kw):
    return ops.AxisRopeConfig(**{**dict(mode="plain", theta=500000.0, scale=1.0, sections=sections), **kw})


def _append(sc, rope, q_out=None, **over):
    m = sc.meta
    n = sc.q.shape[0]
    g = torch.Generator().manual_seed(5)
    k, v = (torch.randn((n, sc.hkv, sc.d), generator=g).to(sc.dtype).cuda() for _ in range(2))
    pool = sc.pool.cuda()
    a = dict(q=sc.q.cuda(), k=k, v=v, pos_ids=torch.randint(0, 99999, (len(rope.sections), n), generator=g, dtype=torch.int32).cuda(),
             batch_indices=dev(np.repeat(np.arange(len(m.qo_indptr) - 1), np.diff(m.qo_indptr)).astype(np.int32)),
             positions=dev(np.concatenate([np.arange(x) for x in np.diff(m.qo_indptr)]).astype(np.int32)),
             paged_kv_cache=pool, kv_indices=dev(m.kv_indices), kv_indptr=dev(m.kv_indptr),
             kv_last_page_len=dev(m.kv_last_page_len), rope=rope, q_out=q_out)
    a.update(over)
    return ops.rope_axes_append_paged_kv_cache(**a), a["paged_kv_cache"]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hq, hkv, lens", [(8, 2, (1, 1, 1)), (6, 3, (5, 0, 33)), (32, 8, (900, 700))])
def test_append_is_the_same_either_way(dtype, hq, hkv, lens):
    sc = make_scenario(hq, hkv, 128, dtype, [(20, n) for n in lens])
    rope = _axes()
    slow, slow_pool = _append(sc, rope)  # the first call of a configuration lays out its table
    fast, fast_pool = _append(sc, rope)
    assert torch.equal(slow, fast) and torch.equal(slow_pool, fast_pool)
    assert not torch.equal(fast_pool, sc.pool.cuda())
    wide = torch.full((sc.q.shape[0], hq, 160), 7.0, dtype=dtype, device="cuda")
    out = wide[:, :, :128]
    got, pool = _append(sc, rope, q_out=out)
    assert got is out and torch.equal(out, slow) and torch.equal(pool, slow_pool) and bool((wide[:, :, 128:] == 7).all())
    in_place = sc.q.cuda()
    got, pool = _append(sc, rope, q=in_place, q_out=in_place)
    assert got is in_place and torch.equal(in_place, slow) and torch.equal(pool, slow_pool)
    strided = torch.zeros((sc.q.shape[0], hq, 2, 128), dtype=dtype, device="cuda")
    strided[:, :, 1] = sc.q.cuda()
    got, _ = _append(sc, rope, q=strided[:, :, 1])
    assert torch.equal(got, slow) and got.is_contiguous()
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
def test_append_refuses_the_same_either_way():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(20, 3), (4, 2)])
    n = 5
    rope = _axes()
    _append(sc, rope)
    i32 = lambda *shape: torch.zeros(shape, dtype=torch.int32, device="cuda")  # noqa: E731
    z = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device="cuda")  # noqa: E731
    for over in (dict(q=z(n, 8, 64)), dict(q=z(n - 1, 8, 128)), dict(q=z(n, 8, 128, dtype=torch.float16)), dict(q=sc.q),
                 dict(k=z(n, 3, 128)), dict(k=z(n, 2, 256)[:, :, ::2]), dict(v=z(n, 2, 64)), dict(v=z(n, 2, 128, dtype=torch.float32)),
                 dict(pos_ids=i32(2, n)), dict(pos_ids=i32(3, n - 1)), dict(pos_ids=i32(3, n).long()), dict(pos_ids=i32(n, 3).T),
                 dict(batch_indices=i32(n - 1)), dict(positions=i32(n - 1)), dict(positions=i32(n).long()),
                 dict(kv_indices=i32(64)[::2]), dict(kv_indptr=i32(3).long()), dict(kv_indptr=i32(0)),
                 dict(paged_kv_cache=z(64, 2, 16, 3, 128)), dict(paged_kv_cache=z(64, 3, 16, 2, 128)),
                 dict(paged_kv_cache=z(64, 2, 16, 2, 128, dtype=torch.float16)), dict(paged_kv_cache=sc.pool),
                 dict(paged_kv_cache=(sc.pool, sc.pool)), dict(q_out=z(n, 8, 64)), dict(q_out=z(n, 8, 128, dtype=torch.float16)),
                 dict(k=z(n, 2, 128).double(), v=z(n, 2, 128).double(), q=z(n, 8, 128).double()), dict(v=None), dict(k=None)):
        for config in (rope, _axes()):
            with pytest.raises(ValueError):
                _append(sc, config, **over)
    with torch.no_grad():
        same, _ = _append(sc, rope)
    assert same.shape == (n, 8, 128)


@pytest.mark.gpu
def test_an_output_that_does_not_fit_raises_the_allocators_error():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(20, 3), (4, 2)])
    rope = _axes()
    _append(sc, rope)
    wide = torch.zeros((1, 1, 128), dtype=torch.bfloat16, device="cuda").expand(5, 1 << 29, 128)  # 687 GB of output
    for config in (rope, _axes()):
        with pytest.raises(torch.OutOfMemoryError):
            _append(sc, config, q=wide)
    again, _ = _append(sc, rope)
    assert again.shape == (5, 8, 128) and ops.device_error("cuda") is None


def _decode_wrapper(sc, kind):
    m = sc.meta
    ws = torch.empty(64 << 20, dtype=torch.uint8, device="cuda")
    tables = (dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), sc.hq, sc.hkv, sc.d, sc.page_size)
    if kind == "prefix":
        w = ops.BatchSharedPrefixDecodeWrapper(ws)
        w.plan(*tables, q_data_type=sc.dtype)
    else:
        w = ops.BatchDecodeWithPagedKVCacheWrapper(ws)
        w.plan(*tables, window_left=60, first_tokens=3, q_data_type=sc.dtype)
    return w


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["prefix", "first"])
@pytest.mark.parametrize("dtype, d", [(torch.bfloat16, 128), (torch.float16, 128), (torch.float32, 64)])
def test_decode_is_the_same_either_way(kind, dtype, d):
    sc = make_scenario(8, 2, d, dtype, [(c, 1) for c in (3, 200, 77, 1000)])
    w = _decode_wrapper(sc, kind)
    q, pool = sc.q.cuda(), sc.pool.cuda()
    slow, _ = w.run(q, pool, return_lse=True)
    fast = w.run(q, pool)
    assert torch.equal(slow, fast)
    out = torch.empty_like(q)
    assert w.run(q, pool, out=out) is out and torch.equal(out, slow)
    wide = torch.zeros((4, 8, 2, d), dtype=dtype, device="cuda")
    wide[:, :, 1] = q
    assert torch.equal(w.run(wide[:, :, 1], pool), slow)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = w.run(q, pool)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(again, slow)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = w.run(q, pool)
    for _ in range(3):
        captured.zero_()
        graph.replay()
        assert torch.equal(captured, slow)
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["prefix", "first"])
def test_decode_refuses_the_same_either_way(kind):
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(c, 1) for c in (3, 200)])
    w = _decode_wrapper(sc, kind)
    q, pool = sc.q.cuda(), sc.pool.cuda()
    for args in ((q[:1], pool), (q[:, :4], pool), (q.half(), pool), (sc.q, pool), (q, sc.pool), (q, pool.half()), (q, pool[:, :, :8]),
                 (q, (pool, pool)), (None, pool), (q.repeat(1, 1, 2)[:, :, ::2], pool)):
        for lse in (False, True):
            with pytest.raises(ValueError):
                w.run(*args, return_lse=lse)
    for out in (q.half(), q[:1], torch.empty((2, 8, 256), dtype=q.dtype, device="cuda")[:, :, ::2], sc.q):
        for lse in (False, True):
            with pytest.raises(ValueError):
                w.run(q, pool, out=out, return_lse=lse)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype, hq, hkv, d", [(torch.bfloat16, 8, 2, 128), (torch.float16, 6, 2, 128), (torch.float32, 4, 4, 64)])
def test_prefill_is_the_same_either_way(causal, dtype, hq, hkv, d):
    sc = make_scenario(hq, hkv, d, dtype, [(3, 5), (200, 70), (0, 130)])
    m = sc.meta
    w = ops.BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    w.plan(dev(m.qo_indptr), dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), hq, hkv, d, sc.page_size,
           causal=causal, window_left=60, first_tokens=3, q_data_type=dtype)
    q, pool = sc.q.cuda(), sc.pool.cuda()
    slow, _ = w.run(q, pool, return_lse=True)
    assert torch.equal(w.run(q, pool), slow)
    out = torch.empty_like(q)
    assert w.run(q, pool, out=out) is out and torch.equal(out, slow)
    wide = torch.zeros((q.shape[0], hq, 2, d), dtype=dtype, device="cuda")
    wide[:, :, 1] = q
    assert torch.equal(w.run(wide[:, :, 1], pool), slow)
    bigger = torch.cat([pool, pool[:3]])  # another number of pages: the work list is built again
    assert torch.equal(w.run(q, bigger), slow) and torch.equal(w.run(q, pool), slow)
    for args in ((q[:, :2], pool), (sc.q, pool), (q, sc.pool), (q, (pool, pool)), (None, pool), (q.double(), pool),
                 (q, pool[:, :, :8])):
        for lse in (False, True):
            with pytest.raises((ValueError, AttributeError) if args[0] is None else ValueError):
                w.run(*args, return_lse=lse)
    assert ops.device_error("cuda") is None
