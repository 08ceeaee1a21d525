"""A sliding window behind which the first tokens of a context stay visible: decode and prefill."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from pie_b200 import _lib, ops
from tests import plain64 as P
from tests.util import dev, make_scenario


def _workspace(mib=64):
    return torch.empty(mib << 20, dtype=torch.uint8, device="cuda")


def _decode(sc, window, first, **run):
    m = sc.meta
    w = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
    w.plan(dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), sc.hq, sc.hkv, sc.d, sc.page_size,
           window_left=window, first_tokens=first, q_data_type=sc.dtype)
    return w.run(sc.q.cuda(), sc.pool.cuda(), return_lse=True, **run)


def _prefill(sc, window, first, causal=True, wrapper=ops.BatchPrefillWithPagedKVCacheWrapper, **run):
    m = sc.meta
    w = wrapper(_workspace())
    w.plan(dev(m.qo_indptr), dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), sc.hq, sc.hkv, sc.d,
           sc.page_size, causal=causal, window_left=window, first_tokens=first, q_data_type=sc.dtype)
    return w.run(sc.q.cuda(), sc.pool.cuda(), return_lse=True, **run)


def _check(sc, got, window, first, causal=True, **kw):
    m = sc.meta
    ref = P.attend(sc.q, sc.pool, m.qo_indptr, m.kv_indptr, m.kv_indices, m.kv_last_page_len, causal=causal,
                   window_left=window, first_tokens=first, **kw)
    assert ops.device_error("cuda") is None
    P.check_attention(got[0], got[1], sc.q, sc.pool, ref)


def _poison_unseen(sc, window, first):
    """NaN in every K and V row that no query token of a request sees, -1 for the ids of pages that hold only such
    rows (and no first token)."""
    m, ps = sc.meta, sc.page_size
    lens = P.kv_lens(m.kv_indptr, m.kv_last_page_len, ps)
    ids = m.kv_indices.copy()
    for b, kv in enumerate(lens):
        new = int(m.qo_indptr[b + 1] - m.qo_indptr[b])
        low = max(0, kv - new - window)
        for i in range(int(m.kv_indptr[b]), int(m.kv_indptr[b + 1])):
            t0 = (i - int(m.kv_indptr[b])) * ps
            page = int(m.kv_indices[i])
            seen = [t for t in range(t0, t0 + ps) if t < kv and (t < first or t >= low)]
            for t in set(range(t0, t0 + ps)) - set(seen):
                sc.pool[page, :, t - t0] = math.nan
            if not seen:
                ids[i] = -1
    m.kv_indices = ids


# ---- on the CPU: refusals
def test_the_library_refuses_on_the_host():
    L, one = _lib.lib, C.c_void_p(256)
    o = _lib.AttnOptions()
    o.window_left, o.first_tokens = 15, -1
    call = lambda: L.piekv_decode_run_opt(one, 128, 128, one, one, None, one, one, one, 1, 8, 4, 128, 16, 8, 2, 1.0, one,  # noqa: E731
                                          1 << 24, None, None, C.byref(o))
    assert call() > 0 and b"first_tokens" in L.piekv_last_error_string()
    o.first_tokens = 4
    rp = _lib.RopeParams()
    rc = L.piekv_decode_step_fused_opt(one, one, one, 128, 128, 128, 128, 128, 128, one, one, one, None, one, one, one, 1, 8,
                                       4, 128, 16, 8, 2, C.byref(rp), 1.0, one, 1 << 24, None, None, C.byref(o))
    assert rc > 0 and b"first_tokens" in L.piekv_last_error_string()
    rc = L.piekv_prefill_run_opt(one, 128, 128, one, one, None, one, one, one, one, one, 64, 1, 1, 1, 1, 8, 4, 128, 16, 8, 2,
                                 1.0, one, 1 << 24, None, None, C.byref(o))
    assert rc > 0 and b"mask" in L.piekv_last_error_string()
    assert L.piekv_decode_first_tokens_workspace_bytes(64, 32, 8, 128) >= 65536
    assert L.piekv_decode_first_tokens_workspace_bytes(-1, 32, 8, 128) == 0


def test_first_tokens_are_checked():
    assert ops._check_first_tokens(4, 10) == 4
    assert ops._check_first_tokens(2 ** 40, 10) == 2 ** 31 - 1
    assert ops._check_first_tokens(4, -1) == 0  # nothing is hidden without a window
    with pytest.raises(ValueError, match="first_tokens"):
        ops._check_first_tokens(-1, 10)


# ---- decode
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, hkv", [(32, 8), (8, 8), (4, 4), (16, 2), (6, 2), (5, 1), (16, 1), (12, 12), (9, 3), (20, 10),
                                     (40, 2)])
@pytest.mark.parametrize("window, first", [(63, 4), (0, 1), (100, 37), (15, 64)])
def test_decode(dtype, hq, hkv, window, first):
    ctx = [0, 1, 15, 16, 17, 63, 64, 66, 67, 68, 69, 100, 137, 300, 1000]
    sc = make_scenario(hq, hkv, 128, dtype, [(c, 1) for c in ctx], seed=hq + window)
    _poison_unseen(sc, window, first)
    _check(sc, _decode(sc, window, first), window, first)


@pytest.mark.gpu
@pytest.mark.parametrize("d, page_size, dtype", [(64, 16, torch.bfloat16), (128, 16, torch.float32), (256, 8, torch.float16),
                                                 (40, 5, torch.float32)])
def test_decode_other_shapes(d, page_size, dtype):
    sc = make_scenario(6, 3, d, dtype, [(c, 1) for c in (0, 4, 15, 40, 41, 90, 200)], page_size=page_size)
    _poison_unseen(sc, 20, 3)
    _check(sc, _decode(sc, 20, 3), 20, 3)


@pytest.mark.gpu
@pytest.mark.parametrize("ctx, window, first, hkv", [
    ([30000], 20000, 16, 8), ([9000, 3, 8000], 4095, 5000, 4), ([5000] * 3, 4999, 1, 1), ([700], 511, 4, 8),
    ([2000 + 37 * i for i in range(40)], 1023, 4, 2)])
def test_decode_long_contexts_are_split(ctx, window, first, hkv):
    sc = make_scenario(4 * hkv, hkv, 128, torch.bfloat16, [(c, 1) for c in ctx], seed=3)
    _check(sc, _decode(sc, window, first), window, first)


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [1100, 2500])
def test_decode_many_requests(batch):
    sc = make_scenario(2, 1, 128, torch.bfloat16, [((7 * i) % 90, 1) for i in range(batch)])
    _check(sc, _decode(sc, 30, 2), 30, 2)


@pytest.mark.gpu
def test_decode_empty_requests_sinks_strides_and_scale():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(0, 0), (70, 1), (0, 0), (5, 1), (0, 0)])
    m = sc.meta
    # one query row per request, also of those that hold nothing
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((5, 8, 2, 128), generator=g).to(torch.bfloat16)
    sc.q = wide[:, :, 0]
    m.qo_indptr = np.arange(6, dtype=np.int32)
    sinks = torch.randn(8, generator=g) * 3
    w = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
    w.plan(dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), 8, 2, 128, 16, window_left=20, first_tokens=3,
           q_data_type=torch.bfloat16)
    q = wide.cuda()[:, :, 0]
    assert not q.is_contiguous()
    got = w.run(q, sc.pool.cuda(), return_lse=True, sinks=sinks.cuda(), sm_scale=0.3)
    ref = P.attend(sc.q, sc.pool, m.qo_indptr, m.kv_indptr, m.kv_indices, m.kv_last_page_len, sm_scale=0.3, window_left=20,
                   first_tokens=3, sinks=sinks)
    P.check_attention(got[0], got[1], sc.q, sc.pool, ref, scale=0.3)
    assert (got[0][0] == 0).all() and torch.isinf(got[1][0]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("window, first", [(2 ** 31 - 1, 3), (5, 2 ** 31 - 1), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_the_largest_numbers(window, first):
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(c, 1) for c in (3, 50, 300)])
    _check(sc, _decode(sc, window, first), -1, 0)
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(3, 40), (200, 70)])
    _check(sc, _prefill(sc, window, first), -1, 0)
    sc = make_scenario(9, 3, 128, torch.bfloat16, [(0, 40)])
    sc.meta.kv_indptr[1], sc.meta.kv_last_page_len[0] = 1, 9  # more query tokens than keys
    _check(sc, _prefill(sc, window, first), -1, 0)


@pytest.mark.gpu
def test_decode_nan_in_sight_comes_out():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(2000, 1), (300, 1)])
    clean = _decode(sc, 1500, 4)[0]
    sc.pool[sc.meta.kv_indices[100], 0, 3, 1] = math.nan  # inside the first request's window, kv head 1
    out = _decode(sc, 1500, 4)[0]
    assert torch.isnan(out[0, 4:]).all()
    assert torch.equal(out[0, :4], clean[0, :4]) and torch.equal(out[1], clean[1])


@pytest.mark.gpu
def test_decode_without_effect_equals_the_plain_call():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(c, 1) for c in (3, 50, 300)])
    m = sc.meta
    w = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
    w.plan(dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), 8, 2, 128, 16, q_data_type=torch.bfloat16)
    plain = w.run(sc.q.cuda(), sc.pool.cuda())
    w.plan(dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), 8, 2, 128, 16, q_data_type=torch.bfloat16,
           first_tokens=9)  # no window: nothing is hidden
    assert torch.equal(plain, w.run(sc.q.cuda(), sc.pool.cuda()))
    _check(sc, _decode(sc, 5000, 9), -1, 0)  # a window wider than every context


@pytest.mark.gpu
def test_decode_graph_with_changing_tables_and_streams():
    sc = make_scenario(16, 4, 128, torch.bfloat16, [(c, 1) for c in (700, 31, 64, 900)], num_pages=400)
    m = sc.meta
    indptr, last = dev(m.kv_indptr), dev(m.kv_last_page_len)
    indices = torch.zeros(400, dtype=torch.int32, device="cuda")
    indices[: len(m.kv_indices)] = dev(m.kv_indices)
    pool, q = sc.pool.cuda(), sc.q.cuda()
    out = torch.empty_like(q)
    w = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace(), use_cuda_graph=True, paged_kv_indptr_buffer=indptr,
                                               paged_kv_indices_buffer=indices, paged_kv_last_page_len_buffer=last)
    w.plan(indptr, indices, last, 16, 4, 128, 16, window_left=100, first_tokens=5, q_data_type=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w.run(q, pool, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(q, pool, out=out)
    for seed, ctx in enumerate(((700, 31, 64, 900), (3, 1000, 500, 1), (0, 0, 0, 0))):
        nx = make_scenario(16, 4, 128, torch.bfloat16, [(c, 1) for c in ctx], num_pages=400, perm_seed=seed)
        nm = nx.meta
        indptr.copy_(dev(nm.kv_indptr))
        indices[: len(nm.kv_indices)] = dev(nm.kv_indices)
        last.copy_(dev(nm.kv_last_page_len))
        out.fill_(5.0)
        for _ in range(2):
            graph.replay()
        ref = P.attend(sc.q, sc.pool, nm.qo_indptr, nm.kv_indptr, nm.kv_indices, nm.kv_last_page_len, window_left=100,
                       first_tokens=5)
        P.check_attention(out, None, sc.q, sc.pool, ref)
    assert not w.workspace_buffer[: ops.COUNTER_BYTES].any()


@pytest.mark.gpu
def test_decode_results_are_reproducible():
    sc = make_scenario(32, 8, 128, torch.bfloat16, [(900 + 100 * i, 1) for i in range(9)], seed=2)
    first = _decode(sc, 700, 4)
    for _ in range(3):
        again = _decode(sc, 700, 4)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


@pytest.mark.gpu
def test_decode_bad_pages_are_reported():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(200, 1)])
    sc.meta.kv_indices[-1] = 9999
    ops.device_error("cuda")
    _decode(sc, 50, 4)
    assert ops.device_error("cuda")["code"] == 3
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(200, 1)])
    sc.meta.kv_last_page_len[0] = 17
    _decode(sc, 50, 4)
    assert ops.device_error("cuda")["code"] == 4


# ---- prefill
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, hkv", [(8, 2), (4, 4), (6, 2), (2, 1), (5, 1), (6, 1), (16, 2), (10, 1), (16, 1), (20, 1)])
@pytest.mark.parametrize("window, first", [(63, 4), (0, 1), (200, 130), (15, 300)])
def test_prefill(dtype, hq, hkv, window, first):
    sc = make_scenario(hq, hkv, 128, dtype, [(0, 1), (0, 17), (5, 128), (700, 129), (300, 1), (511, 256), (40, 0), (1000, 3)],
                       seed=hq + window)
    _poison_unseen(sc, window, first)
    _check(sc, _prefill(sc, window, first), window, first)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d, page_size, dtype", [(128, 16, torch.bfloat16), (64, 16, torch.bfloat16),
                                                 (128, 8, torch.float32)])
def test_prefill_other_shapes_and_not_causal(causal, d, page_size, dtype):
    sc = make_scenario(4, 2, d, dtype, [(0, 33), (150, 20), (400, 140)], page_size=page_size)
    _check(sc, _prefill(sc, 50, 7, causal=causal), 50, 7, causal=causal)


@pytest.mark.gpu
def test_prefill_long_context():
    sc = make_scenario(4, 1, 128, torch.bfloat16, [(9000, 300), (0, 2100)], seed=5)
    _check(sc, _prefill(sc, 1023, 4), 1023, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.1, 0.0])
@pytest.mark.parametrize("hq, hkv", [(8, 2), (6, 2)])
def test_scales_that_are_not_positive(scale, hq, hkv):
    for new in (1, 40):
        sc = make_scenario(hq, hkv, 128, torch.bfloat16, [(200, new), (0, new), (33, new)])
        m = sc.meta
        got = (_decode if new == 1 else _prefill)(sc, 50, 5, sm_scale=scale)
        ref = P.attend(sc.q, sc.pool, m.qo_indptr, m.kv_indptr, m.kv_indices, m.kv_last_page_len, sm_scale=scale,
                       window_left=50, first_tokens=5)
        P.check_attention(got[0], got[1], sc.q, sc.pool, ref, scale=abs(scale))


@pytest.mark.gpu
def test_prefill_sinks_and_the_sink_wrapper():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(300, 40), (0, 150)])
    g = torch.Generator().manual_seed(1)
    sinks = torch.randn(8, generator=g) * 3
    _check(sc, _prefill(sc, 60, 4, sinks=sinks.cuda()), 60, 4, sinks=sinks)
    _check(sc, _prefill(sc, 60, 4, wrapper=ops.BatchAttentionWithAttentionSinkWrapper, sinks=sinks.cuda()), 60, 4,
           sinks=sinks)


@pytest.mark.gpu
def test_prefill_query_rows_longer_than_the_context():
    """More query tokens than cached ones (a caller that has not appended): rows before the context see nothing."""
    sc = make_scenario(4, 2, 128, torch.bfloat16, [(0, 40)])
    sc.meta.kv_indptr[1] = 1
    sc.meta.kv_last_page_len[0] = 9
    out, lse = _prefill(sc, 4, 2)
    m = sc.meta
    ref = P.attend(sc.q, sc.pool, m.qo_indptr, m.kv_indptr, m.kv_indices, m.kv_last_page_len, window_left=4, first_tokens=2)
    P.check_attention(out, lse, sc.q, sc.pool, ref)
    assert (out[:31] == 0).all() and torch.isinf(lse[:31]).all()


@pytest.mark.gpu
def test_prefill_and_decode_agree_and_masks_are_refused():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(c, 1) for c in (300, 20, 90)])
    a, b = _decode(sc, 40, 3), _prefill(sc, 40, 3)
    # two kernels, each within its tolerance of the same value
    ref = P.attend(sc.q, sc.pool, sc.meta.qo_indptr, sc.meta.kv_indptr, sc.meta.kv_indices, sc.meta.kv_last_page_len,
                   window_left=40, first_tokens=3)
    for got in (a, b):
        P.check_attention(got[0], got[1], sc.q, sc.pool, ref)
    m = sc.meta
    w = ops.BatchPrefillWithPagedKVCacheWrapper(_workspace())
    tables = (dev(m.qo_indptr), dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), 8, 2, 128, 16)
    with pytest.raises(ValueError, match="first_tokens"):
        w.plan(*tables, window_left=4, first_tokens=1, custom_mask=torch.ones(10, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError, match="first_tokens"):
        w.plan(*tables, window_left=4, first_tokens=-2)
    w.plan(*tables, causal=True, window_left=4, first_tokens=1, q_data_type=torch.bfloat16)
    with pytest.raises(ValueError, match="packed mask"):
        w.export_custom_mask(3, sc.num_pages)
    d = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
    d.plan(tables[1], tables[2], tables[3], 8, 2, 128, 16, window_left=4, first_tokens=1, q_data_type=torch.bfloat16)
    with pytest.raises(ValueError, match="first_tokens"):
        d.run_fused(sc.q.cuda(), sc.k.cuda(), sc.v.cuda(), dev(m.pos_ids), sc.pool.cuda())
    small = ops.BatchDecodeWithPagedKVCacheWrapper(torch.empty(ops.COUNTER_BYTES, dtype=torch.uint8, device="cuda"))
    need = _lib.lib.piekv_decode_first_tokens_workspace_bytes(3, 8, 2, 128)
    if need > ops.COUNTER_BYTES:
        with pytest.raises(ValueError, match="too small"):
            small.plan(tables[1], tables[2], tables[3], 8, 2, 128, 16, window_left=4, first_tokens=1,
                       q_data_type=torch.bfloat16)
