"""Decode attention for groups of requests whose page lists start with the same pages."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from pie_b200 import _lib, ops, pages
from pie_b200 import workloads as W
from tests import plain64 as P
from tests.util import dev


def _workspace(mib=128):
    return torch.empty(mib << 20, dtype=torch.uint8, device="cuda")


class Batch:
    """Groups given as (shared full pages, [tokens of each request behind them]); seeded pool, NaN in stale rows."""

    def __init__(self, groups, hq, hkv, d=128, dtype=torch.bfloat16, page_size=16, seed=0, spare=5):
        self.hq, self.hkv, self.d, self.dtype, self.page_size = hq, hkv, d, dtype, page_size
        need = sum(s + sum(-(-t // page_size) for t in tails) for s, tails in groups) + spare
        deck = list(W.seeded_perm(need, seed))
        self.lists, self.lens, ends = [], [], [0]
        for shared, tails in groups:
            head = [deck.pop() for _ in range(shared)]
            for t in tails:
                self.lists.append(head + [deck.pop() for _ in range(-(-t // page_size))])
                self.lens.append(shared * page_size + t)
            ends.append(ends[-1] + len(tails))
        self.ends = np.array(ends, dtype=np.int32)
        self.pool = W.randn((need, 2, page_size, hkv, d), seed + 1, dtype)
        self.q = W.randn((len(self.lists), hq, d), seed + 2, dtype)
        for pages_, n in zip(self.lists, self.lens):
            if n % page_size:
                self.pool[pages_[-1], :, n % page_size:] = math.nan
        self.tables()

    def tables(self):
        self.indptr = np.cumsum([0] + [len(x) for x in self.lists]).astype(np.int32)
        self.indices = np.array([p for x in self.lists for p in x] + [0], dtype=np.int32)
        self.last = np.array([(n - 1) % self.page_size + 1 if n else 0 for n in self.lens], dtype=np.int32)

    def plan(self, w, groups="own", **kw):
        ends = dev(self.ends) if isinstance(groups, str) else groups
        w.plan(dev(self.indptr), dev(self.indices), dev(self.last), self.hq, self.hkv, self.d, self.page_size,
               group_indptr=ends, q_data_type=self.dtype, **kw)
        return w

    def reference(self, **kw):
        return P.attend(self.q, self.pool, np.arange(len(self.lens) + 1), self.indptr, self.indices, self.last, **kw)

    def check(self, got, **kw):
        P.check_attention(got[0], got[1], self.q, self.pool, self.reference(**kw), scale=kw.get("sm_scale"))


def _run(b, **kw):
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()))
    return w.run(b.q.cuda(), b.pool.cuda(), return_lse=True, **kw)


# ---- on the CPU: refusals
def _args(**kw):
    a = _lib.SharedPrefixArgs()
    for name, value in {**dict(kv_indptr=256, kv_indices=256, kv_last_page_len=256, group_indptr=256, plan=256,
                               plan_bytes=1 << 30, workspace=256, workspace_bytes=1 << 30, batch=4, num_groups=1,
                               num_qo_heads=8, num_kv_heads=2, head_dim=128, page_size=16, num_pages=8, dtype=2,
                               max_splits=4, q=256, pool=256, out=256, q_stride_n=1024, q_stride_h=128,
                               sm_scale=0.1), **kw}.items():
        setattr(a, name, value)
    return a


@pytest.mark.parametrize("kw, text", [
    (dict(dtype=5), b"dtype"), (dict(batch=-1), b"negative"), (dict(num_qo_heads=7), b"multiple"), (dict(head_dim=0), b"head_dim"),
    (dict(max_splits=0), b"max_splits"), (dict(max_splits=65), b"max_splits"), (dict(num_groups=0), b"groups"),
    (dict(group_indptr=None), b"null"), (dict(kv_indices=None), b"null"), (dict(plan=None), b"plan"),
    (dict(plan_bytes=8), b"plan too small"), (dict(plan=264), b"aligned"),
])
def test_plan_and_run_refuse_on_the_host(kw, text):
    L = _lib.lib
    for call in (L.piekv_shared_prefix_plan, L.piekv_shared_prefix_run):
        assert call(C.byref(_args(**kw)), None) > 0 and text in L.piekv_last_error_string()


def test_run_refuses_on_the_host():
    L = _lib.lib
    for kw, text in ((dict(q=None), b"null"), (dict(num_pages=0), b"num_pages"), (dict(out=None), b"null")):
        assert L.piekv_shared_prefix_run(C.byref(_args(**kw)), None) > 0 and text in L.piekv_last_error_string()
    assert L.piekv_shared_prefix_run(None, None) > 0
    assert L.piekv_shared_prefix_plan(C.byref(_args(batch=0)), None) == 0
    assert L.piekv_shared_prefix_run(C.byref(_args(batch=0)), None) == 0
    assert L.piekv_shared_prefix_plan_bytes(-1, 1, 8, 2) == 0 and L.piekv_shared_prefix_workspace_bytes(4, 8, 2, 128, 0) == 0
    assert L.piekv_shared_prefix_workspace_bytes(4, 8, 2, 128, 1) >= ops.COUNTER_BYTES


def test_run_before_plan_and_cpu_tensors():
    with pytest.raises(ValueError, match="CUDA"):
        ops.BatchSharedPrefixDecodeWrapper(torch.zeros(1 << 20, dtype=torch.uint8))
    w = ops.BatchSharedPrefixDecodeWrapper.__new__(ops.BatchSharedPrefixDecodeWrapper)
    w._plan = None
    for call in (w.replan, lambda: w.run(None, None)):
        with pytest.raises(RuntimeError, match="plan"):
            call()


# ---- on the GPU
HEADS = [(32, 8), (8, 8), (4, 1), (6, 2), (40, 8), (16, 1), (16, 2), (9, 3), (12, 12), (20, 10)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, hkv", HEADS)
def test_groups_of_every_kind(dtype, hq, hkv):
    b = Batch([(70, [1, 16, 17, 40]),            # a prefix that ends inside a 128-token tile
               (16, [200, 5, 31]),               # one that ends with it
               (0, [3, 300]),                    # nothing shared
               (33, [77]),                       # alone
               (100, [0, 0, 1, 0, 64]),          # requests that hold the prefix only
               (1, [1, 2]),                      # one page
               (12, [10] * 9)], hq, hkv, dtype=dtype, seed=hq)
    got = _run(b)
    assert ops.device_error("cuda") is None
    b.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("members, hq, hkv", [(1, 32, 8), (2, 8, 2), (31, 32, 8), (32, 32, 8), (33, 32, 8), (64, 32, 8),
                                              (65, 32, 8), (100, 16, 1), (128, 16, 2), (300, 4, 1), (257, 3, 3)])
def test_row_tiles(members, hq, hkv):
    """Query rows of a group (requests x heads of a kv head) below, at and above the 128-row tiles."""
    b = Batch([(40, [(5 * i) % 37 for i in range(members)])], hq, hkv, seed=members)
    got = _run(b)
    assert ops.device_error("cuda") is None
    b.check(got)


@pytest.mark.gpu
@pytest.mark.parametrize("shared, tails, hq, hkv", [(1000, [9, 700, 1], 32, 8), (2500, [3, 4], 4, 1), (640, [5000, 2, 4000], 16, 4),
                                                    (300, [100] * 70, 8, 2)])
def test_long_prefixes_and_long_tails(shared, tails, hq, hkv):
    b = Batch([(shared, tails)], hq, hkv, seed=3)
    b.check(_run(b))


@pytest.mark.gpu
@pytest.mark.parametrize("batch_groups", [400, 700])
def test_many_groups(batch_groups):
    b = Batch([(9 + i % 5, [1 + (i + j) % 40 for j in range(1 + i % 4)]) for i in range(batch_groups)], 4, 2, seed=1)
    b.check(_run(b))


@pytest.mark.gpu
@pytest.mark.parametrize("d, page_size, dtype, hq, hkv", [(64, 16, torch.bfloat16, 8, 2), (128, 16, torch.float32, 8, 2),
                                                          (128, 8, torch.float16, 8, 2), (256, 16, torch.bfloat16, 4, 2),
                                                          (128, 16, torch.bfloat16, 24, 1), (20, 3, torch.float32, 6, 3)])
def test_shapes_of_the_general_kernel(d, page_size, dtype, hq, hkv):
    b = Batch([(20, [1, 30]), (0, [7]), (11, [40, 0, 2])], hq, hkv, d=d, dtype=dtype, page_size=page_size)
    b.check(_run(b))


@pytest.mark.gpu
def test_any_grouping_gives_the_ordinary_result():
    """What is shared is found from the page lists: a wrong or missing grouping changes nothing but the speed."""
    b = Batch([(70, [1, 16, 40]), (50, [9, 8]), (0, [30, 20])], 16, 4, seed=5)
    q, pool = b.q.cuda(), b.pool.cuda()
    for ends in (None, np.array([0, 7]), np.array([0, 2, 3, 7]), np.array([0, 1, 2, 3, 4, 5, 6, 7]), np.array([0, 0, 3, 3, 5, 7, 7])):
        w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()),
                   groups=None if ends is None else dev(ends.astype(np.int32)))
        b.check(w.run(q, pool, return_lse=True))
    assert ops.device_error("cuda") is None
    for ends in ([1, 3, 7], [0, 3, 6], [0, 5, 3, 7], [0, 3, 8], [-4, 3, 7]):  # not a grouping of the batch: said, and nothing shared
        ops.device_error("cuda")
        w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()), groups=dev(np.array(ends, dtype=np.int32)))
        got = w.run(q, pool, return_lse=True)
        assert ops.device_error("cuda")["code"] == 7
        b.check(got)


@pytest.mark.gpu
def test_lists_that_part_early_and_empty_requests():
    b = Batch([(64, [20, 30, 40]), (40, [5, 6])], 8, 2, seed=6)
    b.lists[1][37] = b.lists[2][-2]       # the second request leaves the first's pages at page 37 (a full page)
    b.lists[4] = []                       # a request without pages in a group
    b.lens[4] = 0
    b.tables()
    got = _run(b)
    b.check(got)
    assert (got[0][4] == 0).all() and torch.isinf(got[1][4]).all()
    empty = Batch([(0, [0, 0])], 8, 2)
    out, lse = _run(empty)
    assert (out == 0).all() and torch.isinf(lse).all()


@pytest.mark.gpu
def test_sinks_scale_strides_and_out():
    b = Batch([(30, [10, 20, 30]), (5, [1])], 8, 2, seed=7)
    g = torch.Generator().manual_seed(1)
    sinks = torch.randn(8, generator=g) * 3
    wide = torch.randn((4, 8, 2, 128), generator=g).to(torch.bfloat16)
    b.q = wide[:, :, 1]
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()), sm_scale=0.2)
    out = torch.empty((4, 8, 128), dtype=torch.bfloat16, device="cuda")
    q = wide.cuda()[:, :, 1]
    got = w.run(q, b.pool.cuda(), out=out, return_lse=True, sinks=sinks.cuda())
    assert got[0] is out
    b.check(got, sinks=sinks, sm_scale=0.2)
    b.check(w.run(q, b.pool.cuda(), return_lse=True, sm_scale=0.05), sm_scale=0.05)
    same = b.q[:1].cuda().expand(4, 8, 128)  # one row for all requests: stride 0
    b2, b.q = b.q, same.cpu()
    b.check(w.run(same, b.pool.cuda(), return_lse=True), sm_scale=0.2)
    b.q = b2
    odd = torch.empty(4 * 8 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(4, 8, 128)  # 2-byte aligned rows
    odd.copy_(q)
    b.check(w.run(odd, b.pool.cuda(), return_lse=True), sm_scale=0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-30])
def test_scales_that_are_not_positive(scale):
    b = Batch([(30, [5, 40, 0]), (0, [9])], 8, 2)
    got = _run(b, sm_scale=scale)
    P.check_attention(got[0], got[1], b.q, b.pool, b.reference(sm_scale=scale), scale=abs(scale))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq, hkv", [(32, 8), (8, 1), (6, 2), (5, 1), (16, 1), (4, 4), (14, 2), (3, 1)])
def test_few_rows_behind_long_prefixes(dtype, hq, hkv):
    """Groups whose rows fill a quarter of a tile or less, and one more than that; prefixes that end inside a quarter."""
    full = 32 // (hq // hkv)
    b = Batch([(32, [3, 40]), (33, [1] * full), (130, [5, 0, 70]), (67, [2] * (full + 1)), (300, [1, 2, 3, 4]), (40, [9])],
              hq, hkv, dtype=dtype, seed=hq)
    got = _run(b)
    assert ops.device_error("cuda") is None
    b.check(got)
    again = _run(b)
    assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


@pytest.mark.gpu
def test_nan_behind_few_rows_comes_out():
    b = Batch([(80, [5, 20, 3]), (64, [1, 9])], 8, 2)
    for page, part in ((int(b.lists[0][37]), 0), (int(b.lists[0][70]), 1)):
        pool = b.pool.clone()
        pool[page, part, 3, 1, 11] = float("nan")
        w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()))
        got = w.run(b.q.cuda(), pool.cuda()).cpu().float()
        bad = torch.isnan(got)
        assert bool(bad[:3, 4:, 11].all()) and not bool(bad[3:].any()) and not bool(bad[:3, :4].any())


@pytest.mark.gpu
def test_large_scores_and_peaked_rows():
    """Scores in the hundreds: the join of prefix and suffix must not overflow, whichever part holds the maximum."""
    b = Batch([(40, [20, 50, 0])], 8, 2, seed=8)
    b.pool[b.lists[0][3], 0] *= 30
    b.pool[b.lists[1][-1], 0, :2] *= 60
    b.check(_run(b))


@pytest.mark.gpu
def test_graph_with_plan_and_layers_while_tables_change():
    b = Batch([(50, [9, 30, 2]), (20, [40, 40])], 16, 4, seed=9, spare=200)
    indptr, last, ends = dev(b.indptr), dev(b.last), dev(b.ends)
    indices = torch.zeros(2000, dtype=torch.int32, device="cuda")
    indices[: len(b.indices)] = dev(b.indices)
    pools = [b.pool.cuda(), (b.pool * 0.5).cuda()]
    q = b.q.cuda()
    outs = [torch.empty_like(q) for _ in pools]
    w = ops.BatchSharedPrefixDecodeWrapper(_workspace())
    other = ops.BatchDecodeWithPagedKVCacheWrapper(w.workspace_buffer)  # shares the workspace
    w.plan(indptr, indices, last, 16, 4, 128, 16, group_indptr=ends, q_data_type=torch.bfloat16)
    other.plan(indptr, indices, last, 16, 4, 128, 16, q_data_type=torch.bfloat16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        w.replan()
        for pool, out in zip(pools, outs):
            w.run(q, pool, out=out)
            other.run(q, pool)

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    b.check((outs[0], None))
    for seed, groups in enumerate(([(50, [9, 30, 2]), (20, [40, 40])], [(3, [200, 100]), (60, [1, 2, 3])], [(0, [1] * 5)])):
        n = Batch(groups, 16, 4, seed=9)
        n.pool, n.q = b.pool, b.q
        n.pool = torch.nan_to_num(n.pool)
        pools[0].copy_(n.pool)
        pools[1].copy_(n.pool * 0.5)
        indptr.copy_(dev(n.indptr))
        indices[: len(n.indices)] = dev(n.indices)
        last.copy_(dev(n.last))
        if len(n.ends) == 3:
            ends.copy_(dev(n.ends))
        else:
            ends.copy_(dev(np.array([0, 2, 5], dtype=np.int32)))
        for out in outs:
            out.fill_(9.0)
        graph.replay()
        graph.replay()
        assert ops.device_error("cuda") is None
        n.check((outs[0], None))
        half = n.pool
        n.pool = half * 0.5
        n.check((outs[1], None))
        n.pool = half
    assert not w.workspace_buffer[: ops.COUNTER_BYTES].any()


@pytest.mark.gpu
def test_reproducible_and_two_streams_with_workspaces_of_their_own():
    b = Batch([(200, [100 + 7 * i for i in range(20)])], 32, 8, seed=10)
    q, pool = b.q.cuda(), b.pool.cuda()
    ws = [b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace())) for _ in range(2)]
    first = ws[0].run(q, pool)
    streams = [torch.cuda.Stream() for _ in ws]
    torch.cuda.synchronize()
    results = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            results.append(ws[i % 2].run(q, pool))
    torch.cuda.synchronize()
    assert all(torch.equal(first, r) for r in results)


@pytest.mark.gpu
def test_small_workspaces():
    b = Batch([(400, [10, 20])], 8, 2, seed=11)
    need = _lib.lib.piekv_shared_prefix_workspace_bytes(2, 8, 2, 128, 1)
    tight = torch.empty(need, dtype=torch.uint8, device="cuda")
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(tight))
    b.check(w.run(b.q.cuda(), b.pool.cuda(), return_lse=True))
    if need > ops.COUNTER_BYTES:
        with pytest.raises(ValueError, match="too small"):
            b.plan(ops.BatchSharedPrefixDecodeWrapper(tight[:-256]))


@pytest.mark.gpu
@pytest.mark.parametrize("splits", [1, 2, 4, 6, 9])
def test_workspaces_with_room_for_few_pieces(splits):
    b = Batch([(260, [10] * 70), (150, [5, 6]), (90, [33] * 40), (0, [40, 2])], 8, 2, seed=13)
    n = len(b.lens)
    need = _lib.lib.piekv_shared_prefix_workspace_bytes(n, 8, 2, 128, splits)
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(torch.empty(need, dtype=torch.uint8, device="cuda")))
    b.check(w.run(b.q.cuda(), b.pool.cuda(), return_lse=True))
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    """Group counts, lengths and head counts at random: wherever the shares of the prefixes' tiles happen to be cut."""
    rng = np.random.default_rng(seed)
    hkv = int(rng.choice([1, 2, 3, 4, 8]))
    hq = hkv * int(rng.choice([1, 2, 3, 4, 7, 8, 12]))
    groups = []
    for _ in range(int(rng.integers(1, 12))):
        members = int(rng.integers(1, 40 if rng.random() < 0.3 else 6))
        groups.append((int(rng.integers(0, 220)), [int(x) for x in rng.integers(0, 90, members)]))
    b = Batch(groups, hq, hkv, dtype=torch.float16 if seed % 2 else torch.bfloat16, seed=seed)
    b.check(_run(b))
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
def test_no_requests_and_nan_in_sight():
    b = Batch([(0, [])], 8, 2)
    w = b.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()))
    out, lse = w.run(b.q.cuda(), b.pool.cuda(), return_lse=True)
    assert out.shape == (0, 8, 128) and lse.shape == (0, 8)
    # NaN that a request does see comes out, whichever part it is in and however the parts are cut, and only there
    b = Batch([(300, [700, 20, 30]), (300, [3, 4])], 8, 2, seed=14)
    clean = _run(b)[0]
    b.pool[b.lists[1][-1], 0, 1] = math.nan       # own page of request 1
    b.pool[b.lists[3][200], 0, 2, 1] = math.nan   # shared page of requests 3 and 4, kv head 1
    out = _run(b)[0]
    assert torch.isnan(out[1]).all() and torch.isnan(out[3:, 4:]).all()
    assert torch.equal(out[0], clean[0]) and torch.equal(out[2], clean[2]) and torch.equal(out[3:, :4], clean[3:, :4])


@pytest.mark.gpu
def test_bad_page_ids_are_reported():
    b = Batch([(30, [10, 20])], 8, 2, seed=12)
    for x in b.lists:
        x[4] = 10 ** 6
    b.tables()
    ops.device_error("cuda")
    _run(b)
    assert ops.device_error("cuda")["code"] == 3
    b = Batch([(30, [10, 20])], 8, 2, seed=12)
    b.lists[0][-1] = -1
    b.tables()
    _run(b)
    assert ops.device_error("cuda")["code"] == 3


@pytest.mark.gpu
def test_refusals_on_the_device():
    b = Batch([(3, [10, 20])], 8, 2)
    w = ops.BatchSharedPrefixDecodeWrapper(_workspace())
    with pytest.raises(ValueError, match="window"):
        b.plan(w, window_left=4)
    b.hkv = 0
    with pytest.raises(ValueError, match="multiple"):
        b.plan(w)
    b.hkv = 2
    with pytest.raises(ValueError, match="group_indptr"):
        b.plan(w, groups=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="int32"):
        b.plan(w, groups=torch.zeros(2, device="cuda"))
    b.plan(w)
    q, pool = b.q.cuda(), b.pool.cuda()
    with pytest.raises(ValueError, match="plan"):
        w.run(q[:1], pool)
    with pytest.raises(ValueError, match="planned"):
        w.run(q.half(), pool.half())
    with pytest.raises(ValueError, match="cache"):
        w.run(q, pool[:, :, :8].contiguous())
    with pytest.raises(ValueError, match="sinks"):
        w.run(q, pool, sinks=torch.zeros(3, device="cuda"))
    with pytest.raises(ValueError, match="out"):
        w.run(q, pool, out=torch.empty((2, 8, 128), device="cuda"))


@pytest.mark.gpu
def test_forked_contexts_from_the_device_page_table():
    """The path a beam search takes: a context written with positions on three axes, forked on the device, every beam
    grown by a token of its own, then one shared-prefix decode over the table's own output; the same batch through a
    window with first tokens."""
    hq, hkv, d, beams = 8, 2, 128, 4
    table = pages.DevicePageTable(num_pages=64, max_requests=8, pages_per_request=32)
    pool = torch.zeros((64, 2, 16, hkv, d), dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    rope = ops.AxisRopeConfig(sections=(16, 24, 24), mode="plain", theta=10000.0, scale=1.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731

    def append(meta, n_new):
        ptr, idx, last = meta
        b = len(n_new)
        qo = i32([0] + list(np.cumsum(n_new)))
        n = sum(n_new)
        lens = ops.get_seq_lens(ptr, last, 16)
        bi, slots = ops.get_batch_indices_positions(qo, lens, n)
        q, k, v = rnd(n, hq, d), rnd(n, hkv, d), rnd(n, hkv, d)
        pos = torch.stack([slots, slots // 3, slots % 7]).contiguous()
        return ops.rope_axes_append_paged_kv_cache(q, k, v, pos, bi, slots, pool, idx, ptr, last, rope), b

    prompt = 300
    append(table.grow(i32([0]), prompt)[:3], [prompt])
    for child in range(1, beams):
        src, dst, valid = table.fork(i32([0]), i32([child]))
        ops.copy_kv_pages(pool, src, dst, valid)
    for _ in range(20):
        m = table.grow(i32(list(range(beams))), 1)
        q, _ = append(m[:3], [1] * beams)
    indptr, kv_indices, last, _ = m
    w = ops.BatchSharedPrefixDecodeWrapper(_workspace())
    w.plan(indptr, kv_indices, last, hq, hkv, d, 16, q_data_type=torch.bfloat16)
    got = w.run(q, pool, return_lse=True)
    n_pages = int(indptr[-1])
    args = (q.cpu(), pool.cpu(), np.arange(beams + 1), indptr.cpu().numpy(), kv_indices[:n_pages].cpu().numpy(),
            last.cpu().numpy())
    P.check_attention(got[0], got[1], args[0], args[1], P.attend(*args))
    plain = ops.BatchDecodeWithPagedKVCacheWrapper(_workspace())
    plain.plan(indptr, kv_indices, last, hq, hkv, d, 16, window_left=63, first_tokens=4, q_data_type=torch.bfloat16)
    got = plain.run(q, pool, return_lse=True)
    P.check_attention(got[0], got[1], args[0], args[1], P.attend(*args, window_left=63, first_tokens=4))
    assert ops.device_error("cuda") is None


@pytest.mark.gpu
def test_captured_runs_outlive_later_plans_of_other_batches():
    first = Batch([(60, [9, 30, 2, 5] * 8)], 16, 4, seed=21)
    others = [Batch([(20, [4, 40])], 8, 2, seed=22), Batch([(70, [3] * 64)], 32, 8, seed=23), first]
    w = first.plan(ops.BatchSharedPrefixDecodeWrapper(_workspace()), groups=None)  # (a grouping that plan() makes itself)
    q, pool = first.q.cuda(), first.pool.cuda()
    out = torch.empty_like(q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.replan()
        w.run(q, pool, out=out)
    layer = torch.cuda.CUDAGraph()
    with torch.cuda.graph(layer):
        again = w.run(q, pool)
    for b in others:
        b.plan(w)
        b.check(w.run(b.q.cuda(), b.pool.cuda(), return_lse=True))
        for g, result in ((layer, again), (graph, out)):
            result.fill_(9.0)
            g.replay()
            assert ops.device_error("cuda") is None
            first.check((result, None))


@pytest.mark.gpu
def test_a_plan_that_was_only_captured_runs_eagerly_too():
    b = Batch([(60, [9, 30, 2]), (5, [1, 2])], 16, 4, seed=24)
    w = ops.BatchSharedPrefixDecodeWrapper(_workspace())
    tables = [dev(x) for x in (b.indptr, b.indices, b.last)]
    ends, q, pool = dev(b.ends), b.q.cuda(), b.pool.cuda()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.plan(*tables, 16, 4, 128, 16, group_indptr=ends, q_data_type=torch.bfloat16)
        captured = w.run(q, pool)
    b.check(w.run(q, pool, return_lse=True))
    graph.replay()
    b.check((captured, None))
    b.check((w.run(q, pool), None))
    assert ops.device_error("cuda") is None
