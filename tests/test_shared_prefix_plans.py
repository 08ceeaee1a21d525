"""Whose memory a shared-prefix plan is: what a captured call points to stays as it was built, on the CPU with a stand-in
for the device."""
import weakref

import pytest
import torch

from pie_b200 import _lib, ops


class FakeLib:
    """The library, with the two calls that would launch something recorded instead."""

    def __init__(self):
        self.calls, self.status = [], 0

    def __getattr__(self, name):
        return getattr(_lib.lib, name)

    def _record(self, what, args):
        args = getattr(args, "_obj", args)  # byref() or the struct
        self.calls.append((what, _lib.SharedPrefixArgs.from_buffer_copy(args)))
        return self.status

    def piekv_shared_prefix_plan(self, args, stream):
        return self._record("plan", args)

    def piekv_shared_prefix_run(self, args, stream):
        return self._record("run", args)


@pytest.fixture
def device(monkeypatch):
    fake = FakeLib()
    fake.capturing = False
    word = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(ops, "lib", fake)
    monkeypatch.setattr(ops, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(ops, "_err_word", lambda dev: word)
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: fake.capturing)
    return fake


HQ, HKV, D, PAGE = 8, 2, 128, 16
POOL = torch.zeros((4, 2, PAGE, HKV, D), dtype=torch.bfloat16)


def _wrapper():
    return ops.BatchSharedPrefixDecodeWrapper(torch.empty(8 << 20, dtype=torch.uint8))


def _plan(w, batch, groups=None):
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    w.plan(i32(batch + 1), i32(batch + 1), i32(batch), HQ, HKV, D, PAGE, group_indptr=None if groups is None else i32(groups + 1),
           q_data_type=torch.bfloat16)


def _run(w, batch):
    return w.run(torch.zeros((batch, HQ, D), dtype=torch.bfloat16), POOL)


@pytest.mark.parametrize("what", ["run", "replan", "plan"])
def test_what_was_captured_keeps_its_plan(device, what):
    w = _wrapper()
    if what != "plan":
        _plan(w, 60)
    device.capturing = True
    if what == "plan":
        _plan(w, 60)
    elif what == "replan":
        w.replan()
    if what != "replan":
        _run(w, 60)
    device.capturing = False
    captured = device.calls[-1][1]
    tables = [weakref.ref(t) for t in w._plan["keep"]]
    for batch in (7, 60, 61, 7):
        _plan(w, batch)
        _run(w, batch)
        for _, later in device.calls[-2:]:
            assert later.plan + later.plan_bytes <= captured.plan or captured.plan + captured.plan_bytes <= later.plan
    assert all(t() is not None for t in tables)  # the page table, and the grouping that plan() made itself


def test_plans_that_nothing_captured_share_one_buffer(device):
    w = _wrapper()
    _plan(w, 200)
    for batch in range(1, 60):
        _plan(w, batch)
        _run(w, batch)
    assert len({a.plan for _, a in device.calls}) == 1


def test_a_captured_plan_is_kept_once(device):
    w = _wrapper()
    _plan(w, 20)
    device.capturing = True
    for _ in range(80):  # a layer each
        _run(w, 20)
    device.capturing = False
    first = device.calls[-1][1].plan
    _plan(w, 20)
    _plan(w, 20)
    assert device.calls[-1][1].plan == device.calls[-2][1].plan != first


def test_a_plan_that_was_only_captured_is_built_before_an_eager_run(device):
    w = _wrapper()
    device.capturing = True
    _plan(w, 9)
    _run(w, 9)
    device.capturing = False
    assert [c for c, _ in device.calls] == ["plan", "run"]
    _run(w, 9)  # the buffer holds nothing yet
    _run(w, 9)
    assert [c for c, _ in device.calls] == ["plan", "run", "plan", "run", "run"]
    assert len({a.plan for _, a in device.calls}) == 1


def test_a_plan_that_could_not_be_built_is_none(device):
    w = _wrapper()
    _plan(w, 9)
    device.status = 1
    with pytest.raises(ValueError):
        _plan(w, 5)
    device.status = 0
    for batch in (5, 9):
        with pytest.raises(RuntimeError, match="plan"):
            _run(w, batch)
    _plan(w, 5)
    _run(w, 5)


# ---- into how many pieces a prefix may be cut: as many as the workspace has room for, and not one more
@pytest.mark.parametrize("batch, hq, hkv", [(21, 1, 1), (14, 12, 4), (7, 24, 8), (23, 12, 2), (1, 1, 1), (5, 3, 1), (64, 32, 8)])
def test_a_plan_has_room_for_the_pieces_it_names(device, batch, hq, hkv):
    need = lambda splits: ops.lib.piekv_shared_prefix_workspace_bytes(batch, hq, hkv, D, splits)  # noqa: E731
    most = _lib.SHARED_PREFIX_MAX_SPLITS
    i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
    sizes = {need(1), need(most), need(most) + 12345}
    for splits in range(1, most):
        sizes |= {need(splits + 1) - 1, need(splits + 1), (need(splits) + need(splits + 1)) // 2}
    whole = torch.empty(max(sizes), dtype=torch.uint8)
    w = ops.BatchSharedPrefixDecodeWrapper(whole)
    for have in sorted(sizes):
        w.workspace_buffer = whole[:have]
        w.plan(i32(batch + 1), i32(batch + 1), i32(batch), hq, hkv, D, PAGE, q_data_type=torch.bfloat16)
        splits = device.calls[-1][1].max_splits
        assert need(splits) <= have and (splits == most or have < need(splits + 1)), (have, splits)
    w.workspace_buffer = whole[:need(1) - 1]
    with pytest.raises(ValueError, match="workspace_buffer too small"):
        w.plan(i32(batch + 1), i32(batch + 1), i32(batch), hq, hkv, D, PAGE, q_data_type=torch.bfloat16)


@pytest.mark.gpu
def test_runs_where_the_workspace_holds_its_pieces_exactly():
    lens = [3 + 5 * i for i in range(21)]
    pages = torch.arange(400, dtype=torch.int32, device="cuda")
    pool = torch.randn((400, 2, PAGE, 1, D), device="cuda").to(torch.bfloat16)
    q = torch.randn((21, 1, D), device="cuda").to(torch.bfloat16)
    lists = [list(range(300)) + [300 + i] for i in range(21)]
    indptr = torch.arange(22, dtype=torch.int32, device="cuda") * 301
    indices = pages[torch.tensor(sum(lists, []), device="cuda")]
    last = torch.tensor([(n - 1) % 16 + 1 for n in lens], dtype=torch.int32, device="cuda")
    results = []
    for splits in (1, 2, 3, 33, 52, 63, 64):
        have = _lib.lib.piekv_shared_prefix_workspace_bytes(21, 1, 1, D, splits)
        for extra in (0, 1, 255, 10240):
            w = ops.BatchSharedPrefixDecodeWrapper(torch.empty(have + extra, dtype=torch.uint8, device="cuda"))
            w.plan(indptr, indices, last, 1, 1, D, PAGE, q_data_type=torch.bfloat16)
            results.append(w.run(q, pool))
    plain = ops.BatchDecodeWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
    plain.plan(indptr, indices, last, 1, 1, D, PAGE, q_data_type=torch.bfloat16)
    want = plain.run(q, pool).float()
    # both round P (2^-8 of |v| <= 6 at most, averaged over ~4800 tokens) and the output (half a step of bf16)
    for got in results:
        assert (got.float() - want).abs().max().item() <= 2 * (2 ** -8 * 6 + 2 ** -9)
    assert ops.device_error("cuda") is None


def test_a_buffer_that_became_too_small_stays(device):
    """A run on another stream than the buffer's may still read it."""
    w = ops.BatchSharedPrefixDecodeWrapper(torch.empty(256 << 20, dtype=torch.uint8))
    _plan(w, 3)
    first = weakref.ref(w._plan["buffer"])
    small = device.calls[-1][1]
    for batch in (20000, 100000, 3):
        i32 = lambda n: torch.zeros(n, dtype=torch.int32)  # noqa: E731
        w.plan(i32(batch + 1), i32(batch + 1), i32(batch), 1, 1, D, PAGE, q_data_type=torch.bfloat16)
    assert first() is not None
    for _, a in device.calls[1:]:
        assert a.plan + a.plan_bytes <= small.plan or small.plan + small.plan_bytes <= a.plan
    sizes = {a.plan: a.plan_bytes for _, a in device.calls}
    assert len(sizes) <= 3


def test_the_grouping_that_plan_makes_lives_in_the_plan_buffer(device):
    w = _wrapper()
    for batch in (5, 300, 0):
        _plan(w, batch)
        a, buffer = device.calls[-1][1], w._plan["buffer"]
        assert a.plan + a.plan_bytes <= a.group_indptr <= buffer.data_ptr() + buffer.numel() - 8
        assert w._plan["keep"][3].tolist() == [0, batch] and w._plan["keep"][3].data_ptr() == a.group_indptr
        assert a.plan == buffer.data_ptr() and a.num_groups == 1


@pytest.mark.parametrize("kind", ["prefix", "decode", "prefill"])
def test_a_plan_holds_the_workspace_that_it_names(device, monkeypatch, kind):
    monkeypatch.setattr(ops, "_err_ptr", lambda index: 0)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    ws = torch.empty(32 << 20, dtype=torch.uint8)
    tables = (i32(0, 2), i32(0, 1), i32(4), HQ, HKV, D, PAGE)
    extra = dict(window_left=60, first_tokens=3, q_data_type=torch.bfloat16)
    if kind == "prefix":
        w = ops.BatchSharedPrefixDecodeWrapper(ws)
        w.plan(*tables, q_data_type=torch.bfloat16)
    elif kind == "decode":
        w = ops.BatchDecodeWithPagedKVCacheWrapper(ws)
        w.plan(*tables, **extra)
    else:
        w = ops.BatchPrefillWithPagedKVCacheWrapper(ws)
        w.plan(i32(0, 1), *tables, **extra)
    held = weakref.ref(ws)
    w.workspace_buffer = torch.empty(32 << 20, dtype=torch.uint8)  # for the next plan()
    del ws
    assert held() is not None
