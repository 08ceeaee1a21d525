"""A prefill plan that was only captured is not there yet for an eager run; on the CPU with a stand-in for the device."""
import pytest
import torch

from pie_b200 import _lib, ops


class FakeLib:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        return getattr(_lib.lib, name)

    def piekv_prefill_plan_opt(self, *args):
        self.calls.append("plan")
        return 0

    def piekv_prefill_run_opt(self, *args):
        self.calls.append("run")
        return 0


@pytest.fixture
def device(monkeypatch):
    fake = FakeLib()
    fake.capturing = False
    word = torch.zeros(4, dtype=torch.int32)
    monkeypatch.setattr(ops, "lib", fake)
    monkeypatch.setattr(ops, "_require_cuda", lambda t, name: None)
    monkeypatch.setattr(ops, "_err_word", lambda dev: word)
    monkeypatch.setattr(ops, "_err_ptr", lambda index: word.data_ptr())
    monkeypatch.setattr(ops, "_stream", lambda dev: 0)
    monkeypatch.setattr(ops, "_stream_of", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: fake.capturing)
    return fake


@pytest.mark.parametrize("extra", [dict(), dict(window_left=60, first_tokens=3)])
def test_a_plan_that_was_only_captured_is_built_before_an_eager_run(device, extra):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pool, q = torch.zeros((4, 2, 16, 2, 128), dtype=torch.bfloat16), torch.zeros((20, 8, 128), dtype=torch.bfloat16)
    w = ops.BatchPrefillWithPagedKVCacheWrapper(torch.empty(32 << 20, dtype=torch.uint8))
    w.plan(i32(0, 20), i32(0, 2), i32(0, 1), i32(4), 8, 2, 128, 16, causal=True, q_data_type=torch.bfloat16, **extra)
    device.capturing = True
    w.run(q, pool)
    w.run(q, pool)  # the next layer of the same graph
    assert device.calls == ["plan", "run", "run"]
    device.capturing = False
    w.run(q, pool)
    w.run(q, pool)
    assert device.calls[3:] == ["plan", "run", "run"]
    device.capturing = True
    w.run(q, pool)  # built: a graph may point to it
    assert device.calls[6:] == ["run"]


@pytest.mark.parametrize("extra", [dict(), dict(window_left=60, first_tokens=3)])
def test_work_list_and_run_use_the_workspace_of_the_plan(device, monkeypatch, extra):
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    pool, q = torch.zeros((4, 2, 16, 2, 128), dtype=torch.bfloat16), torch.zeros((20, 8, 128), dtype=torch.bfloat16)
    named = []
    monkeypatch.setattr(FakeLib, "piekv_prefill_plan_opt", lambda self, *args: named.append(args[-4]) or 0)
    monkeypatch.setattr(FakeLib, "piekv_prefill_run_opt", lambda self, *args: named.append(args[-5]) or 0)
    first, second = (torch.empty(32 << 20, dtype=torch.uint8) for _ in range(2))
    w = ops.BatchPrefillWithPagedKVCacheWrapper(first)
    tables = (i32(0, 20), i32(0, 2), i32(0, 1), i32(4), 8, 2, 128, 16)
    w.plan(*tables, causal=True, q_data_type=torch.bfloat16, **extra)
    w.run(q, pool)
    w.workspace_buffer = second
    w.run(q, pool)
    w.run(q, torch.cat([pool, pool]))
    assert set(named) == {first.data_ptr()} and len(named) == 5
    w.plan(*tables, causal=True, q_data_type=torch.bfloat16, **extra)
    w.run(q, pool)
    assert set(named[5:]) == {second.data_ptr()} and len(named) == 7
