"""What a call points to while another thread changes its configuration, and that the native way takes ordinary calls."""
import gc
import weakref

import pytest
import torch

from pie_b200 import _calls, ops
from tests.test_gpu_calls import _append, _axes
from tests.util import make_scenario


def test_a_table_outlives_a_change_of_its_configuration(monkeypatch):
    rope = _axes()
    table = weakref.ref(rope.prepared())
    alive = []

    class Calls:
        @staticmethod
        def rope_axes_append(*args):
            rope.theta = 10000.0  # as another thread may at any moment: the configuration drops its table
            gc.collect()
            alive.append(table() is not None)

    monkeypatch.setattr(ops, "_calls", Calls)
    ops.rope_axes_append_paged_kv_cache(*[None] * 10, rope)
    assert alive == [True] and rope.__dict__["_table"] is None


def test_a_table_is_taken_as_an_object_only():
    table = _axes().prepared()
    t, i = torch.zeros(2, 2, 8), torch.zeros(2, dtype=torch.int32)
    rest = (t, t, t, i.view(1, 2), i, i, torch.zeros(1, 2, 16, 2, 8), i, i, None)
    for given in (table, bytes(table), b"short", 1, None):
        assert _calls.rope_axes_append(given, *rest) is False


@pytest.mark.gpu
def test_the_native_append_takes_an_ordinary_call():
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(20, 3), (4, 2)])
    rope = _axes()
    want, pool = _append(sc, rope)
    called = []
    native = _calls.rope_axes_append

    class Calls:
        @staticmethod
        def rope_axes_append(table, *rest):
            called.append(native(table, *rest))
            return called[-1]

    saved, ops._calls = ops._calls, Calls
    try:
        got, got_pool = _append(sc, rope)
    finally:
        ops._calls = saved
    assert called[0] is got and torch.equal(got, want) and torch.equal(got_pool, pool)
