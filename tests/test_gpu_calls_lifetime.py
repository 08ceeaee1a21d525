"""What a call points to while another thread changes its configuration, and that the native way takes ordinary calls."""
import gc
import weakref

import pytest
import torch

from pie_b200 import _calls, _lib, ops
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


def test_a_table_laid_out_while_the_configuration_changes_is_not_kept(monkeypatch):
    rope, changed = _axes(), _axes(theta=10000.0)

    class Lib:
        """The library, with another thread's assignment while a table is laid out."""

        def __getattr__(self, name):
            return getattr(_lib.lib, name)

        def piekv_rope_axes_prepare(self, *args):
            status = _lib.lib.piekv_rope_axes_prepare(*args)
            rope.theta = 10000.0
            return status

    with monkeypatch.context() as m:
        m.setattr(ops, "lib", Lib())
        rope.prepared()
    assert list(rope.prepared().turn) == list(changed.prepared().turn)


def test_an_assignment_is_seen_whatever_reads_in_the_middle_of_it(monkeypatch):
    rope, changed = _axes(), _axes(sections=(24, 20, 20))
    rope.prepared()

    class Sections(list):
        """Another thread's call between an assignment's steps: the new value is converted in the middle."""

        def __iter__(self):
            rope.prepared()
            return super().__iter__()

    rope.sections = Sections((24, 20, 20))
    assert list(rope.prepared().axis) == list(changed.prepared().axis)
    seen = []

    class Calls:
        rope_axes_append = staticmethod(lambda table, *rest: seen.append(list(table.axis)))

    monkeypatch.setattr(ops, "_calls", Calls)
    ops.rope_axes_append_paged_kv_cache(*[None] * 10, rope)
    assert seen == [list(changed.prepared().axis)]


def test_a_cos_sin_table_whose_storage_was_replaced_is_looked_at_again(monkeypatch):
    monkeypatch.setattr(ops, "_require_cuda", lambda t, name: None)
    values = torch.zeros(100, 128)
    rope = _axes(mode="table", cos_sin_table=values)
    first = rope.prepared()
    assert first.table_len == 100 and first.cos_sin_table == values.data_ptr() and rope.prepared() is first
    values.data = torch.zeros(10, 128)
    assert rope.prepared().table_len == 10 and rope.prepared().cos_sin_table == values.data_ptr()
