"""The package without, or with an unfitting, native way into the short calls: every operator works, through Python."""
import importlib.util
import os
import subprocess
import sys
import warnings

import pytest
import torch

from tests.conftest import ROOT
from tests.test_gpu_calls import _append, _axes, _decode_wrapper
from tests.util import dev, make_scenario

PRELUDE = "import sys, types, warnings\nimport torch\n"
USE = """
import pie_b200
from pie_b200 import ops
for name in pie_b200.__all__:
    assert getattr(pie_b200, name) is not None
assert ops.lib.piekv_version() > 0 and ops.device_error is not None
assert len(ops.AxisRopeConfig(mode='plain', sections=(4, 2, 2)).prepared().turn) == 128
print('usable', ops.native_calls_loaded())
"""


def _python(code):
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    return r.returncode, r.stdout, r.stderr


@pytest.mark.parametrize("how", [
    "sys.modules['pie_b200._calls'] = None\n",  # not there, or of another interpreter
    "m = types.ModuleType('pie_b200._calls'); m.torch_version = '1.0'; sys.modules['pie_b200._calls'] = m\n",  # of another torch
])
def test_the_package_loads_without_it_and_says_so(how):
    rc, out, err = _python(PRELUDE + "warnings.simplefilter('always')\n" + how + USE)
    assert rc == 0, err
    assert "usable False" in out and "RuntimeWarning" in err and "pie_b200/build.py" in err


def test_the_package_loads_with_it_without_a_word():
    rc, out, err = _python(PRELUDE + "warnings.simplefilter('error')\n" + USE)
    assert rc == 0, err
    assert "usable True" in out and "pie_b200" not in err


def _build_module():
    spec = importlib.util.spec_from_file_location("_build_under_test", os.path.join(ROOT, "pie_b200", "build.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_it_is_built_again_for_another_torch(monkeypatch):
    build = _build_module()
    monkeypatch.setattr(build, "_stale", lambda target, deps: False)
    assert not build._calls_stale([])
    monkeypatch.setattr(build, "_torch_version", lambda: "9.9.9")
    assert build._calls_stale([])


@pytest.mark.gpu
def test_the_short_calls_give_the_same_through_python(monkeypatch):
    from pie_b200 import ops

    assert ops.native_calls_loaded()
    sc = make_scenario(8, 2, 128, torch.bfloat16, [(c, 1) for c in (3, 200, 77, 1000)])
    chunks = make_scenario(8, 2, 128, torch.bfloat16, [(3, 5), (200, 70)])
    rope = _axes()

    def results():
        out = [_decode_wrapper(sc, kind).run(sc.q.cuda(), sc.pool.cuda()) for kind in ("prefix", "first")]
        m = chunks.meta
        w = ops.BatchPrefillWithPagedKVCacheWrapper(torch.empty(64 << 20, dtype=torch.uint8, device="cuda"))
        w.plan(dev(m.qo_indptr), dev(m.kv_indptr), dev(m.kv_indices), dev(m.kv_last_page_len), 8, 2, 128, 16,
               causal=True, window_left=60, first_tokens=3, q_data_type=torch.bfloat16)
        out += [w.run(chunks.q.cuda(), chunks.pool.cuda()) for _ in range(2)]
        _append(chunks, rope)
        return out + list(_append(chunks, rope))

    native = results()
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")
        monkeypatch.setattr(ops, "_calls", ops._NoCalls())
    assert all(torch.equal(a, b) for a, b in zip(native, results()))
    assert not ops.native_calls_loaded() and ops.device_error("cuda") is None
