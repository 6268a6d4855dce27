"""The measured cases as a caller runs them: a state is ready when it is handed out, a pass is complete and checked after
its plan has been finished."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

CASES = [{"kind": "product", "rows": 300, "inner": 200, "outer": 136, "dtype": "f32", "act": "relu"},
         {"kind": "roundtrip", "rows": 500, "inner": 129, "dtype": "f32", "format": "mx8"},
         {"kind": "weights", "rows": 700, "inner": 100, "outer": 72, "dtype": "f32"},
         {"kind": "activation", "rows": 400, "inner": 96, "dtype": "f32", "act": "relu"}]


@pytest.fixture
def operators():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("perf_operators", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("case", CASES, ids=lambda c: c["kind"])
def test_a_finished_pass_is_the_plain_form(operators, case):
    """Without any wait for the device but the plan's own.  The plain form adds in 32 bits like the kernels: both are within
    K 2^-23 of the sum of magnitudes, K at most 700 and the magnitudes at most 100 times the largest result here."""
    operators.own = True
    state = operators.prepare(case, 3)
    for _ in range(3):
        got = operators.run(state)
    state["plan"].finish()
    got = got.clone()
    operators.own = False
    want = operators.run(operators.prepare(case, 3))
    assert got.dtype == want.dtype and got.shape == want.shape
    if case["kind"] in ("roundtrip", "activation"):
        assert torch.equal(got, want)
    else:
        assert (got - want).abs().max() <= 2 * 700 * 2.0 ** -23 * 100 * want.abs().max()
