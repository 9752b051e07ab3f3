"""The measured cases' library form follows torch's current stream, and that stream follows it."""
import importlib.util
import os
import sys

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["rope_step", "cache_step", "attend_few"])
def test_the_library_form_is_ordered_with_torch(name):
    import torch
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("measured_cases", path)
    cases = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = cases
    spec.loader.exec_module(cases)
    case = next(c for c in cases.listed() if c["name"] == name)
    before = torch.cuda.current_stream()
    inputs = {"rope": ["x"], "cache": ["k", "v"], "attend": ["q"]}[case["op"]]
    slow = torch.zeros(1 << 28, device="cuda")
    try:
        cases.own = True
        side = torch.cuda.Stream()
        for stream in (None, side):  # as prepare() leaves it, and under a stream of the program's own
            state = cases.prepare(case, 1)
            codes = {n: state[n].clone() for n in state if n.endswith(("_codes", "_scale"))}
            torch.cuda.synchronize()
            want = cases.run(state)
            torch.cuda.synchronize()
            want = [w.clone() for w in (want if isinstance(want, tuple) else [want])]
            for n in codes:
                state[n].copy_(codes[n])
            source = {n: state[n].clone() for n in inputs}
            for n in inputs:
                state[n].zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                slow.add_(1.0)
                for n in inputs:
                    state[n].copy_(source[n])
                got = cases.run(state)
                got = [g.clone() for g in (got if isinstance(got, tuple) else [got])]
            torch.cuda.synchronize()
            assert all(torch.equal(g, w) for g, w in zip(got, want))
    finally:
        cases.own = False
        torch.cuda.set_stream(before)
