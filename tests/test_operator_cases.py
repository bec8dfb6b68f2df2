"""perf/operators.py: every kind and option of its cases, the calls a user makes
against the plain forms and the float64 results (torch operations, no GPU)."""

import importlib.util
import random
from pathlib import Path

import pytest
import torch

from cyclic_flow_attention import _native
from cyclic_flow_attention.ops import residual, vocab


@pytest.fixture
def operators(monkeypatch):
    path = Path(__file__).resolve().parents[1] / "perf" / "operators.py"
    spec = importlib.util.spec_from_file_location("measured_operators", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "DEV", "cpu")
    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    for ops in (vocab, residual):  # as where torch has to see the calls
        monkeypatch.setattr(ops, "kernel_ok", lambda *tensors: False)
    return module


CASES = ([dict(kind="score", rows=9, vocab=37, top=top, dtype="fp32", masked=masked, train=train)
          for top in (0, 3) for masked in (False, True) for train in (False, True)]
         + [dict(kind="loss", B=2, T=7, vocab=19, dtype="fp32")]
         + [dict(kind="embed", N=15, vocab=11, width=6, dtype="fp32", scale=2.0, pad=pad, train=train)
            for pad in (-1, 2) for train in (False, True)]
         + [dict(kind="join", rows=5, width=12, dtype="fp32", scale=0.5, post=post, gate=gate, train=train)
            for post in (False, True) for gate in (False, True) for train in (False, True)])


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_calls_plain_forms_and_exact_results_agree(operators, case):
    operators.own = False
    plain = operators.run(operators.prepare(case, 3))
    operators.own = True
    state = operators.prepare(case, 3)
    own = operators.run(state)
    exact = operators.exact(case, 3)
    assert len(own) == len(plain) == len(exact) and all(torch.equal(a, b) for a, b in zip(own, operators.run(state)))
    for a, b, e in zip(own, plain, exact):
        assert a.shape == b.shape == e.shape and a.dtype == b.dtype and not a.requires_grad
        if not a.dtype.is_floating_point:
            assert torch.equal(a, b) and torch.equal(a, e)
            continue
        for got in (a, b):  # fp32 sums of at most 37 terms
            assert (got.double() - e).abs().max() <= 2.0**-16 * (1 + e.abs().max())


def test_drawn_cases_are_of_the_listed_kinds(operators):
    listed, rng = operators.listed(), random.Random(5)
    assert len({c["name"] for c in listed}) == len(listed)
    keys = {c["kind"]: set(c) - {"name"} for c in listed}
    for _ in range(50):
        case = operators.draw(rng)
        assert set(case) == keys[case["kind"]] and all(v > 0 for v in operators.work(case).values())
