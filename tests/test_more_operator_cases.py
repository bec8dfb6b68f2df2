"""perf/more_operators.py: every kind and option of its cases, the calls a user
makes against the plain forms and the float64 results (torch operations, no GPU)."""

import importlib.util
import random
from pathlib import Path

import pytest
import torch

from cyclic_flow_attention import _native
from cyclic_flow_attention.ops import distill, sampling


@pytest.fixture
def operators(monkeypatch):
    path = Path(__file__).resolve().parents[1] / "perf" / "more_operators.py"
    spec = importlib.util.spec_from_file_location("more_measured_operators", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    monkeypatch.setattr(module, "DEV", "cpu")
    monkeypatch.setattr(_native, "require_device", lambda *tensors: tensors[0].device)
    for ops in (distill, sampling):  # as where torch has to see the calls
        monkeypatch.setattr(ops, "kernel_ok", lambda *tensors: False)
    return module


_ADJUST = dict(B=3, vocab=77, L=20, dtype="fp32")
CASES = ([dict(kind="adjust", T=T, bias=bias, mask=mask, train=train, **_ADJUST)
          for T in (1, 4) for bias in ("", "dense", "tokens") for mask in ("", "bool", "bits") for train in (False, True)]
         + [dict(kind="step", T=1, bias="tokens", mask=mask, train=False, k=k, p=p, **_ADJUST)
            for mask in ("", "bits") for k in (0, 9) for p in (1.0, 0.8)]
         + [dict(kind="sample", rows=9, vocab=65, k=k, p=p, least=least, mixed=mixed, dtype="fp32")
            for k in (0, 7) for p in (1.0, 0.7) for least in (0.0, 0.05) for mixed in (False, True)]
         + [dict(kind="distill", B=2, T=6, vocab=41, k=k, temperature=T, tail=tail, weights=weights, dtype="fp32")
            for k in (1, 5) for T, tail in ((1.0, False), (2.0, False), (1.0, True)) for weights in (False, True)])


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
        assert a.shape == b.shape and a.dtype == b.dtype and not a.requires_grad
        if e is None:  # a token drawn from logits that differ by an fp32 rounding here and there
            e = b.double() if b.dtype.is_floating_point else b
        assert a.shape == e.shape
        if not a.dtype.is_floating_point:
            assert torch.equal(a, b) and torch.equal(a, e)
            continue
        for got in (a, b):  # fp32 sums of at most 77 terms
            fine = e.isfinite()
            assert torch.equal(got[~fine].double(), e[~fine])
            assert (got[fine].double() - e[fine]).abs().max() <= 2.0**-16 * (1 + e[fine].abs().max())


def test_drawn_cases_are_of_the_listed_kinds(operators):
    listed, rng = operators.listed(), random.Random(5)
    assert len({c["name"] for c in listed}) == len(listed)
    keys = {c["kind"]: set(c) - {"name"} for c in listed}
    for _ in range(50):
        case = operators.draw(rng)
        assert set(case) == keys[case["kind"]] and all(v > 0 for v in operators.work(case).values())
