"""The cases of ``perf/operators.py`` at small sizes on the CPU: the plain form and the
package's eager path against the file's own float64."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

from perf import operators as cases

#: rounding of the results, and of their inputs' products in the eager path
TOL = {"float32": 1e-5, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def flat(outputs):
    return [outputs] if torch.is_tensor(outputs) else list(outputs)


def check(case, monkeypatch, seed=3):
    if torch.cuda.is_available():
        monkeypatch.setattr(cases, "_device", lambda: torch.device("cpu"))
    want = flat(cases.exact(case, seed))
    state = cases.prepare(case, seed)
    for own in (False, True):
        monkeypatch.setattr(cases, "own", own)
        got = [x.double() for x in flat(cases.run(state))]
        assert len(got) == len(want)
        for i, (x, y) in enumerate(zip(got, want)):
            norm = y.norm().item()
            err = (x - y).norm().item()
            assert err <= 2 * TOL[case["dtype"]] * norm, (own, i, err / norm)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("batch", [1, 2, 3])
@pytest.mark.parametrize("k_len", [1, 40, 240, 300])
def test_a_new_token_on_its_cache(monkeypatch, batch, dtype, k_len):
    """Whatever the batch, the new token stands after its cached ones."""
    check(cases._attention("", dtype, batch, 2, 1, 1, k_len, 16, bidirectional=False, ragged=True,
                           train=False), monkeypatch)


@pytest.mark.parametrize("case", [
    cases._attention("", "float32", 4, 2, 2, 9, 9, 6, grid=(3, 3), windows=2),
    cases._attention("", "float32", 2, 2, 1, 40, 40, 8, causal=True, bidirectional=False),
    cases._attention("", "float16", 3, 2, 2, 33, 33, 8, ragged=True, train=False),
    cases._bias("", "float32", 2, 12, 12, grid=(3, 4)),
    cases._bias("", "float32", 3, 17, 29),
    cases._bias("", "float32", 3, 29, 17, bidirectional=False),
    cases._orthogonalize("", "float32", 2, 20, 9),
    cases._orthogonalize("", "float32", 1, 9, 20, steps=6, polar=True),
], ids=lambda c: f"{c['op']}-{c['dtype']}")
def test_each_form(monkeypatch, case):
    check(case, monkeypatch)


def test_draws_are_of_the_listed_kinds():
    rng = random.Random(5)
    keys = {c["op"]: set(c) - {"name"} for c in cases.listed()}
    drawn = [cases.draw(rng) for _ in range(60)]
    assert all(set(c) == keys[c["op"]] for c in drawn)
    assert any(c["op"] == "attention" and c["q_len"] == 1 and c["batch"] == 1
               for c in (cases.draw(rng) for _ in range(2000)))
    assert np.isfinite([cases.work(c)["flops"] for c in drawn]).all()
