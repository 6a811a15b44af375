"""The timed cases of perf/operators.py: what they list and draw, and on the GPU that a pass
through the kernels and one of the plain form give the operator's answer.

Tolerance, of the norm of the difference from the 64-bit answer: the rounding of the output
(2^-9 relative in bfloat16, 2^-12 in float16, at most and mean-free), and for attention that
of the probabilities, of the same size and independent of one another: twice that together.
"""
import random

import pytest
import torch

from perf import operators

UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -20}


def test_listed_and_drawn_cases():
    cases = operators.listed()
    assert len({c["name"] for c in cases}) == len(cases)
    rng = random.Random(5)
    drawn = [operators.draw(rng) for _ in range(60)]
    assert {c["op"] for c in drawn} == {c["op"] for c in cases}
    for case in cases + drawn:
        work = operators.work(case)
        assert work["bytes"] > 0 and work["flops"] > 0


@pytest.mark.gpu
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("case", operators.listed(), ids=lambda c: c["name"])
def test_a_pass_gives_the_answer(case, own, monkeypatch):
    monkeypatch.setattr(operators, "own", own)
    got, want = operators.run(operators.prepare(case, 3)), operators.exact(case, 3)
    got, want = ([t] if torch.is_tensor(t) else t for t in (got, want))
    assert len(got) == len(want)
    for a, b in zip(got, want):
        assert a.isfinite().all()
        if b is not None:
            assert a.shape == b.shape
            assert float((a.double() - b).norm() / b.norm()) < UNIT[case["dtype"]]
