"""The performance cases of a decoding step (perf/operators.py): what the library gives against the cases' definition in 64 bits.

Bounds. bf16 results: a rounding of 2^-8 of each value at most, so of their norm. Codes: v comes from bf16 by one rounding, so its codes and
scales are the definition's. k is normed and rotated in fp32, off by 2^-16 of the magnitudes that are added, 1.5 of the value or so; the
step between codes is 2^-4 of a value at least. So a code may be one step off, and 2 * 1.5 * 2^-16 / 2^-4 < 2^-10 of them may be."""
import importlib.util
import os
import random

import pytest
import torch

pytestmark = pytest.mark.gpu
SPEC = importlib.util.spec_from_file_location("operator_cases", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py"))
ops = importlib.util.module_from_spec(SPEC)
SPEC.loader.exec_module(ops)
ops.own = True
CASES = ops.listed()
DRAWN = [ops.draw(random.Random(seed)) for seed in range(24)]


def check(case, seed):
    got, want = ops.run(ops.prepare(case, seed)), ops.exact(case, seed)
    if case["kind"] != "append":
        assert float((got.double() - want).norm()) <= 2.0 ** -8 * float(want.norm())
        return
    assert float((got["q"].double() - want["q"]).norm()) <= 2.0 ** -8 * float(want["q"].norm())
    assert torch.equal(got["v_scale"].double(), want["v_scale"]) and torch.equal(got["v"].double(), want["v"])
    same = got["k_scale"].double() == want["k_scale"]
    assert float((~same).float().mean()) <= 2.0 ** -10
    have, meant = got["k"].double()[same], want["k"][same]
    off = have != meant
    step = torch.maximum(meant.abs(), have.abs()) * 2.0 ** -3 + 2.0 ** -9
    assert bool(((have - meant).abs() <= step).all()) and float(off.float().mean()) <= 2.0 ** -10


@pytest.mark.parametrize("case", CASES, ids=[c["name"] for c in CASES])
def test_listed_cases(case):
    check(case, 3)


@pytest.mark.parametrize("case", DRAWN, ids=["_".join(str(v) for v in c.values()) for c in DRAWN])
def test_drawn_cases(case):
    check(case, 4)
