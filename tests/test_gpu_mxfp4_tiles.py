"""Experts' products on large tiles with three workgroups a CU: more tiles than two
workgroups a CU take in a round, with rows of whole stages and of a part of one,
f32 and bf16 results, rows by token and in order.  Whole numbers, exact in any
order of f32 sums (see test_gpu_mxfp4_mm.py, whose plain forms these are)."""
import pytest

import test_gpu_mxfp4_mm as mm
from test_gpu_mxfp4_mm import M  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

EXPERTS = [(1000, 8, 60, 700, 256), (1000, 8, 60, 700, 288), (1000, 8, 60, 700, 32), (900, 8, 61, 769, 544)]


@pytest.mark.parametrize("ids", ["spread", "hot", "dropped"])
@pytest.mark.parametrize("kind", ["mxfp4", "bf16"])
@pytest.mark.parametrize("tokens,per_token,experts,out,inp", EXPERTS)
def test_experts_whole_numbers_are_exact(M, tokens, per_token, experts, out, inp, kind, ids):  # noqa: F811
    mm.test_experts_whole_numbers_are_exact(M, tokens, per_token, experts, out, inp, kind, ids)
