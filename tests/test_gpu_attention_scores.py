"""query_attention's scores at the ends of their range: caps from a few units to the largest that is taken."""
import pytest
import torch

from tests.test_gpu_query_attention import BF16, F16, F32, IDS, check, inputs

pytestmark = pytest.mark.gpu


# A cap far above the scores leaves them as they are.
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("mask,distance", [("none", False), ("random", False), ("documents", True)])
@pytest.mark.parametrize("cap", (1e-3, 200.0, 256.0, 257.0, 1e4, 1e6, 1e9, 1e30))
def test_caps_of_any_size(cap, mask, distance, dtype):
    check(inputs(1, 150, 150, 2, 1, 32, dtype, mask=mask, distance=distance, seed=41), cap=cap)


# Scores of up to some hundred, on both sides of where a cap of 300 or 1000 bends them.
@pytest.mark.parametrize("dtype", (F32, F16, BF16), ids=IDS.get)
@pytest.mark.parametrize("cap", (300.0, 1000.0))
def test_scores_that_a_large_cap_bends(cap, dtype):
    t = inputs(1, 150, 150, 2, 2, 16, dtype, seed=42)
    check(t, scale=20.0, cap=cap)
    check(t, scale=-1.0, cap=cap)
