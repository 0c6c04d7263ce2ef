"""Steps over a paged cache where kernels have to agree on what they hold and whose rows they are: wide groups, few single tokens, rows that are masked out, numbers that are not finite.
Against the formulas in 64 bits (paged_oracle.py, which derives the tolerances)."""
import pytest
import torch

import paged_oracle as oracle
from paged_oracle import F64, make
from test_gpu_paged import E, K, call, check, formula, launch, on_gpu, path, same  # noqa: F401 (fixtures)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weights", [False, True])
@pytest.mark.parametrize("per,hs", [(17, 64), (20, 128), (32, 64), (33, 128), (48, 128), (71, 64), (128, 64), (129, 128)])
@pytest.mark.parametrize("cached", [[300], [4100] * 16, [5, 0, 2000]], ids=["one", "many", "unequal"])
def test_single_tokens_of_wide_groups(K, formula, weights, per, hs, cached):
    if per > 32:   # (they go to the tensor memory however few the keys are)
        cached = cached[:4]
    d = make([(1, n) for n in cached], 1, per, hs, 64, weights=weights, seed=per)
    check(call(K, d), formula(d))
