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


@pytest.mark.parametrize("tune,per,rows,n", [(1, 4, 100, 40), (3, 4, 100, 40), (0, 130, 9, 60), (1, 1, 4096, 200)])
@pytest.mark.parametrize("weights", [False, True])
def test_sequences_that_share_rows(E, tune, per, rows, n, weights):
    """More items than the step's rows can come to: none is done, and nothing is read of results that nobody left."""
    G, hs = 2, 64
    d = make([(rows, 20)], G, per, hs, 16, weights=weights, seed=rows)
    first = d["seqs"][0].tolist()
    d["seqs"] = torch.tensor([first] * n, dtype=torch.int32)
    d["row_seq"] = torch.arange(rows, dtype=torch.int32) % n
    d["max_rows"] = rows
    ref = oracle.step({**d, "seqs": d["seqs"][:1]})
    before = E.attn_paged_tune(tune)
    try:
        junk = torch.full((1 << 26,), float("nan"), device="cuda")   # what a workspace may find in its place
        del junk
        out, k, v, kw = call(E, d)
    finally:
        E.attn_paged_tune(before)
    assert not out.any() and same(k.cpu(), ref[2]) and same(v.cpu(), ref[3])
    if weights:
        at = d["pages"][first[3]]
        want = d["kw"].clone()
        for j in range(20, 20 + rows):
            want[at[j // 16], :, j % 16] = 0.0
        assert same(kw.cpu(), want)


@pytest.mark.parametrize("weights", [False, True])
def test_sequences_that_share_rows_on_the_tensor_memory(E, weights):
    rows, n, G, hs, length = 4096, 4096, 32, 64, 100000
    r = torch.Generator(device="cuda").manual_seed(1)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")
    qkv = torch.randn(rows, 3 * G * hs, device="cuda", generator=r).bfloat16()
    table = torch.full((1, 391), -1, dtype=torch.int32, device="cuda")
    k, v = (torch.ones(2, G, 256, hs, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    kw = torch.ones(2, G, 256, device="cuda") if weights else None
    cos, sin = torch.ones(rows, hs, device="cuda"), torch.zeros(rows, hs, device="cuda")
    junk = torch.full((1 << 27,), float("nan"), device="cuda")
    del junk
    out = E.attn_paged(qkv, cos, sin, torch.arange(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, dtype=torch.int32, device="cuda"), i32(0, rows, length - rows, 0).expand(n, 4).contiguous(),
                       table, k, v, G, G, hs, hs, max_rows=rows, max_length=length, key_weights=kw)
    assert not out.any() and (k == 1).all() and (v == 1).all() and (kw is None or (kw == 1).all())
