"""What a step over a paged cache asks for, on the host: sizes of the workspace show which kernels take it."""
import pytest

from lit_gpt_b200 import _cabi as C


@pytest.fixture
def need():
    """(sequences and rows of one token each, groups, heads of a group, head size, max_length, weights) -> bytes; none where one launch does all."""
    return lambda n, groups, per, hs, length, weights=0: C.load().b200_attn_paged_workspace_bytes(n, n, groups * per, groups, hs, 1, length, weights)


@pytest.mark.parametrize("hs", [64, 128])
@pytest.mark.parametrize("n,length", [(1, 256), (1, 300), (2, 2000), (16, 4000)])
def test_one_launch_takes_no_more_heads_than_it_holds(need, hs, n, length):
    """The kernel that does a step of single tokens in one launch has room for 16 heads of a group."""
    assert need(1, 1, 16, hs, 300) == 0
    for per in (17, 20, 31, 32, 33, 48, 64, 71, 128, 129, 200):
        assert need(n, 1, per, hs, length) > 0, per
