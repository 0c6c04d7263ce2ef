"""PagedSession where a caller asks for what one seldom does."""
import pytest
import torch

from test_gpu_answers import along, toy

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["nf4", None])
@torch.inference_mode()
def test_places_named_twice_or_out_of_order(golden, mode):
    """Rows come in the order of a request's tokens, as often as they are named -- in portions and in captured steps of single tokens too.  Every row is the oracle's of its place."""
    from lit_gpt_b200.generate.serve import PagedSession

    model, rc, pw, _ = toy(golden, mode)
    g = torch.Generator().manual_seed(5)
    a, b = (torch.randint(1, 500, (n,), generator=g) for n in (23, 12))
    (la, ta), (lb, tb) = along(model, rc, pw, a, 1), along(model, rc, pw, b, 1)   # logits behind every token but the last

    def check(got, rows_a, rows_b):
        want = torch.cat([la[rows_a], lb[rows_b]])
        assert got.shape == want.shape and (got.cpu() - want).abs().max() <= max(ta, tb)

    a, b = a.tolist(), b.tolist()
    for portion in (4096, 7):
        s = PagedSession(model, 12, 16, portion=portion)
        check(s.step([("a", a[:20], [19, 3, 3, 0, 19, 19]), ("b", b[:9], iter((8, 0, 8)))]), [0, 3, 3, 19, 19, 19], [0, 8, 8])
        check(s.step([("a", [a[20]], [0, 0]), ("b", [b[9]], [0])]), [20, 20], [9])
        check(s.step([("a", [a[21]], [0, 0]), ("b", [b[10]], [])]), [21, 21], [])   # as many rows as requests
