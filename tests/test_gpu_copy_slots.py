"""Copies between the slots of caches and states (csrc/slots.cu): bit for bit what indexing makes of them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from lit_gpt_b200 import kernels

    return kernels


def noise(*shape, dtype=torch.float32):
    size = torch.empty(0, dtype=dtype).element_size()
    return torch.randint(0, 256, (*shape[:-1], shape[-1] * size), dtype=torch.uint8, device="cuda").view(dtype)   # any bits, NaN among them


def check(K, tensors, src, dst, lengths=None):
    want = [t.clone() for t in tensors]
    for t in want:
        for i, (a, b) in enumerate(zip(src, dst)):
            n = t.shape[1] if lengths is None else lengths[i]
            t[b, :n] = t[a, :n]
    K.copy_slots(tensors, src, dst, lengths)
    for t, w in zip(tensors, want):
        assert torch.equal(t.view(torch.uint8), w.view(torch.uint8))


@pytest.mark.parametrize("shapes", [[(1, 1)], [(3, 6144), (1, 262144)], [(1000, 33)], [(7, 5, 11)], [(4096, 576)], [(1024, 512), (5, 3), (1, 16385)]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.uint8])
def test_forks_and_moves(K, shapes, dtype):
    tensors = [noise(6, *s, dtype=dtype) for s in shapes]
    check(K, tensors, [4], [0])
    check(K, tensors, [0, 0, 0], [5, 3, 1])
    check(K, tensors, [2, 1, 2], [5, 4, 3])


@pytest.mark.parametrize("lengths", [[0, 1, 2], [64, 64, 64], [7, 63, 30]])
@pytest.mark.parametrize("cols", [576, 129, 1])
def test_leading_positions(K, lengths, cols):
    tensors = [noise(8, 64, cols, dtype=torch.bfloat16), noise(8, 100, 2 * cols, dtype=torch.float32)]
    check(K, tensors, [1, 1, 6], [0, 3, 2], lengths)


def test_more_tensors_groups_and_copies_than_a_launch_takes(K):
    tensors = [noise(700, 3, 1 + i % 5) for i in range(300)]
    src = [i % 150 for i in range(500)]
    check(K, tensors, src, [200 + i for i in range(500)])
    check(K, tensors, [7] * 400, [100 + i for i in range(400)])


def test_misaligned_buffers(K):
    big = noise(6 * 65 * 3 + 7, dtype=torch.uint8)
    for off in (1, 2, 4):
        check(K, [big[off : off + 6 * 65 * 3].view(6, 65, 3)], [0, 0], [5, 2])


def test_offsets_past_32_bits(K):
    t = torch.zeros(3, 1, 1_200_000_000, dtype=torch.bfloat16, device="cuda")
    t[0, 0, -5:] = 1.5
    t[0, 0, 123] = 2.5
    K.copy_slots([t], [0], [2])
    assert t[2, 0, -5:].tolist() == [1.5] * 5 and t[2, 0, 123] == 2.5 and not t[1].any() and t[2].count_nonzero() == 6


def test_nothing_to_do(K):
    t = noise(3, 4, 5)
    check(K, [t], [], [])
    check(K, [t], [0], [1], [0])
    K.copy_slots([], [0], [1])


def test_captured(K):
    t = noise(4, 10, 100)
    K.copy_slots([t], [0], [3])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        K.copy_slots([t], [0, 0], [1, 2])
    t[0] = 1.0
    graph.replay()
    assert (t[:3] == 1.0).all() and not (t[3] == 1.0).all()


def test_refusals(K):
    t = noise(4, 10, 6)
    before = t.clone()
    for args in (([t], [0], [4]), ([t], [-1], [1]), ([t], [0, 1], [2, 2]), ([t], [0, 2], [2, 3]), ([t], [1], [1]), ([t], [0], [1], [11]), ([t], [0], [1], [-1]), ([t], [0, 1], [2]),
                 ([t], [0], [1], []), ([t.transpose(1, 2)], [0], [1]), ([t, t[:3]], [0], [1]), ([t[0, 0]], [0], [1]), ([t.cpu()], [0], [1]), ([t[:, :0]], [0], [1])):
        with pytest.raises(K.C.B200Error):
            K.copy_slots(*args)
    assert torch.equal(t.view(torch.uint8), before.view(torch.uint8))
