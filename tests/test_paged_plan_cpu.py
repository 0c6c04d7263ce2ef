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


def test_a_list_of_single_tokens_is_sized_by_its_sequences():
    """A token beside a chunk: the chunk's rows are none of the list's, whose sequences have one item of a group each."""
    need = C.load().b200_attn_paged_workspace_bytes
    G, per, hs = 8, 4, 128
    for chunk, length in ((512, 3001), (16384, 20000)):
        rows = 32 + chunk
        tiles, blocks = 33 * G * -(-length // 32), 148 * 2 * 256
        most = (tiles * 8 * 32 * 4                      # scores of 8 queries and 32 keys a tile
                + (33 * G + 148 * 7) * 8 * (hs + 2) * 4   # results of an item and worker
                + blocks * (hs + 2) * 4                 # the tensor memory's
                + rows * per * G * (2 * hs + 4)         # queries and their sums
                + (1 << 20))
        assert need(rows, 33, G * per, G, hs, chunk, length, 1) <= most
    # weights from kept scores: they are part of the workspace, and not given up for the rows of a chunk
    assert need(32 + 16384, 33, G * per, G, hs, 16384, 20000, 1) - need(32 + 16384, 33, G * per, G, hs, 16384, 20000, 0) > 33 * G * (20000 // 32) * 8 * 32 * 4


def test_a_token_beside_a_long_chunk_over_many_keys_is_not_refused():
    import ctypes

    args = dict(qkv=0x10000, cos=0x10000, sin=0x10000, table_dtype=C.F32, table_rows=64, rope_n_elem=64, row_pos=0x10000, row_seq=0x10000, seqs=0x10000, n_seqs=2, pages=0x10000,
                pages_ld=1 << 13, table_seqs=4, max_pages=1 << 13, pool=20, page=128, k_pages=0x10000, v_pages=0x10000, k_page_stride=2048, k_group_stride=1024, v_page_stride=2048,
                v_group_stride=1024, out=0x10000, rows=16385, max_rows=16384, max_length=1 << 20, n_head=32, n_groups=32, head_size=64, workspace=0x10000, workspace_bytes=16)
    assert C.load().b200_attn_paged(ctypes.byref(C.AttnPagedArgs(**args)), None) == 1
    assert "workspace too small" in C.load().b200_last_error().decode()   # (what the call gets to: it has nothing against the step's size)


def test_a_paged_step_over_several_devices_is_refused():
    import torch

    from lit_gpt_b200 import GPT, Config
    from lit_gpt_b200.model import PagedKVCache
    from lit_gpt_b200.ragged import PagedStep

    config = Config(n_layer=2, n_head=2, n_embd=128, vocab_size=50, block_size=32)
    model = GPT(config)
    model.transformer.h[1].to("meta")
    for b in model.transformer.h:
        b.attn.kv_cache = PagedKVCache(config, 4, 16)
    z = torch.zeros(1, dtype=torch.int32)
    step = PagedStep(seqs=z.expand(1, 4), row_pos=z, row_seq=z, table=z[None], max_rows=1, max_length=16)
    with pytest.raises(NotImplementedError, match="one GPU"):
        model.paged_step(z, step)
    assert all(b.attn.kv_cache.step is None for b in model.transformer.h)
