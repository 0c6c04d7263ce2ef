"""A paged cache, what needs no GPU: refusals of the C entry points before any launch."""
import ctypes

import pytest
import torch

from lit_gpt_b200 import _cabi as C
from lit_gpt_b200 import kernels as K

FAKE = 0x10000   # never read: every call here is refused first


def refused(rc, text):
    assert rc == 1 and text in C.load().b200_last_error().decode(), (rc, C.load().b200_last_error())


def test_attention_arguments_are_checked():
    lib = C.load()
    ok = dict(qkv=FAKE, cos=FAKE, sin=FAKE, table_dtype=C.F32, table_rows=64, rope_n_elem=64, row_pos=FAKE, row_seq=FAKE, seqs=FAKE, n_seqs=3, pages=FAKE, pages_ld=8, table_seqs=4,
              max_pages=8, pool=20, page=16, k_pages=FAKE, v_pages=FAKE, k_page_stride=2048, k_group_stride=1024, v_page_stride=2048, v_group_stride=1024, out=FAKE, rows=5,
              max_rows=3, max_length=128, n_head=4, n_groups=2, head_size=64, workspace=FAKE, workspace_bytes=1 << 30)
    call = lambda **kw: lib.b200_attn_paged(ctypes.byref(C.AttnPagedArgs(**{**ok, **kw})), None)
    for kw, text in ((dict(head_size=80), "head size"), (dict(n_head=5), "heads"), (dict(rows=0), "rows"), (dict(n_seqs=0), "sequences"), (dict(rows=1 << 23), "too many rows"),
                     (dict(max_rows=0), "of up to 0 rows"), (dict(max_rows=6), "of up to 6 rows"), (dict(page=8), "pages of 8"), (dict(page=48), "pages of 48"), (dict(page=512), "pages of 512"),
                     (dict(pool=0), "no pages"), (dict(max_pages=0), "no pages"), (dict(pages_ld=7), "page table"), (dict(max_length=129), "129 keys"), (dict(max_length=0), "0 keys"),
                     (dict(qkv=None), "null"), (dict(row_seq=None), "null"), (dict(pages=None), "null"), (dict(v_pages=None), "null"), (dict(out=None), "null"), (dict(rope_n_elem=66), "rope"),
                     (dict(rope_n_elem=3), "rope"), (dict(cos=None), "tables"), (dict(table_rows=0), "tables"), (dict(table_preselected=1, table_rows=4), "preselected"),
                     (dict(table_dtype=C.F16), "tables"), (dict(k_pages=FAKE + 2), "16-byte"), (dict(v_group_stride=1028), "16-byte"), (dict(seqs=FAKE + 4), "16-byte"), (dict(out=FAKE + 8), "16-byte"),
                     (dict(key_weights=FAKE + 2), "16-byte"), (dict(workspace_bytes=16), "workspace"),
                     (dict(rows=1 << 20, max_rows=1 << 20, max_length=1 << 29, max_pages=1 << 25, pages_ld=1 << 25), "too many keys"),
                     (dict(rows=1 << 20, max_rows=1, max_length=1 << 29, max_pages=1 << 25, pages_ld=1 << 25), "too many keys")):
        refused(call(**kw), text)
    refused(lib.b200_attn_paged(None, None), "null")
    need = lib.b200_attn_paged_workspace_bytes
    assert need(5, 3, 4, 2, 64, 3, 128, 0) > 0 and need(5, 3, 4, 2, 64, 3, 128, 1) > need(5, 3, 4, 2, 64, 3, 128, 0)
    for bad in ((0, 3, 4, 2, 64, 3, 128, 0), (5, 0, 4, 2, 64, 3, 128, 0), (5, 3, 4, 3, 64, 3, 128, 0), (5, 3, 4, 2, 80, 3, 128, 0), (5, 3, 4, 2, 64, 6, 128, 0), (5, 3, 4, 2, 64, 3, 0, 0)):
        assert need(*bad) == 0


def test_eviction_arguments_are_checked():
    lib = C.load()
    ok = dict(k_pages=FAKE, v_pages=FAKE, k_page_stride=2048, k_group_stride=1024, v_page_stride=2048, v_group_stride=1024, key_weights=FAKE, pages=FAKE, pages_ld=8, table_seqs=4,
              max_pages=8, pool=20, page=16, lengths=FAKE, lengths_out=2 * FAKE, n_seqs=3, n_groups=2, head_size=64, keep=50, first=4, recent=10, max_length=128, workspace=FAKE,
              workspace_bytes=1 << 30)
    call = lambda **kw: lib.b200_evict_paged(ctypes.byref(C.EvictPagedArgs(**{**ok, **kw})), None)
    for kw, text in ((dict(head_size=80), "head size"), (dict(n_seqs=0), "0 sequences"), (dict(n_groups=1 << 23), "groups"), (dict(page=24), "pages of 24"), (dict(pool=0), "no pages"),
                     (dict(n_seqs=5), "page table of 4 rows"), (dict(max_length=129), "129 keys"), (dict(keep=0), "to keep"), (dict(first=-1), "to keep"), (dict(recent=47), "to keep"),
                     (dict(key_weights=None), "null"), (dict(lengths=None), "null"), (dict(lengths_out=None), "null"), (dict(lengths_out=FAKE), "in the place"),
                     (dict(k_pages=FAKE + 8), "16-byte"), (dict(k_page_stride=2050), "16-byte"), (dict(workspace_bytes=8, keep=30000, max_length=60000, max_pages=8000, pages_ld=8000), "workspace")):
        refused(call(**kw), text)
    refused(lib.b200_evict_paged(None, None), "null")
    need = lib.b200_evict_paged_workspace_bytes
    assert need(3, 2, 30000, 60000, 16) == (3 * 2 * 30000 + 3) * 4 and need(3, 2, 50, 128, 16) == 0 and need(3, 2, 0, 128, 16) == 0


def test_packed_arguments_are_the_structures():
    import struct

    for cls, fmt in ((C.AttnPagedArgs, C.ATTN_PAGED_PACKED), (C.EvictPagedArgs, C.EVICT_PAGED_PACKED)):
        n = len(cls._fields_)
        assert struct.calcsize(fmt) == ctypes.sizeof(cls) and struct.pack(fmt, *range(1, n + 1)) == bytes(cls(*range(1, n + 1)))


def test_tensors_on_the_cpu_are_refused():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    i32 = torch.int32
    with pytest.raises(C.B200Error, match="CUDA"):
        K.attn_paged(z(3, 512), z(9, 64), z(9, 64), z(3, dtype=i32), z(3, dtype=i32), z(1, 4, dtype=i32), z(1, 4, dtype=i32), z(5, 2, 16, 64), z(5, 2, 16, 64), 4, 2, 64, 64, max_rows=3,
                     max_length=20)
    with pytest.raises(C.B200Error, match="CUDA"):
        K.evict_paged(z(5, 2, 16, 64), z(5, 2, 16, 64), z(5, 2, 16, dtype=torch.float32), z(1, 4, dtype=i32), z(1, dtype=i32), 20, max_length=40)


def test_page_layouts_are_checked():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
    k, table, kw = z(5, 2, 16, 64), z(1, 4, dtype=torch.int32), z(5, 2, 16, dtype=torch.float32)
    check = lambda k=k, v=k, kw=kw, table=table, G=2, hs=64: K._pages_of("it", k, v, kw, table, G, hs)
    assert check() == (5, 16, 2048, 1024, 2048, 1024)
    both = z(5, 2, 2, 16, 64)
    assert check(both[:, 0], both[:, 1])[2:] == (4096, 1024, 4096, 1024)
    across = z(2, 5, 16, 64).transpose(0, 1)
    assert check(across, across)[2:] == (1024, 5120, 1024, 5120)
    for kw_, text in ((dict(k=k.half()), "bfloat16"), (dict(G=3), "bfloat16"), (dict(hs=128), "bfloat16"), (dict(v=z(5, 2, 32, 64)), "bfloat16"), (dict(k=z(5, 2, 64, 16).transpose(2, 3)), "rows of a page"),
                      (dict(k=z(5, 2, 16, 128)[..., :64]), "rows of a page"), (dict(k=z(1, 2, 16, 64).expand(5, 2, 16, 64)), "overlap"), (dict(k=z(5, 1, 16, 64).expand(5, 2, 16, 64)), "overlap"),
                      (dict(kw=kw.double()), "key_weights"), (dict(kw=kw[:4]), "key_weights"), (dict(kw=z(5, 16, 2, dtype=torch.float32).transpose(1, 2)), "key_weights"),
                      (dict(table=table.long()), "page table"), (dict(table=table[0]), "page table"), (dict(table=z(4, 1, dtype=torch.int32).expand(4, 3)), "page table")):
        with pytest.raises(C.B200Error, match=text):
            check(**kw_)
