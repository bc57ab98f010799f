"""CPU tests of the paged cache entry points: every argument that the host can see to be wrong is refused before
anything is launched (there is no GPU here, so a call that got past its checks would report a CUDA error)."""
import ctypes as C

import pytest

from instantcua_b200 import _lib as L

A = 1 << 20  # an aligned address that is never followed


def pages(**kw):
    d = dict(k=A, v=A, dtype=L.KV_F16, n_kv=2, page_size=16, n_pages=4)
    return L.IcuaKvPages(**{**d, **kw})


def seqs(**kw):
    d = dict(n_seqs=2, total_q=3, max_q=2, max_kv=40, cu_q=A, kv_len=A, page_table=A, max_pages=4)
    return L.IcuaKvSeqs(**{**d, **kw})


def rows(**kw):
    d = dict(qkv=A, qkv_dtype=L.DT_F32, n_q=4, eps=1e-6, q_out=A, q_dtype=L.DT_F16)
    return L.IcuaKvRows(**{**d, **kw})


def attn(**kw):
    d = dict(q=A, out=A, dtype=L.DT_F16, n_q=4, scratch=A, scratch_bytes=1 << 40)
    return L.IcuaAttnPaged(**{**d, **kw})


BAD_PAGES = [dict(k=None), dict(v=None), dict(k=A + 8), dict(v=A + 4), dict(dtype=3), dict(dtype=-1), dict(n_kv=0), dict(n_kv=129),
             dict(page_size=0), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(n_pages=-1), dict(n_pages=0),
             dict(dtype=L.KV_Q8), dict(dtype=L.KV_Q8, k_scale=A), dict(dtype=L.KV_Q8, k_scale=A, v_scale=A + 4),
             dict(page_rows=32), dict(head_rows=16), dict(page_rows=16, head_rows=8), dict(page_rows=-32, head_rows=16),
             dict(page_rows=24, head_rows=16), dict(page_rows=32, head_rows=24),
             dict(n_pages=2**31 - 1), dict(page_rows=2**60, head_rows=16), dict(page_rows=32, head_rows=2**62)]
BAD_SEQS = [dict(n_seqs=-1), dict(n_seqs=1025), dict(total_q=-1), dict(max_q=-1), dict(max_kv=-1), dict(max_pages=-1), dict(cu_q=None),
            dict(kv_len=None), dict(page_table=None), dict(cu_q=A + 2), dict(page_table=A + 1), dict(max_pages=1 << 28)]
BAD_ROWS = [dict(qkv=None), dict(qkv=A + 4), dict(qkv_dtype=3), dict(qkv_dtype=-1), dict(n_q=-1), dict(n_q=257), dict(q_dtype=L.DT_F32),
            dict(q_dtype=L.DT_BF16), dict(qkv_stride=8), dict(qkv_stride=1028), dict(qkv_stride=-2048), dict(q_stride=500),
            dict(q_stride=516), dict(q_out=A + 2), dict(q_norm=A + 4), dict(k_norm=A + 8), dict(rope=A + 8), dict(rope_rows=A + 2),
            dict(rope=A, rope_len=-1), dict(eps=-1.0), dict(eps=float("nan"))]
BAD_ATTN = [dict(q=None), dict(out=None), dict(q=A + 2), dict(out=A + 8), dict(dtype=L.DT_F32), dict(dtype=L.DT_BF16), dict(n_q=0),
            dict(n_q=1), dict(n_q=5), dict(n_q=258), dict(q_stride=8), dict(q_stride=516), dict(out_stride=-512), dict(scale=-1.0),
            dict(scale=float("nan")), dict(scale=float("inf")), dict(scratch=None), dict(scratch=A + 4), dict(scratch_bytes=16)]


def refused(status):
    assert status == L.ERR_INVALID, (status, L.lib().icua_global_error())
    assert L.lib().icua_global_error()


@pytest.mark.parametrize("kw", BAD_PAGES, ids=str)
def test_bad_cache_is_refused(kw):
    lib, p, s = L.lib(), pages(**kw), seqs()
    refused(lib.icua_kv_write(C.byref(p), C.byref(s), C.byref(rows()), None, None))
    refused(lib.icua_kv_read(C.byref(p), C.byref(s), A, A, L.DT_F16, None, None))
    refused(lib.icua_attn_paged(C.byref(p), C.byref(s), C.byref(attn()), None, None))
    assert lib.icua_attn_paged_scratch_bytes(C.byref(p), C.byref(s), 4) == 0


@pytest.mark.parametrize("kw", BAD_SEQS, ids=str)
def test_bad_batch_is_refused(kw):
    lib, p, s = L.lib(), pages(), seqs(**kw)
    refused(lib.icua_kv_write(C.byref(p), C.byref(s), C.byref(rows()), None, None))
    refused(lib.icua_kv_read(C.byref(p), C.byref(s), A, A, L.DT_F16, None, None))
    refused(lib.icua_attn_paged(C.byref(p), C.byref(s), C.byref(attn()), None, None))


@pytest.mark.parametrize("kw", BAD_ROWS, ids=str)
def test_bad_rows_are_refused(kw):
    refused(L.lib().icua_kv_write(C.byref(pages()), C.byref(seqs()), C.byref(rows(**kw)), None, None))


@pytest.mark.parametrize("kw", BAD_ATTN, ids=str)
def test_bad_attention_arguments_are_refused(kw):
    refused(L.lib().icua_attn_paged(C.byref(pages()), C.byref(seqs()), C.byref(attn(**kw)), None, None))


def test_null_descriptors_outputs_and_flags():
    lib, p, s = L.lib(), C.byref(pages()), C.byref(seqs())
    refused(lib.icua_kv_write(None, s, C.byref(rows()), None, None))
    refused(lib.icua_kv_write(p, None, C.byref(rows()), None, None))
    refused(lib.icua_kv_write(p, s, None, None, None))
    refused(lib.icua_kv_write(p, s, C.byref(rows()), A + 2, None))
    refused(lib.icua_kv_read(p, s, None, None, L.DT_F16, None, None))
    refused(lib.icua_kv_read(p, s, A + 8, A, L.DT_F16, None, None))
    refused(lib.icua_kv_read(p, s, A, A, 3, None, None))
    refused(lib.icua_attn_paged(p, s, None, None, None))
    refused(lib.icua_attn_paged(p, s, C.byref(attn()), A + 1, None))
    big = seqs(total_q=2**31 - 1)
    refused(lib.icua_attn_paged(p, C.byref(big), C.byref(attn()), None, None))


def test_types_go_together():
    lib = L.lib()
    for cache, typ in ((L.KV_F16, L.DT_BF16), (L.KV_BF16, L.DT_F16)):
        refused(lib.icua_attn_paged(C.byref(pages(dtype=cache)), C.byref(seqs()), C.byref(attn(dtype=typ)), None, None))
        refused(lib.icua_kv_write(C.byref(pages(dtype=cache)), C.byref(seqs()), C.byref(rows(q_dtype=typ)), None, None))


def test_empty_batches_are_no_work():
    """No sequence or no row: nothing to launch, so it succeeds without a GPU."""
    lib, p = L.lib(), C.byref(pages())
    for s in (seqs(n_seqs=0), seqs(total_q=0), seqs(n_seqs=0, cu_q=None, kv_len=None, page_table=None)):
        assert lib.icua_kv_write(p, C.byref(s), C.byref(rows()), None, None) == L.OK
        assert lib.icua_kv_read(p, C.byref(s), A, A, L.DT_F32, None, None) == L.OK
        assert lib.icua_attn_paged(p, C.byref(s), C.byref(attn()), None, None) == L.OK


@pytest.mark.parametrize("total_q,n_q", [(32768, 128), (65536, 64), (1 << 20, 64)])
def test_long_prompts_with_wide_tables_are_taken(total_q, n_q):
    """The size limit counts rows of short sequences only: whole prompts beside a page table for a million positions."""
    p = pages(n_kv=8, page_size=256)
    s = seqs(n_seqs=1, total_q=total_q, max_q=total_q, max_kv=total_q, max_pages=4096)
    assert L.lib().icua_attn_paged_scratch_bytes(C.byref(p), C.byref(s), n_q) > 0


def test_batches_past_the_counters_are_refused():
    p = C.byref(pages(n_kv=128, page_size=256))
    for s in (seqs(n_seqs=1024, total_q=1024, max_pages=1 << 22),   # 1,024 x 128 items over 2^30 positions
              seqs(n_seqs=1, total_q=1 << 25, max_q=1 << 25)):      # 2^25 tokens x 64 heads a kv head
        n_q = 128 if s.n_seqs > 1 else 256
        if s.n_seqs == 1:
            p = C.byref(pages(n_kv=4))
        assert L.lib().icua_attn_paged_scratch_bytes(p, C.byref(s), n_q) == 0
        refused(L.lib().icua_attn_paged(p, C.byref(s), C.byref(attn(n_q=n_q)), None, None))


def test_scale_stays_finite_in_units_of_log2():
    """scale * log2(e) passes fp32's largest number from 2.36e38 on: scores of 0 would turn into NaN."""
    for scale in (2.4e38, 2.9e38):
        refused(L.lib().icua_attn_paged(C.byref(pages()), C.byref(seqs()), C.byref(attn(scale=scale)), None, None))
    assert L.lib().icua_attn_paged(C.byref(pages()), C.byref(seqs(n_seqs=0)), C.byref(attn(scale=2.3e38)), None, None) == L.OK


def test_in_place_attention_keeps_the_stride():
    """out = q with another token stride would write over rows of q that are still to be read."""
    lib, p = L.lib(), C.byref(pages())
    for kw in (dict(q_stride=520), dict(out_stride=1024), dict(q_stride=1024, out_stride=520)):
        refused(lib.icua_attn_paged(p, C.byref(seqs()), C.byref(attn(**kw)), None, None))
    for kw in (dict(), dict(q_stride=520, out_stride=520), dict(q_stride=512), dict(out_stride=520, out=2 * A)):
        assert lib.icua_attn_paged(p, C.byref(seqs(n_seqs=0)), C.byref(attn(**kw)), None, None) == L.OK
