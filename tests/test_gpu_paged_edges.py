"""GPU tests of calls of the paged K/V cache operators that the ordinary ones do not make: whole halves of a tile without
a position, entries that contradict each other far back in a batch, hints and sizes at their ends."""
import ctypes as C

import pytest
import torch

from _paged import Cache, check_close, ptr
from instantcua_b200 import _lib as L

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [(F16, F16), (BF16, BF16), ("q8", F16), ("q8", BF16)]


@pytest.fixture(autouse=True)
def _gpu(require_gpu):
    pass


def name(v):
    return {F16: "f16", BF16: "bf16", F32: "f32"}.get(v, v) if not isinstance(v, (list, tuple)) else None


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv", [([300], [100]), ([300], [204]), ([200], [0]), ([64, 300, 1], [0, 110, 5]), ([257] * 9, [130] * 9)], ids=str)
def test_halves_of_a_tile_without_a_position(n, kv, cache, typ):
    """256 query rows a tile, four heads a token: tiles and halves of tiles whose tokens all lie before the cache's first
    position get zeros, the rows behind them their attention, also in place and every time.  At most 256 positions: a tile's
    keys are one share, so that its rows are written where they are computed."""
    c = Cache(n, kv, cache=cache, typ=typ, n_kv=2, n_q=8, seed=sum(n)).fill()
    assert max(kv) <= 256
    q = (c.randn(c.total, 8, 128) * 2).to(typ)
    want, bound = c.attend64(q)
    first = c.attend(q, torch.full_like(q, 6.0))
    check_close(first, want, bound)
    at = 0
    for a, b in zip(n, kv):
        assert (first[at:at + max(0, a - b)] == 0).all()
        at += a
    for _ in range(20):
        same = q.clone()
        c.attend(same, same)
        assert torch.equal(same, first)
    assert c.flags() == 0


@pytest.mark.parametrize("typ", [F16, BF16], ids=name)
@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e3])
@pytest.mark.parametrize("n", [1, 3, 9, 90])
def test_zero_v_rows_among_others(n, size, typ):
    """Rows of zeros in V, as icua_kv_write leaves them in a q8 cache, among rows of one small (or large) size: they count in
    the sum and hide nothing.  Every third key has one, the first and the last among them."""
    total = n + 63
    c = Cache([total], [total], cache="q8", typ=typ, n_kv=2, n_q=8)
    qkv = c.randn(total, 12, 128)
    qkv[:, 10:] = (1 + 0.1 * qkv[:, 10:]) * size
    qkv[::3, 10:] = 0
    qkv[-1, 10:] = 0
    c.write(qkv.view(total, -1), None)
    assert (c.read(F32)[1][::3] == 0).all()
    c.n, c.total = [n], n
    c.cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = c.randn(n, 8, 128).to(typ)
    out = c.attend(q)
    want, bound = c.attend64(q)
    check_close(out, want, bound)
    assert c.flags() == 0


@pytest.mark.parametrize("change", ["length", "offset"])
@pytest.mark.parametrize("n", [[40] * 40, [20] * 600, [300] + [1] * 70], ids=lambda n: f"{len(n)}")
def test_attention_flags_contradictions_anywhere_in_a_batch(n, change):
    """A sequence far behind the first 32 of a batch that contradicts itself is flagged and left alone, whichever kernels the
    batch goes through."""
    kv = [x + 10 for x in n]
    c = Cache(n, kv, n_kv=2, n_q=4).fill()
    q = c.randn(c.total, 4, 128).half()
    clean = c.attend(q).clone()
    assert c.flags() == 0
    if change == "length":
        s = len(n) - 5
        c.kv_len[s] = -5
        gone = slice(sum(n[:s]), sum(n[:s + 1]))
    else:
        c.cu[len(n)] = c.total + 1
        gone = slice(c.total - n[-1], c.total)
    out = c.attend(q, torch.full_like(q, 7))
    assert c.flags() == L.FLAG_SEQ
    assert (out[gone] == 7).all()
    out[gone] = clean[gone]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("cache", [F16, "q8"], ids=name)
@pytest.mark.parametrize("seqs", [3, 80])
@pytest.mark.parametrize("length", [-1, 1 << 29])
def test_write_and_read_flag_idle_sequences_that_contradict_themselves(seqs, length, cache):
    """An idle sequence with an impossible length: no token looks it up, the flag is set all the same, and the other
    sequences' rows are written and read."""
    n = [1] * seqs
    n[seqs - 2] = 0
    c = Cache(n, [9] * seqs, cache=cache, junk=2.0).fill()
    qkv = c.randn(c.total, 8 * 128)
    c.write(qkv, None)
    clean = c.read(F16)
    assert c.flags() == 0
    c.kv_len[seqs - 2] = length
    got = c.read(F16)
    assert c.flags() == L.FLAG_SEQ
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    c.err.zero_()
    c.fill()
    c.write(qkv, None)
    assert c.flags() == L.FLAG_SEQ
    got = c.read(F16)
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])


def test_write_and_read_flag_offsets_that_no_token_meets():
    """cu_q = 0, 4, 2, 2, 6: sequence 1 descends, and no row's lookup ends at it."""
    c = Cache([2, 0, 0, 4], [20] * 4, junk=2.0).fill()
    c.cu.copy_(torch.tensor([0, 4, 2, 2, 6]))
    c.write(c.randn(6, 8 * 128), None)
    assert c.flags() == L.FLAG_SEQ
    c.err.zero_()
    c.read(F16)
    assert c.flags() == L.FLAG_SEQ


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
def test_more_tokens_promised_than_any_sequence_has(cache, typ):
    """max_q far above every sequence's tokens: the tensor-core kernel and its join find nothing to do.  Calls that follow one
    another in the stream with other offsets each attend their own batch, and flag their own contradictions."""
    n, kv = [1, 3, 2, 0], [3000, 700, 40, 9]
    c = Cache(n, kv, cache=cache, typ=typ, n_kv=2, n_q=8).fill()
    q = (c.randn(c.total, 8, 128) * 2).to(typ)
    want, bound = c.attend64(q)
    good, idle, bad = c.cu.clone(), torch.zeros_like(c.cu), c.kv_len.clone()
    bad[3] = -7
    sc = c.scratch(max_q=500)
    for _ in range(20):
        c.cu.copy_(good)
        out = c.attend(q, torch.full_like(q, 5.0), max_q=500, scratch=sc)
        c.cu.copy_(idle)
        none = c.attend(q, torch.full_like(q, 5.0), max_q=500, scratch=sc)
        assert (none == 5).all()
        check_close(out, want, bound)
    assert c.flags() == 0
    c.cu.copy_(good)
    c.kv_len.copy_(bad)
    check_close(c.attend(q, max_q=500, scratch=sc), want, bound)
    assert c.flags() == L.FLAG_SEQ


def test_offsets_that_claim_rows_over_and_over():
    """Descending offsets under which 683 of 1,024 sequences claim the same 64 rows, over nearly two million positions each,
    with more rows a sequence than max_q says: 683 x 2 tiles x 128 heads x 30,360 blocks pass 32 bits.  Nothing is followed
    or written, the flag is set."""
    c = Cache([1], [5], n_kv=128, n_q=128)
    pages, q = 7590, c.randn(64, 128, 128).half()
    c.ps, c.n_pages, c.total, c.max_pages = 256, 1, 64, pages
    c.k, c.v = (torch.zeros(128 * 256, 128, device="cuda", dtype=F16) for _ in range(2))
    c.cu = torch.tensor([0, 32, 64] * 341 + [0, 32], dtype=torch.int32, device="cuda")
    c.kv_len = torch.full((1024,), pages * 256, dtype=torch.int32, device="cuda")
    c.table = torch.full((1024, pages), -1, dtype=torch.int32, device="cuda")
    assert int((c.cu[1:] > c.cu[:-1]).sum()) * 2 * 128 * (pages * 256 // 64) > 2**32
    out = c.attend(q, torch.full_like(q, 7.0), n_seqs=1024, max_q=16, max_kv=pages * 256)
    assert c.flags() == L.FLAG_SEQ
    assert (out == 7).all()


def test_a_chunk_beside_a_table_for_a_million_positions():
    """40 tokens of 128 heads over 8 kv heads with a page table of 2^20 positions, in a batch padded to 32,768 rows."""
    c = Cache([40], [300], n_kv=8, n_q=128, ps=256, pad=32728, max_pages=4096).fill()
    q = c.randn(c.total, 128, 128).half()
    out = c.attend(q, max_q=c.total)
    want, bound = c.attend64(q)
    check_close(out[:40], want[:40], bound[:40])
    assert c.flags() == 0


@pytest.mark.parametrize("n,kv", [([200], [9000]), ([1, 60], [5000, 700]), ([1], [3000])], ids=str)
def test_the_largest_length_hint(n, kv):
    """max_kv up to 2^31 - 1 splits the keys as any other hint above all lengths does: the same bits."""
    c = Cache(n, kv).fill()
    q = c.randn(c.total, 4, 128).half()
    want = c.attend(q, max_kv=1 << 20)
    for hint in (2**31 - 256, 2**31 - 255, 2**31 - 1):
        assert torch.equal(c.attend(q, max_kv=hint), want)


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv", [([300], [300]), ([300], [9000]), ([200, 3, 1], [250, 40, 2000])], ids=str)
def test_a_wait_that_gives_up_leaves_nan_rows_and_a_flag(n, kv, cache, typ):
    """The tensor-core kernel's last wait with a limit of no polls: its rows become NaN (written at once, or through the join
    of key shares), with and without a flag word; the others and the next call are as ever."""
    c = Cache(n, kv, cache=cache, typ=typ, n_kv=2, n_q=8).fill()
    q = (c.randn(c.total, 8, 128) * 2).to(typ)
    want = c.attend(q).clone()
    lib = L.lib()
    try:
        L.check(lib.icua_set_wait_limit(0))
        lost = c.attend(q, torch.full_like(q, 7.0))
        assert c.flags() == L.FLAG_WAIT
        err, c.err = c.err, None
        silent = c.attend(q, torch.full_like(q, 7.0))
        c.err = err
        torch.cuda.synchronize()
    finally:
        L.check(lib.icua_set_wait_limit(1 << 22))
    for out in (lost, silent):
        assert out[:n[0]].isnan().all() and torch.equal(out[n[0]:], want[n[0]:])
    c.err.zero_()
    assert torch.equal(c.attend(q), want) and c.flags() == 0


POINTERS = ["k", "v", "k_scale", "v_scale", "cu_q", "kv_len", "page_table", "err_dev"]


@pytest.mark.parametrize("call,bad", [(c, b) for c, own in (("write", ["qkv", "q_out", "q_norm", "k_norm", "rope", "rope_rows"]),
                                                            ("read", ["k_out", "v_out"]), ("attend", ["q", "out", "scratch"]))
                                      for b in POINTERS + own])
def test_every_pointer_to_host_memory_is_refused(call, bad):
    """Each pointer of each call in pageable host memory: refused by name before anything is launched."""
    c = Cache([2], [5], cache="q8").fill()
    host = torch.zeros(1 << 18)
    at = (host.data_ptr() + 255) // 256 * 256

    def pick(name, t):
        return at if name == bad else ptr(t)

    pages = c.pages(**{x: at for x in POINTERS[:4] if x == bad})
    seqs = c.seqs(**{x: at for x in POINTERS[4:7] if x == bad})
    err, lib = pick("err_dev", c.err), L.lib()
    rows, w, rope = c.randn(2, 8, 128), torch.ones(128, device="cuda"), torch.zeros(8, 64, 2, device="cuda")
    idx, q, out = torch.zeros(2, dtype=torch.int32, device="cuda"), c.randn(2, 4, 128).half(), torch.zeros(2, 4, 128, device="cuda").half()
    before = c.k.clone()
    if call == "write":
        r = L.IcuaKvRows(qkv=pick("qkv", rows), qkv_dtype=L.DT_F32, n_q=4, q_norm=pick("q_norm", w), k_norm=pick("k_norm", w), eps=1e-6,
                         rope=pick("rope", rope), rope_rows=pick("rope_rows", idx), rope_len=8, q_out=pick("q_out", out), q_dtype=L.DT_F16)
        status = lib.icua_kv_write(C.byref(pages), C.byref(seqs), C.byref(r), err, None)
    elif call == "read":
        kv = torch.zeros(2, 2, 128, device="cuda").half()
        status = lib.icua_kv_read(C.byref(pages), C.byref(seqs), pick("k_out", kv), pick("v_out", kv), L.DT_F16, err, None)
    else:
        sc, need = c.scratch()
        a = L.IcuaAttnPaged(q=pick("q", q), out=pick("out", out), dtype=L.DT_F16, n_q=4, scratch=pick("scratch", sc), scratch_bytes=need)
        status = lib.icua_attn_paged(C.byref(pages), C.byref(seqs), C.byref(a), err, None)
    assert status == L.ERR_INVALID
    assert b"is not device memory" in lib.icua_global_error()
    torch.cuda.synchronize()
    assert torch.equal(c.k, before) and (out == 0).all()


def test_lengths_and_tables_in_pinned_host_memory():
    """The small arrays where the device reads them in place."""
    c = Cache([3, 1], [40, 700], n_kv=2, n_q=8).fill()
    q = c.randn(4, 8, 128).half()
    want = c.attend(q).clone()
    c.cu, c.kv_len, c.table = (x.cpu().pin_memory() for x in (c.cu, c.kv_len, c.table))
    assert torch.equal(c.attend(q), want) and c.flags() == 0


def test_calls_from_several_threads():
    """Eight threads, a stream, a batch and a scratch each, all making their first calls together."""
    from concurrent.futures import ThreadPoolExecutor

    caches, qs, wants = [], [], []
    for i in range(8):
        c = Cache([1 + 40 * (i % 2), 1], [300 + i, 5000 - 600 * i], n_kv=1 + i % 3, n_q=6, cache="q8" if i % 4 == 3 else F16).fill()
        caches.append(c)
        qs.append((c.randn(c.total, 6, 128) * 2).half())
        wants.append(c.attend(qs[-1]).clone())
    torch.cuda.synchronize()

    def work(i):
        st = torch.cuda.Stream()
        bad = 0
        with torch.cuda.stream(st):
            sc = caches[i].scratch()
            st.synchronize()
            for _ in range(50):
                out = caches[i].attend(qs[i], scratch=sc)
                caches[i].read(F16)
                st.synchronize()
                bad += not torch.equal(out, wants[i])
        return bad

    with ThreadPoolExecutor(8) as pool:
        assert list(pool.map(work, range(8))) == [0] * 8
    assert all(c.flags() == 0 for c in caches)


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("items", [(1, 1), (1, 2), (3, 8), (12, 8)], ids=str)
def test_drafts_of_few_and_many_items_below_1024_positions(items, cache, typ):
    """28 and 8 rows an item around the lengths where the work's split changes with the number of items."""
    s, n_kv = items
    for kv in (255, 257, 449, 1000, 1024):
        for n, group in ((7, 4), (1, 8)):
            c = Cache([n] * s, [max(n, kv - 13 * i) for i in range(s)], n_kv=n_kv, n_q=group * n_kv, cache=cache, typ=typ, seed=kv).fill()
            q = (c.randn(c.total, c.n_q, 128) * 2).to(typ)
            want, bound = c.attend64(q)
            check_close(c.attend(q), want, bound, f"{kv} positions, {n} tokens")
            assert c.flags() == 0
