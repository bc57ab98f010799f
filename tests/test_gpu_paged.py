"""GPU tests of the paged K/V cache operators (icua_kv_write, icua_kv_read, icua_attn_paged) against the formulas in 64
bits, at the sizes and masks where they can go wrong."""
import ctypes as C

import pytest
import torch

from _paged import DT, HD, Cache, check_close, ptr
from instantcua_b200 import _lib as L

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
TYPES = [(F16, F16), (BF16, BF16), ("q8", F16), ("q8", BF16)]


@pytest.fixture(autouse=True)
def _gpu(require_gpu):
    pass


def name(v):
    return {F16: "f16", BF16: "bf16", F32: "f32"}.get(v, v) if not isinstance(v, (list, tuple)) else None


# ---- write and read back ----------------------------------------------------------------------------------------------
def turn64(x, w, cs, eps):
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    if cs is None:
        return x
    a, b, c, s = x[..., :64], x[..., 64:], cs[:, None, :, 0].double(), cs[:, None, :, 1].double()
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def rope_table(n):
    ang = torch.arange(n, device="cuda", dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(64, device="cuda").double() / 64)
    return torch.stack((ang.cos(), ang.sin()), -1).float().contiguous()


WRITES = [
    # new tokens, positions, options
    ([1], [1], {}),
    ([1], [4097], dict(ps=64, n_kv=8, n_q=16)),
    ([3, 0, 18, 1], [3, 7, 40, 16], dict(ps=32, pad=5)),
    ([37, 200], [53, 200], dict(ps=128, n_kv=1, n_q=7, layout="lines")),
    ([700, 801], [700, 900], dict(ps=256, n_kv=8, n_q=16)),  # four vectors per half-warp
    ([0, 0, 1] * 30, [0, 5, 1] * 30, dict(n_kv=3, n_q=3)),   # more sequences than one round of the lookup
]


@pytest.mark.parametrize("inp", [F32, BF16, F16], ids=name)
@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv,opt", WRITES, ids=[str(i) for i in range(len(WRITES))])
@pytest.mark.parametrize("mode", ["norm+rope", "rope rows", "plain"])
def test_write_and_read_back(n, kv, opt, cache, typ, inp, mode):
    c = Cache(n, kv, cache=cache, typ=typ, junk=3.0, **opt)
    real, nq, nk = sum(n), c.n_q, c.n_kv
    stride = (nq + 2 * nk) * HD + 8
    qkv = torch.empty(c.total, stride, device="cuda", dtype=inp)
    qkv.copy_(c.randn(c.total, stride) * 3)
    if real > 2:
        qkv[1] = 0  # a token of zeros
    q_out = torch.full((c.total, nq * HD + 16), 5.0, device="cuda", dtype=typ)
    w = (1 + 0.3 * c.randn(HD), 1 + 0.3 * c.randn(HD)) if mode != "plain" else (None, None)
    rope = rope_table(max(kv) + 3) if mode != "plain" else None
    rows = torch.randint(0, max(kv) + 3, (c.total,), device="cuda", dtype=torch.int32) if mode == "rope rows" else None
    before = [c.k.clone(), c.v.clone()]
    c.write(qkv, q_out, q_norm=w[0], k_norm=w[1], rope=rope, rope_rows=rows, qkv_stride=stride, q_stride=nq * HD + 16)
    assert c.flags() == 0
    pos = torch.cat([torch.arange(b - a, b, device="cuda") for a, b in zip(n, kv)])
    x = qkv[:real, :stride - 8].double().view(real, nq + 2 * nk, HD)
    cs = None if rope is None else rope[rows[:real].long() if rows is not None else pos]
    q64, k64, v64 = turn64(x[:, :nq], w[0], cs, 1e-6), turn64(x[:, nq:nq + nk], w[1], cs, 1e-6), x[:, nq + nk:]
    # fp32 arithmetic: the norm's sum of 128 squares, its root and three products, then two products and a sum of the pair
    fp32 = 2.0 ** -24 * 160

    def pair(y):
        return y.abs() + y.roll(64, -1).abs()

    def rounded(y, t):
        h = torch.finfo(t).eps / 2
        return fp32 * pair(y) + h * (y.abs() + fp32 * pair(y)) + (2.0 ** -25 if t == F16 else 0)

    check_close(q_out[:real, :nq * HD].reshape(real, nq, HD), q64, rounded(q64, typ), "q")
    assert (q_out[:, nq * HD:] == 5).all() and (q_out[real:] == 5).all()  # gaps and rows behind the last sequence
    k32, v32 = c.read(F32, fill=9.0)
    for got, want, what in ((k32, k64, "k"), (v32, v64, "v")):
        assert (got[real:] == 9).all()
        got = got[:real]
        if cache == "q8":
            step = want.abs().amax(-1, keepdim=True) / 127
            # a code is off by half a step, the scale by the fp32 error of the row's largest value
            check_close(got, want, step * (0.5 + 127 * fp32 * 2 + 1e-4) + fp32 * pair(want) + 1e-30, what)
        else:
            check_close(got, want, rounded(want, cache), what)
        for t in (F16, BF16):  # the other types are one rounding of the same values
            a, b = c.read(t)
            assert torch.equal((a if what == "k" else b)[:real], got.to(t))
    # rows of nobody's new tokens stayed as they were
    mine = torch.zeros(c.k.shape[0], dtype=torch.bool, device="cuda")
    for s in range(len(n)):
        mine[c.cells(s, torch.arange(kv[s] - n[s], kv[s], device="cuda")).flatten()] = True
    assert torch.equal(c.k[~mine], before[0][~mine]) and torch.equal(c.v[~mine], before[1][~mine])


def test_q8_rows_of_zeros_tiny_values_nan_and_inf():
    c = Cache([6], [6], cache="q8", n_kv=1, n_q=1, junk=0.0)
    qkv = torch.zeros(6, 3 * HD, device="cuda")
    qkv[1] = torch.linspace(-1e-38, 1e-38, 3 * HD, device="cuda")   # scale below the normal numbers
    qkv[2] = torch.linspace(-1, 1, 3 * HD, device="cuda") * 3e38
    qkv[3, 2 * HD + 5] = float("nan")
    qkv[4, HD + 7] = float("inf")
    qkv[5, 2 * HD:] = -4.0
    c.write(qkv, None)
    k, v = c.read(F32)
    assert (k[0] == 0).all() and (v[0] == 0).all()
    for i in (1, 2):
        for got, want in ((k[i, 0], qkv[i, HD:2 * HD]), (v[i, 0], qkv[i, 2 * HD:])):
            assert ((got.double() - want.double()).abs() <= want.double().abs().max() / 127 * 0.502 + 1e-44).all()
    assert v[3].isnan().all() and not k[3].isnan().any()
    assert k[4].isnan().all() and not v[4].isnan().any()
    assert (v[5] + 4).abs().max() <= 4 * 2.0 ** -23


# ---- attention --------------------------------------------------------------------------------------------------------
ATTN = [
    # one token each: length one, below / at / above a page and a block, long enough to be shared by many CTAs
    ([1], [1], {}),
    ([1], [150], dict(n_kv=8, n_q=16)),
    ([1] * 7, [15, 16, 17, 63, 64, 65, 129], dict(ps=16)),
    ([1, 1], [5000, 3], dict(ps=64, n_kv=8, n_q=16)),
    ([1] * 40, [1 + 53 * i for i in range(40)], dict(ps=32, n_kv=4, n_q=32)),
    ([1], [20011], dict(ps=256, n_kv=1, n_q=16)),
    # idle sequences, empty ones, a token without any position, rows behind the last sequence
    ([0, 1, 0, 2, 0], [0, 9, 77, 200, 0], dict(pad=9)),
    ([1, 3, 1], [0, 1, 30], dict(ps=32)),
    # drafts: rows that fill a part of a tile, exactly one, and cross into the next
    ([2, 3, 4, 5], [100, 3, 260, 77], dict(n_kv=2, n_q=8)),
    ([7] * 5, [7, 60, 300, 1000, 2049], dict(n_kv=4, n_q=16, ps=128)),
    ([4, 5], [400, 500], dict(n_kv=2, n_q=6)),
    # odd groups: one query head per kv head, seven, all of sixteen, 128
    ([1, 9], [77, 9], dict(n_kv=3, n_q=3)),
    ([3, 1], [50, 301], dict(n_kv=1, n_q=7)),
    ([1, 2], [2000, 31], dict(n_kv=1, n_q=128)),
    # chunks and prompts
    ([20], [20], {}),
    ([64, 65, 63], [64, 200, 63], dict(n_kv=2, n_q=4)),
    ([130, 1, 257], [1000, 700, 257], dict(n_kv=2, n_q=8, ps=64, pad=3)),
    ([500], [2777], dict(n_kv=1, n_q=1, ps=32)),
    ([300, 33], [300, 5000], dict(n_kv=8, n_q=16, layout="lines")),
    ([1024], [1024], dict(n_kv=2, n_q=8, ps=128)),
    # tokens without a position among those that have one, in a draft and in a chunk
    ([9, 3, 2], [4, 0, 50], dict(n_kv=2, n_q=6)),
    ([100, 70, 300], [40, 0, 270], dict(n_kv=2, n_q=8)),
    # the widest groups: 256 query rows from one token
    ([1, 3], [200, 1000], dict(n_kv=1, n_q=256)),
]


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv,opt", ATTN, ids=[str(i) for i in range(len(ATTN))])
def test_attention_against_64_bits(n, kv, opt, cache, typ):
    c = Cache(n, kv, cache=cache, typ=typ, seed=len(n) + sum(kv), **opt).fill(scale=2.0)
    q = (c.randn(c.total, c.n_q, HD) * 2).to(typ)
    out = torch.full_like(q, 6.0)
    c.attend(q, out)
    assert c.flags() == 0
    want, bound = c.attend64(q)
    real = sum(n)
    check_close(out[:real], want[:real], bound[:real])
    assert (out[real:] == 6).all()
    again = c.attend(q, torch.zeros_like(q))
    assert torch.equal(again[:real], out[:real])  # the same bits every time


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
def test_peaked_and_extreme_scores(cache, typ):
    """Scores hundreds apart (one key takes all), maxima that rise with every block, V rows of very different sizes."""
    n, kv = [1, 40, 1], [700, 900, 333]
    c = Cache(n, kv, cache=cache, typ=typ, n_kv=2, n_q=4)
    ks = [c.randn(x, 2, HD) * torch.linspace(0.1, 6.0, x, device="cuda")[:, None, None] for x in kv]
    vs = [c.randn(x, 2, HD) * 10 ** (4 * torch.rand(x, 2, 1, device="cuda", generator=c.g) - 3) for x in kv]
    c.fill(ks, vs)
    q = (c.randn(c.total, 4, HD) * 4).to(typ)
    out = c.attend(q, scale=0.3)
    want, bound = c.attend64(q, 0.3)
    check_close(out, want, bound)


# ---- what a call may meet ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv", [([1, 1], [300, 500]), ([1], [9000]), ([9, 1], [300, 500]), ([150, 2], [700, 500])], ids=str)
def test_nan_and_infinity_reach_the_rows_that_see_them(n, kv, cache, typ):
    """A NaN query row, a NaN key of one sequence: NaN in exactly the rows that see it, nothing elsewhere."""
    c = Cache(n, kv, cache=cache, typ=typ).fill()
    q = c.randn(c.total, c.n_q, HD).to(typ)
    clean = c.attend(q).clone()
    q[0, 1] = float("nan")
    got = c.attend(q)
    assert got[0, 1].isnan().all()
    got[0, 1] = clean[0, 1]
    assert torch.equal(got, clean)
    q[0, 1] = 0
    cell = c.cells(0, torch.tensor([3], device="cuda"))[0, 1]  # position 3, kv head 1: seen by every token of sequence 0
    if cache == "q8":
        c.ks[cell] = float("nan")
    else:
        c.k[cell, 5] = float("nan")
    got = c.attend(q)
    assert got[:n[0], 2:].isnan().all() and not got[:n[0], :2].isnan().any() and not got[n[0]:].isnan().any()


@pytest.mark.parametrize("n", [1, 3, 90])
def test_a_later_tokens_poisoned_q8_row_does_not_reach_earlier_tokens(n):
    c = Cache([n], [n + 40], cache="q8").fill()
    q = c.randn(n, c.n_q, HD).half()
    clean = c.attend(q).clone()
    cell = c.cells(0, torch.tensor([n + 39], device="cuda"))[0]
    c.ks[cell], c.vs[cell] = float("nan"), float("nan")
    c.k[cell], c.v[cell] = 0, 0  # as icua_kv_write leaves a row that holds a NaN
    got = c.attend(q)
    assert got[n - 1].isnan().all() and torch.equal(got[:n - 1], clean[:n - 1])


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n", [[1, 1, 1], [5, 5, 5], [100, 40, 1]], ids=str)
def test_bad_pages_and_sequences_are_left_out_and_flagged(n, cache, typ):
    """Entries that only the device can see: nothing is read or written through them, the other sequences' rows do not
    change, the flags tell."""
    kv = [210, 205, 300]
    c = Cache(n, kv, cache=cache, typ=typ, junk=2.0).fill()
    q = c.randn(c.total, c.n_q, HD).to(typ)
    clean = c.attend(q).clone()
    assert c.flags() == 0
    rows = slice(n[0], n[0] + n[1])
    good = c.table.clone()
    for page in (-1, c.n_pages, -2**31, 2**31 - 1):
        c.table[1, 2] = page  # positions 32 .. 47 of sequence 1 are masked
        got = c.attend(q)
        assert c.flags() == L.FLAG_PAGE
        assert torch.equal(got[:n[0]], clean[:n[0]]) and torch.equal(got[n[0] + n[1]:], clean[n[0] + n[1]:])
        k, v = c.read(F32)
        c.err.zero_()
    c.table.copy_(good)
    # the same keys hidden by hand: scores of -inf through a second cache without them
    keep = torch.cat([torch.arange(32, device="cuda"), torch.arange(48, kv[1], device="cuda")])
    ks, vs = c.rows64("k", 1, keep), c.rows64("v", 1, keep)
    scale = 128 ** -0.5
    p = torch.einsum("thd,khd->thk", q[rows].double(), ks.repeat_interleave(2, 1)) * scale
    see = keep[None, :] <= (kv[1] - n[1] + torch.arange(n[1], device="cuda"))[:, None]
    p = torch.softmax(p.masked_fill(~see[:, None], -float("inf")), -1)
    want = torch.einsum("thk,khd->thd", p, vs.repeat_interleave(2, 1))
    _, bound = c.attend64(q)
    check_close(got[rows], want, bound[rows] * 2)
    # sequences that contradict themselves count as empty
    for change, undo in ((lambda: c.kv_len.__setitem__(1, -5), lambda: c.kv_len.__setitem__(1, kv[1])),
                         (lambda: c.kv_len.__setitem__(1, 2**31 - 1), lambda: c.kv_len.__setitem__(1, kv[1]))):
        change()
        out = c.attend(q, torch.full_like(q, 7))
        assert c.flags() == L.FLAG_SEQ
        assert torch.equal(out[:n[0]], clean[:n[0]]) and (out[rows] == 7).all() and torch.equal(out[rows.stop:], clean[rows.stop:])
        undo()
        c.err.zero_()
    c.cu[3] = c.total + 50  # past the row arrays
    out = c.attend(q, torch.full_like(q, 7))
    assert c.flags() == L.FLAG_SEQ and (out[rows.stop:] == 7).all() and torch.equal(out[:rows.stop], clean[:rows.stop])


def test_write_leaves_out_what_has_no_place():
    c = Cache([3, 2, 2], [20, 40, 1], cache=F16, n_kv=1, n_q=1, junk=4.0, ps=16)
    qkv = c.randn(7, 3 * HD)
    rope, rows = rope_table(8), torch.tensor([0, 7, 8, -1, 3, 0, 0], dtype=torch.int32, device="cuda")
    q = torch.full((7, HD), 9.0, device="cuda").half()
    c.table[1, 2] = -7  # the page of sequence 1's new tokens
    before = c.k.clone()
    c.write(qkv, q, rope=rope, rope_rows=rows)
    assert c.flags() == L.FLAG_SEQ | L.FLAG_PAGE
    # left out: tokens 2 and 3 (no table row), 5 (no position); token 4's cached row has no page, its q is written
    assert [bool((q[i] == 9).all()) for i in range(7)] == [False, False, True, True, False, True, False]
    changed = (c.k != before).any(-1).nonzero().flatten().tolist()
    want = c.cells(0, torch.tensor([17, 18], device="cuda")).flatten().tolist() + c.cells(2, torch.tensor([0], device="cuda")).flatten().tolist()
    assert sorted(changed) == sorted(want)


def test_more_tokens_than_promised():
    """max_q below a sequence's tokens: flagged and left alone where only the few-rows kernel runs, attended otherwise."""
    c = Cache([40, 1], [60, 60]).fill()
    q = c.randn(41, c.n_q, HD).half()
    want = c.attend(q).clone()
    out = c.attend(q, torch.full_like(q, 3), max_q=1)
    assert c.flags() == L.FLAG_SEQ
    assert (out[:40] == 3).all() and torch.equal(out[40], want[40])


@pytest.mark.parametrize("n,kv", [([1] * 3, [900, 50, 7000]), ([6, 1], [80, 4000]), ([200, 1, 70], [300, 900, 2000])], ids=str)
def test_strides_in_place_streams_and_graphs(n, kv):
    """q and out as slices of wider rows, out = q, a side stream, a captured call replayed with other lengths, two captured
    graphs with a scratch each running side by side."""
    c = Cache(n, kv, n_kv=2, n_q=8, typ=BF16, cache=BF16).fill()
    q = (c.randn(c.total, 8, HD) * 2).bfloat16()
    want = c.attend(q).clone()
    wide = torch.zeros(c.total, 8 * HD + 72, device="cuda", dtype=BF16)
    wide[:, :8 * HD] = q.view(c.total, -1)
    out = torch.full((c.total, 8 * HD + 8), 5.0, device="cuda", dtype=BF16)
    c.attend(wide, out, q_stride=8 * HD + 72, out_stride=8 * HD + 8)
    assert torch.equal(out[:, :8 * HD].reshape_as(q), want) and (out[:, 8 * HD:] == 5).all()
    same = q.clone()
    assert torch.equal(c.attend(same, same), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.attend(q, torch.zeros_like(q))
    side.synchronize()
    assert torch.equal(got, want)
    # capture; lengths change between replays, within what the descriptors say
    graphs, outs, keep = [], [], []
    for _ in range(2):
        g, o, sc = torch.cuda.CUDAGraph(), torch.zeros_like(q), c.scratch()
        with torch.cuda.graph(g):
            c.attend(q, o, scratch=sc)
        graphs.append(g)
        outs.append(o)
        keep.append(sc)
    torch.cuda.synchronize()
    c.kv_len -= 3
    c.kv = [x - 3 for x in kv]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for st in streams:
        st.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    ref, bound = c.attend64(q)
    for o in outs:
        check_close(o, ref, bound)
    assert torch.equal(outs[0], outs[1])


@pytest.mark.parametrize("cache", [F16, "q8"], ids=name)
def test_pool_offsets_past_32_bits(cache):
    """Pages at the far end of a pool of more than 2^32 bytes."""
    ps, n_kv, far = 256, 8, 9000 if cache == F16 else 18000
    c = Cache([1, 40], [300, 700], cache=cache, n_kv=n_kv, n_q=16, ps=ps, junk=0.0)
    small = [c.k, c.v, c.ks, c.vs]
    c.fill(scale=1.5)
    q = c.randn(41, 16, HD).half()
    want = c.attend(q).clone()
    rows = n_kv * ps
    assert far * rows * small[0].shape[1] * small[0].element_size() > 2**32
    for nm in ("k", "v", "ks", "vs"):
        t = getattr(c, nm)
        if t is not None:
            big = torch.empty((far + c.n_pages) * rows, *t.shape[1:], device="cuda", dtype=t.dtype)
            big[far * rows:] = t
            setattr(c, nm, big)
    c.table += far
    c.n_pages += far
    got = c.attend(q)
    assert c.flags() == 0 and torch.equal(got, want)
    k, v = c.read(F16)
    for x, w in ((k, "k"), (v, "v")):
        for s, (a, b) in enumerate(((0, 1), (1, 41))):
            pos = torch.arange(c.kv[s] - (b - a), c.kv[s], device="cuda")
            assert torch.equal(x[a:b], c.rows64(w, s, pos).half())
    qkv = c.randn(41, 32 * HD)
    c.write(qkv, None)
    k2, v2 = c.read(F32)
    assert (v2.view(41, -1) - qkv.view(41, 32, HD)[:, 24:].reshape(41, -1)).abs().max() < 0.04


def test_host_memory_is_refused():
    c = Cache([1], [5]).fill()
    q = c.randn(1, c.n_q, HD).half()
    for bad in ("k", "q"):
        host = torch.zeros(1 << 16, dtype=F16)
        p = c.pages(**({"k": ptr(host)} if bad == "k" else {}))
        sc, need = c.scratch()
        a = L.IcuaAttnPaged(q=ptr(host if bad == "q" else q), out=ptr(q), dtype=DT[F16], n_q=c.n_q, scratch=ptr(sc), scratch_bytes=need)
        assert L.lib().icua_attn_paged(C.byref(p), C.byref(c.seqs()), C.byref(a), None, None) == L.ERR_INVALID
        assert b"device memory" in L.lib().icua_global_error()


# ---- together ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
def test_prompts_then_decoding_together(cache, typ):
    """Three prompts written and attended in one call, then twelve single tokens for each, against causal attention over
    everything so far in 64 bits (from the rows the cache gives back)."""
    n_kv, n_q, ps = 2, 6, 16
    prompt, steps = [130, 1, 47], 12
    cap = [p + steps for p in prompt]
    c = Cache(prompt, cap, n_kv=n_kv, n_q=n_q, cache=cache, typ=typ, ps=ps)
    rope, w = rope_table(max(cap)), [1 + 0.2 * c.randn(HD), 1 + 0.2 * c.randn(HD)]
    done = [0, 0, 0]
    for step in range(1 + steps):
        n = prompt if step == 0 else [1, 1, 1]
        done = [a + b for a, b in zip(done, n)]
        c.n, c.kv, c.total = n, done, sum(n)
        c.cu = torch.tensor([0] + n).cumsum(0).to(torch.int32).cuda()
        c.kv_len = torch.tensor(done, dtype=torch.int32).cuda()
        qkv = c.randn(c.total, (n_q + 2 * n_kv) * HD) * 1.5
        q = torch.zeros(c.total, n_q, HD, device="cuda", dtype=typ)
        c.write(qkv, q, q_norm=w[0], k_norm=w[1], rope=rope)
        out = c.attend(q)
        assert c.flags() == 0
        want, bound = c.attend64(q)
        check_close(out, want, bound, f"step {step}")
        v32 = c.read(F32)[1]
        step_size = qkv.view(c.total, -1, HD)[:, n_q + n_kv:].abs().amax(-1, keepdim=True)
        half = 0.502 / 127 if cache == "q8" else torch.finfo(cache).eps / 2
        assert ((v32 - qkv.view(c.total, -1, HD)[:, n_q + n_kv:]).abs() <= half * step_size).all()


@pytest.mark.parametrize("cache,typ", TYPES, ids=name)
@pytest.mark.parametrize("n,kv", [([1] * 5, [700, 3, 5000, 64, 0]), ([6, 1, 3], [400, 6000, 3]), ([1], [9000]),
                                  ([90, 5, 1, 0], [90, 3000, 12, 7])], ids=str)
def test_the_length_hint_changes_no_result(n, kv, cache, typ):
    """max_kv only steers the split: far too small and far too large values give the same attention."""
    c = Cache(n, kv, cache=cache, typ=typ, n_kv=2, n_q=8).fill(scale=2.0)
    q = (c.randn(c.total, 8, HD) * 2).to(typ)
    want, bound = c.attend64(q)
    for hint in (0, 1, 1024, 4096, 1 << 20):
        check_close(c.attend(q, max_kv=hint), want, bound, f"max_kv {hint}")
    assert c.flags() == 0


@pytest.mark.parametrize("n", [1, 2, 100])
def test_v_rows_of_wildly_different_sizes(n):
    """Half of the probability on a row 10^32 times smaller than the other's: it adds nothing to the result, but it counts."""
    c = Cache([n], [n + 63], cache="q8", typ=BF16, n_kv=1, n_q=1)
    total = n + 63
    ks = torch.zeros(total, 1, HD, device="cuda")
    vs = torch.ones(total, 1, HD, device="cuda")
    vs[::2] *= 1e-32
    c.fill([ks], [vs * 3])
    q = c.randn(n, 1, HD).bfloat16()
    out = c.attend(q)
    pos = torch.arange(63, total, device="cuda")
    want = 3.0 * ((pos + 1) // 2).double() / (pos + 1).double()
    assert ((out.double() - want[:, None, None]).abs() <= want[:, None, None] * 2.0 ** -7).all()
