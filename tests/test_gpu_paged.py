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
