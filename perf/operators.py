"""Measured cases of the paged K/V cache operators: writing new tokens into the cache (per-head norms, rotation,
quantisation), reading it back, and the attention of new tokens over it.

The cache is a pool of pages, [page][kv head][position][128].  16-bit rows hold their sixteen 16-byte chunks in the
engine's cache order (chunk c at place c ^ (position & 7)); 8-bit rows hold int8 codes in plain order and one fp32
scale each.  A sequence's new tokens are its last ones: token i of n sits at position kv_len - n + i.
"""
import ctypes as C
import math
import random

import torch

own = False

HD = 128
_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_DT = {"f32": 0, "bf16": 1, "f16": 2}
_KV = {"f16": 0, "bf16": 1, "q8": 2}


# ---- cases -----------------------------------------------------------------------------------------------------
def _case(name, op, **kw):
    c = dict(op=op, nq=16, nkv=8, typ="f16", cache="f16", inp="f32", ps=16, seqs=1, qmin=1, qmax=1, cmin=0, cmax=0, pad=0,
             idle=0, mrope=False, mix=1)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the first tokens after a short prompt of one session: only latency counts
        _case("attn_decode_short", "attn", cmin=150, cmax=150),
        # batch-1 decode at 4K context, the benchmark's cache type
        _case("attn_decode_4k", "attn", typ="bf16", cache="bf16", ps=64, cmin=4095, cmax=4095),
        # 64 sessions at about 2K positions each (the batched benchmark), 8-bit cache
        _case("attn_decode_64x2k_q8", "attn", cache="q8", ps=32, seqs=64, cmin=1900, cmax=2100),
        # a serving batch of very different lengths, groups of four heads
        _case("attn_decode_ragged", "attn", nq=32, typ="bf16", cache="bf16", seqs=48, cmin=3, cmax=16000, mix=5),
        # drafted tokens checked together: a few new tokens for each of many sessions
        _case("attn_draft_24x7", "attn", nq=32, seqs=24, qmin=7, qmax=7, cmin=700, cmax=5000, ps=32),
        # a document's next chunk over a long 8-bit cache
        _case("attn_chunk_500_over_8k_q8", "attn", typ="bf16", cache="q8", ps=64, qmin=500, qmax=500, cmin=8001, cmax=8001),
        # prompts of different lengths and running sessions in one step; rows behind the last sequence
        _case("attn_mixed_step", "attn", seqs=12, qmin=1, qmax=600, cmin=0, cmax=3900, pad=37, mix=3),
        # one long prompt
        _case("attn_prompt_8k", "attn", nq=32, typ="bf16", cache="bf16", ps=128, qmin=8192, qmax=8192),
        # one token of one session into the engine's cache type
        _case("write_token", "write", cmin=4095, cmax=4095),
        # a prefill step's tokens into an 8-bit cache, each with its own row of the rotation table, and their rows back
        _case("write_prefill_q8", "write", nq=32, typ="bf16", cache="q8", inp="bf16", seqs=9, qmin=100, qmax=4000, cmin=0, cmax=900,
              ps=32, mrope=True, mix=2),
        # a few cached tokens handed to another program
        _case("read_few", "read", typ="bf16", cache="bf16", seqs=3, qmin=5, qmax=40, cmin=0, cmax=300),
        # 64 sessions' whole caches taken out
        _case("read_64x2k_q8", "read", cache="q8", ps=32, seqs=64, qmin=1901, qmax=2101),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _lens(case):
    """New tokens and earlier positions of each sequence: from the case alone."""
    r = random.Random(case["mix"])
    n = [_log(r, case["qmin"], case["qmax"]) for _ in range(case["seqs"])]
    c = [_log(r, case["cmin"] + 1, case["cmax"] + 1) - 1 for _ in range(case["seqs"])]
    if case["idle"]:  # sequences of the batch that bring no token this time
        n = [0 if i % case["idle"] == case["idle"] - 1 else x for i, x in enumerate(n)]
    return n, c


def _fits(case):
    n, c = _lens(case)
    kv = max(a + b for a, b in zip(n, c))
    if sum(a + b for a, b in zip(n, c)) * case["nkv"] > 6_000_000:
        return False
    if case["op"] == "attn":
        return case["seqs"] * case["nq"] * max(n) * kv <= 2_200_000_000 and case["seqs"] * kv * case["nkv"] <= 8_000_000
    return sum(n) * (case["nkv"] if case["op"] == "read" else case["nq"] + 2 * case["nkv"]) <= 1_200_000


def draw(rng):
    while True:
        op = rng.choice(["attn", "attn", "attn", "attn", "write", "read"])
        typ = rng.choice(["f16", "bf16"])
        nkv = rng.choice([1, 2, 4, 8, 8])
        case = _case(None, op, nkv=nkv, nq=nkv * rng.choice([1, 2, 2, 3, 4, 5, 7, 8, 16]), typ=typ,
                     cache=rng.choice([typ, "q8"]), inp=rng.choice(["f32", typ]), ps=rng.choice([16, 32, 64, 128, 256]),
                     seqs=_log(rng, 1, 100), pad=rng.choice([0, 0, rng.randint(1, 90)]), idle=rng.choice([0, 0, 0, 2, 3]), mrope=rng.random() < 0.3,
                     mix=rng.randrange(1 << 20))
        new = rng.choice([1, 1, _log(rng, 2, 12), _log(rng, 8, 6000)])
        case["qmin"], case["qmax"] = rng.choice([1, new, max(1, new // 3)]), new
        ctx = _log(rng, 1, 120_000) - 1
        case["cmin"], case["cmax"] = rng.choice([0, ctx, ctx // 2]), ctx
        if rng.random() < 0.25:  # prompts without a past
            case["cmin"] = case["cmax"] = 0
        if op == "read":
            case["qmax"] = _log(rng, 1, 20_000)
            case["qmin"] = min(case["qmin"], case["qmax"])
        if case["seqs"] < case["idle"]:
            case["idle"] = 0
        if _fits(case):
            return case


def work(case):
    n, c = _lens(case)
    new, kv = sum(n), sum(n) + sum(c)
    el = 2
    row = HD + 4 if case["cache"] == "q8" else 2 * HD  # one cached row
    nq, nkv = case["nq"], case["nkv"]
    if case["op"] == "attn":
        pairs = sum(a * b + a * (a + 1) // 2 for a, b in zip(n, c))
        return {"bytes": 2 * kv * nkv * row + 2 * new * nq * HD * el, "flops": 4 * HD * nq * pairs}
    if case["op"] == "read":
        return {"bytes": 2 * new * nkv * (row + HD * el), "flops": 2 * new * nkv * HD}
    inp = 4 if case["inp"] == "f32" else 2
    b = new * ((nq + 2 * nkv) * HD * inp + nq * HD * el + 2 * nkv * row)
    if case["cache"] == "q8":  # read back
        b += 2 * new * nkv * (row + HD * el)
    return {"bytes": b, "flops": new * (nq + nkv) * HD * 8}


# ---- what a program has in hand ---------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    cpu = torch.Generator().manual_seed(seed)
    n, c = _lens(case)
    nq, nkv, ps = case["nq"], case["nkv"], case["ps"]
    typ, ns = _T[case["typ"]], case["seqs"]
    kv = [a + b for a, b in zip(n, c)]
    pages = [-(-x // ps) for x in kv]
    n_pages, max_pages = sum(pages) + 3, max(pages) + 1
    order = torch.randperm(n_pages, generator=cpu)[: sum(pages)].to(torch.int32)
    table = torch.full((ns, max_pages), -1, dtype=torch.int32)  # entries behind a sequence's end name no page
    cut = torch.tensor(pages)
    table[torch.arange(max_pages)[None, :] < cut[:, None]] = order
    cu = torch.tensor([0] + n).cumsum(0).to(torch.int32)
    total = sum(n) + case["pad"]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32).to(dtype)

    s = dict(case=case, table=table.to(dev), cu=cu.to(dev), kv_len=torch.tensor(kv, dtype=torch.int32, device=dev), total=total,
             max_q=max(n), max_kv=max(kv), max_pages=max_pages, n_pages=n_pages)
    shape = (n_pages, nkv, ps, HD)
    # cached keys are normalised and rotated vectors, values plain projections; rows of no sequence hold what was there before
    if case["cache"] == "q8":
        for x in ("k", "v"):
            s[x] = torch.randint(-127, 128, shape, device=dev, generator=g, dtype=torch.int8)
            s[x + "_scale"] = torch.rand(shape[:3], device=dev, generator=g) * 0.02 + 0.008
    else:
        for x in ("k", "v"):
            s[x] = normal(*shape, dtype=typ)
    if case["op"] == "attn":
        s["q"] = normal(total, nq, HD, dtype=typ)
        s["q"] *= 1.7
        s["out"] = torch.zeros(total, nq, HD, device=dev, dtype=typ)
    else:
        s["k_out"] = torch.zeros(total, nkv, HD, device=dev, dtype=typ)
        s["v_out"] = torch.zeros(total, nkv, HD, device=dev, dtype=typ)
    if case["op"] == "write":
        s["qkv"] = normal(total, nq + 2 * nkv, HD, dtype=_T[case["inp"]])
        s["q_norm"] = 1 + 0.2 * normal(HD)
        s["k_norm"] = 1 + 0.2 * normal(HD)
        top = max(kv) + 40
        freq = 5e6 ** (-torch.arange(64, device=dev, dtype=torch.float64) / 64)
        angle = torch.arange(top, device=dev, dtype=torch.float64)[:, None] * freq
        s["rope"] = torch.stack((angle.cos(), angle.sin()), -1).to(torch.float32).contiguous()
        # image rows turn by their place in the grid: a row of the table for each token
        s["rope_rows"] = torch.randint(0, top, (total,), device=dev, generator=g, dtype=torch.int32) if case["mrope"] else None
        s["q_out"] = torch.zeros(total, nq, HD, device=dev, dtype=typ)
    if own:
        s["call"] = _bind(s)
    return s


# ---- plain form ---------------------------------------------------------------------------------------------------
def _tokens(s):
    """For each row: its sequence, its position, and whether it is any sequence's."""
    cu, kv = s["cu"].long(), s["kv_len"].long()
    t = torch.arange(s["total"], device=cu.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = seq < kv.numel()
    seq = seq.clamp(max=kv.numel() - 1)
    return seq, kv[seq] - (cu[seq + 1] - cu[seq]) + t - cu[seq], real


def _cells(s, seq, pos):
    """Row of the pool, viewed as [rows, 128], of every kv head at positions `pos` of sequences `seq`: [..., nkv]."""
    ps, nkv = s["case"]["ps"], s["case"]["nkv"]
    page = s["table"].long()[seq, pos // ps]
    return (page[..., None] * nkv + torch.arange(nkv, device=pos.device)) * ps + (pos % ps)[..., None]


def _order(pos):
    """Where element d of a 16-bit row at position pos is kept."""
    d = torch.arange(HD, device=pos.device)
    return (((d // 8) ^ (pos[..., None] % 8)) * 8) + d % 8


def _fetch(s, which, seq, pos):
    """Cached rows in 32 bits, [..., nkv, 128]."""
    cell = _cells(s, seq, pos)
    x = s[which].view(-1, HD)[cell]
    if s["case"]["cache"] == "q8":
        return x.float() * s[which + "_scale"].view(-1)[cell][..., None]
    return torch.gather(x, -1, _order(pos)[..., None, :].expand(x.shape)).float()


def _plain_attn(s):
    case = s["case"]
    nq, nkv, ns = case["nq"], case["nkv"], case["seqs"]
    grp, mq, mk = nq // nkv, s["max_q"], s["max_kv"]
    seq, pos, real = _tokens(s)
    j = torch.arange(mk, device=pos.device)
    all_seq = torch.arange(ns, device=pos.device)[:, None].expand(ns, mk)
    held = j[None, :] < s["kv_len"][:, None]
    at = torch.where(held, j[None, :], 0)
    k = _fetch(s, "k", all_seq, at).permute(0, 2, 3, 1)  # [seq, kv head, 128, key]
    v = _fetch(s, "v", all_seq, at).permute(0, 2, 1, 3)
    seq, pos = seq[real], pos[real]
    i = pos - (s["kv_len"][seq] - (s["cu"][seq + 1] - s["cu"][seq]))  # place among the sequence's new tokens
    q = torch.zeros(ns, mq, nq, HD, device=pos.device)
    q[seq, i] = s["q"][real].float()
    q = q.view(ns, mq, nkv, grp, HD).permute(0, 2, 1, 3, 4).reshape(ns, nkv, mq * grp, HD)
    p = torch.matmul(q, k).view(ns, nkv, mq, grp, mk)
    p *= 1.0 / math.sqrt(HD)
    last = torch.full((ns, mq), -1, device=pos.device, dtype=torch.long)
    last[seq, i] = pos
    p.masked_fill_((j > last[..., None])[:, None, :, None, :], -math.inf)
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(ns, nkv, mq * grp, mk), v).view(ns, nkv, mq, grp, HD)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 2, 1, 3, 4).reshape(ns, mq, nq, HD)
    out = torch.zeros_like(s["q"])
    out[real] = o[seq, i].to(out.dtype)
    return out


def _norm_turn(x, w, cs):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    a, b, c, t = x[..., :64], x[..., 64:], cs[:, None, :, 0], cs[:, None, :, 1]
    return torch.cat((a * c - b * t, b * c + a * t), -1)


def _plain_write(s):
    case = s["case"]
    nq, nkv = case["nq"], case["nkv"]
    typ = _T[case["typ"]]
    seq, pos, real = _tokens(s)
    seq, pos = seq[real], pos[real]
    x = s["qkv"][real].float()
    cs = s["rope"][s["rope_rows"][real].long() if s["rope_rows"] is not None else pos]
    q_out = torch.zeros_like(s["q_out"])
    q_out[real] = _norm_turn(x[:, :nq], s["q_norm"], cs).to(typ)
    rows = {"k": _norm_turn(x[:, nq:nq + nkv], s["k_norm"], cs), "v": x[:, nq + nkv:]}
    cell = _cells(s, seq, pos)
    if case["cache"] != "q8":
        place = _order(pos)[:, None, :].expand(-1, nkv, -1)
        keep = {w: torch.empty_like(r).scatter_(-1, place, r) for w, r in rows.items()}
        s["k"].view(-1, HD)[cell] = keep["k"].to(typ)
        s["v"].view(-1, HD)[cell] = keep["v"].to(typ)
        return q_out, s["k"], s["v"]
    scale = {w: r.abs().amax(-1) / 127.0 for w, r in rows.items()}
    scale = {w: torch.where(r == 0, 1.0, r) for w, r in scale.items()}
    code = {w: torch.round(rows[w] / scale[w][..., None]) for w in rows}
    s["k"].view(-1, HD)[cell] = code["k"].to(torch.int8)
    s["v"].view(-1, HD)[cell] = code["v"].to(torch.int8)
    s["k_scale"].view(-1)[cell] = scale["k"]
    s["v_scale"].view(-1)[cell] = scale["v"]
    return (q_out, *_plain_read(s))


def _plain_read(s):
    seq, pos, real = _tokens(s)
    k, v = torch.zeros_like(s["k_out"]), torch.zeros_like(s["v_out"])
    k[real] = _fetch(s, "k", seq[real], pos[real]).to(k.dtype)
    v[real] = _fetch(s, "v", seq[real], pos[real]).to(v.dtype)
    return k, v


# ---- the framework's calls ----------------------------------------------------------------------------------------
def _bind(s):
    """The descriptors that a program keeps for its cache, its batch and its row buffers."""
    from instantcua_b200 import _lib as L

    case, lib = s["case"], L.lib()
    ptr = lambda x: None if x is None else x.data_ptr()  # noqa: E731
    pages = L.IcuaKvPages(k=ptr(s["k"]), v=ptr(s["v"]), k_scale=ptr(s.get("k_scale")), v_scale=ptr(s.get("v_scale")),
                          dtype=_KV[case["cache"]], n_kv=case["nkv"], page_size=case["ps"], n_pages=s["n_pages"])
    seqs = L.IcuaKvSeqs(n_seqs=case["seqs"], total_q=s["total"], max_q=s["max_q"], max_kv=s["max_kv"], cu_q=ptr(s["cu"]),
                        kv_len=ptr(s["kv_len"]), page_table=ptr(s["table"]), max_pages=s["max_pages"])
    d = dict(lib=lib, check=L.check, pages=C.byref(pages), seqs=C.byref(seqs), keep=[pages, seqs])
    if case["op"] == "attn":
        need = lib.icua_attn_paged_scratch_bytes(C.byref(pages), C.byref(seqs), case["nq"])
        d["scratch"] = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
        args = L.IcuaAttnPaged(q=ptr(s["q"]), out=ptr(s["out"]), dtype=_DT[case["typ"]], n_q=case["nq"],
                               scratch=ptr(d["scratch"]), scratch_bytes=need)
    else:
        args = L.IcuaKvRows(qkv=ptr(s.get("qkv")), qkv_dtype=_DT[case["inp"]], n_q=case["nq"], q_norm=ptr(s.get("q_norm")),
                            k_norm=ptr(s.get("k_norm")), eps=1e-6, rope=ptr(s.get("rope")), rope_rows=ptr(s.get("rope_rows")),
                            rope_len=s["rope"].shape[0] if "rope" in s else 0, q_out=ptr(s.get("q_out")),
                            q_dtype=_DT[case["typ"]])
        d["read"] = (ptr(s["k_out"]), ptr(s["v_out"]), _DT[case["typ"]])
    d["keep"].append(args)
    d["args"] = C.byref(args)
    return d


def _own_run(s):
    d, op = s["call"], s["case"]["op"]
    lib, stream = d["lib"], torch.cuda.current_stream().cuda_stream
    if op == "attn":
        d["check"](lib.icua_attn_paged(d["pages"], d["seqs"], d["args"], None, stream))
        return s["out"]
    if op == "read":
        d["check"](lib.icua_kv_read(d["pages"], d["seqs"], *d["read"], None, stream))
        return s["k_out"], s["v_out"]
    d["check"](lib.icua_kv_write(d["pages"], d["seqs"], d["args"], None, stream))
    if s["case"]["cache"] != "q8":
        return s["q_out"], s["k"], s["v"]
    d["check"](lib.icua_kv_read(d["pages"], d["seqs"], *d["read"], None, stream))
    return s["q_out"], s["k_out"], s["v_out"]


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attn, "write": _plain_write, "read": _plain_read}[state["case"]["op"]](state)


# ---- 64 bits ------------------------------------------------------------------------------------------------------
def _line(s, which, b, first, last):
    """Positions [first, last) of sequence b in 64 bits, [kv head, positions, 128], page by page."""
    case, ps = s["case"], s["case"]["ps"]
    table = s["table"][b].tolist()
    part = []
    for p in range(first // ps, -(-last // ps)):
        x = s[which][table[p]].double()
        if case["cache"] == "q8":
            x = x * s[which + "_scale"][table[p]].double()[..., None]
        else:
            x = x.view(case["nkv"], ps // 8, 8, 16, 8)
            x = torch.stack([x[:, :, r][:, :, [c ^ r for c in range(16)]] for r in range(8)], 2).reshape(case["nkv"], ps, HD)
        part.append(x)
    x = torch.cat(part, 1) if part else torch.zeros(case["nkv"], 0, HD, dtype=torch.float64, device="cuda")
    lo = first // ps * ps
    return x[:, first - lo:last - lo]


def exact(case, seed):
    s = prepare(case, seed)
    n, c = _lens(case)
    nq, nkv = case["nq"], case["nkv"]
    grp = nq // nkv
    dev, f8 = "cuda", torch.float64
    if case["op"] == "attn":
        out = torch.zeros(s["total"], nq, HD, dtype=f8, device=dev)
        row = 0
        for b in range(case["seqs"]):
            k, v = (_line(s, w, b, 0, n[b] + c[b]).repeat_interleave(grp, 0) for w in ("k", "v"))
            for a in range(0, n[b], 512):
                e = min(n[b], a + 512)
                q = s["q"][row + a:row + e].double().transpose(0, 1)
                see = c[b] + e
                z = q @ k[:, :see].transpose(1, 2) / math.sqrt(HD)
                hide = torch.ones(e - a, see, dtype=torch.bool, device=dev).triu(c[b] + a + 1)
                out[row + a:row + e] = (torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v[:, :see]).transpose(0, 1)
            row += n[b]
        return out
    if case["op"] == "read":
        got = [torch.zeros(s["total"], nkv, HD, dtype=f8, device=dev) for _ in range(2)]
        row = 0
        for b in range(case["seqs"]):
            for w, o in zip(("k", "v"), got):
                o[row:row + n[b]] = _line(s, w, b, c[b], c[b] + n[b]).transpose(0, 1)
            row += n[b]
        return tuple(got)
    q_out = torch.zeros(s["total"], nq, HD, dtype=f8, device=dev)
    k_out, v_out = (torch.zeros(s["total"], nkv, HD, dtype=f8, device=dev) for _ in range(2))
    row = 0
    for b in range(case["seqs"]):
        x = s["qkv"][row:row + n[b]].double()
        at = s["rope_rows"][row:row + n[b]].long() if s["rope_rows"] is not None else torch.arange(c[b], c[b] + n[b], device=dev)
        turn = torch.view_as_complex(s["rope"].double()[at])[:, None]

        def head(y, w):
            y = y / (y.pow(2).sum(-1, keepdim=True) / HD + 1e-6).sqrt() * w.double()
            z = torch.complex(y[..., :64].contiguous(), y[..., 64:].contiguous()) * turn
            return torch.cat((z.real, z.imag), -1)

        q_out[row:row + n[b]] = head(x[:, :nq], s["q_norm"])
        k_out[row:row + n[b]] = head(x[:, nq:nq + nkv], s["k_norm"])
        v_out[row:row + n[b]] = x[:, nq + nkv:]
        row += n[b]
    if case["cache"] == "q8":
        for o in (k_out, v_out):
            step = o.abs().max(-1, keepdim=True).values / 127
            step[step == 0] = 1
            o.copy_((o / step).round() * step)
        return q_out, k_out, v_out
    pool = {"k": s["k"].double(), "v": s["v"].double()}
    row, ps = 0, case["ps"]
    for b in range(case["seqs"]):
        pos = torch.arange(c[b], c[b] + n[b], device=dev)
        page, r = s["table"][b].long()[pos // ps], pos % ps
        for w, o in (("k", k_out), ("v", v_out)):
            x = o[row:row + n[b]].view(n[b], nkv, 16, 8)
            for chunk in range(16):
                at = ((chunk ^ (pos % 8)) * 8)[:, None] + torch.arange(8, device=dev)
                pool[w][page[:, None, None], torch.arange(nkv, device=dev)[None, :, None], r[:, None, None], at[:, None, :]] = x[:, :, chunk]
        row += n[b]
    return q_out, pool["k"], pool["v"]
