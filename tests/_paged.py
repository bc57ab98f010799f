"""A paged cache with its batch on the GPU, the calls on it, and the operators in 64 bits."""
import ctypes as C

import torch

from instantcua_b200 import _lib as L

HD = 128
DT = {torch.float32: L.DT_F32, torch.bfloat16: L.DT_BF16, torch.float16: L.DT_F16}
KV = {torch.float16: L.KV_F16, torch.bfloat16: L.KV_BF16, "q8": L.KV_Q8}


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """n: new tokens per sequence, kv: positions per sequence.  layout "pages": dense pages; "lines": pages laid over
    [head][positions][128] caches (page_rows = page size, head_rows = positions of all pages).  Rows of no sequence, and
    rows behind a sequence's end, hold `junk`."""

    def __init__(self, n, kv, *, n_kv=2, n_q=4, cache=torch.float16, typ=torch.float16, ps=16, pad=0, layout="pages",
                 junk=float("nan"), seed=0, max_pages=None):
        self.n, self.kv, self.n_kv, self.n_q, self.cache, self.typ, self.ps = list(n), list(kv), n_kv, n_q, cache, typ, ps
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g = g
        cpu = torch.Generator().manual_seed(seed + 1)
        pages = [-(-x // ps) for x in kv]
        self.n_pages = sum(pages) + 2
        self.max_pages = max_pages or max(pages + [1]) + 1
        order = torch.randperm(self.n_pages, generator=cpu)[: sum(pages)].tolist()
        table = torch.full((len(kv), self.max_pages), 1 << 30, dtype=torch.int32)
        at = 0
        for s, c in enumerate(pages):
            table[s, :c] = torch.tensor(order[at:at + c], dtype=torch.int32)
            at += c
        self.table = table.cuda()
        self.cu = torch.tensor([0] + list(n)).cumsum(0).to(torch.int32).cuda()
        self.kv_len = torch.tensor(list(kv), dtype=torch.int32).cuda()
        self.total = sum(n) + pad
        rows = self.n_pages * n_kv * ps
        if layout == "pages":
            self.page_rows, self.head_rows = n_kv * ps, ps
        else:
            self.page_rows, self.head_rows = ps, self.n_pages * ps
        self.strides = (0, 0) if layout == "pages" else (self.page_rows, self.head_rows)
        if cache == "q8":
            self.k = torch.randint(-128, 128, (rows, HD), device="cuda", generator=g, dtype=torch.int8)
            self.v = torch.randint(-128, 128, (rows, HD), device="cuda", generator=g, dtype=torch.int8)
            self.ks = torch.full((rows,), junk, device="cuda")
            self.vs = torch.full((rows,), junk, device="cuda")
        else:
            self.k = torch.full((rows, HD), junk, device="cuda", dtype=cache)
            self.v = torch.full((rows, HD), junk, device="cuda", dtype=cache)
            self.ks = self.vs = None
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")

    def randn(self, *shape):
        return torch.randn(*shape, device="cuda", generator=self.g)

    def cells(self, s, pos):
        """Pool rows [positions, kv head]."""
        page = self.table[s].long()[pos // self.ps]
        return page[:, None] * self.page_rows + torch.arange(self.n_kv, device="cuda") * self.head_rows + (pos % self.ps)[:, None]

    def fill(self, k=None, v=None, scale=1.0):
        """Puts values into every position of every sequence (given [sequence][positions, kv head, 128] lists, or random)."""
        for s, length in enumerate(self.kv):
            pos = torch.arange(length, device="cuda")
            cell = self.cells(s, pos)
            for name, given, mul in (("k", k, 1.0), ("v", v, scale)):
                x = given[s] if given is not None else self.randn(length, self.n_kv, HD) * mul
                if self.cache == "q8":
                    sc = x.abs().amax(-1) / 127
                    sc = torch.where(sc == 0, 1.0, sc)
                    getattr(self, name)[cell] = torch.round(x / sc[..., None]).to(torch.int8)
                    getattr(self, name + "s")[cell] = sc
                else:
                    d = torch.arange(HD, device="cuda")
                    place = ((d // 8) ^ (pos[:, None] % 8)) * 8 + d % 8
                    y = torch.empty_like(x).scatter_(-1, place[:, None, :].expand_as(x), x)
                    getattr(self, name)[cell] = y.to(self.cache)
        return self

    def rows64(self, which, s, pos):
        """Cached values of sequence s at positions pos, 64 bits [positions, kv head, 128]."""
        cell = self.cells(s, pos)
        x = getattr(self, which)[cell].double()
        if self.cache == "q8":
            return x * getattr(self, which + "s")[cell].double()[..., None]
        d = torch.arange(HD, device="cuda")
        place = ((d // 8) ^ (pos[:, None] % 8)) * 8 + d % 8
        return torch.gather(x, -1, place[:, None, :].expand_as(x))

    # ---- descriptors and calls
    def pages(self, **kw):
        d = dict(k=ptr(self.k), v=ptr(self.v), k_scale=ptr(self.ks), v_scale=ptr(self.vs), dtype=KV[self.cache], n_kv=self.n_kv,
                 page_size=self.ps, n_pages=self.n_pages, page_rows=self.strides[0], head_rows=self.strides[1])
        return L.IcuaKvPages(**{**d, **kw})

    def seqs(self, **kw):
        d = dict(n_seqs=len(self.n), total_q=self.total, max_q=max(self.n + [0]), max_kv=max(self.kv + [0]), cu_q=ptr(self.cu),
                 kv_len=ptr(self.kv_len), page_table=ptr(self.table), max_pages=self.max_pages)
        return L.IcuaKvSeqs(**{**d, **kw})

    def write(self, qkv, q_out, *, q_norm=None, k_norm=None, eps=1e-6, rope=None, rope_rows=None, qkv_stride=0, q_stride=0,
              stream=None):
        rows = L.IcuaKvRows(qkv=ptr(qkv), qkv_stride=qkv_stride, qkv_dtype=DT[qkv.dtype], n_q=self.n_q, q_norm=ptr(q_norm),
                            k_norm=ptr(k_norm), eps=eps, rope=ptr(rope), rope_rows=ptr(rope_rows),
                            rope_len=0 if rope is None else rope.shape[0], q_out=ptr(q_out), q_stride=q_stride,
                            q_dtype=DT[self.typ])
        L.check(L.lib().icua_kv_write(C.byref(self.pages()), C.byref(self.seqs()), C.byref(rows), ptr(self.err), stream))

    def read(self, dtype, k_out=None, v_out=None, fill=0.0):
        if k_out is None and v_out is None:
            k_out = torch.full((self.total, self.n_kv, HD), fill, device="cuda", dtype=dtype)
            v_out = torch.full_like(k_out, fill)
        L.check(L.lib().icua_kv_read(C.byref(self.pages()), C.byref(self.seqs()), ptr(k_out), ptr(v_out), DT[dtype], ptr(self.err),
                                     torch.cuda.current_stream().cuda_stream))
        return k_out, v_out

    def scratch(self, **kw):
        need = L.lib().icua_attn_paged_scratch_bytes(C.byref(self.pages()), C.byref(self.seqs(**kw)), self.n_q)
        assert need > 0
        return torch.full((need // 4 + 4,), float("nan"), device="cuda"), need

    def attend(self, q, out=None, *, scale=0.0, q_stride=0, out_stride=0, scratch=None, stream=None, **kw):
        out = torch.zeros_like(q) if out is None else out
        buf, need = scratch or self.scratch(**kw)
        a = L.IcuaAttnPaged(q=ptr(q), out=ptr(out), q_stride=q_stride, out_stride=out_stride, dtype=DT[self.typ], n_q=self.n_q,
                            scale=scale, scratch=ptr(buf), scratch_bytes=need)
        st = torch.cuda.current_stream().cuda_stream if stream is None else stream
        L.check(L.lib().icua_attn_paged(C.byref(self.pages()), C.byref(self.seqs(**kw)), C.byref(a), ptr(self.err), st))
        self.keep = buf
        return out

    def flags(self):
        torch.cuda.synchronize()
        return int(self.err.item())

    # ---- 64 bits
    def attend64(self, q, scale=None):
        """(output, bound) of the attention, by the formula in 64 bits.

        The bound, per element: the kernel rounds each probability (half a step of the type, relative to it) and the
        result (half a step); scores are fp32 sums of 128 products (128 roundings of 2^-24 relative to the sum of
        magnitudes, entering numerator and denominator), the exponential and the running sums fp32: per step of 16 keys
        2^-22 of the sum of magnitudes at most, and 32 steps' worth for scales, maxima and the join of parts.  Weights
        relative to the largest one (of p, or of p times the V scale in a q8 cache) that are below the type's normal
        numbers are off by up to 2^-25 in fp16 (half a subnormal step) and by up to 2^-126 in bf16 (the exponential
        flushes to zero there): for each key at most that much of the largest |v|."""
        scale = 128 ** -0.5 if scale is None else scale
        half = torch.finfo(self.typ).eps / 2
        tiny = 2.0 ** -25 if self.typ == torch.float16 else 2.0 ** -126
        out = torch.zeros(self.total, self.n_q, HD, dtype=torch.float64, device="cuda")
        bound = torch.zeros_like(out)
        grp, row = self.n_q // self.n_kv, 0
        for s, (n, kv) in enumerate(zip(self.n, self.kv)):
            pos = torch.arange(kv, device="cuda")
            k = self.rows64("k", s, pos).repeat_interleave(grp, 1).permute(1, 0, 2)
            v = self.rows64("v", s, pos).repeat_interleave(grp, 1).permute(1, 0, 2)
            for a in range(0, n, 256):
                e = min(n, a + 256)
                x = q[row + a:row + e].double().permute(1, 0, 2)
                z = x @ k.transpose(1, 2) * scale
                mag = (x.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * scale if kv else z.sum(-1, keepdim=True)
                see = pos[None, :] <= (kv - n + torch.arange(a, e, device="cuda"))[:, None]
                z = z.masked_fill(~see, -float("inf"))
                any_ = see.any(-1)[None, :, None]
                top = torch.where(any_, z.amax(-1, keepdim=True) if kv else z.sum(-1, keepdim=True), 0.0)
                p = torch.exp(z - top)
                p = p / torch.where(any_, p.sum(-1, keepdim=True), 1.0)
                o, m = p @ v, p @ v.abs()
                fp32 = 2 * 128 * 2.0 ** -24 * mag + (kv / 16 + 32) * 2.0 ** -22
                b = (half + fp32) * m + (tiny * kv * float(v.abs().max()) if kv else 0.0)
                out[row + a:row + e] = o.permute(1, 0, 2)
                bound[row + a:row + e] = (b + half * (o.abs() + b) + 2.0 ** -25 * (self.typ == torch.float16)).permute(1, 0, 2)
            row += n
        return out, bound


def check_close(got, want, bound, what=""):
    bad = ~((got.double() - want).abs() <= bound)  # (a NaN is bad)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}, " \
        f"worst {float(((got.double() - want).abs() / bound.clamp_min(1e-300)).nan_to_num(1e9).max()):.3g} x the bound"
