// Attention of new tokens over a paged K/V cache, few query rows per kv head (single tokens, drafts):
// warp-level MMA, memory bound.
//
//   o_i = sum_{j <= pos_i} softmax_j(scale q_i . k_j) v_j,   pos_i = kv_len - n + i
//
// The n new tokens of a sequence and the G = n_q / n_kv query heads of a kv head form n G query rows
// over the same keys (row r = token r / G, head r % G); an item is 16 of them over one (sequence, kv
// head), the M of mma.sync.m16n8k16, so every K/V byte is read once for all rows of the tile.
//
// Bound: HBM (4 G FLOP per cached byte and row).  What follows from it:
// * The items' blocks (64 keys, 128 in a q8 cache) are dealt evenly over the CTAs, two or three per SM, as one
//   line: by the real lengths, read on the device, so a batch of very different lengths leaves no SM
//   idle.  A CTA that holds a part of an item writes (max, sum, output) to the workspace, and
//   paged_attn_join_kernel folds an item's parts in the order of their keys: the same bits every run.
// * Each of the four warps streams its own sixteen (q8: 32) rows of a block through a ring of two or three
//   slots with 16-byte cp.async, and runs its own online softmax; only the end of an item meets in
//   shared memory.  Rows behind the sequence's end are never read: cp.async fills zeros, so whatever a
//   page still holds there (NaN included) cannot reach a sum.
// * q8 rows are converted in registers, exactly: code -> 16-bit float by placing the byte in the
//   mantissa of 1024 (fp16) or 128 / 256 (bf16) and subtracting.  The scales add no rounding of their own: the
//   K scale multiplies the fp32 score; the V scale enters the exponent, p' = 2^(s + log2 vs - m') with
//   m' the running maximum of that sum, so the 16-bit operand of the P V product lies in [0, 256] whatever
//   the scales are, and the row sum is l = sum p' / vs.  (In fp16 a p' below 2^-14 is a subnormal number, off by
//   up to 2^-25: less than that much of the largest |v| that counts.)
// The running maximum is only moved (and the output rescaled) when a score exceeds it by more than 2^8: the
// rescale is then rare, and p below 256 is as precise in 16 bits as p below 1.
// Scores, maxima, sums and outputs are fp32; p is rounded once to the 16-bit type of q.
//
// Measured on a B200 (6.54 TB/s by copy): 48 single tokens over 3 .. 16,000 positions, 32:8 heads, bf16, 76 us =
// 5.5 TB/s; 64 over about 2,000 positions, 16:8 heads, q8, 72 us = 3.8 TB/s, bound by the conversions (half of
// the issue slots at three warps per scheduler); 24 drafts of 7 tokens, 32:8 heads, fp16, 56 us = 3.5 TB/s, bound
// by latency (the two tiles' registers leave two warps per scheduler); one token over 4,096 positions, 16:8
// heads, bf16, in a cluster per kv head 10.3 us against 12.3 us dealt as a line and joined.
#pragma once
#include "paged.cuh"
#include "tcgen05.cuh"

namespace icua {

constexpr int PA_ROWS_MAX = 32;   // query rows per item: 16 or 32
constexpr int pa_warps(int cl) { return cl > 1 ? 8 : 4; }  // (a cluster's CTAs have their SM to themselves)
constexpr int PA_ITEM = 3;        // (ragged decode / drafts of the figures above: 1: 85 / 59 us, 2: 76 / 58, 4: 76 / 55)
constexpr int PA_CLUSTER = 8;     // CTAs that share an item in the small-batch form
constexpr int PA_MAX_CTAS = 480;  // workspace slots are laid out for so many
constexpr int PA_MAX_SEQS = 1024;
// What a CTA leaves for the join: the item that it began and did not end.
struct PaSplit {
    int n_parts;  // CTAs that worked on it (0: nothing to join), this one first
    int first, rows;  // the tile's first row among the sequence's, its rows
    int q0, h;
    int pad[3];
};
constexpr int PA_PART = PA_ROWS_MAX * HD + 2 * PA_ROWS_MAX;  // floats of a part: o[32][128], m[32], l[32]

struct PagedAttnParams {
    PagesView pages;
    SeqsView seqs;
    const void* q;
    void* out;
    long long q_stride, out_stride;
    int group;
    float scale_log2;  // softmax scale x log2(e)
    int max_rows;      // sequences with more rows (n G) than this belong to another kernel,
    int alone;         //   or, when there is none in this call, break the caller's max_q (ERR_SEQ)
    float* part;       // [gridDim.x][2][PA_PART]: 0 = an item begun by an earlier CTA, 1 = an item begun here
    PaSplit* split;    // [gridDim.x]
    int* err;
};

constexpr int pa_keys(bool q8) { return q8 ? 32 : 16; }  // rows of a warp's slot
constexpr int pa_block(bool q8, int cl) { return pa_warps(cl) * pa_keys(q8); }
constexpr int pa_slot(bool q8) { return q8 ? 32 * 2 * HD + 2 * 32 * 4 : 16 * 2 * HD * 2; }
// CTAs per SM and ring slots per warp.  Sixteen rows of a q8 cache: three CTAs (their fragments' conversion is
// a chain of dependent instructions, which more warps hide), with the q fragments in shared memory to fit the
// registers.  Else two, which stream a 16-bit cache at HBM speed.
constexpr int pa_ctas(bool q8, int mt, int cl) { return cl > 1 ? 1 : q8 && mt == 1 ? 3 : 2; }
constexpr int pa_ns(bool q8, int mt, int cl) { return pa_ctas(q8, mt, cl) == 2 ? 3 : 2; }
constexpr bool pa_q_in_smem(bool q8, int mt) { return mt > 1 || q8; }
constexpr int pa_smem(bool q8, int mt, int cl) {
    return pa_warps(cl) * pa_ns(q8, mt, cl) * pa_slot(q8) + (pa_q_in_smem(q8, mt) ? mt * 16 * 2 * HD : 0) + (cl == 1 ? (PA_MAX_SEQS + 1) * 4 : 0);
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The float that CTA `rank` of the cluster has where `here` is in this one.
__device__ __forceinline__ float ld_cluster(const float* here, uint32_t rank) {
    const uint32_t a = smem_u32(here);
    uint32_t ra;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(a), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(ra));
    return v;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two int8 codes in bytes 0 and 2 of w (anything in bytes 1 and 3) as a pair of 16-bit floats, exactly.
template <typename T>
__device__ __forceinline__ uint32_t codes_to_pair(uint32_t w);
template <>
__device__ __forceinline__ uint32_t codes_to_pair<__half>(uint32_t w) {
    // 1024 + (code + 128), minus 1152
    const uint32_t u = (w & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&u), __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <>
__device__ __forceinline__ uint32_t codes_to_pair<__nv_bfloat16>(uint32_t w) {
    // 128 + the low seven bits, minus 128 or, for a negative code, 256
    const uint32_t a = (w & 0x007f007fu) | 0x43004300u, b = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}

__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// The line of work: sequence s holds items(s) (item = kv head x tiles + tile) of PA_ITEM + nb(s) units, the
// first PA_ITEM for beginning and ending an item, then one per block of keys.  (Without them the CTAs that get
// the short sequences of a ragged batch have several times the others' work.)
struct PaWork {
    int n, kv, q0, tiles, nb, items;
    __device__ __forceinline__ int units() const { return nb + PA_ITEM; }
};
__device__ __forceinline__ PaWork pa_work(const SeqsView& S, int ps_shift, int n_kv, int group, int max_rows, int tile_rows,
                                          int block, int s, int* err, bool alone = false) {
    const SeqInfo q = load_seq(S, ps_shift, s, err);
    PaWork w{q.n, q.kv, q.q0, 0, 0, 0};
    const long long rows = (long long)q.n * group;
    if (rows > 0 && rows <= max_rows) {
        w.tiles = (int)((rows + tile_rows - 1) / tile_rows);
        w.items = w.tiles * n_kv;
        w.nb = max(1, (q.kv + block - 1) / block);  // an item without keys still writes its (zero) rows
    } else if (rows > 0 && alone && err) {
        atomicOr(err, ERR_SEQ);
    }
    return w;
}

__device__ __forceinline__ uint32_t add_sat(uint32_t a, uint32_t b) { return a + b < a ? 0xffffffffu : a + b; }

// pre[s] = units before sequence s, pre[n_seqs] = all of them.  `warp_tot` holds one word per warp.  Offsets that
// contradict each other can claim the same rows many times over, so that the units pass 32 bits although the call's
// check of its sizes holds: the sums stop at the largest word, and such a batch counts as one without tokens.
template <int THREADS>
__device__ __forceinline__ uint32_t pa_prefix(const SeqsView& S, int ps_shift, int n_kv, int group, int max_rows, int tile_rows,
                                              int block, uint32_t* pre, uint32_t* warp_tot, int* err, bool alone = false) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t base = 0;
    for (int s0 = 0; s0 < S.n_seqs; s0 += THREADS) {
        const int s = s0 + tid;
        uint32_t w = 0;
        if (s < S.n_seqs) {
            const PaWork k = pa_work(S, ps_shift, n_kv, group, max_rows, tile_rows, block, s, err, alone);
            w = (uint32_t)min((unsigned long long)k.items * (unsigned long long)k.units(), 0xffffffffull);
        }
        uint32_t x = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x = add_sat(x, y);
        }
        if (lane == 31) warp_tot[warp] = x;
        __syncthreads();
        uint32_t before = base, all = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) {
            if (i < warp) before += warp_tot[i];
            all = add_sat(all, warp_tot[i]);
        }
        if (s < S.n_seqs) pre[s] = before + x - w;
        base = add_sat(base, all);
        __syncthreads();
    }
    if (base == 0xffffffffu) {
        if (tid == 0 && err) atomicOr(err, ERR_SEQ);
        return 0;
    }
    if (tid == 0) pre[S.n_seqs] = base;
    __syncthreads();
    return base;
}

__device__ __forceinline__ int pa_find(const uint32_t* pre, int n, uint32_t x) {  // last s with pre[s] <= x
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int m = (lo + hi) >> 1;
        if (pre[m] <= x) lo = m;
        else hi = m;
    }
    return lo;
}

// The line dealt to the CTAs: the first r take q + 1 blocks, the others q (none past the end of a line
// that is shorter than the grid).
struct PaDeal {
    uint32_t q, r;
    __device__ __forceinline__ PaDeal(uint32_t total, uint32_t ctas) : q(total / ctas), r(total % ctas) {}
    __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * q + min(c, r); }
    __device__ __forceinline__ uint32_t cta_of(uint32_t x) const {
        const uint32_t lead = r * (q + 1);
        return x < lead ? x / (q + 1) : r + (x - lead) / max(q, 1u);
    }
};

// MT: tiles of sixteen query rows per item that share every K and V fragment.
// CL = 1: the line and a join.  CL > 1 (few sequences of moderate length): the cluster's CL CTAs share one item,
// (sequence, kv head) of the cluster's number, and join its parts through distributed shared memory.  CL = 0
// (many short sequences): a CTA per item.  The last two are one launch without workspace, for calls whose
// time is latency.
template <typename T, bool Q8, int MT, int CL>
__global__ void __launch_bounds__(32 * pa_warps(CL), pa_ctas(Q8, MT, CL)) paged_attn_kernel(const PagedAttnParams p) {
    constexpr bool LINE = CL == 1;
    constexpr int CN = CL > 1 ? CL : 1;  // CTAs that share an item
    constexpr int PA_WARPS = pa_warps(CL), PA_THREADS = 32 * PA_WARPS, PA_NS = pa_ns(Q8, MT, CL);
    constexpr bool QS = pa_q_in_smem(Q8, MT);
    constexpr int KEYS = pa_keys(Q8), BLOCK = pa_block(Q8, CL), SLOT = pa_slot(Q8), NT = KEYS / 8, ROWS = 16 * MT;
    constexpr int ROW = Q8 ? HD : 2 * HD;  // bytes of a cached row
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float ml[PA_WARPS][2][ROWS];
    __shared__ float ml_c[2][ROWS];  // CL > 1: this CTA's part's
    __shared__ uint32_t warp_tot[PA_WARPS];
    uint8_t* q_tile = smem + PA_WARPS * PA_NS * SLOT;  // QS: the rows of the item, 256 B each, chunk c at c ^ (row & 7)
    uint32_t* pre = reinterpret_cast<uint32_t*>(q_tile + (QS ? ROWS * 2 * HD : 0));
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int ps_shift = p.pages.ps_shift, n_kv = p.pages.n_kv, G = p.group;

    struct Cursor {  // a block of keys of an item
        int s, item, b;
        PaWork w;
    };
    auto work_of = [&](int s, int* err) { return pa_work(p.seqs, ps_shift, n_kv, G, p.max_rows, ROWS, BLOCK, s, err, p.alone != 0); };
    Cursor f{}, end{};  // this CTA's first block, and the one after its last
    if (LINE) {
        const uint32_t total = pa_prefix<PA_THREADS>(p.seqs, ps_shift, n_kv, G, p.max_rows, ROWS, BLOCK, pre, warp_tot,
                                                     blockIdx.x == 0 ? p.err : nullptr, p.alone != 0);
        const PaDeal deal(total, gridDim.x);
        const uint32_t x0 = deal.begin(blockIdx.x), x1 = deal.begin(blockIdx.x + 1);
        // the item of this CTA's last unit is its to be joined when its first block is here and its end is not
        PaSplit sp{};
        if (x0 < x1) {
            const int s = pa_find(pre, p.seqs.n_seqs, x1 - 1);
            const PaWork w = work_of(s, nullptr);
            const uint32_t u = w.units(), item = (x1 - 1 - pre[s]) / u, i0 = pre[s] + item * u, i1 = i0 + u;
            if (i0 + PA_ITEM >= x0 && i0 + PA_ITEM < x1 && i1 > x1) {
                sp.n_parts = (int)(deal.cta_of(i1 - 1) - blockIdx.x) + 1;
                sp.h = item / w.tiles;
                sp.first = (item % w.tiles) * ROWS;
                sp.rows = min(ROWS, w.n * G - sp.first);
                sp.q0 = w.q0;
            }
        }
        if (tid == 0) p.split[blockIdx.x] = sp;
        pdl_launch_dependents();
        if (x0 >= x1) {
            pdl_wait();  // (see the end)
            return;
        }
        auto at = [&](uint32_t x) {  // the first block at or behind unit x
            Cursor c;
            c.s = pa_find(pre, p.seqs.n_seqs, x);
            c.w = work_of(c.s, nullptr);
            const uint32_t y = x - pre[c.s], u = c.w.units();
            c.item = (int)(y / u);
            c.b = max(0, (int)(y % u) - PA_ITEM);
            return c;
        };
        f = at(x0);
        if (x1 < total) end = at(x1);
        else end.s = -1;
    } else {
        const int item = blockIdx.x / CN, rank = blockIdx.x % CN;
        f.s = item / n_kv;
        f.w = work_of(f.s, rank == 0 && item % n_kv == 0 ? p.err : nullptr);
        if (f.w.items == 0) {  // (the whole cluster)
            if (CL == 0) pdl_wait();  // (see the end)
            return;
        }
        f.item = item % n_kv;  // (one tile: max_rows is ROWS)
        end = f;
        f.b = (int)((long long)f.w.nb * rank / CN);
        end.b = (int)((long long)f.w.nb * (rank + 1) / CN);
    }
    auto at_end = [&](const Cursor& c) { return c.s == end.s && c.item == end.item && c.b == end.b; };
    auto next_item = [&](Cursor& c) {  // the next one's first block; behind the last item: s = -1, as in `end`
        c.b = 0;
        if (++c.item == c.w.items) {
            c.item = 0;
            do {
                ++c.s;
            } while (c.s < p.seqs.n_seqs && pre[c.s + 1] == pre[c.s]);
            if (c.s == p.seqs.n_seqs) c.s = -1;
            else c.w = work_of(c.s, nullptr);
        }
    };
    Cursor c = f;

    uint8_t* ring = smem + warp * PA_NS * SLOT;
    const uint32_t ring_u = smem_u32(ring);
    bool more = !at_end(f);
    // page table entries of the block to request next, read one request ahead (-2: past the sequence's end)
    int entry[KEYS / 16];
    auto look = [&]() {
#pragma unroll
        for (int part = 0; part < KEYS / 16; ++part) {
            const int r0 = f.b * BLOCK + warp * KEYS + 16 * part;
            entry[part] = more && r0 < f.w.kv ? p.seqs.table[(long long)f.s * p.seqs.max_pages + (r0 >> ps_shift)] : -2;
        }
    };
    look();
    uint32_t dead = 0;  // slots (q8: half slots) whose page does not exist
    // Requests this warp's rows of the next block of the line into ring slot `slot`.
    auto fetch = [&](int slot) {
        if (more) {
            const int h = f.item / f.w.tiles, k0 = f.b * BLOCK + warp * KEYS;
            const uint32_t dst = ring_u + slot * SLOT;
#pragma unroll
            for (int part = 0; part < KEYS / 16; ++part) {  // sixteen rows lie in one page
                const int r0 = k0 + 16 * part;
                const int page = entry[part];
                long long row = -1;
                if ((unsigned)page < (unsigned)p.pages.n_pages)
                    row = page * p.pages.page_rows + h * p.pages.head_rows + (r0 & ((1 << ps_shift) - 1));
                else if (page != -2 && lane == 0 && p.err)
                    atomicOr(p.err, ERR_PAGE);
                const uint32_t bit = 1u << (slot * 2 + part);
                dead = row < 0 ? dead | bit : dead & ~bit;
                const int left = row < 0 ? 0 : f.w.kv - r0;  // rows of the sequence from here on
                const long long base = row < 0 ? 0 : row;
                // (sixteen rows lie in one page, so a row behind the sequence's end still has an address; it is not read)
                const uint8_t *ks = p.pages.k + base * ROW + lane * 16, *vs = p.pages.v + base * ROW + lane * 16;
                if (!Q8) {
                    const uint32_t d = dst + lane * 16;
                    if (left >= 16) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            cp_async16(d + i * 512, ks + i * 512);
                            cp_async16(d + KEYS * ROW + i * 512, vs + i * 512);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const bool real = 2 * i + (lane >> 4) < left;
                            cp_async16(d + i * 512, ks + i * 512, real);
                            cp_async16(d + KEYS * ROW + i * 512, vs + i * 512, real);
                        }
                    }
                } else {
                    // chunk c of row r goes to c ^ 4 (r & 1) for K and c ^ 2 ((r >> 1) & 3) for V: the places that
                    // make the fragment reads below free of bank conflicts
                    const int c = lane & 7, q = lane >> 3;
                    const uint32_t dk = dst + (16 * part + q) * ROW + ((c ^ ((q & 1) << 2)) << 4);
                    const uint32_t dv = dst + (KEYS + 16 * part + q) * ROW + ((c ^ ((q >> 1) << 1)) << 4);
                    if (left >= 16) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {  // rows 4 i + q
                            cp_async16(dk + i * 512, ks + i * 512);
                            cp_async16((dv ^ ((i & 1) << 6)) + i * 512, vs + i * 512);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool real = 4 * i + q < left;
                            cp_async16(dk + i * 512, ks + i * 512, real);
                            cp_async16((dv ^ ((i & 1) << 6)) + i * 512, vs + i * 512, real);
                        }
                    }
                    if (lane < 8) {  // scales: a quad that reaches past the sequence's end is read whole (same page)
                        const int e = (lane & 3) * 4;
                        const bool real = e < left;
                        const float* src = lane < 4 ? p.pages.ks : p.pages.vs;
                        cp_async16(dst + 2 * KEYS * ROW + (lane >> 2) * KEYS * 4 + (16 * part + e) * 4,
                                   real ? src + base + e : src, real);
                    }
                }
            }
            if (++f.b == f.w.nb && (LINE || f.b != end.b)) next_item(f);
            more = !at_end(f);
            look();
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < PA_NS; ++i) fetch(i);

    int slot = 0;
    bool again = !LINE || !at_end(c);  // (a CTA of a cluster without a block still takes part in the join)
    while (again) {
        const int h = c.item / c.w.tiles, tile = c.item - h * c.w.tiles;
        const int b0 = c.b, b1 = c.s == end.s && c.item == end.item ? end.b : c.w.nb;
        // this lane's rows g and g + 8 of every sixteen: last visible positions
        const int rows = c.w.n * G;
        auto q_row = [&](int r) {  // row r of the item (rows past the end: the last one, never stored)
            const int rr = min(tile * ROWS + r, rows - 1);
            return reinterpret_cast<const T*>(p.q) + (c.w.q0 + rr / G) * p.q_stride + (h * G + rr % G) * HD;
        };
        int lim[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = tile * ROWS + 16 * mt + g + 8 * i;
                lim[mt][i] = c.w.kv - c.w.n + min(r, rows - 1) / G;  // (rows past the end: the last one's)
            }
        // A fragments of q.  In a q8 cache a lane's K codes are 32-bit words of four dimensions d0 .. d0 + 3, used
        // as the pairs (d0, d0 + 2) and (d0 + 1, d0 + 3), so q takes the same order: word 2 t + 16 ks of a row
        // holds the first pair of d0 = 64 (ks / 4) + 16 t + 4 (ks % 4), word 2 t + 16 ks + 8 the second.
        uint32_t qa[QS ? 1 : 8][4];
        if (!QS) {
            const T* qp[2] = {q_row(g), q_row(g + 8)};
#pragma unroll
            for (int ks = 0; ks < 8; ++ks)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    qa[QS ? 0 : ks][i] = *reinterpret_cast<const uint32_t*>(qp[i] + 16 * ks + 2 * t);
                    qa[QS ? 0 : ks][2 + i] = *reinterpret_cast<const uint32_t*>(qp[i] + 16 * ks + 2 * t + 8);
                }
        } else {
            // (the barriers at the end of an item are behind every read of the tile before)
            for (int e = tid; e < ROWS * 16; e += PA_THREADS) {
                const int r = e >> 4, ch = e & 15;
                const uint4 v = *reinterpret_cast<const uint4*>(q_row(r) + 8 * ch);
                if (!Q8) {
                    *reinterpret_cast<uint4*>(q_tile + r * 256 + ((ch ^ (r & 7)) << 4)) = v;
                } else {
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int f = 0; f < 2; ++f) {  // dimensions 8 ch + 4 f ..
                        const int d = 8 * ch + 4 * f, ks = 4 * (d >> 6) + ((d >> 2) & 3), tt = (d >> 4) & 3;
                        uint8_t* qr = q_tile + r * 256 + 4 * tt;
                        *reinterpret_cast<uint32_t*>(qr + (((2 * ks) ^ (r & 7)) << 4)) = prmt(w[2 * f], w[2 * f + 1], 0x5410);
                        *reinterpret_cast<uint32_t*>(qr + (((2 * ks + 1) ^ (r & 7)) << 4)) = prmt(w[2 * f], w[2 * f + 1], 0x7632);
                    }
                }
            }
            __syncthreads();
        }
        const uint32_t q_u = smem_u32(q_tile);
        auto q_frag = [&](int mt, int ks, uint32_t (&a)[4]) {
            if (!QS) {
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = qa[QS ? 0 : ks][i];
            } else {  // rows 0-7 / 8-15 of chunk 2 ks, then of 2 ks + 1
                const int r = 16 * mt + (lane & 15);
                ldsm_x4(a, q_u + r * 256 + (((2 * ks + (lane >> 4)) ^ (r & 7)) << 4));
            }
        };
        float m[MT][2], l[MT][2], o[MT][16][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            m[mt][0] = m[mt][1] = -INFINITY;
            l[mt][0] = l[mt][1] = 0.f;
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[mt][j][i] = 0.f;
        }

        for (int b = b0; b < b1; ++b) {
            cp_async_wait<PA_NS - 1>();
            __syncwarp();
            const uint32_t sk = ring_u + slot * SLOT, sv = sk + KEYS * ROW;
            const uint8_t* sp = ring + slot * SLOT;
            const int k0 = b * BLOCK + warp * KEYS;
            if (k0 < c.w.kv) {
                float s[MT][NT][4] = {};
                if (!Q8) {
                    // matrices: keys 0-7 / dims 0-7, keys 0-7 / dims 8-15, keys 8-15 / ...
                    const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        uint32_t kb[4];
                        ldsm_x4(kb, sk + row * ROW + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            uint32_t a[4];
                            q_frag(mt, ks, a);
                            mma_kv<T>(s[mt][0], a, kb[0], kb[1]);
                            mma_kv<T>(s[mt][1], a, kb[2], kb[3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        uint4 w4[NT];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
                            w4[nt] = *reinterpret_cast<const uint4*>(sp + (8 * nt + g) * ROW + (((t + 4 * half) ^ ((g & 1) << 2)) << 4));
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                uint32_t a[4];
                                q_frag(mt, 4 * half + i, a);
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    const uint32_t w = i == 0 ? w4[nt].x : i == 1 ? w4[nt].y : i == 2 ? w4[nt].z : w4[nt].w;
                                    mma_kv<T>(s[mt][nt], a, codes_to_pair<T>(w), codes_to_pair<T>(w >> 8));
                                }
                            }
                    }
                }
                // columns of this lane: keys 8 nt + 2t, + 1
                float inv[2 * NT];
                if (Q8) {
                    const float* kscale = reinterpret_cast<const float*>(sp + 2 * KEYS * ROW);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        const float2 a = *reinterpret_cast<const float2*>(kscale + 8 * nt + 2 * t);
                        const float2 v = *reinterpret_cast<const float2*>(kscale + KEYS + 8 * nt + 2 * t);
                        const float av[2] = {a.x, a.y}, vv[2] = {v.x, v.y};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            // a NaN scale (a poisoned row) reaches the rows that see it through the score; a masked
                            // one adds 0 x 0 to their sums.  Scales below 1e-30 count as that: p' must not fall
                            // under fp32's range while p / vs still counts in the sum
                            const float vs = vv[e] < 1e-30f ? 1e-30f : vv[e];
                            const float add = lg2_approx(vs), mul = av[e] * p.scale_log2;
                            inv[2 * nt + e] = vs == vs ? rcp_approx(vs) : 0.f;
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) {
                                s[mt][nt][e] = fmaf(s[mt][nt][e], mul, add);
                                s[mt][nt][2 + e] = fmaf(s[mt][nt][2 + e], mul, add);
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[mt][nt][e] *= p.scale_log2;
                }
                // Every step is taken for all tiles before the next one, and the two branches are uniform: the tiles'
                // chains of dependent instructions overlap.
                const uint32_t gone = (dead >> (2 * slot)) & 3u;
                int low = lim[0][0];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) low = min(low, min(lim[mt][0], lim[mt][1]));
                if (gone || __any_sync(0xffffffffu, k0 + KEYS - 1 > low)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (k0 + 8 * nt + 2 * t + (e & 1) > lim[mt][e >> 1] || (gone >> (nt >> 1)) & 1u) s[mt][nt][e] = -INFINITY;
                }
                float bm[MT][2];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // (a NaN among the scores becomes the maximum, and the row's result)
                        bm[mt][i] = max_nan(s[mt][0][2 * i], s[mt][0][2 * i + 1]);
#pragma unroll
                        for (int nt = 1; nt < NT; ++nt) bm[mt][i] = max_nan(bm[mt][i], s[mt][nt][2 * i], s[mt][nt][2 * i + 1]);
                    }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1)
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) bm[mt][i] = max_nan(bm[mt][i], __shfl_xor_sync(0xffffffffu, bm[mt][i], x));
                auto moves = [&](int mt, int i) { return !(bm[mt][i] <= m[mt][i] + 8.f) && bm[mt][i] != -INFINITY; };
                bool any = false;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) any |= moves(mt, 0) || moves(mt, 1);
                if (__any_sync(0xffffffffu, any)) {
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const float mn = moves(mt, i) ? bm[mt][i] : m[mt][i];
                            const float corr = m[mt][i] == -INFINITY ? 0.f : ex2_approx(m[mt][i] - mn);
                            m[mt][i] = mn;
                            l[mt][i] *= corr;
#pragma unroll
                            for (int j = 0; j < 16; ++j) {
                                o[mt][j][2 * i] *= corr;
                                o[mt][j][2 * i + 1] *= corr;
                            }
                        }
                }
                uint32_t pa[MT][NT / 2][4];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float ms = m[mt][i] == -INFINITY ? 0.f : m[mt][i];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float e0 = ex2_approx(s[mt][nt][2 * i] - ms), e1 = ex2_approx(s[mt][nt][2 * i + 1] - ms);
                            l[mt][i] += Q8 ? fmaf(e0, inv[2 * nt], e1 * inv[2 * nt + 1]) : e0 + e1;
                            pa[mt][nt >> 1][2 * (nt & 1) + i] = pack_f<T>(e0, e1);
                        }
                    }
                if (!Q8) {
                    const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t vb[4];  // keys 0-7 / 8-15 of dims 16j .. 16j + 7, then of 16j + 8 ..
                        ldsm_x4_trans(vb, sv + row * ROW + (((2 * j + (lane >> 4)) ^ (row & 7)) << 4));
#pragma unroll
                        for (int mt = 0; mt < MT; ++mt) {
                            mma_kv<T>(o[mt][2 * j], pa[mt][0], vb[0], vb[1]);
                            mma_kv<T>(o[mt][2 * j + 1], pa[mt][0], vb[2], vb[3]);
                        }
                    }
                } else {
                    // column n of product j is dimension 16 n + j: lane g's chunk of a row holds all sixteen
#pragma unroll
                    for (int part = 0; part < NT / 2; ++part) {
                        uint32_t w[4][4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int r = 2 * t + (i & 1) + 8 * (i >> 1);
                            const uint4 v = *reinterpret_cast<const uint4*>(sp + KEYS * ROW + (16 * part + r) * ROW +
                                                                            ((g ^ (((r >> 1) & 3) << 1)) << 4));
                            w[i][0] = v.x; w[i][1] = v.y; w[i][2] = v.z; w[i][3] = v.w;
                        }
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint32_t sel = 0x0400 | (j & 3) << 8 | (j & 3);  // byte j of the two keys
                            const uint32_t b0 = codes_to_pair<T>(prmt(w[0][j >> 2], w[1][j >> 2], sel));
                            const uint32_t b1 = codes_to_pair<T>(prmt(w[2][j >> 2], w[3][j >> 2], sel));
#pragma unroll
                            for (int mt = 0; mt < MT; ++mt) mma_kv<T>(o[mt][j], pa[mt][part], b0, b1);
                        }
                    }
                }
            }
            __syncwarp();
            if (b + 1 < b1) {
                fetch(slot);
                slot = slot + 1 == PA_NS ? 0 : slot + 1;
            }
        }
        // the end of the item, or of this CTA's share of it: sixteen rows at a time the warps meet in the
        // slots they have just used up ([16][128] fp32 each; float4 column c4 of row r at
        // c4 ^ 2 ((c4 >> 3) & 3) ^ (r & 1))
        float* mine = reinterpret_cast<float*>(ring + slot * SLOT);
        const bool whole = b0 == 0 && b1 == c.w.nb;
        if (CL > 1) cp_async_wait<0>();  // (nothing more was requested; the next slot of warp 0 takes this CTA's part)
        float* part_c = reinterpret_cast<float*>(smem + (slot + 1 == PA_NS ? 0 : slot + 1) * SLOT);
        float* pt = p.part + (size_t)(2 * blockIdx.x + (b0 == 0 ? 1 : 0)) * PA_PART;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            if (mt > 0) __syncthreads();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
                l[mt][i] += __shfl_xor_sync(0xffffffffu, l[mt][i], 2);
                if (t == 0) {
                    ml[warp][0][16 * mt + g + 8 * i] = m[mt][i];
                    ml[warp][1][16 * mt + g + 8 * i] = l[mt][i];
                }
                const int r = g + 8 * i;
                auto place = [&](int c4) { return mine + r * HD + 4 * (c4 ^ (((c4 >> 3) & 3) << 1) ^ (r & 1)); };
                if (!Q8) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        *reinterpret_cast<float2*>(place(2 * j + (t >> 1)) + 2 * (t & 1)) =
                            make_float2(o[mt][j][2 * i], o[mt][j][2 * i + 1]);
                } else {
#pragma unroll
                    for (int e = 0; e < 2; ++e)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<float4*>(place(8 * t + 4 * e + j)) =
                                make_float4(o[mt][4 * j][2 * i + e], o[mt][4 * j + 1][2 * i + e], o[mt][4 * j + 2][2 * i + e],
                                            o[mt][4 * j + 3][2 * i + e]);
                }
            }
            __syncthreads();
            constexpr int TPR = PA_THREADS / 16;  // threads a row, chunks of eight columns in turn
            const int r = tid / TPR, rt = 16 * mt + r;
            const int rr = tile * ROWS + rt;
            if (rr < rows) {
                float mm = ml[0][0][rt];
#pragma unroll
                for (int w = 1; w < PA_WARPS; ++w) mm = max_nan(mm, ml[w][0][rt]);
                float fw[PA_WARPS], ll = 0.f;
#pragma unroll
                for (int w = 0; w < PA_WARPS; ++w) {
                    fw[w] = mm == -INFINITY ? 0.f : ex2_approx(ml[w][0][rt] - mm);
                    ll = fmaf(fw[w], ml[w][1][rt], ll);
                }
                const float il = mm == -INFINITY ? 0.f : 1.0f / ll;
                T* dst = reinterpret_cast<T*>(p.out) + (c.w.q0 + rr / G) * p.out_stride + (h * G + rr % G) * HD;
#pragma unroll
                for (int i = 0; i < 16 / TPR; ++i) {
                    const int col = 8 * (tid % TPR + TPR * i);
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int c4 = col / 4 + e;
                        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < PA_WARPS; ++w) {
                            const float4 v = *reinterpret_cast<const float4*>(
                                reinterpret_cast<const float*>(smem + (w * PA_NS + slot) * SLOT) + r * HD +
                                4 * (c4 ^ (((c4 >> 3) & 3) << 1) ^ (r & 1)));
                            a.x = fmaf(fw[w], v.x, a.x);
                            a.y = fmaf(fw[w], v.y, a.y);
                            a.z = fmaf(fw[w], v.z, a.z);
                            a.w = fmaf(fw[w], v.w, a.w);
                        }
                        y[4 * e] = a.x; y[4 * e + 1] = a.y; y[4 * e + 2] = a.z; y[4 * e + 3] = a.w;
                    }
                    if (CL > 1) {
                        store8<float>(part_c + r * HD + col, y);
                    } else if (whole) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] *= il;
                        store8<T>(dst + col, y);
                    } else {
                        store8<float>(pt + rt * HD + col, y);
                    }
                }
                if (CL > 1 && tid % TPR == 0) {
                    ml_c[0][rt] = mm;
                    ml_c[1][rt] = ll;
                }
                if (LINE && !whole && tid % TPR == 0) {
                    pt[PA_ROWS_MAX * HD + rt] = mm;
                    pt[PA_ROWS_MAX * HD + PA_ROWS_MAX + rt] = ll;
                }
            }
        }
        if (CL == 0) break;  // (the one item is whole, and nothing more was requested)
        if constexpr (CL > 1) {
            // every CTA's part is in its own shared memory: CTA `rank` folds columns [16 rank, 16 rank + 16) of all
            cluster_barrier();
            const int r = tid >> 3, rr = tile * ROWS + r, rank = blockIdx.x % CL;
            const int col = (HD / CL) * rank + 2 * (tid & 7);
            if (tid < 128 && rr < rows) {
                float pm[CL], pl[CL], px[CL], py[CL];
#pragma unroll
                for (int k = 0; k < CL; ++k) {
                    pm[k] = ld_cluster(&ml_c[0][r], k);
                    pl[k] = ld_cluster(&ml_c[1][r], k);
                    // (the slot that holds a CTA's part depends on how many blocks it had)
                    const int n = (int)((long long)c.w.nb * (k + 1) / CL) - (int)((long long)c.w.nb * k / CL);
                    const int sl = (max(n - 1, 0) + 1) % PA_NS;
                    const float* pk = reinterpret_cast<const float*>(smem + sl * SLOT) + r * HD + col;
                    px[k] = ld_cluster(pk, k);
                    py[k] = ld_cluster(pk + 1, k);
                }
                float mm = pm[0];
#pragma unroll
                for (int k = 1; k < CL; ++k) mm = max_nan(mm, pm[k]);
                float ll = 0.f, ax = 0.f, ay = 0.f;
#pragma unroll
                for (int k = 0; k < CL; ++k) {
                    const float fk = pm[k] == -INFINITY ? 0.f : ex2_approx(pm[k] - mm);
                    ll = fmaf(fk, pl[k], ll);
                    ax = fmaf(fk, px[k], ax);
                    ay = fmaf(fk, py[k], ay);
                }
                const float il = mm == -INFINITY ? 0.f : 1.0f / ll;
                T* dst = reinterpret_cast<T*>(p.out) + (c.w.q0 + rr / G) * p.out_stride + (h * G + rr % G) * HD + col;
                *reinterpret_cast<uint32_t*>(dst) = pack_f<T>(ax * il, ay * il);
            }
            cluster_barrier();  // (no CTA leaves while its part is being read)
            return;
        }
        __syncthreads();
        fetch(slot);
        slot = slot + 1 == PA_NS ? 0 : slot + 1;
        c.b = b1;
        if (b1 == c.w.nb) next_item(c);
        again = !at_end(c);
    }
    cp_async_wait<0>();
    // A mixed batch's tensor-core kernel may still run: this grid then started beside it (they share no rows) and
    // is not done before it, so that whatever follows in the stream comes after both.
    pdl_wait();
}

// Folds the parts of the items that more than one CTA of paged_attn_kernel worked on: CTA c takes the item
// that c began and did not end, one of gridDim.y groups of its rows each (a long item has dozens of parts).  Eight
// warps: with few rows several warps share one (each takes every W-th part, eight in flight) and meet in
// shared memory; the grouping depends on the sizes alone, so the bits do too.
constexpr int PJ_WARPS = 8;
template <typename T>
__global__ void __launch_bounds__(PJ_WARPS * 32) paged_attn_join_kernel(const PagedAttnParams p) {
    __shared__ float4 acc_s[PJ_WARPS][32];
    __shared__ float ml_s[PJ_WARPS][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.group;
    pdl_wait();
    const PaSplit sp = p.split[blockIdx.x];
    const int group = (sp.rows + gridDim.y - 1) / gridDim.y, lo = blockIdx.y * group, hi = min(sp.rows, lo + group);
    if (sp.n_parts == 0 || lo >= hi) return;
    int log_r = 0;  // rows at a time, a power of two; W warps a row
    while (log_r < 3 && (1 << log_r) < hi - lo) ++log_r;
    const int W = PJ_WARPS >> log_r, piece = warp >> log_r;
    for (int r0 = lo; r0 < hi; r0 += 1 << log_r) {
        const int r = r0 + (warp & ((1 << log_r) - 1));
        float m = -INFINITY, l = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < hi) {
            for (int k0 = piece; k0 < sp.n_parts; k0 += 8 * W) {
                float pm[8], pl[8];
                float4 v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const int k = k0 + u * W;
                    pm[u] = -INFINITY;
                    if (k < sp.n_parts) {
                        const float* pt = p.part + (size_t)(2 * (blockIdx.x + k) + (k == 0 ? 1 : 0)) * PA_PART;
                        pm[u] = pt[PA_ROWS_MAX * HD + r];
                        pl[u] = pt[PA_ROWS_MAX * HD + PA_ROWS_MAX + r];
                        v[u] = *reinterpret_cast<const float4*>(pt + r * HD + 4 * lane);
                    }
                }
                float mn = m;
#pragma unroll
                for (int u = 0; u < 8; ++u) mn = max_nan(mn, pm[u]);
                const float f0 = m == -INFINITY ? 0.f : ex2_approx(m - mn);
                m = mn;
                l *= f0;
                a.x *= f0; a.y *= f0; a.z *= f0; a.w *= f0;
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (pm[u] != -INFINITY) {
                        const float f = ex2_approx(pm[u] - mn);
                        l = fmaf(pl[u], f, l);
                        a.x = fmaf(v[u].x, f, a.x);
                        a.y = fmaf(v[u].y, f, a.y);
                        a.z = fmaf(v[u].z, f, a.z);
                        a.w = fmaf(v[u].w, f, a.w);
                    }
            }
        }
        if (W > 1) {  // (once: the rows are fewer than the warps)
            acc_s[warp][lane] = a;
            if (lane == 0) {
                ml_s[warp][0] = m;
                ml_s[warp][1] = l;
            }
            __syncthreads();
            if (piece == 0)
                for (int k = 1; k < W; ++k) {
                    const int o = (k << log_r) + warp;
                    const float pm = ml_s[o][0];
                    if (pm == -INFINITY) continue;
                    const float mn = max_nan(m, pm), f0 = m == -INFINITY ? 0.f : ex2_approx(m - mn), f1 = ex2_approx(pm - mn);
                    const float4 v = acc_s[o][lane];
                    m = mn;
                    l = l * f0 + ml_s[o][1] * f1;
                    a.x = a.x * f0 + v.x * f1;
                    a.y = a.y * f0 + v.y * f1;
                    a.z = a.z * f0 + v.z * f1;
                    a.w = a.w * f0 + v.w * f1;
                }
        }
        if (piece == 0 && r < hi) {
            const float il = m == -INFINITY ? 0.f : 1.0f / l;
            const int rr = sp.first + r;
            T* dst = reinterpret_cast<T*>(p.out) + (sp.q0 + rr / G) * p.out_stride + (sp.h * G + rr % G) * HD + 4 * lane;
            *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f<T>(a.x * il, a.y * il), pack_f<T>(a.z * il, a.w * il));
        }
    }
}

}  // namespace icua
