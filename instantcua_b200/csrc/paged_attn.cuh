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
// * The items' blocks (64 keys, 128 in a q8 cache) are dealt evenly over the CTAs, two per SM, as one
//   line: by the real lengths, read on the device, so a batch of very different lengths leaves no SM
//   idle.  A CTA that holds a part of an item writes (max, sum, output) to the workspace, and
//   paged_attn_join_kernel folds an item's parts in the order of their keys: the same bits every run.
// * Each of the four warps streams its own sixteen (q8: 32) rows of a block through a ring of three
//   slots with 16-byte cp.async, and runs its own online softmax; only the end of an item meets in
//   shared memory.  Rows behind the sequence's end are never read: cp.async fills zeros, so whatever a
//   page still holds there (NaN included) cannot reach a sum.
// * q8 rows are converted in registers, exactly: code -> 16-bit float by placing the byte in the
//   mantissa of 1024 (fp16) or 128 / 256 (bf16) and subtracting.  The scales never round anything: the
//   K scale multiplies the fp32 score; the V scale enters the exponent, p' = 2^(s + log2 vs - m') with
//   m' the running maximum of that sum, so the 16-bit operand of the P V product lies in [0, 1] whatever
//   the scales are, and the row sum is l = sum p' / vs.
// Scores, maxima, sums and outputs are fp32; p is rounded once to the 16-bit type of q.
#pragma once
#include "paged.cuh"
#include "tcgen05.cuh"

namespace icua {

constexpr int PA_ROWS = 16;       // query rows per item
constexpr int PA_WARPS = 4;
constexpr int PA_THREADS = PA_WARPS * 32;
constexpr int PA_NS = 3;          // ring slots per warp
constexpr int PA_MAX_CTAS = 320;  // workspace slots are laid out for so many
constexpr int PA_MAX_SEQS = 1024;
constexpr int PA_PART = PA_ROWS * HD + 2 * PA_ROWS;  // floats of a part: o[16][128], m[16], l[16]

struct PagedAttnParams {
    PagesView pages;
    SeqsView seqs;
    const void* q;
    void* out;
    long long q_stride, out_stride;
    int n_q, group;
    float scale_log2;  // softmax scale x log2(e)
    int max_rows;      // sequences with more rows (n G) than this belong to another kernel,
    int alone;         //   or, when there is none in this call, break the caller's max_q (ERR_SEQ)
    float* part;       // [gridDim.x][2][PA_PART]: 0 = an item begun by an earlier CTA, 1 = an item begun here
    int* err;
};

constexpr int pa_keys(bool q8) { return q8 ? 32 : 16; }  // rows of a warp's slot
constexpr int pa_block(bool q8) { return PA_WARPS * pa_keys(q8); }
constexpr int pa_slot(bool q8) { return q8 ? 32 * 2 * HD + 2 * 32 * 4 : 16 * 2 * HD * 2; }
constexpr int pa_smem(bool q8) { return PA_WARPS * PA_NS * pa_slot(q8) + (PA_MAX_SEQS + 1) * 4; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
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

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t r;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
    return r;
}

// The line of blocks: sequence s holds items(s) x nb(s) of them, item = kv head x tiles + tile.
struct PaWork {
    int n, kv, q0, tiles, nb, items;
};
__device__ __forceinline__ PaWork pa_work(const SeqsView& S, int ps_shift, int n_kv, int group, int max_rows, int block, int s,
                                          int* err, bool alone = false) {
    const SeqInfo q = load_seq(S, ps_shift, s, err);
    PaWork w{q.n, q.kv, q.q0, 0, 0, 0};
    const long long rows = (long long)q.n * group;
    if (rows > 0 && rows <= max_rows) {
        w.tiles = (int)((rows + PA_ROWS - 1) / PA_ROWS);
        w.items = w.tiles * n_kv;
        w.nb = max(1, (q.kv + block - 1) / block);  // an item without keys still writes its (zero) rows
    } else if (rows > 0 && alone && err) {
        atomicOr(err, ERR_SEQ);
    }
    return w;
}

// pre[s] = blocks before sequence s, pre[n_seqs] = all of them.  `warp_tot` holds one word per warp.
template <int THREADS>
__device__ __forceinline__ uint32_t pa_prefix(const SeqsView& S, int ps_shift, int n_kv, int group, int max_rows, int block,
                                              uint32_t* pre, uint32_t* warp_tot, int* err, bool alone = false) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint32_t base = 0;
    for (int s0 = 0; s0 < S.n_seqs; s0 += THREADS) {
        const int s = s0 + tid;
        uint32_t w = 0;
        if (s < S.n_seqs) {
            const PaWork k = pa_work(S, ps_shift, n_kv, group, max_rows, block, s, err, alone);
            w = (uint32_t)k.items * (uint32_t)k.nb;
        }
        uint32_t x = w;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (lane == 31) warp_tot[warp] = x;
        __syncthreads();
        uint32_t before = base, all = 0;
#pragma unroll
        for (int i = 0; i < THREADS / 32; ++i) {
            if (i < warp) before += warp_tot[i];
            all += warp_tot[i];
        }
        if (s < S.n_seqs) pre[s] = before + x - w;
        base += all;
        __syncthreads();
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

template <typename T, bool Q8>
__global__ void __launch_bounds__(PA_THREADS, 2) paged_attn_kernel(const PagedAttnParams p) {
    constexpr int KEYS = pa_keys(Q8), BLOCK = pa_block(Q8), SLOT = pa_slot(Q8);
    constexpr int ROW = Q8 ? HD : 2 * HD;  // bytes of a cached row
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float ml[PA_WARPS][2][PA_ROWS];
    __shared__ uint32_t warp_tot[PA_WARPS];
    uint32_t* pre = reinterpret_cast<uint32_t*>(smem + PA_WARPS * PA_NS * SLOT);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int ps_shift = p.pages.ps_shift, n_kv = p.pages.n_kv, G = p.group;
    const uint32_t total =
        pa_prefix<PA_THREADS>(p.seqs, ps_shift, n_kv, G, p.max_rows, BLOCK, pre, warp_tot, blockIdx.x == 0 ? p.err : nullptr,
                               p.alone != 0);
    const PaDeal deal(total, gridDim.x);
    const uint32_t x0 = deal.begin(blockIdx.x), x1 = deal.begin(blockIdx.x + 1);
    pdl_launch_dependents();
    if (x0 >= x1) return;

    struct Cursor {  // a block of the line
        int s, item, b;
        PaWork w;
    };
    auto at = [&](uint32_t x) {
        Cursor c;
        c.s = pa_find(pre, p.seqs.n_seqs, x);
        c.w = pa_work(p.seqs, ps_shift, n_kv, G, p.max_rows, BLOCK, c.s, nullptr);
        const uint32_t y = x - pre[c.s];
        c.item = (int)(y / (uint32_t)c.w.nb);
        c.b = (int)(y % (uint32_t)c.w.nb);
        return c;
    };
    auto next_item = [&](Cursor& c) {  // only called while blocks are left
        c.b = 0;
        if (++c.item == c.w.items) {
            c.item = 0;
            do {
                ++c.s;
            } while (pre[c.s + 1] == pre[c.s]);
            c.w = pa_work(p.seqs, ps_shift, n_kv, G, p.max_rows, BLOCK, c.s, nullptr);
        }
    };

    uint8_t* ring = smem + warp * PA_NS * SLOT;
    const uint32_t ring_u = smem_u32(ring);
    Cursor f = at(x0);
    uint32_t fx = x0;
    uint32_t dead = 0;  // slots (q8: half slots) whose page does not exist
    // Requests this warp's rows of the next block of the line into ring slot `slot`.
    auto fetch = [&](int slot) {
        if (fx < x1) {
            const int h = f.item / f.w.tiles, k0 = f.b * BLOCK + warp * KEYS;
            const uint32_t dst = ring_u + slot * SLOT;
#pragma unroll
            for (int part = 0; part < KEYS / 16; ++part) {  // sixteen rows lie in one page
                const int r0 = k0 + 16 * part;
                long long row = -1;
                if (r0 < f.w.kv) row = page_row(p.pages, p.seqs, f.s, h, r0, lane == 0 ? p.err : nullptr);
                const uint32_t bit = 1u << (slot * 2 + part);
                dead = row < 0 ? dead | bit : dead & ~bit;
                const int left = row < 0 ? 0 : f.w.kv - r0;  // rows of the sequence from here on
                const long long base = row < 0 ? 0 : row;
                if (!Q8) {
                    const uint8_t *ks = p.pages.k + base * ROW + lane * 16, *vs = p.pages.v + base * ROW + lane * 16;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const bool real = 2 * i + (lane >> 4) < left;
                        cp_async16(dst + i * 512 + lane * 16, real ? ks + i * 512 : p.pages.k, real);
                        cp_async16(dst + KEYS * ROW + i * 512 + lane * 16, real ? vs + i * 512 : p.pages.v, real);
                    }
                } else {
                    // chunk c of row r goes to c ^ 4 (r & 1) for K and c ^ 2 ((r >> 1) & 3) for V: the places that
                    // make the fragment reads below free of bank conflicts
                    const int c = lane & 7;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 4 * i + (lane >> 3);
                        const bool real = r < left;
                        const uint32_t at_row = dst + (16 * part + r) * ROW;
                        const long long off = (base + r) * ROW + c * 16;
                        cp_async16(at_row + ((c ^ ((r & 1) << 2)) << 4), real ? p.pages.k + off : p.pages.k, real);
                        cp_async16(at_row + KEYS * ROW + ((c ^ (((r >> 1) & 3) << 1)) << 4), real ? p.pages.v + off : p.pages.v,
                                   real);
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
            ++fx;
            if (++f.b == f.w.nb && fx < x1) next_item(f);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < PA_NS; ++i) fetch(i);

    Cursor c = at(x0);
    uint32_t x = x0;
    int slot = 0;
    while (x < x1) {
        const int h = c.item / c.w.tiles, tile = c.item - h * c.w.tiles;
        const int b0 = c.b, b1 = (int)min((uint32_t)c.w.nb, c.b + (x1 - x));
        // this lane's rows g and g + 8: query pointers and last visible positions
        const int rows = c.w.n * G;
        const T* qp[2];
        int lim[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = tile * PA_ROWS + g + 8 * i;
            const int tok = min(r, rows - 1) / G, hd = min(r, rows - 1) % G;
            qp[i] = reinterpret_cast<const T*>(p.q) + (c.w.q0 + tok) * p.q_stride + (h * G + hd) * HD;
            lim[i] = r < rows ? c.w.kv - c.w.n + tok : -1;
        }
        uint32_t qa[8][4];
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            if (!Q8) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    qa[ks][i] = *reinterpret_cast<const uint32_t*>(qp[i] + 16 * ks + 2 * t);
                    qa[ks][2 + i] = *reinterpret_cast<const uint32_t*>(qp[i] + 16 * ks + 2 * t + 8);
                }
            } else {
                // a lane's K codes are 32-bit words of four dimensions d0 .. d0 + 3, used as (d0, d0 + 2) and
                // (d0 + 1, d0 + 3): the same order here
                const int d0 = (ks < 4 ? 0 : 64) + 16 * t + 4 * (ks & 3);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint2 v = *reinterpret_cast<const uint2*>(qp[i] + d0);
                    qa[ks][i] = prmt(v.x, v.y, 0x5410);
                    qa[ks][2 + i] = prmt(v.x, v.y, 0x7632);
                }
            }
        }
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        float o[16][4];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[j][i] = 0.f;

        for (int b = b0; b < b1; ++b) {
            cp_async_wait<PA_NS - 1>();
            __syncwarp();
            const uint32_t sk = ring_u + slot * SLOT, sv = sk + KEYS * ROW;
            const uint8_t* sp = ring + slot * SLOT;
#pragma unroll
            for (int part = 0; part < KEYS / 16; ++part) {
                const int k0 = b * BLOCK + warp * KEYS + 16 * part;
                if (k0 >= c.w.kv || (dead >> (slot * 2 + part)) & 1) continue;
                float s[2][4] = {};
                if (!Q8) {
                    // matrices: keys 0-7 / dims 0-7, keys 0-7 / dims 8-15, keys 8-15 / ...
                    const int row = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        uint32_t kb[4];
                        ldsm_x4(kb, sk + row * ROW + (((2 * ks + ((lane >> 3) & 1)) ^ (row & 7)) << 4));
                        mma_kv<T>(s[0], qa[ks], kb[0], kb[1]);
                        mma_kv<T>(s[1], qa[ks], kb[2], kb[3]);
                    }
                } else {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const int r = 8 * nt + g;
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const uint4 v = *reinterpret_cast<const uint4*>(sp + (16 * part + r) * ROW +
                                                                            (((t + 4 * half) ^ ((r & 1) << 2)) << 4));
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                mma_kv<T>(s[nt], qa[4 * half + i], codes_to_pair<T>(w[i]), codes_to_pair<T>(w[i] >> 8));
                        }
                    }
                }
                // columns of this lane: keys 2t, 2t + 1, 2t + 8, 2t + 9
                float inv[4];
                if (Q8) {
                    const float* kscale = reinterpret_cast<const float*>(sp + 2 * KEYS * ROW) + 16 * part;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const float2 a = *reinterpret_cast<const float2*>(kscale + 8 * nt + 2 * t);
                        const float2 v = *reinterpret_cast<const float2*>(kscale + KEYS + 8 * nt + 2 * t);
                        const float av[2] = {a.x, a.y}, vv[2] = {v.x, v.y};
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            // a NaN scale (a poisoned row) reaches the rows that see it through the score; a masked
                            // one adds 0 x 0 to their sums
                            const float vs = vv[e] < 1e-37f ? 1e-37f : vv[e];
                            const float add = log2f(vs), mul = av[e] * p.scale_log2;
                            inv[2 * nt + e] = vs == vs ? 1.0f / vs : 0.f;
                            s[nt][e] = fmaf(s[nt][e], mul, add);
                            s[nt][2 + e] = fmaf(s[nt][2 + e], mul, add);
                        }
                    }
                } else {
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[nt][e] *= p.scale_log2;
                }
                float mn[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float bm = -INFINITY;
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float& v = s[nt][2 * i + e];
                            v = k0 + 8 * nt + 2 * t + e <= lim[i] ? v : -INFINITY;
                            bm = fmaxf(bm, v);
                        }
                    bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
                    bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
                    mn[i] = fmaxf(m[i], bm);
                }
                if (__any_sync(0xffffffffu, mn[0] > m[0] || mn[1] > m[1])) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const float corr = m[i] == -INFINITY ? 0.f : exp2f(m[i] - mn[i]);
                        m[i] = mn[i];
                        l[i] *= corr;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            o[j][2 * i] *= corr;
                            o[j][2 * i + 1] *= corr;
                        }
                    }
                }
                uint32_t pa[4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float ms = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
                    for (int nt = 0; nt < 2; ++nt) {
                        const float e0 = ex2_approx(s[nt][2 * i] - ms), e1 = ex2_approx(s[nt][2 * i + 1] - ms);
                        l[i] += Q8 ? fmaf(e0, inv[2 * nt], e1 * inv[2 * nt + 1]) : e0 + e1;
                        pa[2 * nt + i] = pack_f<T>(e0, e1);
                    }
                }
                if (!Q8) {
                    const int row = (lane & 7) + (((lane >> 3) & 1) << 3);
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        uint32_t vb[4];  // keys 0-7 / 8-15 of dims 16j .. 16j + 7, then of 16j + 8 ..
                        ldsm_x4_trans(vb, sv + row * ROW + (((2 * j + (lane >> 4)) ^ (row & 7)) << 4));
                        mma_kv<T>(o[2 * j], pa, vb[0], vb[1]);
                        mma_kv<T>(o[2 * j + 1], pa, vb[2], vb[3]);
                    }
                } else {
                    // column n of product j is dimension 16 n + j: lane g's chunk of a row holds all sixteen
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
                        const uint32_t sel = 0x0040 << 4 | (j & 3) << 8 | (j & 3);  // bytes j of the two keys
                        mma_kv<T>(o[j], pa, codes_to_pair<T>(prmt(w[0][j >> 2], w[1][j >> 2], sel)),
                                  codes_to_pair<T>(prmt(w[2][j >> 2], w[3][j >> 2], sel)));
                    }
                }
            }
            __syncwarp();
            if (b + 1 < b1) {
                fetch(slot);
                slot = slot + 1 == PA_NS ? 0 : slot + 1;
            }
        }
        // the end of the item, or of this CTA's share of it: the warps meet in the slots they have just
        // used up ([16][128] fp32 each; float4 column c4 of row r at c4 ^ 2 ((c4 >> 3) & 3) ^ (r & 1))
        float* mine = reinterpret_cast<float*>(ring + slot * SLOT);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
            if (t == 0) {
                ml[warp][0][g + 8 * i] = m[i];
                ml[warp][1][g + 8 * i] = l[i];
            }
            const int r = g + 8 * i;
            auto place = [&](int c4) { return mine + r * HD + 4 * (c4 ^ (((c4 >> 3) & 3) << 1) ^ (r & 1)); };
            if (!Q8) {
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    *reinterpret_cast<float2*>(place(2 * j + (t >> 1)) + 2 * (t & 1)) = make_float2(o[j][2 * i], o[j][2 * i + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<float4*>(place(8 * t + 4 * e + j)) =
                            make_float4(o[4 * j][2 * i + e], o[4 * j + 1][2 * i + e], o[4 * j + 2][2 * i + e], o[4 * j + 3][2 * i + e]);
            }
        }
        __syncthreads();
        {
            const int r = tid >> 3;  // eight threads a row, sixteen columns each
            float mm = ml[0][0][r];
#pragma unroll
            for (int w = 1; w < PA_WARPS; ++w) mm = fmaxf(mm, ml[w][0][r]);
            float fw[PA_WARPS], ll = 0.f;
#pragma unroll
            for (int w = 0; w < PA_WARPS; ++w) {
                fw[w] = mm == -INFINITY ? 0.f : exp2f(ml[w][0][r] - mm);
                ll = fmaf(fw[w], ml[w][1][r], ll);
            }
            const bool whole = b0 == 0 && b1 == c.w.nb;
            const float il = mm == -INFINITY ? 0.f : 1.0f / ll;
            const int rr = tile * PA_ROWS + r;
            float* pt = p.part + (size_t)(2 * blockIdx.x + (b0 == 0 ? 1 : 0)) * PA_PART;
            T* dst = reinterpret_cast<T*>(p.out) + (c.w.q0 + rr / G) * p.out_stride + (h * G + rr % G) * HD;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int col = 8 * ((tid & 7) + 8 * i);
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
                if (rr < rows) {
                    if (whole) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] *= il;
                        store8<T>(dst + col, y);
                    } else {
                        store8<float>(pt + r * HD + col, y);
                    }
                }
            }
            if (!whole && (tid & 7) == 0) {
                pt[PA_ROWS * HD + r] = mm;
                pt[PA_ROWS * HD + PA_ROWS + r] = ll;
            }
        }
        __syncthreads();
        fetch(slot);
        slot = slot + 1 == PA_NS ? 0 : slot + 1;
        x += b1 - b0;
        if (x < x1) next_item(c);
    }
    cp_async_wait<0>();
}

// Folds the parts of the items that more than one CTA of paged_attn_kernel (grid `ctas`, the same
// arguments) worked on, in the order of their keys.  CTA c takes the item that c began and did not end.
template <typename T, int BLOCK>
__global__ void __launch_bounds__(PA_THREADS) paged_attn_join_kernel(const PagedAttnParams p, int ctas) {
    __shared__ uint32_t pre[PA_MAX_SEQS + 1];
    __shared__ uint32_t warp_tot[PA_WARPS];
    const int tid = threadIdx.x, G = p.group;
    const uint32_t total = pa_prefix<PA_THREADS>(p.seqs, p.pages.ps_shift, p.pages.n_kv, G, p.max_rows, BLOCK, pre, warp_tot, nullptr);
    const PaDeal deal(total, ctas);
    const uint32_t c0 = blockIdx.x, x0 = deal.begin(c0), x1 = deal.begin(c0 + 1);
    if (x0 >= x1) return;
    const int s = pa_find(pre, p.seqs.n_seqs, x1 - 1);
    const PaWork w = pa_work(p.seqs, p.pages.ps_shift, p.pages.n_kv, G, p.max_rows, BLOCK, s, nullptr);
    const uint32_t item = (x1 - 1 - pre[s]) / w.nb, i0 = pre[s] + item * w.nb, i1 = i0 + w.nb;
    if (i0 < x0 || i1 <= x1) return;
    const uint32_t c1 = deal.cta_of(i1 - 1);
    const int h = item / w.tiles, tile = item % w.tiles, rows = min(PA_ROWS, w.n * G - tile * PA_ROWS);
    pdl_wait();
    // thread = four columns of every fourth row
    for (int r = tid >> 5; r < rows; r += PA_THREADS / 32) {
        const int col = 4 * (tid & 31);
        float m = -INFINITY, l = 0.f;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (uint32_t c = c0; c <= c1; ++c) {
            const float* pt = p.part + (size_t)(2 * c + (c == c0 ? 1 : 0)) * PA_PART;
            const float pm = pt[PA_ROWS * HD + r], pl = pt[PA_ROWS * HD + PA_ROWS + r];
            const float4 v = *reinterpret_cast<const float4*>(pt + r * HD + col);
            const float mn = fmaxf(m, pm);
            const float f0 = m == -INFINITY ? 0.f : exp2f(m - mn), f1 = pm == -INFINITY ? 0.f : exp2f(pm - mn);
            m = mn;
            l = l * f0 + pl * f1;
            a.x = a.x * f0 + v.x * f1;
            a.y = a.y * f0 + v.y * f1;
            a.z = a.z * f0 + v.z * f1;
            a.w = a.w * f0 + v.w * f1;
        }
        const float il = m == -INFINITY ? 0.f : 1.0f / l;
        const int rr = tile * PA_ROWS + r;
        T* dst = reinterpret_cast<T*>(p.out) + (w.q0 + rr / G) * p.out_stride + (h * G + rr % G) * HD + col;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_f<T>(a.x * il, a.y * il), pack_f<T>(a.z * il, a.w * il));
    }
}

}  // namespace icua
