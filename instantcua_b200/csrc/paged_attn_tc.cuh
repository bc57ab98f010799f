// Attention of chunks and prompts over a paged K/V cache on the 5th-generation tensor cores.
//
// The n G query rows of a (sequence, kv head) (row r = token r / G, head r % G) are cut into tiles of 2
// x 128; one CTA takes a tile over all its keys, or over a share of them (n_split) when there are fewer
// tiles than SMs.  Per block of 128 keys and half t:
//   S_t = Q_t K^T     (M = 128, N = 128, K = 128; both operands K-major in shared memory)
//   P_t = 2^(S_t scale log2(e) - m)   in the 16-bit type of q, written over S_t in tensor memory, 64 keys
//                                     at a time so that the product with V starts early
//   O_t += P_t V      (A = P_t from tensor memory, B = V as it lies in the cache: MN-major)
// warps 0-3 / 4-7  softmax of half 0 / 1, one thread per row (tensor-memory lane)
// warp 8           tensor memory, and every product
// warps 12-15      bring the q rows and the K / V blocks: 16-bit rows by cp.async into the 128-byte
//                  swizzle (which is the cache's own row order), q8 rows through registers, converted
//                  exactly; rows past the sequence's end and of pages that do not exist are zeros
// While one half's softmax runs, the tensor core works for the other half.  The running maximum is
// only moved (and O_t rescaled in tensor memory) when a score exceeds it by more than 2^8: P then stays
// below 256, which the 16-bit types hold as precisely as 1, and the rescale is rare.
// q8 caches: the scales enter as in paged_attn.cuh, as three fp32 factors per key.
// Bound: the chain of one half's block (softmax about 1,950 clocks, then P V and the next scores 1,150), of
// which two run against each other: about 3,200 clocks per 256 x 128 scores, where the exponentials (16 per
// clock and SM) and the products (64 clocks per M128 N128 K16 step) take 2,048 each.  Measured on a B200 (1,629
// TFLOP/s by library GEMM): a prompt of 8,192 tokens, 32:8 heads, bf16, in 0.544 ms = 1,010 TFLOP/s; a chunk of
// 500 over 8,001 positions, 16:8 heads, fp16 51 us, q8 86 us (74 from L2), there bound by the four converting warps
// (1,800 clocks per 128 rows) and by the factors' shared-memory reads.  Tried and slower: part of the exponentials as
// polynomials on the FMA pipe (560 against 549 us), two threads per row (575), rows as matrix fragments (608).
// Every wait is bounded: one that gives up raises ERR_WAIT_PREFILL, the half's rows become NaN, and the CTA still
// drains its copies and products and frees its tensor memory.
#pragma once
#include "paged_attn.cuh"

namespace icua {

constexpr int PC_BK = 128;
constexpr int PC_ROWS = 256;
constexpr int PC_THREADS = 16 * 32;
// Registers per thread after the split of the launch's 512 x 128: softmax, products, producers.
constexpr int PC_REGS_SOFTMAX = 184, PC_REGS_MMA = 56, PC_REGS_LOAD = 88;
static_assert(2 * PC_REGS_SOFTMAX + PC_REGS_MMA + PC_REGS_LOAD <= 512, "the split draws on the launch's registers");
constexpr int PC_TMEM_COLS = 512;  // S / P of the halves at 0, 128; O at 256, 384
constexpr int PC_PART = PC_ROWS * HD + 2 * PC_ROWS;  // floats of a part: o[256][128], m[256], l[256]

// K and V blocks in turn (item 2 i: K of block i, 2 i + 1: V) through one ring of tiles.
template <bool Q8>
struct PcSmem {
    static constexpr int NS = Q8 ? 4 : 5;
    static constexpr int q_off = 0;                       // 2 halves x [2][128 rows][128 B]
    static constexpr int kv_off = 65536;                  // NS x [2][128 keys][128 B]
    static constexpr int c_off = kv_off + NS * 32768;     // q8: 4 x (mul, add, inv)[128]
    static constexpr int bar_off = c_off + (Q8 ? 4 * 3 * 512 : 0);
    static constexpr int total = bar_off + 24 * 8;
    static constexpr int alloc = total + 1024;
};
// Place of an item in the ring.
template <int NS>
struct PcRing {
    int slot = 0;
    uint32_t lap = 0;
    __device__ __forceinline__ void next() {
        if (++slot == NS) {
            slot = 0;
            ++lap;
        }
    }
    __device__ __forceinline__ uint32_t full_phase() const { return lap & 1; }
    __device__ __forceinline__ uint32_t empty_phase() const { return (lap - 1) & 1; }  // laps after the first
};

struct PagedTcParams {
    PagesView pages;
    SeqsView seqs;
    const void* q;
    void* out;
    long long q_stride, out_stride;
    int group;
    float scale_log2;
    int min_rows;  // sequences with at most so many rows belong to the other kernel
    int n_split;
    uint32_t polls;  // limit of the last wait of a half's softmax
    float* part;   // [gridDim.x][PC_PART] when n_split > 1
    int* err;
};

template <typename T>
__host__ __device__ constexpr uint32_t pc_idesc(bool b_mn) {
    return umma_idesc_f16(128, 128) | (std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u) | (b_mn ? 1u << 16 : 0u);
}

// Products of the 128-byte swizzle with the descriptors' changing words alone in registers (the upper one
// is the same for all K-major operands, and one other for V).  Issued by the lane that `one` marks, from a
// warp that stays together: the operands then live in uniform registers and an issue costs little more
// than the instruction itself.
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r;
}
constexpr uint32_t PC_DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ void pc_mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 a, {%1, %3};\n\t"
        "mov.b64 b, {%2, %3};\n\t@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d),
        "r"(a_lo), "r"(b_lo), "n"(PC_DESC_HI), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}
__device__ __forceinline__ void pc_mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate, uint32_t one) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\tmov.b64 b, {%2, %3};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d),
        "r"(a), "r"(b_lo), "n"(PC_DESC_HI), "r"(idesc), "r"(accumulate), "r"(one)
        : "memory");
}

// Whether the phase has completed (try_wait would suspend the thread until it has, or for a while).
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Two fp32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 32 columns from `taddr` into v[OFF ..]; complete after tmem_wait_ld.
template <int OFF, int N>
__device__ __forceinline__ void tmem_ld32_async(uint32_t taddr, float (&v)[N]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[OFF + 0]), "=f"(v[OFF + 1]), "=f"(v[OFF + 2]), "=f"(v[OFF + 3]), "=f"(v[OFF + 4]), "=f"(v[OFF + 5]),
          "=f"(v[OFF + 6]), "=f"(v[OFF + 7]), "=f"(v[OFF + 8]), "=f"(v[OFF + 9]), "=f"(v[OFF + 10]), "=f"(v[OFF + 11]),
          "=f"(v[OFF + 12]), "=f"(v[OFF + 13]), "=f"(v[OFF + 14]), "=f"(v[OFF + 15]), "=f"(v[OFF + 16]), "=f"(v[OFF + 17]),
          "=f"(v[OFF + 18]), "=f"(v[OFF + 19]), "=f"(v[OFF + 20]), "=f"(v[OFF + 21]), "=f"(v[OFF + 22]), "=f"(v[OFF + 23]),
          "=f"(v[OFF + 24]), "=f"(v[OFF + 25]), "=f"(v[OFF + 26]), "=f"(v[OFF + 27]), "=f"(v[OFF + 28]), "=f"(v[OFF + 29]),
          "=f"(v[OFF + 30]), "=f"(v[OFF + 31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, float (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
        : "r"(taddr)
        : "memory");
}
// (the values pass through, so that no use of them moves above the wait)
template <int N>
__device__ __forceinline__ void tmem_wait_ld(float (&v)[N]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Tile of the grid: which rows of which sequence, and the keys its share covers.
struct PcTile {
    int s, q0, n, kv, row0;  // row0: first of the tile's 256 query rows
    int j0, j1, last;        // blocks of keys [j0, j1); the last key any row sees
};

// The y-th tile of the batch, found by one warp: the last tile of every sequence (they see the most keys), then
// the last but one of each, and so on, 32 sequences at a time; CTAs start in this order, so the long ones do
// first.  False past the last one.
__device__ __forceinline__ bool pc_find(const SeqsView& S, int ps_shift, int G, int min_rows, int y, int lane, PcTile& t) {
    int before = 0;
    for (int s0 = 0; s0 < S.n_seqs; s0 += 32) {
        SeqInfo q{0, 0, 0};
        if (s0 + lane < S.n_seqs) q = load_seq(S, ps_shift, s0 + lane, nullptr);
        const int rows = q.n * G;
        const int tiles = rows > min_rows ? (rows + PC_ROWS - 1) / PC_ROWS : 0;
        const int all = __reduce_add_sync(0xffffffffu, tiles);
        if (y < before + all) {
            // the turn: the most r with y at or behind the first r tiles of every sequence
            unsigned has = __ballot_sync(0xffffffffu, tiles > 0);
            int lo = y - before;  // (one sequence: its tiles in turn)
            if (has & (has - 1)) {
                int hi = __reduce_max_sync(0xffffffffu, tiles);
                lo = 0;
                while (hi - lo > 1) {
                    const int r = (lo + hi) >> 1;
                    if (y - before >= __reduce_add_sync(0xffffffffu, min(tiles, r))) lo = r;
                    else hi = r;
                }
                int i = y - before - __reduce_add_sync(0xffffffffu, min(tiles, lo));
                has = __ballot_sync(0xffffffffu, tiles > lo);
                for (; i > 0; --i) has &= has - 1;
            }
            const int src = __ffs(has) - 1;
            t.s = s0 + src;
            t.q0 = __shfl_sync(0xffffffffu, q.q0, src);
            t.n = __shfl_sync(0xffffffffu, q.n, src);
            t.kv = __shfl_sync(0xffffffffu, q.kv, src);
            t.row0 = (__shfl_sync(0xffffffffu, tiles, src) - 1 - lo) * PC_ROWS;
            return true;
        }
        before += all;
    }
    return false;
}
__device__ __forceinline__ void pc_share(PcTile& t, int G, int split, int n_split) {
    t.last = t.kv - t.n + min(t.row0 + PC_ROWS - 1, t.n * G - 1) / G;
    const int nb = t.last < 0 ? 0 : t.last / PC_BK + 1;
    t.j0 = (int)((long long)nb * split / n_split);
    t.j1 = (int)((long long)nb * (split + 1) / n_split);
}

// Grid: n_kv x n_split x (a bound of the) tiles, kv head fastest.
template <typename T, bool Q8>
__global__ void __launch_bounds__(PC_THREADS, 1) paged_attn_tc_kernel(const PagedTcParams p) {
    using S = PcSmem<Q8>;
    constexpr int NS = S::NS;
    extern __shared__ uint8_t smem_raw[];
    __shared__ PcTile tile_s;
    __shared__ int live_s;
    __shared__ uint32_t tmem_slot;
    const uint32_t base_u = smem_u32(smem_raw);
    uint8_t* smem = smem_raw + (((base_u + 1023u) & ~1023u) - base_u);
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::bar_off);
    uint64_t *q_full = bars, *done = bars + 1, *s_full = bars + 2, *p_full = bars + 4, *o_full = bars + 8, *c_full = bars + 10,
             *kv_full = bars + 14, *kv_empty = bars + 14 + NS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_kv = p.pages.n_kv, G = p.group, ps_shift = p.pages.ps_shift;
    const int h = blockIdx.x % n_kv, split = (blockIdx.x / n_kv) % p.n_split, y = blockIdx.x / (n_kv * p.n_split);

    if (warp == 0) {
        PcTile t{};
        const bool live = pc_find(p.seqs, ps_shift, G, p.min_rows, y, lane, t);
        if (live) pc_share(t, G, split, p.n_split);
        if (lane == 0) {
            tile_s = t;
            live_s = live;
        }
    } else if (warp == 8) {
        tmem_alloc(&tmem_slot, PC_TMEM_COLS);
        tmem_relinquish();
    } else if (warp == 2 && blockIdx.x == 0) {  // (the tile search ends at the tile, not at the last sequence)
        check_seqs(p.seqs, ps_shift, lane, p.err);
    } else if (threadIdx.x == 32) {
        mbar_init(q_full, 128);
        for (int i = 0; i < 2; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&p_full[2 + i], 4);
            mbar_init(&o_full[i], 1);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&c_full[i], 128);
        for (int i = 0; i < NS; ++i) {
            mbar_init(&kv_full[i], 128);
            mbar_init(&kv_empty[i], 1);
        }
        mbar_init(done, 1);
        fence_mbar_init();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = tmem_slot;
    if (!live_s) {
        if (warp == 8) tmem_dealloc(tmem, PC_TMEM_COLS);
        return;
    }
    const PcTile t = tile_s;
    const int rows = t.n * G, nblk = t.j1 - t.j0;
    // blocks of the half: its last row sees no further
    auto half_blocks = [&](int hf) {
        const int r0 = t.row0 + 128 * hf;
        if (r0 >= rows) return 0;
        const int last = t.kv - t.n + min(r0 + 127, rows - 1) / G;
        return last < 0 ? 0 : max(0, min(t.j1, last / PC_BK + 1) - t.j0);
    };

    if (warp >= 12) {
        reg_dec<PC_REGS_LOAD>();
        // ---- producers -----------------------------------------------------------------------------
        const int w = warp - 12;
        bool ok = true;
        // This warp's keys 32 w .. 32 w + 31 of a block lie in two pages at most, sixteen each.  The table is
        // read one block ahead (raw entries; -2: past the sequence's end).
        const int* table = p.seqs.table + (long long)t.s * p.seqs.max_pages;
        auto entry = [&](int j, int part) -> int {
            const int pos = j * PC_BK + 32 * w + 16 * part;
            return j < t.j1 && pos < t.kv ? table[pos >> ps_shift] : -2;
        };
        // pool row of the first of the sixteen keys (all ones: none of them is to be read)
        auto row_of = [&](int page, int j, int part) -> uint32_t {
            if ((unsigned)page >= (unsigned)p.pages.n_pages) {
                if (page != -2 && lane == 0 && p.err) atomicOr(p.err, ERR_PAGE);
                return 0xffffffffu;
            }
            const int pos = j * PC_BK + 32 * w + 16 * part;
            return (uint32_t)(page * p.pages.page_rows + h * p.pages.head_rows + (pos & ((1 << ps_shift) - 1)));
        };
        int ahead[2] = {entry(t.j0, 0), entry(t.j0, 1)};
        // the q rows first; they are announced like the copies that follow them
        {
            const T* qrow[2];
            bool real[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // this warp's rows 64 w + lane, + 32
                const int R = t.row0 + 64 * w + 32 * i + lane;
                real[i] = R < rows;
                const int tok = min(R, rows - 1) / G, hd = min(R, rows - 1) % G;
                qrow[i] = reinterpret_cast<const T*>(p.q) + (t.q0 + tok) * p.q_stride + (h * G + hd) * HD;
            }
            const uint32_t qs = smem_u32(smem + S::q_off);
            const int c = lane & 15;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int src = 2 * k + (lane >> 4);
                    const unsigned long long a = __shfl_sync(0xffffffffu, (unsigned long long)qrow[i], src);
                    const bool rl = __shfl_sync(0xffffffffu, (int)real[i], src);
                    const int R = 64 * w + 32 * i + src;  // row of the tile: half R / 128
                    cp_async16(qs + (R >> 7) * 32768 + (c >> 3) * 16384 + (R & 127) * 128 + (((c & 7) ^ (R & 7)) << 4),
                               reinterpret_cast<const uint8_t*>(a) + c * 16, rl);
                }
            cp_async_commit();
        }
        if (!Q8) {
            const int c = lane & 15;
            // rows 2 k + lane / 16 of each sixteen; `left`: the sequence's keys from the first one on
            auto issue = [&](uint8_t* dst, const uint8_t* pool, const uint32_t (&row)[2], int left) {
                const uint32_t d = smem_u32(dst) + (c >> 3) * 16384 + (c & 7) * 16 + (32 * w + (lane >> 4)) * 128;
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const bool there = row[part] != 0xffffffffu;
                    const uint8_t* src = pool + (there ? (size_t)row[part] * 256 : 0) + lane * 16;
                    const int n = there ? left - 16 * part - (lane >> 4) : 0;
#pragma unroll
                    for (int k = 0; k < 8; ++k) cp_async16(d + part * 2048 + k * 256, src + (2 * k < n ? k * 512 : 0), 2 * k < n);
                }
                cp_async_commit();
            };
            // Copies are announced two items behind, three in flight, so that their latency is covered; a
            // producer that has to wait for room announces everything first.
            PcRing<NS> put, tell;
            int untold = 1;
            bool q_told = false;
            auto tell_one = [&]() {
                fence_proxy_async_smem();
                --untold;
                if (!q_told) {
                    q_told = true;
                    mbar_arrive(q_full);
                    return;
                }
                mbar_arrive(&kv_full[tell.slot]);
                tell.next();
            };
            for (int i = 0; ok && i < nblk; ++i) {
                const int j = t.j0 + i;
                const uint32_t row[2] = {row_of(ahead[0], j, 0), row_of(ahead[1], j, 1)};
                ahead[0] = entry(j + 1, 0);
                ahead[1] = entry(j + 1, 1);
#pragma unroll
                for (int kv = 0; kv < 2; ++kv) {
                    if (put.lap > 0 && !__all_sync(0xffffffffu, mbar_test(&kv_empty[put.slot], put.empty_phase()))) {
                        cp_async_wait<0>();
                        while (untold > 0) tell_one();
                        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&kv_empty[put.slot], put.empty_phase()))) {
                            ok = false;
                            break;
                        }
                    }
                    issue(smem + S::kv_off + put.slot * 32768, kv ? p.pages.v : p.pages.k, row, t.kv - j * PC_BK - 32 * w);
                    put.next();
                    ++untold;
                    cp_async_wait<2>();
                    while (untold > 2) tell_one();
                }
            }
            cp_async_wait<0>();
            while (untold > 0) tell_one();
        } else {
            // eight 16-byte loads a lane: rows 4 i + lane / 8 of the warp's 32, chunk lane % 8
            const int c = lane & 7;
            uint4 rk[8], rv[8];
            auto load = [&](uint4 (&raw)[8], const uint8_t* pool, const uint32_t (&row)[2], int left) {
#pragma unroll
                for (int part = 0; part < 2; ++part) {
                    const bool there = row[part] != 0xffffffffu;
                    const uint8_t* src = pool + (there ? (size_t)row[part] * HD : 0) + lane * 16;
                    const int n = there ? left - 16 * part - (lane >> 3) : 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        raw[4 * part + i] = make_uint4(0, 0, 0, 0);
                        if (4 * i < n) raw[4 * part + i] = *reinterpret_cast<const uint4*>(src + i * 512);
                    }
                }
            };
            // 16 codes become two chunks of the 128-byte swizzle; the two halves of the row in turn, so that
            // eight lanes store to eight different bank groups
            auto store = [&](uint8_t* dst, const uint4 (&raw)[8]) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int R = 32 * w + 4 * i + (lane >> 3);
                    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                    uint32_t y[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        y[2 * e] = codes_to_pair<T>(prmt(x[e], 0, 0x0100));
                        y[2 * e + 1] = codes_to_pair<T>(prmt(x[e], 0, 0x0302));
                    }
                    uint8_t* d = dst + (c >> 2) * 16384 + R * 128;
                    const int p0 = 2 * (c & 3);
                    const bool odd = c >> 2;
                    const uint4 lo = make_uint4(y[0], y[1], y[2], y[3]), hi = make_uint4(y[4], y[5], y[6], y[7]);
                    *reinterpret_cast<uint4*>(d + (((p0 + odd) ^ (R & 7)) << 4)) = odd ? hi : lo;
                    *reinterpret_cast<uint4*>(d + (((p0 + !odd) ^ (R & 7)) << 4)) = odd ? lo : hi;
                }
            };
            PcRing<NS> put;
            auto room = [&]() {
                return put.lap == 0 || __all_sync(0xffffffffu, mbar_wait_bounded(&kv_empty[put.slot], put.empty_phase()));
            };
            uint32_t row[2] = {row_of(ahead[0], t.j0, 0), row_of(ahead[1], t.j0, 1)};
            if (nblk > 0) load(rk, p.pages.k, row, t.kv - t.j0 * PC_BK - 32 * w);
            cp_async_wait<0>();
            fence_proxy_async_smem();
            mbar_arrive(q_full);
            for (int i = 0; i < nblk; ++i) {
                const int j = t.j0 + i, left = t.kv - j * PC_BK - 32 * w;
                ahead[0] = entry(j + 1, 0);
                ahead[1] = entry(j + 1, 1);
                load(rv, p.pages.v, row, left);
                const uint32_t mine = lane < 16 ? row[0] : row[1];
                const bool rl = mine != 0xffffffffu && lane < left;
                const float ksc = rl ? p.pages.ks[mine + (lane & 15)] : 0.f, vsc = rl ? p.pages.vs[mine + (lane & 15)] : 1.f;
                if (!(ok = room())) break;
                store(smem + S::kv_off + put.slot * 32768, rk);
                {
                    // (block i + 4 is stored after the scores of block i + 2, which come after both halves' softmax of i)
                    float* f = reinterpret_cast<float*>(smem + S::c_off) + (i & 3) * 384 + 32 * w + lane;
                    const float vs = vsc < 1e-30f ? 1e-30f : vsc;
                    f[0] = ksc * p.scale_log2;
                    f[128] = lg2_approx(vs);
                    f[256] = vs == vs ? rcp_approx(vs) : 0.f;
                    mbar_arrive(&c_full[i & 3]);
                }
                fence_proxy_async_smem();
                mbar_arrive(&kv_full[put.slot]);
                put.next();
                row[0] = row_of(ahead[0], j + 1, 0);
                row[1] = row_of(ahead[1], j + 1, 1);
                if (i + 1 < nblk) load(rk, p.pages.k, row, left - PC_BK);
                if (!(ok = room())) break;
                store(smem + S::kv_off + put.slot * 32768, rv);
                fence_proxy_async_smem();
                mbar_arrive(&kv_full[put.slot]);
                put.next();
            }
        }
        if (!ok && lane == 0 && p.err) atomicOr(p.err, ERR_WAIT_PREFILL);
    } else if (warp >= 8) {
        reg_dec<PC_REGS_MMA>();
        // ---- products --------------------------------------------------------------------------------
        if (warp == 8) {
            const int nb[2] = {half_blocks(0), half_blocks(1)};
            const uint32_t one = elect_one(), tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint32_t q_lo = ((base_u + 1023u) & ~1023u) >> 4, kv_lo = q_lo + (S::kv_off >> 4);
            constexpr uint32_t id_s = pc_idesc<T>(false), id_o = pc_idesc<T>(true);
            auto wait = [&](uint64_t* bar, uint32_t phase) { return __all_sync(0xffffffffu, mbar_wait_bounded(bar, phase)); };
            auto commit = [&](uint64_t* bar) {
                if (one) tc_commit(bar);
                __syncwarp();
            };
            bool ok = wait(q_full, 0);
            tc_fence_after();
            PcRing<NS> get;  // the next item to wait for
            auto arrived = [&]() {
                if (!wait(&kv_full[get.slot], get.full_phase())) return false;
                get.next();
                return true;
            };
            // (a leading byte offset of 16 bytes is ignored for K-major operands; V's 64-column halves are 16 KB apart)
            auto scores = [&](int hf, int k_slot) {
                const uint32_t a = q_lo + (1u << 16) + hf * 2048, b = kv_lo + (1u << 16) + k_slot * 2048;
#pragma unroll
                for (int ks = 0; ks < 8; ++ks) {
                    const int off = (ks >> 2) * 1024 + 2 * (ks & 3);
                    pc_mma_ss(tm + 128 * hf, a + off, b + off, id_s, ks != 0, one);
                }
                commit(&s_full[hf]);
            };
            if (ok && nblk > 0) {
                ok = arrived();
                tc_fence_after();
                if (ok) {
                    for (int hf = 0; hf < 2; ++hf)
                        if (nb[hf] > 0) scores(hf, 0);
                    commit(&kv_empty[0]);
                }
            }
            for (int i = 0; ok && i < nblk; ++i) {
                const int v_slot = get.slot;
                if (!(ok = arrived())) break;
                const int k_slot = get.slot;
                const uint32_t v_lo = kv_lo + ((16384u >> 4) << 16) + v_slot * 2048;
                bool k_here = false;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf) {
                    if (!ok || i >= nb[hf]) continue;
#pragma unroll
                    for (int part = 0; part < 2; ++part) {  // the keys' first half as soon as its P is there
                        if (!ok || !(ok = wait(&p_full[2 * part + hf], i & 1))) break;
                        tc_fence_after();
#pragma unroll
                        for (int ks = 4 * part; ks < 4 * part + 4; ++ks)
                            pc_mma_ts(tm + 256 + 128 * hf, tm + 128 * hf + 8 * ks, v_lo + 128 * ks, id_o, ks == 0 ? i : 1, one);
                    }
                    if (!ok) break;
                    if (hf == (i < nb[1] ? 1 : 0)) commit(&kv_empty[v_slot]);
                    if (i + 1 < nb[hf]) {
                        if (!k_here && !(ok = arrived())) break;
                        k_here = true;
                        scores(hf, k_slot);
                    } else {
                        commit(&o_full[hf]);
                    }
                }
                if (ok && i + 1 < nblk) commit(&kv_empty[k_slot]);
            }
            if (!ok && one && p.err) atomicOr(p.err, ERR_WAIT_PREFILL);
            commit(done);  // every product issued has completed before tensor memory is freed
            mbar_wait_bounded(done, 0);
        }
    } else {
        reg_inc<PC_REGS_SOFTMAX>();
        // ---- softmax ---------------------------------------------------------------------------------
        const int hf = warp >> 2, quarter = warp & 3;
        const int R = t.row0 + 128 * hf + 32 * quarter + lane;
        const int lim = t.kv - t.n + min(R, rows - 1) / G;  // (rows past the end: the last one's, never stored)
        const int nb = half_blocks(hf);
        const uint32_t s_tm = tmem + 128 * hf + ((uint32_t)(32 * quarter) << 16), o_tm = s_tm + 256;
        float m = -INFINITY;
        float2 l = make_float2(0.f, 0.f);  // sums of the even and of the odd keys
        bool ok = true;
        // whether lanes 0-7's sixteen keys of block i lie in a page that does not exist (read a block ahead)
        const int* table = p.seqs.table + (long long)t.s * p.seqs.max_pages;
        auto entry = [&](int i) {
            const int pos = (t.j0 + i) * PC_BK + 16 * lane;
            return i < nb && lane < 8 && pos < t.kv ? table[pos >> ps_shift] : 0;
        };
        int ahead = entry(0);
        for (int i = 0; i < nb; ++i) {
            const uint32_t gone = __ballot_sync(0xffffffffu, (unsigned)ahead >= (unsigned)p.pages.n_pages);
            ahead = entry(i + 1);
            if (!__all_sync(0xffffffffu, mbar_wait_bounded(&s_full[hf], i & 1))) {
                ok = false;
                break;
            }
            tc_fence_after();
            const int k0 = (t.j0 + i) * PC_BK;
            const bool edge = __any_sync(0xffffffffu, lim < k0 + PC_BK - 1);
            const float* f = reinterpret_cast<const float*>(smem + S::c_off) + (i & 3) * 384;
            if (Q8 && !__all_sync(0xffffffffu, mbar_wait_bounded(&c_full[i & 3], (i >> 2) & 1))) {
                ok = false;
                break;
            }
            float v[128];
            tmem_ld32_async<0>(s_tm, v);
            tmem_ld32_async<32>(s_tm + 32, v);
            tmem_ld32_async<64>(s_tm + 64, v);
            tmem_ld32_async<96>(s_tm + 96, v);
            tmem_wait_ld(v);
            if (Q8) {  // scores in units of log2, with the V scale's logarithm
#pragma unroll
                for (int c = 0; c < 32; ++c) {
                    const float4 a = reinterpret_cast<const float4*>(f)[c], b = reinterpret_cast<const float4*>(f + 128)[c];
                    const float2 x = fma2(make_float2(v[4 * c], v[4 * c + 1]), make_float2(a.x, a.y), make_float2(b.x, b.y));
                    const float2 y = fma2(make_float2(v[4 * c + 2], v[4 * c + 3]), make_float2(a.z, a.w), make_float2(b.z, b.w));
                    v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = y.x; v[4 * c + 3] = y.y;
                }
            }
            if (edge || gone) {
#pragma unroll
                for (int c = 0; c < 128; ++c)
                    if (k0 + c > lim || (gone >> (c >> 4)) & 1u) v[c] = -INFINITY;
            }
            float bm4[4];  // (a NaN among the scores becomes the maximum, and the row's result)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                bm4[c] = max_nan(v[c], v[c + 4]);
#pragma unroll
                for (int e = 8; e < 128; e += 8) bm4[c] = max_nan(bm4[c], v[e + c], v[e + c + 4]);
            }
            const float sl = Q8 ? 1.f : p.scale_log2;
            const float bm = max_nan(max_nan(bm4[0], bm4[1]), bm4[2], bm4[3]) * sl;
            const bool move = !(bm <= m + 8.f) && bm != -INFINITY;  // (from -inf: any score that is seen)
            if (__any_sync(0xffffffffu, move)) {
                const float corr = move ? (m == -INFINITY ? 0.f : ex2_approx(m - bm)) : 1.f;
                if (move) m = bm;
                l.x *= corr;
                l.y *= corr;
                if (i > 0) {  // (O is complete up to the block before: S of this one was issued after it)
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        float x[16];
                        uint32_t r[16];
                        tmem_ld16_async(o_tm + 16 * c, x);
                        tmem_wait_ld(x);
#pragma unroll
                        for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(x[e] * corr);
                        tmem_st16(o_tm + 16 * c, r);
                    }
                }
            }
            const float ms = m == -INFINITY ? 0.f : -m;
            const float2 sl2 = make_float2(sl, sl), ms2 = make_float2(ms, ms);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t r[16];
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int x = 32 * c + 2 * e;
                    float2 z = make_float2(v[x], v[x + 1]);
                    z = Q8 ? add2(z, ms2) : fma2(z, sl2, ms2);
                    z.x = ex2_approx(z.x);
                    z.y = ex2_approx(z.y);
                    if (Q8) l = fma2(z, *reinterpret_cast<const float2*>(f + 256 + x), l);
                    else l = add2(l, z);
                    r[e] = pack_f<T>(z.x, z.y);
                }
                tmem_st16(s_tm + 16 * c, r);
                if (c & 1) {
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[(c & 2) + hf]);
                }
            }
        }
        // The rows go out through the half's q tile: behind its last product or, where no row has a position and so no
        // product runs, behind the copies that fill the tile.
        if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(nb > 0 ? &o_full[hf] : q_full, 0, p.polls))) ok = false;
        tc_fence_after();
        if (!ok) {
            // rows that are lost are NaN, whether or not the caller reads flags
            if (lane == 0 && p.err) atomicOr(p.err, ERR_WAIT_PREFILL);
            if (p.n_split > 1) {  // (the join keeps a NaN maximum)
                float* pt = p.part + (size_t)blockIdx.x * PC_PART + PC_ROWS * HD + 128 * hf + 32 * quarter + lane;
                pt[0] = pt[PC_ROWS] = __int_as_float(0x7fffffff);
            } else if (R < rows) {
                uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (t.q0 + R / G) * p.out_stride + (h * G + R % G) * HD);
                for (int c = 0; c < 16; ++c) dst[c] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
            }
        } else {
            const float sum = l.x + l.y;
            const int rt = 128 * hf + 32 * quarter + lane;  // row of the tile
            if (p.n_split > 1) {  // parts lie [32 chunks of four columns][256 rows]: the warp's stores are contiguous
                float* pt = p.part + (size_t)blockIdx.x * PC_PART;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    if (nb > 0) tmem_ld32(o_tm + 32 * c, v);
#pragma unroll
                    for (int b = 0; b < 8; ++b) {
                        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (nb > 0) x = make_float4(v[4 * b], v[4 * b + 1], v[4 * b + 2], v[4 * b + 3]);
                        *reinterpret_cast<float4*>(pt + ((8 * c + b) * PC_ROWS + rt) * 4) = x;
                    }
                }
                pt[PC_ROWS * HD + rt] = m;
                pt[PC_ROWS * HD + PC_ROWS + rt] = sum;
            } else {
                // through the half's q tile, which no product reads any more (16-byte chunk c of row r at c ^ (r & 15)),
                // so that the warp writes whole rows
                const float il = nb == 0 || m == -INFINITY ? 0.f : 1.0f / sum;
                uint8_t* o_s = smem + S::q_off + rt * 256;
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    float v[32];
                    if (nb > 0) tmem_ld32(o_tm + 32 * c, v);
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        float x[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = il != 0.f ? v[8 * b + e] * il : 0.f;
                        store8<T>(reinterpret_cast<T*>(o_s + (((4 * c + b) ^ (rt & 15)) << 4)), x);
                    }
                }
                __syncwarp();
                const int ch = lane & 15;
#pragma unroll 4
                for (int k = 0; k < 16; ++k) {
                    const int r = 128 * hf + 32 * quarter + 2 * k + (lane >> 4), rr = t.row0 + r;
                    if (rr < rows)
                        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (t.q0 + rr / G) * p.out_stride + (h * G + rr % G) * HD +
                                                  8 * ch) =
                            *reinterpret_cast<const uint4*>(smem + S::q_off + r * 256 + ((ch ^ (r & 15)) << 4));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 8) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, PC_TMEM_COLS);
    }
}

// Folds the n_split parts of every row, in the order of the keys.  Grid: n_kv x tiles x 8; a CTA takes 32 rows, lane
// = row and warp = four chunks of four columns (as the parts lie), and turns them in shared memory to write rows.
template <typename T>
__global__ void __launch_bounds__(256) paged_attn_tc_join_kernel(const PagedTcParams p) {
    __shared__ __align__(16) uint2 o_s[32][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_kv = p.pages.n_kv, G = p.group;
    const int r0 = (blockIdx.x & 7) * 32, h = (blockIdx.x >> 3) % n_kv, y = (blockIdx.x >> 3) / n_kv;
    PcTile t{};
    const bool live = pc_find(p.seqs, p.pages.ps_shift, G, p.min_rows, y, lane, t);
    pdl_wait();  // (every CTA: what follows in the stream relies on this grid not being done before the one it joins)
    if (!live || t.row0 + r0 >= t.n * G) return;
    const float* pt0 = p.part + (size_t)(h + n_kv * p.n_split * y) * PC_PART + r0 + lane;
    float m = -INFINITY, l = 0.f;
    float4 a[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) a[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int z = 0; z < p.n_split; ++z) {
        const float* pt = pt0 + (size_t)n_kv * z * PC_PART;
        const float pm = pt[PC_ROWS * HD], pl = pt[PC_ROWS * HD + PC_ROWS];
        float4 v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
            v[c] = *reinterpret_cast<const float4*>(pt - r0 - lane + ((4 * warp + c) * PC_ROWS + r0 + lane) * 4);
        const float mn = max_nan(m, pm);
        const float f0 = m == -INFINITY ? 0.f : ex2_approx(m - mn), f1 = pm == -INFINITY ? 0.f : ex2_approx(pm - mn);
        m = mn;
        l = l * f0 + pl * f1;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            a[c].x = a[c].x * f0 + v[c].x * f1;
            a[c].y = a[c].y * f0 + v[c].y * f1;
            a[c].z = a[c].z * f0 + v[c].z * f1;
            a[c].w = a[c].w * f0 + v[c].w * f1;
        }
    }
    const float il = m == -INFINITY ? 0.f : 1.0f / l;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        o_s[lane][4 * warp + c] = make_uint2(pack_f<T>(a[c].x * il, a[c].y * il), pack_f<T>(a[c].z * il, a[c].w * il));
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = 4 * warp + k, R = t.row0 + r0 + r;
        if (R < t.n * G)
            *reinterpret_cast<uint2*>(reinterpret_cast<T*>(p.out) + (t.q0 + R / G) * p.out_stride + (h * G + R % G) * HD + 4 * lane) =
                o_s[r][lane];
    }
}

}  // namespace icua
