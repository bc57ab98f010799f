// Paged K/V cache: the kernels that write new tokens into it (per-head norms and rotation in the
// same pass, quantised as they are written) and read them back, and the device view of a cache and
// its batch that these and the attention kernels share.
//
// A page holds page_size positions of every kv head; row (page, head, position in page) is row
// page * page_rows + head * head_rows + position of the K and of the V pool.  16-bit rows are 256 B
// in the engine's cache order (kv_swz); q8 rows are 128 int8 codes in plain order with one fp32
// scale per row in a second array under the same row number.
#pragma once
#include "common.cuh"
#include "warp_mma.cuh"

namespace icua {

enum KvDtype : int { KV_F16 = 0, KV_BF16 = 1, KV_Q8 = 2 };   // ICUA_KV_*
enum RowDtype : int { DT_F32 = 0, DT_BF16 = 1, DT_F16 = 2 };  // ICUA_DT_*

// Flags of the paged kernels in the caller's error word (beside the ERR_WAIT_* ones).
enum : int { ERR_PAGE = 16, ERR_SEQ = 32 };

struct PagesView {
    uint8_t *k, *v;
    float *ks, *vs;
    long long page_rows, head_rows;
    int n_kv, ps_shift, n_pages;
};

struct SeqsView {
    const int *cu_q, *kv_len, *table;
    int n_seqs, total_q, max_pages;
};

struct SeqInfo {
    int q0, n, kv;  // first row, new tokens, positions in all
};

// A sequence's entry, checked: anything that would lead out of the row arrays or the page table
// makes the sequence an empty one and raises ERR_SEQ.
__device__ __forceinline__ SeqInfo load_seq(const SeqsView& S, int ps_shift, int s, int* err) {
    const int q0 = S.cu_q[s], q1 = S.cu_q[s + 1], kv = S.kv_len[s];
    if (q0 < 0 || q1 < q0 || q1 > S.total_q || kv < 0 || kv > ((long long)S.max_pages << ps_shift)) {
        if (err) atomicOr(err, ERR_SEQ);
        return SeqInfo{0, 0, 0};
    }
    return SeqInfo{q0, q1 - q0, kv};
}

// Raises ERR_SEQ if any sequence's entry contradicts itself; one warp.
__device__ __forceinline__ void check_seqs(const SeqsView& S, int ps_shift, int lane, int* err) {
    if (err == nullptr) return;
#pragma unroll 4  // (the loads of four rounds in flight)
    for (int s = lane; s < S.n_seqs; s += 32) load_seq(S, ps_shift, s, err);
}

// First pool row of position pos (any position of one page) of head h in sequence s, or -1 for a
// table entry that names no page.
__device__ __forceinline__ long long page_row(const PagesView& P, const SeqsView& S, int s, int h, int pos, int* err) {
    const int page = S.table[(long long)s * S.max_pages + (pos >> P.ps_shift)];
    if ((unsigned)page >= (unsigned)P.n_pages) {
        if (err) atomicOr(err, ERR_PAGE);
        return -1;
    }
    return page * P.page_rows + h * P.head_rows + (pos & ((1 << P.ps_shift) - 1));
}

// Sequence of row t: the number of sequences that end at or before t (cu_q ascends), counted by
// the whole warp, 32 entries a round.
__device__ __forceinline__ int find_seq(const SeqsView& S, int t, int lane) {
    int c = 0;
    for (int i = 0; i < S.n_seqs; i += 32) {
        const bool le = i + lane < S.n_seqs && S.cu_q[i + lane + 1] <= t;
        const unsigned b = __ballot_sync(0xffffffffu, le);
        c += __popc(b);
        if (b != 0xffffffffu) break;
    }
    return c;
}

// Maxima that keep a NaN.
__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Scale of a V row of zeros.  The attention takes its probabilities relative to the largest product of probability and V
// scale, in 16 bits: with the scale 1 a row that adds nothing would set that maximum and push keys with small V rows
// under fp16's normal numbers (rows of 1e-5 beside one of zeros: up to 63 % off).  2^-60 is below the scales of values down
// to 1e-16, and so far above fp32's smallest numbers that the row still counts in the sum beside V rows of up to 1e12.
constexpr float KV_ZERO_V = 8.673617379884035e-19f;

struct KvWriteParams {
    PagesView pages;
    SeqsView seqs;
    const void* qkv;
    long long qkv_stride;  // elements between the rows of two tokens
    const float *q_norm, *k_norm;
    const float2* rope;
    const int* rope_rows;
    int rope_len, n_q;
    float eps;
    void* q_out;
    long long q_stride;
    int* err;
};

// Eight consecutive elements (one 16-byte chunk of a 16-bit row) as floats.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <>
__device__ __forceinline__ void load8<__half>(const __half* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
}
template <>
__device__ __forceinline__ void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}

template <typename T>
__device__ __forceinline__ uint32_t pack_f(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack_f<__half>(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_f<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_f<T>(x[0], x[1]), pack_f<T>(x[2], x[3]), pack_f<T>(x[4], x[5]), pack_f<T>(x[6], x[7]));
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Four consecutive elements as they lie in memory, as floats, and back.
template <typename T>
struct Raw4 {
    typename std::conditional<sizeof(T) == 4, float4, uint2>::type v;
    __device__ __forceinline__ void load(const T* p) { v = *reinterpret_cast<const decltype(v)*>(p); }
};
template <typename T>
__device__ __forceinline__ void unpack4(const Raw4<T>& raw, float* x) {
    if constexpr (sizeof(T) == 4) {
        x[0] = raw.v.x; x[1] = raw.v.y; x[2] = raw.v.z; x[3] = raw.v.w;
    } else {
        const uint32_t w[2] = {raw.v.x, raw.v.y};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
__device__ __forceinline__ void load4(const float* p, float* x) {
    Raw4<float> raw;
    raw.load(p);
    unpack4(raw, x);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float* x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_f<T>(x[0], x[1]), pack_f<T>(x[2], x[3]));
}
// A half-warp per head vector: lane l holds elements 4 l .. 4 l + 3 and 64 + 4 l .., the two halves of four
// rotation pairs.  y = x rsqrt(mean x^2 + eps) w, then (y_j c - y_{j+64} s, y_{j+64} c + y_j s), in fp32; q rows
// are rounded to the output type, k and v rows to the cache type or to int8 codes: scale = max|x| / 127 in fp32
// and code = x / scale to the nearest, so a code is off by at most half a step (and 2^-15 of one, by the reciprocal
// that x is multiplied with).  A row that holds a NaN or an infinity gets the scale NaN and reads back as NaN
// throughout.  A row of zeros gets the scale 1 (K) or KV_ZERO_V.
// A CTA takes TOK tokens: a warp each looks its sequence, position and page up, then every token's vectors
// are dealt to 16 / TOK half-warps, each with its token's rotation row and the norm weights in registers and
// four vectors' loads in flight.  Bound: HBM for many tokens (each row is read once and written once; TOK = 4
// shares the lookups), latency for few (TOK = 1).  Measured on a B200: 13,081 tokens, 32:8 heads, bf16 into q8, and
// their rows read back by the kernel below, 86 us = 4.4 TB/s (6.54 by copy).
template <typename TI, typename TQ, int KVD, int TOK>
__global__ void __launch_bounds__(256, sizeof(TI) == 4 ? 3 : 4) kv_write_kernel(const KvWriteParams p) {
    using TC = typename std::conditional<KVD == KV_BF16, __nv_bfloat16, __half>::type;
    constexpr int U = 4, STEP = 16 / TOK;
    struct Token {
        long long row;  // pool row of kv head 0, -1: no page
        int pos, rope;  // rope: -1 = the token is left out
    };
    __shared__ Token tok_s[TOK];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 15;
    const int n_kv = p.pages.n_kv;
    if (warp < TOK) {
        const int t = blockIdx.x * TOK + warp;
        const int s = t < p.seqs.total_q ? find_seq(p.seqs, t, lane) : p.seqs.n_seqs;
        if (lane == 0) {
            Token k{-1, 0, -1};
            if (s < p.seqs.n_seqs) {
                const SeqInfo q = load_seq(p.seqs, p.pages.ps_shift, s, p.err);
                k.pos = q.kv - q.n + (t - q.q0);
                if (t >= q.q0 && t < q.q0 + q.n) {
                    const int r = p.rope == nullptr ? 0 : p.rope_rows != nullptr ? p.rope_rows[t] : k.pos;
                    if (k.pos < 0 || (p.rope != nullptr && (unsigned)r >= (unsigned)p.rope_len)) {
                        if (p.err) atomicOr(p.err, ERR_SEQ);  // more new tokens than positions, or no rotation row
                    } else {
                        k.rope = r;
                        k.row = page_row(p.pages, p.seqs, s, 0, k.pos, p.err);
                    }
                }
            }
            tok_s[warp] = k;
        }
    } else if (warp == 7 && blockIdx.x == 0) {  // (sequences whose rows no token looks up are checked too)
        check_seqs(p.seqs, p.pages.ps_shift, lane, p.err);
    }
    __syncthreads();
    const int hw = threadIdx.x >> 4;
    const Token k = tok_s[hw % TOK];
    if (k.rope < 0) return;
    const int t = blockIdx.x * TOK + hw % TOK, pos = k.pos;
    const unsigned mask = lane < 16 ? 0x0000ffffu : 0xffff0000u;  // shuffles stay within the half
    float cs[4], sn[4], w[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        cs[e] = 1.f;
        sn[e] = 0.f;
    }
    if (p.rope != nullptr) {
        const float4* c4 = reinterpret_cast<const float4*>(p.rope + (long long)k.rope * 64 + 4 * l);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float4 c = c4[e];
            cs[2 * e] = c.x; sn[2 * e] = c.y;
            cs[2 * e + 1] = c.z; sn[2 * e + 1] = c.w;
        }
    }
    const TI* row = reinterpret_cast<const TI*>(p.qkv) + (long long)t * p.qkv_stride + 4 * l;
    // Vectors first, first + STEP, .. below end: loads of U at a time, then `finish` for each.
    auto each = [&](int first, int end, auto&& finish) {
#pragma unroll 1
        for (int v0 = first; v0 < end; v0 += U * STEP) {
            Raw4<TI> raw[U][2];
#pragma unroll
            for (int i = 0; i < U; ++i)
                if (v0 + i * STEP < end) {
                    raw[i][0].load(row + (v0 + i * STEP) * HD);
                    raw[i][1].load(row + (v0 + i * STEP) * HD + 64);
                }
#pragma unroll
            for (int i = 0; i < U; ++i) {
                if (v0 + i * STEP >= end) break;
                float x[8];
                unpack4(raw[i][0], x);
                unpack4(raw[i][1], x + 4);
                finish(v0 + i * STEP, x);
            }
        }
    };
    auto norm_turn = [&](float (&x)[8], bool norm) {
        if (norm) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) ss += __shfl_xor_sync(mask, ss, o);
            const float r = rsqrtf(fmaf(ss, 1.f / HD, p.eps));
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float a = x[e], b = x[e + 4];
            x[e] = a * cs[e] - b * sn[e];
            x[e + 4] = b * cs[e] + a * sn[e];
        }
    };
    if (p.q_out != nullptr) {
        const bool norm = p.q_norm != nullptr;
        if (norm) {
            load4(p.q_norm + 4 * l, w);
            load4(p.q_norm + 64 + 4 * l, w + 4);
        }
        TQ* out = reinterpret_cast<TQ*>(p.q_out) + (long long)t * p.q_stride + 4 * l;
        each(hw / TOK, p.n_q, [&](int v, float (&x)[8]) {
            norm_turn(x, norm);
            store4(out + v * HD, x);
            store4(out + v * HD + 64, x + 4);
        });
    }
    if (k.row < 0) return;
    const bool norm = p.k_norm != nullptr;
    if (norm) {
        load4(p.k_norm + 4 * l, w);
        load4(p.k_norm + 64 + 4 * l, w + 4);
    }
    // places of the lane's two fours in a cached 16-bit row: half of chunk l / 2, and of chunk 8 + l / 2
    const int at0 = 8 * ((l >> 1) ^ (pos & 7)) + 4 * (l & 1);
    each(p.n_q + hw / TOK, p.n_q + 2 * n_kv, [&](int v, float (&x)[8]) {
        const bool is_v = v >= p.n_q + n_kv;
        const int h = v - p.n_q - (is_v ? n_kv : 0);
        if (!is_v) norm_turn(x, norm);
        const long long r = k.row + h * p.pages.head_rows;
        uint8_t* pool = is_v ? p.pages.v : p.pages.k;
        if (KVD == KV_Q8) {
            float amax = 0.f;  // (NaN when the row holds one)
#pragma unroll
            for (int e = 0; e < 8; ++e) amax = max_nan(amax, fabsf(x[e]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(mask, amax, o));
            float sc = amax * (1.f / 127.f);
            if (sc == 0.f) sc = is_v ? KV_ZERO_V : 1.f;
            uint32_t c[8];
            if (sc > 1e-30f) {  // x times the reciprocal is within 2^-15 of a step; 1.5 x 2^23 rounds it into the low byte
                const float inv = __fdividef(1.0f, sc);
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e] = __float_as_uint(fmaf(x[e], inv, 12582912.f));
            } else {  // (the reciprocal may pass fp32's range)
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e] = (uint32_t)max(-127, min(127, __float2int_rn(x[e] / sc)));
            }
            const bool bad = !(amax <= 3.402823466e38f);
            uint8_t* o = pool + r * HD + 4 * l;
#pragma unroll
            for (int e = 0; e < 2; ++e)
                *reinterpret_cast<uint32_t*>(o + 64 * e) =
                    bad ? 0u : __byte_perm(__byte_perm(c[4 * e], c[4 * e + 1], 0x0040), __byte_perm(c[4 * e + 2], c[4 * e + 3], 0x0040), 0x5410);
            if (l == 0) (is_v ? p.pages.vs : p.pages.ks)[r] = bad ? __int_as_float(0x7fc00000) : sc;
        } else {
            TC* o = reinterpret_cast<TC*>(pool) + r * HD + at0;
            store4(o, x);
            store4(o + 64, x + 4);
        }
    });
}

struct KvReadParams {
    PagesView pages;
    SeqsView seqs;
    void *k_out, *v_out;
    int n_groups;  // half-warps per token, each for VPT of its 2 n_kv rows
    int* err;
};

// value = code * scale (q8) or the stored 16-bit value, one rounding to the output type.  A row of a
// position that the sequence does not have, or of a table entry that names no page, reads as zeros.
// Bound: HBM; a half-warp has VPT rows of one token in flight (four where that leaves two CTAs per SM).  Measured
// on a B200: 127,780 tokens, 8 kv heads, q8 to fp16, 141 us = 5.6 TB/s, fp16 162 us = 6.5 TB/s (6.54 by copy).
template <typename TO, int KVD, int VPT>
__global__ void __launch_bounds__(256) kv_read_kernel(const KvReadParams p) {
    using TC = typename std::conditional<KVD == KV_BF16, __nv_bfloat16, __half>::type;
    const int lane = threadIdx.x & 31, l = lane & 15;
    const long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) >> 4;
    const int t = (int)(unit / p.n_groups), v0 = (int)(unit % p.n_groups) * VPT;
    if (blockIdx.x == 0 && threadIdx.x >= 224) check_seqs(p.seqs, p.pages.ps_shift, lane, p.err);
    const int ta = __shfl_sync(0xffffffffu, t, 0), tb = __shfl_sync(0xffffffffu, t, 16);
    const int sa = find_seq(p.seqs, ta, lane);
    const int sb = tb == ta ? sa : find_seq(p.seqs, tb, lane);
    const int s = lane < 16 ? sa : sb;
    if (t >= p.seqs.total_q || s >= p.seqs.n_seqs) return;
    const int n_kv = p.pages.n_kv;
    const SeqInfo q = load_seq(p.seqs, p.pages.ps_shift, s, l == 0 ? p.err : nullptr);
    if (t < q.q0 || t >= q.q0 + q.n) return;
    const int pos = q.kv - q.n + (t - q.q0);
    long long crow = -1;
    if (pos >= 0) crow = page_row(p.pages, p.seqs, s, 0, pos, l == 0 ? p.err : nullptr);
    else if (p.err && l == 0) atomicOr(p.err, ERR_SEQ);
    uint4 raw[VPT];
    float sc[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vi = v0 + i, h = vi < n_kv ? vi : vi - n_kv;
        raw[i] = make_uint4(0, 0, 0, 0);
        sc[i] = 0.f;
        if (vi < 2 * n_kv && crow >= 0) {
            const long long r = crow + h * p.pages.head_rows;
            const uint8_t* pool = vi < n_kv ? p.pages.k : p.pages.v;
            if (KVD == KV_Q8) {
                const uint2 c = *reinterpret_cast<const uint2*>(pool + r * HD + 8 * l);
                raw[i].x = c.x;
                raw[i].y = c.y;
                sc[i] = (vi < n_kv ? p.pages.ks : p.pages.vs)[r];
            } else {
                raw[i] = *reinterpret_cast<const uint4*>(pool + r * 2 * HD + 16 * (l ^ (pos & 7)));
            }
        }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vi = v0 + i, h = vi < n_kv ? vi : vi - n_kv;
        if (vi >= 2 * n_kv) break;
        TO* o = reinterpret_cast<TO*>(vi < n_kv ? p.k_out : p.v_out);
        if (o == nullptr) continue;
        float x[8];
        if (KVD == KV_Q8) {
            const uint32_t c[2] = {raw[i].x, raw[i].y};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)(c[e >> 2] >> (8 * (e & 3))) * sc[i];
        } else {
            load8<TC>(reinterpret_cast<const TC*>(&raw[i]), x);
        }
        store8<TO>(o + ((long long)t * n_kv + h) * HD + 8 * l, x);
    }
}

}  // namespace icua
