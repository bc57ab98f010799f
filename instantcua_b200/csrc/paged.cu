// Entry points of the paged K/V cache (include/icua.h): argument checks, choice of the kernel
// variant and launch.  Kernels: paged.cuh (write, read back), paged_attn.cuh and paged_attn_tc.cuh
// (attention of few and of many rows).
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <type_traits>

#include "../../include/icua.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "paged_attn_tc.cuh"

namespace icua_host {
icua_status set_global_error(icua_status s, const char* msg);
std::atomic<uint32_t> paged_wait_polls{1u << 22};  // icua_set_wait_limit
}

using namespace icua;

namespace {

icua_status bad(const char* fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return icua_host::set_global_error(ICUA_ERR_INVALID, buf);
}

icua_status cuda_fail(const char* what, cudaError_t e) {
    char buf[256];
    snprintf(buf, sizeof buf, "%s: %s", what, cudaGetErrorString(e));
    return icua_host::set_global_error(ICUA_ERR_CUDA, buf);
}

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// cuPointerGetAttributes (about 50 ns a pointer; the runtime's call takes 70).
using PointerAttributes = CUresult (*)(unsigned, CUpointer_attribute*, void**, CUdeviceptr);
PointerAttributes pointer_attributes() {
    static const PointerAttributes fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        const cudaError_t e = cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q);
        return e == cudaSuccess && q == cudaDriverEntryPointSuccess ? (PointerAttributes)f : nullptr;
    }();
    return fn;
}

struct Named {
    const void* p;  // NULL: not given
    const char* name;
};
// Pointers that the kernels may follow: memory of the current device, or managed memory; the first two (a pool and a row
// array) no host memory, the others also pinned host memory, which the device reads in place.
icua_status check_device_ptrs(int* dev, std::initializer_list<Named> list) {
    const cudaError_t e = cudaGetDevice(dev);
    if (e != cudaSuccess) return cuda_fail("cudaGetDevice", e);
    const PointerAttributes get = pointer_attributes();
    if (!get) return cuda_fail("cuPointerGetAttributes", cudaErrorSymbolNotFound);
    // (small arrays often share an allocation: a pointer into one that has been looked up is not looked up again)
    struct Range {
        CUdeviceptr begin;
        size_t bytes;
    } seen[16];
    int i = 0, n_seen = 0;
    for (const Named& n : list) {
        const bool host = i++ >= 2;
        if (!n.p) continue;
        const CUdeviceptr p = (CUdeviceptr)n.p;
        bool known = false;
        for (int k = 0; k < n_seen; ++k) known |= p - seen[k].begin < seen[k].bytes;
        if (known) continue;
        unsigned type = 0;
        int at = -1;
        Range r{};
        CUpointer_attribute what[4] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL,
                                       CU_POINTER_ATTRIBUTE_RANGE_START_ADDR, CU_POINTER_ATTRIBUTE_RANGE_SIZE};
        void* to[4] = {&type, &at, &r.begin, &r.bytes};
        if (get(4, what, to, p) != CUDA_SUCCESS) type = 0;
        if (type == CU_MEMORYTYPE_DEVICE && at == *dev) {
            if (n_seen < 16) seen[n_seen++] = r;
            continue;
        }
        if (type == CU_MEMORYTYPE_HOST && host) continue;
        unsigned managed = 0;
        what[0] = CU_POINTER_ATTRIBUTE_IS_MANAGED;
        to[0] = &managed;
        if (type != 0 && get(1, what, to, p) == CUDA_SUCCESS && managed) continue;
        if (type != CU_MEMORYTYPE_DEVICE) return bad("%s is not device memory", n.name);
        return bad("%s is on device %d, the current device is %d", n.name, at, *dev);
    }
    return ICUA_OK;
}

icua_status check_cache(const icua_kv_pages* c, const icua_kv_seqs* s, PagesView* P, SeqsView* S) {
    if (!c || !s) return bad("null argument");
    if (s->n_seqs < 0 || s->n_seqs > PA_MAX_SEQS || s->total_q < 0 || s->max_q < 0 || s->max_kv < 0 || s->max_pages < 0)
        return bad("batch sizes out of range (n_seqs 0..%d, the others not negative)", PA_MAX_SEQS);
    if (c->dtype != ICUA_KV_F16 && c->dtype != ICUA_KV_BF16 && c->dtype != ICUA_KV_Q8) return bad("unknown cache type %d", c->dtype);
    if (c->n_kv < 1 || c->n_kv > 128) return bad("n_kv %d is not in 1..128", c->n_kv);
    int sh = 4;
    while (sh < 8 && (1 << sh) != c->page_size) ++sh;
    if ((1 << sh) != c->page_size) return bad("page_size %d is not 16, 32, 64, 128 or 256", c->page_size);
    if (c->n_pages < 1) return bad("n_pages is below 1");
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16)) return bad("pools are null or not 16-byte aligned");
    if (c->dtype == ICUA_KV_Q8 && (!c->k_scale || !c->v_scale || !aligned(c->k_scale, 16) || !aligned(c->v_scale, 16)))
        return bad("scales of a q8 cache are null or not 16-byte aligned");
    P->page_rows = c->page_rows;
    P->head_rows = c->head_rows;
    if (c->page_rows == 0 && c->head_rows == 0) {
        P->head_rows = c->page_size;
        P->page_rows = (int64_t)c->n_kv * c->page_size;
    }
    if (P->page_rows < c->page_size || P->page_rows % 16 || P->head_rows < c->page_size || P->head_rows % 16)
        return bad("page_rows and head_rows are multiples of 16, at least page_size (or both 0)");
    // (the kernels count pool rows in 32 bits: 2^32 rows are 512 GB)
    if (P->page_rows > UINT32_MAX || P->head_rows > UINT32_MAX ||
        (double)c->n_pages * P->page_rows + (double)c->n_kv * P->head_rows > 4294967295.0)
        return bad("the pool is too large");
    if (s->n_seqs > 0 && (!s->cu_q || !s->kv_len || (s->max_pages > 0 && !s->page_table))) return bad("null batch arrays");
    if (!aligned(s->cu_q, 4) || !aligned(s->kv_len, 4) || !aligned(s->page_table, 4)) return bad("batch arrays are not aligned");
    if ((int64_t)s->max_pages * c->page_size > 1 << 30) return bad("max_pages * page_size is above 2^30");
    P->k = (uint8_t*)c->k;
    P->v = (uint8_t*)c->v;
    P->ks = c->k_scale;
    P->vs = c->v_scale;
    P->n_kv = c->n_kv;
    P->ps_shift = sh;
    P->n_pages = c->n_pages;
    *S = SeqsView{s->cu_q, s->kv_len, s->page_table, s->n_seqs, s->total_q, s->max_pages};
    return ICUA_OK;
}

// What a device is asked once (by whichever threads come first: they find the same).
constexpr int MAX_DEVICES = 64;
int sm_count(int dev) {
    static std::atomic<int> known[MAX_DEVICES];
    const bool in = dev >= 0 && dev < MAX_DEVICES;
    int n = in ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    if (in) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <auto Kernel>
cudaError_t allow_smem(int bytes, int dev) {
    static std::atomic<bool> done[MAX_DEVICES];
    const bool in = dev >= 0 && dev < MAX_DEVICES;
    if (in && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && in) done[dev].store(true, std::memory_order_release);
    return e;
}

// four vectors per half-warp where that still leaves two CTAs (of 16 half-warps) per SM
int vectors_per_unit(int64_t tokens, int n_vec, int n_sm) { return tokens * ((n_vec + 3) / 4) >= 2ll * 16 * n_sm ? 4 : 1; }

// beside: the launch may start while the kernel before it still runs (which it waits for itself).
template <typename P>
cudaError_t launch_on(void (*kernel)(const P), dim3 grid, int block, int smem, cudaStream_t st, bool beside, const P& p) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = beside ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename TI, typename TQ, int KVD>
cudaError_t launch_write(const KvWriteParams& p, int n_sm, cudaStream_t st) {
    // four tokens a CTA once that leaves two CTAs per SM
    if (p.seqs.total_q >= 8 * n_sm)
        return launch_on(kv_write_kernel<TI, TQ, KVD, 4>, dim3((p.seqs.total_q - 1) / 4 + 1), 256, 0, st, false, p);
    return launch_on(kv_write_kernel<TI, TQ, KVD, 1>, dim3(p.seqs.total_q), 256, 0, st, false, p);
}

template <typename TI>
cudaError_t launch_write_in(const KvWriteParams& p, int kvd, int qd, int n_sm, cudaStream_t st) {
    if (kvd == ICUA_KV_F16) return launch_write<TI, __half, KV_F16>(p, n_sm, st);
    if (kvd == ICUA_KV_BF16) return launch_write<TI, __nv_bfloat16, KV_BF16>(p, n_sm, st);
    return qd == ICUA_DT_F16 ? launch_write<TI, __half, KV_Q8>(p, n_sm, st) : launch_write<TI, __nv_bfloat16, KV_Q8>(p, n_sm, st);
}

template <typename TO, int KVD>
cudaError_t launch_read_one(KvReadParams& p, int n_sm, cudaStream_t st) {
    const int n_vec = 2 * p.pages.n_kv;
    const int vpt = vectors_per_unit(p.seqs.total_q, n_vec, n_sm);
    p.n_groups = (n_vec + vpt - 1) / vpt;
    const int64_t grid = ((int64_t)p.seqs.total_q * p.n_groups + 15) / 16;
    return launch_on(vpt == 4 ? kv_read_kernel<TO, KVD, 4> : kv_read_kernel<TO, KVD, 1>, dim3((unsigned)grid), 256, 0, st, false, p);
}

template <typename TO>
cudaError_t launch_read(KvReadParams& p, int kvd, int n_sm, cudaStream_t st) {
    return kvd == ICUA_KV_F16 ? launch_read_one<TO, KV_F16>(p, n_sm, st)
         : kvd == ICUA_KV_BF16 ? launch_read_one<TO, KV_BF16>(p, n_sm, st)
                               : launch_read_one<TO, KV_Q8>(p, n_sm, st);
}

// 16-bit rows of q: the cache's own type where the cache is 16-bit.
bool q_type_fits(int dtype, int kvd) {
    return (dtype == ICUA_DT_F16 && kvd != ICUA_KV_BF16) || (dtype == ICUA_DT_BF16 && kvd != ICUA_KV_F16);
}

// beside: the launch before this one in the stream is the same call's tensor-core kernel.
template <typename T, bool Q8, int MT>
cudaError_t launch_attn(const PagedAttnParams& p, bool beside, int dev, cudaStream_t st) {
    const int smem = pa_smem(Q8, MT, 1);
    cudaError_t e = allow_smem<paged_attn_kernel<T, Q8, MT, 1>>(smem, dev);
    if (e != cudaSuccess) return e;
    const int ctas = std::min(PA_MAX_CTAS, pa_ctas(Q8, MT, 1) * sm_count(dev));
    e = launch_on(paged_attn_kernel<T, Q8, MT, 1>, dim3(ctas), 32 * pa_warps(1), smem, st, beside, p);
    // Items in many parts are joined by four CTAs each (12 sequences of up to 34,000 positions, 2 kv heads: 31 -> 25 us);
    // where the parts are few one does, and the launch stays small (64 sequences of 2,000, 8 kv heads: 72 against 74).
    const int groups = p.seqs.n_seqs * p.pages.n_kv * 4 <= ctas ? 4 : 1;
    return e != cudaSuccess ? e : launch_on(paged_attn_join_kernel<T>, dim3(ctas, groups), PJ_WARPS * 32, 0, st, true, p);
}

// One cluster per (sequence, kv head), one launch.
template <typename T, bool Q8>
cudaError_t launch_attn_cluster(const PagedAttnParams& p, int dev, cudaStream_t st) {
    const int smem = pa_smem(Q8, 1, PA_CLUSTER);
    const cudaError_t e = allow_smem<paged_attn_kernel<T, Q8, 1, PA_CLUSTER>>(smem, dev);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.seqs.n_seqs * p.pages.n_kv * PA_CLUSTER);
    cfg.blockDim = dim3(32 * pa_warps(PA_CLUSTER));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = PA_CLUSTER;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, paged_attn_kernel<T, Q8, 1, PA_CLUSTER>, p);
}

// One CTA per (sequence, kv head), one launch.
template <typename T, bool Q8, int MT>
cudaError_t launch_attn_cta(const PagedAttnParams& p, bool beside, int dev, cudaStream_t st) {
    const int smem = pa_smem(Q8, MT, 0), items = p.seqs.n_seqs * p.pages.n_kv;
    const cudaError_t e = allow_smem<paged_attn_kernel<T, Q8, MT, 0>>(smem, dev);
    if (e != cudaSuccess) return e;
    return launch_on(paged_attn_kernel<T, Q8, MT, 0>, dim3(items), 32 * pa_warps(0), smem, st, beside, p);
}

enum class Share { line, cta, cluster };
template <typename T, bool Q8>
cudaError_t launch_attn_few(const PagedAttnParams& p, Share share, bool one_tile, bool beside, int dev, cudaStream_t st) {
    if (share == Share::cluster) return launch_attn_cluster<T, Q8>(p, dev, st);
    if (share == Share::cta) return one_tile ? launch_attn_cta<T, Q8, 1>(p, beside, dev, st) : launch_attn_cta<T, Q8, 2>(p, beside, dev, st);
    return one_tile ? launch_attn<T, Q8, 1>(p, beside, dev, st) : launch_attn<T, Q8, 2>(p, beside, dev, st);
}

// Sequences with up to PA_ROWS_FEW query rows per kv head go through the warp-MMA kernel, more rows
// through the tensor-core kernel.  (28 rows, 24 sequences of about 2,400 positions: 58 us there, 96 us on the
// tensor core.  With 64 as the border the sequences of a mixed batch that have 33 to 64 rows go through the
// first kernel's tiles of 32 twice: 47.1 against 45.3 us for 12 sequences of 1 to 600 tokens.)
// Up to PA_CLUSTER_KEYS positions a cluster per item serves small batches.  (One token, 8 kv heads, bf16, in a
// graph, cluster against line and join: 512 positions 5.8 / 7.7 us, 2,048 7.1 / 8.6, 4,096 8.9 / 10.8, 8,192 12.7 /
// 12.4, 32,768 36.6 / 30.1; with fewer heads the line, which always has every SM, catches up earlier.)
constexpr int PA_ROWS_FEW = 32;
constexpr int PA_CLUSTER_KEYS = 4096;
// Short ones of the others get a CTA per item, without the line's counting and its join: up to 256 positions, and 8 more
// for each item up to PA_CTA_KEYS, since a batch of few items needs the line to fill the GPU.  (fp16 / q8, in a graph, CTA
// against line.  28 rows: 1 item of 256 positions 9.0 / 8.1 against 10.0 / 10.1 us, of 512 12.9 / 11.8 against 10.1 / 10.1, of
// 1,000 20.8 / 19.0 against 10.8 / 10.4; 24 items of 512 13.3 / 12.2 against 13.5 / 13.1, of 1,000 21.2 / 19.6 against 15.5 /
// 13.5; 64 of 512 13.4 / 12.4 against 16.2 / 16.2, of 1,000 21.4 / 19.9 against 18.8 / 18.9; 128 of 1,000 21.6 / 20.4 against
// 28.4 / 28.4.  8 rows: 24 of 512 9.5 / 9.5 against 10.3 / 10.9, of 1,000 16.0 / 16.0 against 11.0 / 11.6; 64 of 1,000 16.1 / 16.2
// against 14.1 / 15.5; 128 of 1,000 16.2 / 16.5 against 17.2 / 18.5; 296 of 1,000 28.1 / 21.4 against 31.0 / 28.7.)
constexpr int PA_CTA_KEYS = 1024;
int cta_keys(int64_t items) { return (int)std::min<int64_t>(PA_CTA_KEYS, 256 + 8 * items); }
static_assert(PA_ROWS_FEW <= 32, "the kernel's largest tile holds every item");

// Tiles of the tensor-core kernel: a bound from what the host knows, and the shares of the keys that fill
// the SMs when the tiles alone do not (two blocks of keys per share at least).
constexpr int PC_MAX_SHARES = 160;
struct TcGrid {
    int tiles, n_split;
};
TcGrid tc_grid(const icua_kv_seqs* s, int n_kv, int group, int min_rows, int n_sm) {
    const int64_t rows = (int64_t)s->total_q * group;
    TcGrid g;
    g.tiles = (int)(rows / PC_ROWS + std::min<int64_t>(s->n_seqs, rows / (min_rows + 1)));
    const int base = g.tiles * n_kv;
    g.n_split = std::max(1, std::min(std::min(n_sm, PC_MAX_SHARES) / std::max(base, 1), (int)(((int64_t)s->max_kv + 2 * PC_BK - 1) / (2 * PC_BK))));
    return g;
}

template <typename T, bool Q8>
cudaError_t launch_attn_tc(const PagedTcParams& p, int tiles, int dev, cudaStream_t st) {
    cudaError_t e = allow_smem<paged_attn_tc_kernel<T, Q8>>(PcSmem<Q8>::alloc, dev);
    if (e != cudaSuccess) return e;
    e = launch_on(paged_attn_tc_kernel<T, Q8>, dim3(tiles * p.pages.n_kv * p.n_split), PC_THREADS, PcSmem<Q8>::alloc, st, false, p);
    if (e != cudaSuccess || p.n_split == 1) return e;
    return launch_on(paged_attn_tc_join_kernel<T>, dim3(tiles * p.pages.n_kv * 8), 256, 0, st, true, p);
}

constexpr size_t PA_SCRATCH = PA_MAX_CTAS * (2 * PA_PART * sizeof(float) + sizeof(PaSplit));
constexpr size_t PC_SCRATCH = (size_t)PC_MAX_SHARES * PC_PART * sizeof(float);

icua_status check_attn(const icua_kv_pages* pages, const icua_kv_seqs* seqs, int32_t n_q, PagesView* P, SeqsView* S) {
    const icua_status st = check_cache(pages, seqs, P, S);
    if (st != ICUA_OK) return st;
    if (n_q < pages->n_kv || n_q > 256 || n_q % pages->n_kv) return bad("n_q %d is not a multiple of n_kv %d up to 256", n_q, pages->n_kv);
    // rows are counted in 32 bits, and so are the few-rows kernel's blocks of keys over all its items: tiles of sixteen rows
    // at least, of sequences with PA_ROWS_FEW rows at most
    const int64_t rows = (int64_t)seqs->total_q * (n_q / pages->n_kv);
    const double tiles = std::min((double)rows / 16 + seqs->n_seqs, (PA_ROWS_FEW / 16.0) * seqs->n_seqs);
    const double blocks = tiles * pages->n_kv * ((double)seqs->max_pages * pages->page_size / 64 + 1 + PA_ITEM);
    if (rows > INT32_MAX || blocks > 4e9) return bad("the batch is too large: split it");
    return ICUA_OK;
}

}  // namespace

extern "C" {

icua_status icua_kv_write(const icua_kv_pages* pages, const icua_kv_seqs* seqs, const icua_kv_rows* rows, int32_t* err_dev,
                          void* stream) {
    KvWriteParams p{};
    icua_status st = check_cache(pages, seqs, &p.pages, &p.seqs);
    if (st != ICUA_OK) return st;
    if (!rows || !rows->qkv || !aligned(rows->qkv, 16)) return bad("qkv is null or not 16-byte aligned");
    if (rows->qkv_dtype < ICUA_DT_F32 || rows->qkv_dtype > ICUA_DT_F16) return bad("unknown qkv type %d", rows->qkv_dtype);
    if (rows->n_q < 0 || rows->n_q > 256) return bad("n_q %d is not in 0..256", rows->n_q);
    if (!q_type_fits(rows->q_dtype, pages->dtype)) return bad("q type %d does not go with cache type %d", rows->q_dtype, pages->dtype);
    const int64_t width = (int64_t)(rows->n_q + 2 * pages->n_kv) * HD;
    p.qkv_stride = rows->qkv_stride ? rows->qkv_stride : width;
    p.q_stride = rows->q_stride ? rows->q_stride : (int64_t)rows->n_q * HD;
    if (p.qkv_stride < width || p.qkv_stride % 8 || p.q_stride < (int64_t)rows->n_q * HD || p.q_stride % 8)
        return bad("token strides are multiples of 8, at least a row (or 0)");
    if (!aligned(rows->q_out, 16) || !aligned(rows->q_norm, 16) || !aligned(rows->k_norm, 16) || !aligned(rows->rope, 16) ||
        !aligned(rows->rope_rows, 4) || !aligned(err_dev, 4))
        return bad("a row array is not aligned");
    if (rows->rope && rows->rope_len < 0) return bad("rope_len is negative");
    if (!(rows->eps >= 0.f)) return bad("eps is negative or NaN");
    if (seqs->n_seqs == 0 || seqs->total_q == 0) return ICUA_OK;
    int dev = 0;
    const bool scales = pages->dtype == ICUA_KV_Q8;
    st = check_device_ptrs(&dev, {{pages->k, "the K pool"}, {rows->qkv, "the row array"}, {pages->v, "the V pool"},
                                 {scales ? pages->k_scale : nullptr, "k_scale"}, {scales ? pages->v_scale : nullptr, "v_scale"},
                                 {seqs->cu_q, "cu_q"}, {seqs->kv_len, "kv_len"}, {seqs->page_table, "page_table"}, {err_dev, "err_dev"},
                                 {rows->q_norm, "q_norm"}, {rows->k_norm, "k_norm"}, {rows->rope, "rope"},
                                 {rows->rope ? rows->rope_rows : nullptr, "rope_rows"}, {rows->q_out, "q_out"}});
    if (st != ICUA_OK) return st;
    p.qkv = rows->qkv;
    p.q_norm = rows->q_norm;
    p.k_norm = rows->k_norm;
    p.rope = reinterpret_cast<const float2*>(rows->rope);
    p.rope_rows = rows->rope_rows;
    p.rope_len = rows->rope_len;
    p.n_q = rows->n_q;
    p.eps = rows->eps;
    p.q_out = rows->q_out;
    p.err = err_dev;
    cudaStream_t s = (cudaStream_t)stream;
    const int n_sm = sm_count(dev);
    const cudaError_t e = rows->qkv_dtype == ICUA_DT_F32    ? launch_write_in<float>(p, pages->dtype, rows->q_dtype, n_sm, s)
                          : rows->qkv_dtype == ICUA_DT_BF16 ? launch_write_in<__nv_bfloat16>(p, pages->dtype, rows->q_dtype, n_sm, s)
                                                            : launch_write_in<__half>(p, pages->dtype, rows->q_dtype, n_sm, s);
    return e == cudaSuccess ? ICUA_OK : cuda_fail("icua_kv_write", e);
}

icua_status icua_kv_read(const icua_kv_pages* pages, const icua_kv_seqs* seqs, void* k_out, void* v_out, int32_t dtype,
                         int32_t* err_dev, void* stream) {
    KvReadParams p{};
    icua_status st = check_cache(pages, seqs, &p.pages, &p.seqs);
    if (st != ICUA_OK) return st;
    if (dtype < ICUA_DT_F32 || dtype > ICUA_DT_F16) return bad("unknown row type %d", dtype);
    if ((!k_out && !v_out) || !aligned(k_out, 16) || !aligned(v_out, 16) || !aligned(err_dev, 4))
        return bad("both outputs are null, or one is not 16-byte aligned");
    if ((int64_t)seqs->total_q * 2 * pages->n_kv > ((int64_t)16 << 31) - 16) return bad("the batch is too large: split it");
    if (seqs->n_seqs == 0 || seqs->total_q == 0) return ICUA_OK;
    int dev = 0;
    const bool scales = pages->dtype == ICUA_KV_Q8;
    st = check_device_ptrs(&dev, {{pages->k, "the K pool"}, {k_out ? k_out : v_out, "the row array"}, {pages->v, "the V pool"},
                                 {scales ? pages->k_scale : nullptr, "k_scale"}, {scales ? pages->v_scale : nullptr, "v_scale"},
                                 {seqs->cu_q, "cu_q"}, {seqs->kv_len, "kv_len"}, {seqs->page_table, "page_table"}, {err_dev, "err_dev"},
                                 {v_out, "v_out"}});
    if (st != ICUA_OK) return st;
    p.k_out = k_out;
    p.v_out = v_out;
    p.err = err_dev;
    cudaStream_t s = (cudaStream_t)stream;
    const int n_sm = sm_count(dev);
    const cudaError_t e = dtype == ICUA_DT_F32    ? launch_read<float>(p, pages->dtype, n_sm, s)
                          : dtype == ICUA_DT_BF16 ? launch_read<__nv_bfloat16>(p, pages->dtype, n_sm, s)
                                                  : launch_read<__half>(p, pages->dtype, n_sm, s);
    return e == cudaSuccess ? ICUA_OK : cuda_fail("icua_kv_read", e);
}

uint64_t icua_attn_paged_scratch_bytes(const icua_kv_pages* pages, const icua_kv_seqs* seqs, int32_t n_q) {
    PagesView P;
    SeqsView S;
    if (check_attn(pages, seqs, n_q, &P, &S) != ICUA_OK) return 0;
    return PA_SCRATCH + ((int64_t)seqs->max_q * (n_q / pages->n_kv) > PA_ROWS_FEW ? PC_SCRATCH : 0);
}

icua_status icua_attn_paged(const icua_kv_pages* pages, const icua_kv_seqs* seqs, const icua_attn_paged_args* a, int32_t* err_dev,
                            void* stream) {
    PagedAttnParams p{};
    if (!a) return bad("null argument");
    icua_status st = check_attn(pages, seqs, a->n_q, &p.pages, &p.seqs);
    if (st != ICUA_OK) return st;
    if (!a->q || !a->out || !aligned(a->q, 16) || !aligned(a->out, 16) || !aligned(err_dev, 4))
        return bad("q or out is null or not 16-byte aligned");
    if (!q_type_fits(a->dtype, pages->dtype)) return bad("row type %d does not go with cache type %d", a->dtype, pages->dtype);
    p.q_stride = a->q_stride ? a->q_stride : (int64_t)a->n_q * HD;
    p.out_stride = a->out_stride ? a->out_stride : (int64_t)a->n_q * HD;
    if (p.q_stride < (int64_t)a->n_q * HD || p.q_stride % 8 || p.out_stride < (int64_t)a->n_q * HD || p.out_stride % 8)
        return bad("token strides are multiples of 8, at least a row (or 0)");
    // (a row written at its place in out would be another token's q)
    if (a->q == a->out && p.q_stride != p.out_stride && seqs->total_q > 1) return bad("out is q itself, with another token stride");
    p.scale_log2 = (a->scale > 0.f ? a->scale : 0.08838834764831845f) * 1.4426950408889634f;  // (scores in units of log2)
    if (!(a->scale >= 0.f) || !(p.scale_log2 <= FLT_MAX)) return bad("scale is negative or, in units of log2, not finite");
    if (!a->scratch || !aligned(a->scratch, 16) || a->scratch_bytes < icua_attn_paged_scratch_bytes(pages, seqs, a->n_q))
        return bad("scratch is null, not 16-byte aligned or smaller than icua_attn_paged_scratch_bytes");
    if (seqs->n_seqs == 0 || seqs->total_q == 0) return ICUA_OK;
    int dev = 0;
    const bool scales = pages->dtype == ICUA_KV_Q8;
    st = check_device_ptrs(&dev, {{pages->k, "the K pool"}, {a->q, "the row array"}, {pages->v, "the V pool"},
                                 {scales ? pages->k_scale : nullptr, "k_scale"}, {scales ? pages->v_scale : nullptr, "v_scale"},
                                 {seqs->cu_q, "cu_q"}, {seqs->kv_len, "kv_len"}, {seqs->page_table, "page_table"}, {err_dev, "err_dev"},
                                 {a->out, "out"}, {a->scratch, "scratch"}});
    if (st != ICUA_OK) return st;
    p.q = a->q;
    p.out = a->out;
    p.group = a->n_q / pages->n_kv;
    p.max_rows = PA_ROWS_FEW;
    p.part = (float*)a->scratch;
    p.split = (PaSplit*)(p.part + (size_t)PA_MAX_CTAS * 2 * PA_PART);
    p.err = err_dev;
    cudaStream_t s = (cudaStream_t)stream;
    const bool f16 = a->dtype == ICUA_DT_F16, q8 = pages->dtype == ICUA_KV_Q8;
    cudaError_t e = cudaSuccess;
    bool tc_ran = false;
    const bool tc = (int64_t)seqs->max_q * p.group > PA_ROWS_FEW;
    // A batch whose sequences all seem to bring max_q tokens goes there whole, one launch less (a shorter
    // sequence that it holds all the same is then a tile like any other).
    const bool all_tc = tc && (int64_t)seqs->n_seqs * seqs->max_q == seqs->total_q;
    if (tc) {
        PagedTcParams c{};
        c.pages = p.pages;
        c.seqs = p.seqs;
        c.q = p.q;
        c.out = p.out;
        c.q_stride = p.q_stride;
        c.out_stride = p.out_stride;
        c.group = p.group;
        c.scale_log2 = p.scale_log2;
        c.min_rows = all_tc ? 0 : PA_ROWS_FEW;
        c.part = (float*)((uint8_t*)a->scratch + PA_SCRATCH);
        c.err = err_dev;
        const TcGrid g = tc_grid(seqs, pages->n_kv, p.group, c.min_rows, sm_count(dev));
        c.n_split = g.n_split;
        c.polls = icua_host::paged_wait_polls.load(std::memory_order_relaxed);
        tc_ran = g.tiles > 0;
        if (tc_ran)
            e = q8 ? (f16 ? launch_attn_tc<__half, true>(c, g.tiles, dev, s) : launch_attn_tc<__nv_bfloat16, true>(c, g.tiles, dev, s))
                : f16 ? launch_attn_tc<__half, false>(c, g.tiles, dev, s)
                      : launch_attn_tc<__nv_bfloat16, false>(c, g.tiles, dev, s);
    }
    p.alone = !tc;
    if (e == cudaSuccess && !all_tc) {
        const bool one_tile = (int64_t)seqs->max_q * p.group <= 16;
        const int64_t items = (int64_t)seqs->n_seqs * pages->n_kv;
        const bool few = one_tile && items * PA_CLUSTER <= sm_count(dev);
        const Share share = few && seqs->max_kv <= PA_CLUSTER_KEYS ? Share::cluster : seqs->max_kv <= cta_keys(items) ? Share::cta : Share::line;
        if (share != Share::line) p.max_rows = one_tile ? 16 : 32;  // one tile per (sequence, kv head)
        e = q8 ? (f16 ? launch_attn_few<__half, true>(p, share, one_tile, tc_ran, dev, s)
                      : launch_attn_few<__nv_bfloat16, true>(p, share, one_tile, tc_ran, dev, s))
            : f16 ? launch_attn_few<__half, false>(p, share, one_tile, tc_ran, dev, s)
                  : launch_attn_few<__nv_bfloat16, false>(p, share, one_tile, tc_ran, dev, s);
    }
    return e == cudaSuccess ? ICUA_OK : cuda_fail("icua_attn_paged", e);
}

}  // extern "C"
