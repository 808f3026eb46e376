// tb_paged.cuh -- what the paged int8 KV cache operators share: the cache's
// description on the device, the lookup of a row, and the tiles of keys that a
// query sees under a sliding window with first tokens kept.
//
// Pools Kq / Vq int8 [n_pages][page_rows][nKv*hd], Ks / Vs f32
// [n_pages][page_rows][nKv*hd/32]: each page holds rows in the format of the
// contiguous cache (tb_attn.cu), so one page of S_max rows is that cache.  Row r
// of sequence b is line r % page_rows of page table[b][r / page_rows].
#pragma once
#include "tb_internal.h"

namespace {

// error word codes (tb_ctx_device_error): a page number outside the pool, a
// length or a row outside the table, a chunk longer than its sequence
constexpr int ERR_PAGED_PAGE = 0x6c01;
constexpr int ERR_PAGED_LEN = 0x6c02;
// a bounded wait on a copy or an MMA of the CTA's own gave up
constexpr int ERR_PAGED_WAIT = 0x6c03;

constexpr int KT = 32;   // keys a tile: a tile starts on a multiple of KT rows

struct PagedArgs {
    int8_t* Kq;
    float* Ks;
    int8_t* Vq;
    float* Vs;
    const int* table;    // [batch][max_pages]
    int n_pages, log_page, max_pages, batch, nKv;
    int* err;

    __device__ __forceinline__ int cap() const { return max_pages << log_page; }
    // pool row of cache row r of sequence b (r < cap()), -1 for a page outside the pool
    __device__ __forceinline__ int row(int b, int r) const
    {
        const int p = __ldg(table + (long long)b * max_pages + (r >> log_page));
        if ((unsigned)p >= (unsigned)n_pages) {
            atomicExch(err, ERR_PAGED_PAGE);
            return -1;
        }
        return (p << log_page) | (r & ((1 << log_page) - 1));
    }
    // cached rows of a sequence; one that the table cannot hold counts as empty
    __device__ __forceinline__ int checked_len(int n) const
    {
        if (n >= 0 && n <= cap()) return n;
        atomicExch(err, ERR_PAGED_LEN);
        return 0;
    }
};

// The keys that the queries at rows p0 .. p1 see between them (key j <= p, and with a
// window p - j < window or j < sinks): rows [0, sinks) and [lo, p1], as tiles of kt keys.
struct SeenTiles {
    int first, from, count;   // tiles 0 .. first-1, then from .. from+count-first-1

    __device__ __forceinline__ SeenTiles(int p0, int p1, int window, int sinks, int kt = KT)
    {
        const int end = p1 < 0 ? 0 : p1 / kt + 1;
        const int lo = window > 0 && p0 >= window ? p0 - window + 1 : 0;
        from = lo / kt;
        first = min(from, (min(sinks, lo) + kt - 1) / kt);
        count = first + max(0, end - from);
    }
    __device__ __forceinline__ int tile(int i) const { return i < first ? i : from + i - first; }
};

__device__ __forceinline__ bool key_seen(int key, int pos, int window, int sinks)
{
    return key <= pos && (window <= 0 || pos - key < window || key < sinks);
}

// the warp's largest value (NaN left out, as fmaxf does)
__device__ __forceinline__ float redux_max(float v)
{
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// ---- mbarriers and asynchronous copies -------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* b, unsigned count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b)
{
    asm volatile("{\n .reg .b64 st;\n mbarrier.arrive.shared::cta.b64 st, [%0];\n}" ::"r"(smem_u32(b)) : "memory");
}
// whether the phase of this parity has completed (no suspension: half the time of a try_wait
// whose phase has)
__device__ __forceinline__ bool mbar_test(uint64_t* b, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(smem_u32(b)), "r"(parity) : "memory");
    return done != 0;
}
// Waits until the phase of this parity has completed; at most WAIT_TRIES tries of up to
// 1 ms each, after which (or when *abort is up) it returns false.
constexpr int WAIT_TRIES = 1000;
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity, volatile int* abort = nullptr)
{
    const uint32_t a = smem_u32(b);
    for (int it = 0; it < WAIT_TRIES; it++) {
        uint32_t done;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n"
                     " selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done) : "r"(a), "r"(parity), "r"(1000000u) : "memory");
        if (done) return true;
        if (abort && *abort) return false;
    }
    return false;
}
// 16- and 8-byte copies a thread
__device__ __forceinline__ void cp_async16(void* sdst, const void* gsrc)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(sdst)), "l"(gsrc) : "memory");
}
__device__ __forceinline__ void cp_async8(void* sdst, const void* gsrc)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(sdst)), "l"(gsrc) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// The boxes at (x, y) of two 2-D tensor maps into shared memory (x: a multiple of 16 bytes), and the
// bytes that a barrier is to expect: run by a whole warp with uniform operands, one thread issues.
__device__ __forceinline__ void tma_2d_elect(void* dst0, const CUtensorMap* map0, void* dst1, const CUtensorMap* map1, int x,
                                             int y, uint64_t* bar)
{
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%4, %5}], [%6];\n"
                 " @e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%2], [%3, {%4, %5}], [%6];\n}"
                 ::"r"(smem_u32(dst0)), "l"(reinterpret_cast<uint64_t>(map0)), "r"(smem_u32(dst1)),
                   "l"(reinterpret_cast<uint64_t>(map1)), "r"(x), "r"(y), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void mbar_expect_elect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// makes a context's device the current one for a call's launches
struct DeviceGuard {
    int prev = -1;
    bool moved = false;
    explicit DeviceGuard(int device)
    {
        if (cudaGetDevice(&prev) == cudaSuccess && prev != device) moved = cudaSetDevice(device) == cudaSuccess;
    }
    ~DeviceGuard()
    {
        if (moved) cudaSetDevice(prev);
    }
};

inline int paged_check(tb_ctx* ctx, const tb_paged_kv* kv)
{
    TB_REQUIRE(ctx, kv != nullptr, "null cache");
    TB_REQUIRE(ctx, kv->Kq && kv->Ks && kv->Vq && kv->Vs && kv->table, "null cache pointer");
    TB_REQUIRE(ctx, TB_ALIGNED(kv->Kq, 16) && TB_ALIGNED(kv->Vq, 16) && TB_ALIGNED(kv->Ks, 16) &&
                        TB_ALIGNED(kv->Vs, 16), "KV cache must be 16-byte aligned");
    TB_REQUIRE(ctx, kv->page_rows >= 16 && kv->page_rows <= 256 && (kv->page_rows & (kv->page_rows - 1)) == 0,
               "page_rows must be 16, 32, 64, 128 or 256 (got %lld)", (long long)kv->page_rows);
    TB_REQUIRE(ctx, kv->n_pages > 0 && kv->n_pages <= (1LL << 31) / kv->page_rows - 1, "bad page count %lld",
               (long long)kv->n_pages);
    TB_REQUIRE(ctx, kv->max_pages > 0 && kv->max_pages <= (1LL << 30) / kv->page_rows, "bad table width %lld",
               (long long)kv->max_pages);
    TB_REQUIRE(ctx, kv->batch > 0 && kv->batch <= 65535, "batch must be 1..65535 (got %lld)", (long long)kv->batch);
    TB_REQUIRE(ctx, kv->nKv > 0 && kv->nKv <= 1024, "bad kv head count %lld", (long long)kv->nKv);
    TB_REQUIRE(ctx, kv->hd == 64 || kv->hd == 128, "head_dim must be 64 or 128 (got %lld)", (long long)kv->hd);
    return TB_OK;
}

inline int paged_check_heads(tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq)
{
    const int64_t g = nHq > 0 && nHq % kv->nKv == 0 ? nHq / kv->nKv : 0;
    if (g != 1 && g != 2 && g != 4 && g != 8)
        return tb_fail(ctx, TB_ERR_UNSUPPORTED, "nHq/nKv = %lld/%lld not built (1, 2, 4, 8)", (long long)nHq,
                       (long long)kv->nKv);
    return TB_OK;
}

inline PagedArgs paged_args(tb_ctx* ctx, const tb_paged_kv* kv)
{
    PagedArgs a{};
    a.Kq = kv->Kq;
    a.Ks = kv->Ks;
    a.Vq = kv->Vq;
    a.Vs = kv->Vs;
    a.table = kv->table;
    a.n_pages = (int)kv->n_pages;
    a.log_page = __builtin_ctzll((unsigned long long)kv->page_rows);
    a.max_pages = (int)kv->max_pages;
    a.batch = (int)kv->batch;
    a.nKv = (int)kv->nKv;
    a.err = ctx->dev_error;
    return a;
}

}  // namespace
