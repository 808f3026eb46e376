// tb_paged_evict.cu -- shrinks sequences of the paged int8 KV cache to a budget of rows:
// the first `sinks` and the last `recent` rows stay, the rest of the budget goes to the
// rows with the largest accumulated attention weight, and the rows that stay are copied,
// in order, into other pages (so pages shared with other sequences keep their rows).
//
//   score_j = sum over kv heads of weights[b][h][j], in 64 bits (a sum of f32 weights is
//   then exact up to far below their own rounding, so the choice does not depend on the
//   order of the sum); ties go to the lower row
//
// 16 sequences of 8192 rows and below to 2048 (8 heads of 128; 146 MB) take 51 us: scores 5,
// selection 19, copy 27 (5.4 TB/s); one of 131072 rows to 16384 (80 MB) 41, of which scores 5,
// selection 25, copy 10 (one call repeated, its weights in L2; calls over other inputs in turn
// 54 and 48).  Slower: 16 CTAs a sequence (43 us for the long one), the scores formed by the
// selecting clusters (one launch less, but 52, and 2 us more at 2048 rows), 11-bit digits (61).
#include "tb_paged.cuh"

namespace {

constexpr int ST = 1024;          // threads of a selecting CTA
constexpr int DIGIT = 8, BINS = 1 << DIGIT;   // larger digits cost more in reading the other CTAs' counts than they save
constexpr int MAX_CLUSTER = 8;    // CTAs a sequence (portable)
// Table rows a CTA takes before a sequence gets another one.  One CTA, and always eight, a call that keeps an eighth of
// the rows, over 400 MB of inputs in turn: 2048 rows 19.9 and 21.0 us, 4096 22.6 and 22.5, 16384 30.3 and 25.5, 131072
// 168 and 49; 16 sequences of up to 2048 24.5 and 26.8, of up to 8192 40.6 and 39.8; 32 of up to 4096 37.9 and 54.1.
constexpr int SLOTS = 2048;
constexpr int KEPT_KEYS = 16;     // keys a thread holds in registers; those beyond are read again each step

struct EvictArgs {
    PagedArgs kv, dst;
    const int* lens;
    const float* weights;        // [B][nKv][cap]
    int* kept;                   // [B][budget]
    int* new_lens;               // [B]
    float* new_weights;          // [B][nKv][new cap]
    unsigned long long* keys;    // [B][cap]
    int budget, sinks, recent, row_bytes, row_scales;
};

// order of the scores as unsigned numbers; a NaN comes above every number
__device__ __forceinline__ unsigned long long score_key(double s)
{
    if (s != s) return ~0ull;
    const unsigned long long u = (unsigned long long)__double_as_longlong(s + 0.0);
    return (u >> 63) ? ~u : u | (1ull << 63);
}

// not the .aligned form: it follows loops and branches in which a warp's lanes part
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory");
}
// a word of another CTA's shared memory, at the place of `p` in this one's
__device__ __forceinline__ unsigned remote(const void* p, int rank)
{
    uint32_t at;
    unsigned v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}

// scores of the rows that are to be chosen from, as ordered numbers: grid (rows / 256, sequences)
__global__ void __launch_bounds__(256) k_evict_scores(const EvictArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int b = blockIdx.y, cap = a.kv.cap(), nKv = a.kv.nKv;
    const int n = a.kv.checked_len(__ldg(a.lens + b));
    const int j = blockIdx.x * 256 + threadIdx.x;
    if (n <= a.budget || j < a.sinks || j >= n - a.recent) return;
    const float* w = a.weights + (long long)b * nKv * cap + j;
    double s = 0.0;
#pragma unroll 8
    for (int h = 0; h < nKv; h++) s += (double)__ldg(w + (long long)h * cap);
    a.keys[(long long)b * cap + j] = score_key(s);
}

// A cluster a sequence.  Its CTAs share the middle rows (between the first and the last
// ones that stay): the need-th largest score by radix, 8 bits a step from the highest bit in
// which two scores differ (above it a digit would be the same for all, and its additions in
// shared memory would queue) -- each CTA counts its rows' digits, all add up the counts of all
// over distributed shared memory -- until the digit's whole class is needed (three steps where
// scores differ, eight at most), then the rows above it and, in order, as many of its class as
// are still needed.  Bound by the steps' barriers.
__global__ void __launch_bounds__(ST) k_evict_select(const EvictArgs a)
{
    __shared__ unsigned hist[2][BINS];       // two: a step's counts are read while the next one's are made
    __shared__ int wsum[ST / 32];
    __shared__ int found_bin, found_left, found_all;
    __shared__ int wkeep[ST / 32], wtie[ST / 32], mine[2];
    __shared__ unsigned differ[2];           // bits in which this CTA's scores differ from the first one
    tb_pdl_wait();
    tb_pdl_trigger();
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    int rank, ncta;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ncta));
    const int b = blockIdx.x / ncta, cap = a.kv.cap();
    const int n = a.kv.checked_len(__ldg(a.lens + b)), left = min(n, a.budget);
    const int gt = rank * ST + tid, gs = ncta * ST;          // the thread's place in the cluster
    int* kept = a.kept + (long long)b * a.budget;
    if (gt == 0) a.new_lens[b] = left;
    if (n <= a.budget) {
        for (int i = gt; i < a.budget; i += gs) kept[i] = i < n ? i : -1;
        return;
    }
    const int lo = a.sinks, hi = n - a.recent, need = a.budget - a.sinks - a.recent;
    for (int i = gt; i < a.sinks; i += gs) kept[i] = i;
    for (int i = gt; i < a.recent; i += gs) kept[a.budget - a.recent + i] = hi + i;
    if (need == 0) return;
    // this CTA's rows
    const int span = ((hi - lo + ncta - 1) / ncta + 31) & ~31;
    const int j0 = min(hi, lo + rank * span), j1 = min(hi, j0 + span);
    unsigned long long* keys = a.keys + (long long)b * cap;
    unsigned long long own[KEPT_KEYS];
#pragma unroll
    for (int i = 0; i < KEPT_KEYS; i++) {
        const int j = j0 + tid + i * ST;
        own[i] = j < j1 ? keys[j] : 0;
    }
    // the bits that all scores share
    const unsigned long long ref = __ldcg(keys + lo);
    if (tid < 2) differ[tid] = 0;
    __syncthreads();
    {
        unsigned long long d = 0;
#pragma unroll
        for (int i = 0; i < KEPT_KEYS; i++)
            if (j0 + tid + i * ST < j1) d |= own[i] ^ ref;
        for (int j = j0 + tid + KEPT_KEYS * ST; j < j1; j += ST) d |= keys[j] ^ ref;
        const unsigned d0 = __reduce_or_sync(0xffffffffu, (unsigned)d), d1 = __reduce_or_sync(0xffffffffu, (unsigned)(d >> 32));
        if (lane == 0) {
            atomicOr(&differ[0], d0);
            atomicOr(&differ[1], d1);
        }
    }
    cluster_sync();
    unsigned long long all = 0;
#pragma unroll
    for (int r = 0; r < MAX_CLUSTER; r++)
        if (r < ncta) all |= (unsigned long long)remote(&differ[1], r) << 32 | remote(&differ[0], r);
    int shift = 64 - __clzll((long long)all), remaining = need;
    unsigned long long prefix = shift < 64 ? ref >> shift : 0;   // of the class looked at: the key's bits from `shift` on
    for (int step = 0; shift > 0; step++) {
        const int bits = min(DIGIT, shift), next = shift - bits;
        unsigned* cnt = hist[step & 1];
        for (int i = tid; i < BINS; i += ST) cnt[i] = 0;
        __syncthreads();
        auto count = [&](unsigned long long k, int j) {
            if (j < j1 && (shift == 64 || (k >> shift) == prefix)) atomicAdd(&cnt[(k >> next) & ((1u << bits) - 1)], 1u);
        };
#pragma unroll
        for (int i = 0; i < KEPT_KEYS; i++) count(own[i], j0 + tid + i * ST);
        for (int j = j0 + tid + KEPT_KEYS * ST; j < j1; j += ST) count(keys[j], j);
        cluster_sync();
        // classes from the top: thread t < 256 has 255 - t
        int c = 0;
        if (tid < BINS) {
#pragma unroll
            for (int r = 0; r < MAX_CLUSTER; r++)
                if (r < ncta) c += (int)remote(&cnt[BINS - 1 - tid], r);
        }
        int x = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += v;
        }
        if (lane == 31) wsum[wid] = x;
        __syncthreads();
        if (tid < BINS) {
            int above = x - c;
            for (int i = 0; i < wid; i++) above += wsum[i];
            if (above < remaining && remaining <= above + c) {
                found_bin = BINS - 1 - tid;
                found_left = remaining - above;
                found_all = remaining == above + c;
            }
        }
        __syncthreads();
        prefix = (prefix << bits) | (unsigned)found_bin;
        remaining = found_left;
        shift = next;
        if (found_all) break;
    }
    // ---- rows above the class stay, and the first `remaining` of it: a warp a run of rows
    const int run = (span / 32 + ST / 32 - 1) / (ST / 32) * 32, k0 = j0 + wid * run, k1 = min(j1, k0 + run);
    auto look = [&](int j, unsigned& above, unsigned& tie) {
        const unsigned long long k = j < k1 ? keys[j] >> shift : 0;
        above = __ballot_sync(0xffffffffu, j < k1 && k > prefix);
        tie = __ballot_sync(0xffffffffu, j < k1 && k == prefix);
    };
    int na = 0, nt = 0;
#pragma unroll 8
    for (int j = k0; j < k1; j += 32) {
        unsigned above, tie;
        look(j + lane, above, tie);
        na += __popc(above);
        nt += __popc(tie);
    }
    if (lane == 0) {
        wkeep[wid] = na;
        wtie[wid] = nt;
    }
    __syncthreads();
    if (tid < 2) {
        int s = 0;
        for (int i = 0; i < ST / 32; i++) s += tid ? wtie[i] : wkeep[i];
        mine[tid] = s;
    }
    cluster_sync();
    int ka = 0, kt = 0;                       // above and ties before this warp's run
    for (int r = 0; r < rank; r++) {
        ka += (int)remote(&mine[0], r);
        kt += (int)remote(&mine[1], r);
    }
    for (int i = 0; i < wid; i++) {
        ka += wkeep[i];
        kt += wtie[i];
    }
#pragma unroll 8
    for (int j = k0; j < k1; j += 32) {
        unsigned above, tie;
        look(j + lane, above, tie);
        const unsigned low = (1u << lane) - 1;
        const int t = kt + __popc(tie & low);
        const bool keep = ((above >> lane) & 1) || (((tie >> lane) & 1) && t < remaining);
        if (keep) kept[a.sinks + ka + __popc(above & low) + min(t, remaining)] = j + lane;
        ka += __popc(above);
        kt += __popc(tie);
    }
    cluster_sync();                           // no CTA leaves while its counts may be read
}

// A warp CR kept rows at a time, K, V and their scales into the new pages: every load of a
// round before its first store, so the rows' bytes are in flight together.  Then the weights.
constexpr int CR = 4;
__global__ void __launch_bounds__(256) k_evict_copy(const EvictArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int lane = threadIdx.x & 31, warps = (int)(gridDim.x * blockDim.x) >> 5;
    const int gw = (int)(blockIdx.x * blockDim.x + threadIdx.x) >> 5, chunks = a.row_bytes / 16;
    const long long rows = (long long)a.kv.batch * a.budget;
    for (long long i0 = (long long)gw * CR; i0 < rows; i0 += (long long)warps * CR) {
        // lanes 0 .. CR - 1 look the rows up
        long long from = -1, to = -1;
        const long long i = i0 + lane;
        if (lane < CR && i < rows) {
            const int b = (int)(i / a.budget), at = (int)(i - (long long)b * a.budget), j = __ldg(a.kept + i);
            if (j >= 0) {
                from = a.kv.row(b, j);
                to = a.dst.row(b, at);
            }
        }
        long long src[CR], dst[CR];
#pragma unroll
        for (int r = 0; r < CR; r++) {
            src[r] = __shfl_sync(0xffffffffu, from, r);
            dst[r] = __shfl_sync(0xffffffffu, to, r);
            if (src[r] < 0) dst[r] = -1;
        }
        for (int c = lane; c < chunks; c += 32) {
            uint4 k[CR], v[CR];
#pragma unroll
            for (int r = 0; r < CR; r++)
                if (dst[r] >= 0) {
                    k[r] = __ldcs(reinterpret_cast<const uint4*>(a.kv.Kq + src[r] * a.row_bytes) + c);
                    v[r] = __ldcs(reinterpret_cast<const uint4*>(a.kv.Vq + src[r] * a.row_bytes) + c);
                }
#pragma unroll
            for (int r = 0; r < CR; r++)
                if (dst[r] >= 0) {
                    reinterpret_cast<uint4*>(a.dst.Kq + dst[r] * a.row_bytes)[c] = k[r];
                    reinterpret_cast<uint4*>(a.dst.Vq + dst[r] * a.row_bytes)[c] = v[r];
                }
        }
        for (int c = lane; c < a.row_scales; c += 32) {
            float k[CR], v[CR];
#pragma unroll
            for (int r = 0; r < CR; r++)
                if (dst[r] >= 0) {
                    k[r] = __ldcs(a.kv.Ks + src[r] * a.row_scales + c);
                    v[r] = __ldcs(a.kv.Vs + src[r] * a.row_scales + c);
                }
#pragma unroll
            for (int r = 0; r < CR; r++)
                if (dst[r] >= 0) {
                    a.dst.Ks[dst[r] * a.row_scales + c] = k[r];
                    a.dst.Vs[dst[r] * a.row_scales + c] = v[r];
                }
        }
    }
    const int cap = a.kv.cap(), new_cap = a.dst.cap(), nKv = a.kv.nKv;
    // (sequence, head) pairs over the grid's y, rows over x
    for (int bh = blockIdx.x % (a.kv.batch * nKv); bh < a.kv.batch * nKv; bh += gridDim.x) {
        const int part = blockIdx.x / (a.kv.batch * nKv), parts = max(1, (int)gridDim.x / (a.kv.batch * nKv));
        if (part >= parts) break;
        const int* kept = a.kept + (long long)(bh / nKv) * a.budget;
        for (int at = part * 256 + threadIdx.x; at < new_cap; at += parts * 256) {
            const int j = at < a.budget ? __ldg(kept + at) : -1;
            a.new_weights[(long long)bh * new_cap + at] = j >= 0 ? __ldg(a.weights + (long long)bh * cap + j) : 0.0f;
        }
    }
}

}  // namespace

extern "C" {

TB_API int tb_kv_evict_paged_ws(tb_ctx* ctx, const tb_paged_kv* kv, size_t* bytes)
{
    if (!ctx || !bytes) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (rc) return rc;
    *bytes = (size_t)kv->batch * kv->max_pages * kv->page_rows * sizeof(unsigned long long);
    return TB_OK;
}

TB_API int tb_kv_evict_paged_q8(tb_ctx* ctx, const tb_paged_kv* kv, const tb_paged_kv* dst, const int32_t* lens,
                                const float* weights, int32_t* kept, int32_t* new_lens, float* new_weights,
                                int64_t budget, int64_t sinks, int64_t recent, void* ws, size_t ws_bytes)
{
    if (!ctx) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check(ctx, dst);
    if (rc) return rc;
    TB_REQUIRE(ctx, lens && weights && kept && new_lens && new_weights, "null pointer");
    TB_REQUIRE(ctx, kv->nKv == dst->nKv && kv->hd == dst->hd && kv->batch == dst->batch,
               "the new pages must have the cache's heads, head_dim and batch");
    TB_REQUIRE(ctx, sinks >= 0 && recent >= 0 && budget > 0 && sinks + recent <= budget,
               "needs sinks, recent >= 0 and sinks + recent <= budget");
    TB_REQUIRE(ctx, budget <= dst->max_pages * dst->page_rows, "the new table holds %lld rows, less than the budget",
               (long long)(dst->max_pages * dst->page_rows));
    size_t need = 0;
    rc = tb_kv_evict_paged_ws(ctx, kv, &need);
    if (rc) return rc;
    DeviceGuard dev(ctx->device);
    if (!ws) {
        ws = tb_ctx_scratch(ctx, need);
        if (!ws) return TB_ERR_NOMEM;
    } else {
        TB_REQUIRE(ctx, TB_ALIGNED(ws, 256) && ws_bytes >= need, "workspace: %zu bytes, 256-byte aligned, are needed", need);
    }
    EvictArgs a{};
    a.kv = paged_args(ctx, kv);
    a.dst = paged_args(ctx, dst);
    a.lens = lens;
    a.weights = weights;
    a.kept = kept;
    a.new_lens = new_lens;
    a.new_weights = new_weights;
    a.keys = static_cast<unsigned long long*>(ws);
    a.budget = (int)budget;
    a.sinks = (int)sinks;
    a.recent = (int)recent;
    a.row_bytes = (int)(kv->nKv * kv->hd);
    a.row_scales = a.row_bytes / 32;
    // budget == sinks + recent: nothing to choose
    const int64_t cap = kv->max_pages * kv->page_rows;
    cudaError_t e = cudaSuccess;
    if (budget > sinks + recent)
        e = tb_launch(ctx, k_evict_scores, dim3((unsigned)((cap + 255) / 256), (unsigned)kv->batch), dim3(256), 0, a);
    int cluster = 1;
    while (cluster < MAX_CLUSTER && cap > (int64_t)cluster * SLOTS) cluster *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(kv->batch * cluster));
    cfg.blockDim = dim3(ST);
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = ctx->pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, k_evict_select, a);
    if (e == cudaSuccess) e = tb_launch(ctx, k_evict_copy, dim3((unsigned)ctx->num_sms * 8), dim3(256), 0, a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "kv_evict_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}

}  // extern "C"
