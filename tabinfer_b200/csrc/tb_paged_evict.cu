// tb_paged_evict.cu -- shrinks sequences of the paged int8 KV cache to a budget of rows:
// the first `sinks` and the last `recent` rows stay, the rest of the budget goes to the
// rows with the largest accumulated attention weight, and the rows that stay are copied,
// in order, into other pages (so pages shared with other sequences keep their rows).
//
//   score_j = sum over kv heads of weights[b][h][j], in 64 bits (a sum of f32 weights is
//   then exact up to far below their own rounding, so the choice does not depend on the
//   order of the sum); ties go to the lower row
#include "tb_paged.cuh"

namespace {

constexpr int ST = 1024;   // threads of a selecting CTA

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

__global__ void __launch_bounds__(ST) k_evict_select(const EvictArgs a)
{
    __shared__ unsigned hist[256];
    __shared__ unsigned long long prefix;
    __shared__ int remaining, base_kept, base_tie;
    __shared__ int wkept[ST / 32], wtie[ST / 32];
    tb_pdl_wait();
    tb_pdl_trigger();
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int cap = a.kv.cap(), nKv = a.kv.nKv;
    const int n = a.kv.checked_len(__ldg(a.lens + b));
    const int left = min(n, a.budget);
    int* kept = a.kept + (long long)b * a.budget;
    if (tid == 0) a.new_lens[b] = left;
    for (int i = left + tid; i < a.budget; i += ST) kept[i] = -1;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += ST) kept[i] = i;
        return;
    }
    const int lo = a.sinks, hi = n - a.recent, need = a.budget - a.sinks - a.recent;
    unsigned long long* keys = a.keys + (long long)b * cap;
    const float* w = a.weights + (long long)b * nKv * cap;
    for (int j = lo + tid; j < hi; j += ST) {
        double s = 0.0;
        for (int h = 0; h < nKv; h++) s += (double)w[(long long)h * cap + j];
        keys[j] = score_key(s);
    }
    if (tid == 0) {
        prefix = 0;
        remaining = need;
    }
    __syncthreads();
    // the need-th largest key, eight bits at a time from the top
    if (need > 0) {
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            const unsigned long long pre = prefix;
            for (int j = lo + tid; j < hi; j += ST) {
                const unsigned long long k = keys[j];
                if (shift == 56 || (k >> (shift + 8)) == (pre >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                int r = remaining, bin = 255;
                while (bin > 0 && (int)hist[bin] < r) r -= (int)hist[bin--];
                remaining = r;
                prefix = pre | ((unsigned long long)bin << shift);
            }
            __syncthreads();
        }
    }
    const unsigned long long thr = need > 0 ? prefix : ~0ull;
    const int ties = need > 0 ? remaining : 0;
    if (tid == 0) {
        base_kept = 0;
        base_tie = 0;
    }
    __syncthreads();
    for (int j0 = 0; j0 < n; j0 += ST) {
        const int j = j0 + tid;
        bool keep = j < n && (j < lo || j >= hi), tie = false;
        if (j >= lo && j < hi) {
            const unsigned long long k = keys[j];
            tie = ties > 0 && k == thr;
            keep = need > 0 && k > thr;
        }
        const unsigned mt = __ballot_sync(0xffffffffu, tie);
        if (lane == 0) wtie[wid] = __popc(mt);
        __syncthreads();
        int t = base_tie + __popc(mt & ((1u << lane) - 1));
        for (int i = 0; i < wid; i++) t += wtie[i];
        keep = keep || (tie && t < ties);
        const unsigned mk = __ballot_sync(0xffffffffu, keep);
        if (lane == 0) wkept[wid] = __popc(mk);
        __syncthreads();
        int at = base_kept + __popc(mk & ((1u << lane) - 1));
        for (int i = 0; i < wid; i++) at += wkept[i];
        if (keep && at < a.budget) kept[at] = j;
        __syncthreads();
        if (tid == 0) {
            for (int i = 0; i < ST / 32; i++) {
                base_kept += wkept[i];
                base_tie += wtie[i];
            }
        }
        __syncthreads();
    }
}

// a warp a kept row: K, V and their scales into the new page; then the weights
__global__ void __launch_bounds__(256) k_evict_copy(const EvictArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int lane = threadIdx.x & 31;
    const long long rows = (long long)a.kv.batch * a.budget;
    const long long warps = ((long long)gridDim.x * blockDim.x) >> 5;
    for (long long i = (blockIdx.x * (long long)blockDim.x + threadIdx.x) >> 5; i < rows; i += warps) {
        const int b = (int)(i / a.budget), at = (int)(i % a.budget);
        const int j = a.kept[i];
        if (j < 0) continue;
        const int src = a.kv.row(b, j), dst = a.dst.row(b, at);
        if (src < 0 || dst < 0) continue;
        const uint4* k0 = reinterpret_cast<const uint4*>(a.kv.Kq + (long long)src * a.row_bytes);
        const uint4* v0 = reinterpret_cast<const uint4*>(a.kv.Vq + (long long)src * a.row_bytes);
        uint4* k1 = reinterpret_cast<uint4*>(a.dst.Kq + (long long)dst * a.row_bytes);
        uint4* v1 = reinterpret_cast<uint4*>(a.dst.Vq + (long long)dst * a.row_bytes);
        for (int c = lane; c < a.row_bytes / 16; c += 32) {
            k1[c] = k0[c];
            v1[c] = v0[c];
        }
        for (int c = lane; c < a.row_scales; c += 32) {
            a.dst.Ks[(long long)dst * a.row_scales + c] = a.kv.Ks[(long long)src * a.row_scales + c];
            a.dst.Vs[(long long)dst * a.row_scales + c] = a.kv.Vs[(long long)src * a.row_scales + c];
        }
    }
    const int cap = a.kv.cap(), new_cap = a.dst.cap(), nKv = a.kv.nKv;
    const long long all = (long long)a.kv.batch * nKv * new_cap;
    for (long long i = blockIdx.x * (long long)blockDim.x + threadIdx.x; i < all; i += (long long)gridDim.x * blockDim.x) {
        const int at = (int)(i % new_cap);
        const long long bh = i / new_cap;
        const int j = at < a.budget ? a.kept[bh / nKv * a.budget + at] : -1;
        a.new_weights[i] = j >= 0 ? a.weights[bh * cap + j] : 0.0f;
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
    cudaError_t e = tb_launch(ctx, k_evict_select, dim3((unsigned)kv->batch), dim3(ST), 0, a);
    if (e == cudaSuccess) e = tb_launch(ctx, k_evict_copy, dim3((unsigned)ctx->num_sms * 8), dim3(256), 0, a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "kv_evict_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}

}  // extern "C"
