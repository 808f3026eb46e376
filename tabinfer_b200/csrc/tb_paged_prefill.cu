// tb_paged_prefill.cu -- attention of packed prompts or chunks of prompts over the paged
// int8 KV cache: causal, GQA, a sliding window with first tokens kept.
//
// Rows cu[b] .. cu[b+1]-1 of q are the last t_b = cu[b+1]-cu[b] rows of sequence b; query i
// stands at row n_b - t_b + i.  One CTA a (query, kv head): each warp takes 32-key tiles
// with its own running maximum and sum, and the warps meet at the end.
#include <cuda_bf16.h>

#include "tb_attn_dev.cuh"
#include "tb_paged.cuh"

namespace {

constexpr int W = 4, NT = 32 * W;

struct PrefillArgs {
    PagedArgs kv;
    const float* q;         // [T][nHq*HD]
    __nv_bfloat16* out;     // [T][nHq*HD]
    const int* cu;          // [B+1]
    const int* lens;        // [B]
    int T, nHq, window, sinks;
    float qscale;
};

template <int HD, int GRP>
__global__ void __launch_bounds__(NT) k_paged_prefill(const PrefillArgs a)
{
    __shared__ float qs[GRP][HD];
    __shared__ float wo[W][GRP][HD];
    __shared__ float wm[W][GRP], wl[W][GRP];
    tb_pdl_wait();
    tb_pdl_trigger();
    constexpr int NG = HD / 32, DPL = HD / 32;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int nKv = a.kv.nKv, nHq = a.nHq, t = blockIdx.x, h = blockIdx.y;
    int lo = 0, hi = a.kv.batch;             // the sequence with cu[b] <= t < cu[b+1]
    if (t < __ldg(a.cu) || t >= __ldg(a.cu + hi)) return;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (__ldg(a.cu + mid) <= t) lo = mid;
        else hi = mid;
    }
    const int b = lo, first = __ldg(a.cu + b), rows = __ldg(a.cu + b + 1) - first;
    const int n = a.kv.checked_len(__ldg(a.lens + b)), pos = n - rows + t - first;
    if (pos < 0 && tid == 0) atomicExch(a.kv.err, ERR_PAGED_LEN);
    for (int i = tid; i < GRP * HD; i += NT)
        qs[i / HD][i % HD] = a.q[(long long)t * nHq * HD + h * GRP * HD + i] * a.qscale;
    __syncthreads();
    float m[GRP], l[GRP], o[GRP][DPL];
#pragma unroll
    for (int g = 0; g < GRP; g++) {
        m[g] = NEG_BIG;
        l[g] = 0.0f;
#pragma unroll
        for (int i = 0; i < DPL; i++) o[g][i] = 0.0f;
    }
    const SeenTiles seen(pos, pos, a.window, a.sinks);
    for (int i = wid; i < seen.count; i += W) {
        const int key = seen.tile(i) * KT + lane;
        bool ok = key_seen(key, pos, a.window, a.sinks);
        const int row = ok ? a.kv.row(b, key) : -1;
        ok = row >= 0;
        const long long at = (long long)(ok ? row : 0) * nKv * HD + h * HD;
        float s[GRP], p[GRP];
#pragma unroll
        for (int g = 0; g < GRP; g++) s[g] = 0.0f;
        if (ok) {
            for (int G = 0; G < NG; G++) {
                float part[GRP];
#pragma unroll
                for (int g = 0; g < GRP; g++) part[g] = 0.0f;
                for (int d = 0; d < 32; d++) {
                    const float x = (float)a.kv.Kq[at + 32 * G + d];
#pragma unroll
                    for (int g = 0; g < GRP; g++) part[g] = fmaf(x, qs[g][32 * G + d], part[g]);
                }
                const float sc = a.kv.Ks[at / 32 + G] * (1.0f / 127.0f);
#pragma unroll
                for (int g = 0; g < GRP; g++) s[g] = fmaf(part[g], sc, s[g]);
            }
        }
#pragma unroll
        for (int g = 0; g < GRP; g++) {
            const float x = ok ? s[g] : NEG_BIG;
            const float mn = fmaxf(m[g], warp_max(x)), corr = exp2f(m[g] - mn);
            p[g] = ok ? exp2f(x - mn) : 0.0f;
            l[g] = fmaf(l[g], corr, p[g]);
            m[g] = mn;
#pragma unroll
            for (int j = 0; j < DPL; j++) o[g][j] *= corr;
        }
        for (int k = 0; k < KT; k++) {
            const int r = __shfl_sync(0xffffffffu, row, k);
            float pk[GRP];
#pragma unroll
            for (int g = 0; g < GRP; g++) pk[g] = __shfl_sync(0xffffffffu, p[g], k);
            if (r < 0) continue;
            const long long va = (long long)r * nKv * HD + h * HD;
#pragma unroll
            for (int j = 0; j < DPL; j++) {
                const float v = (float)a.kv.Vq[va + 32 * j + lane] * (a.kv.Vs[va / 32 + j] * (1.0f / 127.0f));
#pragma unroll
                for (int g = 0; g < GRP; g++) o[g][j] = fmaf(pk[g], v, o[g][j]);
            }
        }
    }
#pragma unroll
    for (int g = 0; g < GRP; g++) {
        const float lt = warp_sum(l[g]);
        if (lane == 0) {
            wm[wid][g] = m[g];
            wl[wid][g] = lt;
        }
#pragma unroll
        for (int j = 0; j < DPL; j++) wo[wid][g][32 * j + lane] = o[g][j];
    }
    __syncthreads();
    for (int i = tid; i < GRP * HD; i += NT) {
        const int g = i / HD, d = i % HD;
        float M = NEG_BIG, L = 0.0f, O = 0.0f;
#pragma unroll
        for (int k = 0; k < W; k++) M = fmaxf(M, wm[k][g]);
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float e = exp2f(wm[k][g] - M);
            L = fmaf(wl[k][g], e, L);
            O = fmaf(wo[k][g][d], e, O);
        }
        a.out[(long long)t * nHq * HD + (h * GRP + g) * HD + d] = __float2bfloat16_rn(L > 0.0f ? O / L : 0.0f);
    }
}

template <int HD, int GRP>
int launch_prefill(tb_ctx* ctx, const PrefillArgs& a)
{
    cudaError_t e = tb_launch(ctx, k_paged_prefill<HD, GRP>, dim3(a.T, a.kv.nKv), dim3(NT), 0, a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "attn_prefill_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}

}  // namespace

extern "C" {

TB_API int tb_attn_prefill_paged_ws(tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, int64_t T, size_t* bytes)
{
    if (!ctx || !bytes) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check_heads(ctx, kv, nHq);
    if (rc) return rc;
    TB_REQUIRE(ctx, T >= 0 && T < (1LL << 31), "bad row count %lld", (long long)T);
    *bytes = 0;
    return TB_OK;
}

TB_API int tb_attn_prefill_paged_q8(tb_ctx* ctx, const tb_paged_kv* kv, uint16_t* out_bf16, const float* q,
                                    const int32_t* cu, const int32_t* lens, int64_t nHq, int64_t T, int64_t window,
                                    int64_t sinks, void* ws, size_t ws_bytes)
{
    if (!ctx) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check_heads(ctx, kv, nHq);
    if (rc) return rc;
    TB_REQUIRE(ctx, T >= 0 && T < (1LL << 31), "bad row count %lld", (long long)T);
    TB_REQUIRE(ctx, window >= 0 && sinks >= 0, "window and sinks must not be negative");
    if (T == 0) return TB_OK;
    TB_REQUIRE(ctx, out_bf16 && q && cu && lens, "null pointer");
    TB_REQUIRE(ctx, TB_ALIGNED(out_bf16, 16) && TB_ALIGNED(q, 16), "q and out must be 16-byte aligned");
    DeviceGuard dev(ctx->device);
    (void)ws;
    (void)ws_bytes;
    PrefillArgs a{};
    a.kv = paged_args(ctx, kv);
    a.q = q;
    a.out = reinterpret_cast<__nv_bfloat16*>(out_bf16);
    a.cu = cu;
    a.lens = lens;
    a.T = (int)T;
    a.nHq = (int)nHq;
    a.window = (int)std::min<int64_t>(window, 1LL << 30);
    a.sinks = (int)std::min<int64_t>(sinks, 1LL << 30);
    a.qscale = 1.4426950408889634f / sqrtf((float)kv->hd);
    switch ((int)(kv->hd * 10 + nHq / kv->nKv)) {
    case 641: return launch_prefill<64, 1>(ctx, a);
    case 642: return launch_prefill<64, 2>(ctx, a);
    case 644: return launch_prefill<64, 4>(ctx, a);
    case 648: return launch_prefill<64, 8>(ctx, a);
    case 1281: return launch_prefill<128, 1>(ctx, a);
    case 1282: return launch_prefill<128, 2>(ctx, a);
    case 1284: return launch_prefill<128, 4>(ctx, a);
    default: return launch_prefill<128, 8>(ctx, a);
    }
}

}  // extern "C"
