// tb_paged_decode.cu -- attention of one new token a sequence over the paged int8 KV
// cache: ragged lengths, GQA, a sliding window with first tokens kept, and (optionally)
// the keys' attention weights added to an accumulator.
//
//   s_j = q . k_j / sqrt(hd) over the keys seen;  p = softmax(s);  out = sum_j p_j v_j
//   weights[b][kv head][j] += sum over the head's group of p_j
//
// The keys seen are a list of 32-key tiles; W consecutive tiles are a chunk, and the
// chunks of all (sequence, kv head) pairs in order are dealt out evenly to the CTAs, so
// ragged batches and long single sequences fill the machine alike.  A CTA whose range
// holds only a part of a pair's chunks writes (m, l, o) for it (at most two such parts a
// CTA: its first and its last pair); k_paged_combine joins a pair's parts in order, so
// results do not depend on timing.
#include "tb_attn_dev.cuh"
#include "tb_paged.cuh"

namespace {

constexpr int W = 4, NT = 32 * W;

struct DecArgs {
    PagedArgs kv;
    const float* q;        // [B][nHq*HD]
    float* out;            // [B][nHq*HD]
    const int* lens;       // [B]
    float* PO;             // [grid][2][GRP][HD]
    float2* PML;           // [grid][2][GRP]
    float* SC;             // [B][nKv][cap][GRP] scores (log2), when weights are wanted
    float2* ML;            // [B][nHq] final (m, l), when weights are wanted
    float* weights;        // [B][nKv][cap]
    int nHq, window, sinks, grid;
    float qscale;          // log2(e) / sqrt(HD)
};

__device__ __forceinline__ SeenTiles seen_of(const DecArgs& a, int n) { return SeenTiles(n - 1, n - 1, a.window, a.sinks); }
__device__ __forceinline__ int chunks_of(const DecArgs& a, int b)
{
    return (seen_of(a, a.kv.checked_len(__ldg(a.lens + b))).count + W - 1) / W;
}

// Sums of the sequences' chunk counts, by all NT threads: returns the total; the thread
// whose slice of sequences holds chunk index `at` (in units of one kv head's chunks when
// nKv = 1) finds its sequence.  before(b) sums: pass find_b >= 0 to get the sum below
// sequence find_b in *below, else the sequence holding unit `at` of the nKv-fold list.
struct Where {
    long long total;   // chunks of one kv head over all sequences
    int b;             // the sequence found
    long long below;   // chunks of one kv head in the sequences below b
};
__device__ Where locate(const DecArgs& a, int find_b, long long per_of, long long cta)
{
    __shared__ long long sums[NT];
    __shared__ Where found;
    const int tid = threadIdx.x, B = a.kv.batch, slice = (B + NT - 1) / NT;
    const int b0 = min(B, tid * slice), b1 = min(B, b0 + slice);
    long long mine = 0;
    for (int b = b0; b < b1; b++) mine += chunks_of(a, b);
    sums[tid] = mine;
    __syncthreads();
    if (B > slice) {      // more than one slice in use: inclusive scan
        for (int o = 1; o < NT; o <<= 1) {
            const long long v = tid >= o ? sums[tid - o] : 0;
            __syncthreads();
            sums[tid] += v;
            __syncthreads();
        }
    } else if (tid > 0) {
        sums[tid] = sums[0];
    }
    __syncthreads();
    const long long total = sums[NT - 1];
    // the unit looked for, in chunks of the nKv-fold list
    const long long all = total * a.kv.nKv;
    const long long per = per_of > 0 ? (all + per_of - 1) / per_of : 0;
    const long long at = cta * per;
    if (tid == 0) found = Where{total, -1, 0};
    __syncthreads();
    long long below = sums[tid] - mine;
    if (find_b >= 0) {
        if (b0 <= find_b && find_b < b1) {
            for (int b = b0; b < find_b; b++) below += chunks_of(a, b);
            found = Where{total, find_b, below};
        }
    } else if (at < all && below * a.kv.nKv <= at && at < (below + mine) * a.kv.nKv) {
        int b = b0;
        for (; b < b1; b++) {
            const int n = chunks_of(a, b);
            if (at < (below + n) * a.kv.nKv) break;
            below += n;
        }
        found = Where{total, b, below};
    }
    __syncthreads();
    return found;
}

template <int HD, int GRP>
__global__ void __launch_bounds__(NT) k_paged_decode(const DecArgs a)
{
    __shared__ float qs[GRP][HD];
    __shared__ float wo[W][GRP][HD];
    __shared__ float wm[W][GRP], wl[W][GRP];
    tb_pdl_wait();
    tb_pdl_trigger();
    constexpr int NG = HD / 32, DPL = HD / 32;
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const int nKv = a.kv.nKv, nHq = a.nHq, cta = blockIdx.x;
    const Where w = locate(a, -1, a.grid, cta);
    const long long all = w.total * nKv, per = (all + a.grid - 1) / a.grid;
    const long long u0 = cta * per, u1 = min(all, u0 + per);
    if (u0 >= u1) return;
    int b = w.b;
    long long base = w.below * nKv;          // units below sequence b
    for (long long u = u0; u < u1;) {
        const int n = a.kv.checked_len(__ldg(a.lens + b));
        const SeenTiles seen = seen_of(a, n);
        const int nc = (seen.count + W - 1) / W;
        if (u >= base + (long long)nc * nKv) {
            base += (long long)nc * nKv;
            b++;
            continue;
        }
        const int h = (int)((u - base) / nc), c0 = (int)((u - base) % nc);
        const int c1 = (int)min((long long)nc, c0 + (u1 - u));
        __syncthreads();
        for (int i = tid; i < GRP * HD; i += NT)
            qs[i / HD][i % HD] = a.q[(long long)b * nHq * HD + h * GRP * HD + i] * a.qscale;
        __syncthreads();
        float m[GRP], l[GRP], o[GRP][DPL];
#pragma unroll
        for (int g = 0; g < GRP; g++) {
            m[g] = NEG_BIG;
            l[g] = 0.0f;
#pragma unroll
            for (int i = 0; i < DPL; i++) o[g][i] = 0.0f;
        }
        const int t1 = min(seen.count, c1 * W);
        for (int i = c0 * W + wid; i < t1; i += W) {
            const int key = seen.tile(i) * KT + lane;
            bool ok = key_seen(key, n - 1, a.window, a.sinks);
            int row = ok ? a.kv.row(b, key) : -1;
            ok = row >= 0;
            const long long at = (long long)(ok ? row : 0) * nKv * HD + h * HD;
            float s[GRP];
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
            float p[GRP];
#pragma unroll
            for (int g = 0; g < GRP; g++) {
                const float x = ok ? s[g] : NEG_BIG;
                const float mn = fmaxf(m[g], warp_max(x)), corr = exp2f(m[g] - mn);
                p[g] = ok ? exp2f(x - mn) : 0.0f;
                l[g] = fmaf(l[g], corr, p[g]);
                m[g] = mn;
#pragma unroll
                for (int j = 0; j < DPL; j++) o[g][j] *= corr;
                if (a.SC && key < a.kv.cap())
                    a.SC[(((long long)b * nKv + h) * a.kv.cap() + key) * GRP + g] = ok ? x : -INFINITY;
            }
            for (int k = 0; k < KT; k++) {
                const int r = __shfl_sync(0xffffffffu, row, k);
                float pk[GRP];
#pragma unroll
                for (int g = 0; g < GRP; g++) pk[g] = __shfl_sync(0xffffffffu, p[g], k);
                if (r < 0) continue;
                const long long va = (long long)r * nKv * HD + h * HD;
#pragma unroll
                for (int j = 0; j < DPL; j++) {      // lane holds dims 32 j + lane
                    const float v = (float)a.kv.Vq[va + 32 * j + lane] * (a.kv.Vs[va / 32 + j] * (1.0f / 127.0f));
#pragma unroll
                    for (int g = 0; g < GRP; g++) o[g][j] = fmaf(pk[g], v, o[g][j]);
                }
            }
        }
        // ---- the warps' states meet
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
        const bool whole = c0 == 0 && c1 == nc;
        const long long slot = 2LL * cta + (u == u0 ? 0 : 1);
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
            if (whole) {
                a.out[(long long)b * nHq * HD + (h * GRP + g) * HD + d] = L > 0.0f ? O / L : 0.0f;
                if (d == 0 && a.ML) a.ML[(long long)b * nHq + h * GRP + g] = make_float2(M, L);
            } else {
                a.PO[(slot * GRP + g) * HD + d] = O;
                if (d == 0) a.PML[slot * GRP + g] = make_float2(M, L);
            }
        }
        u += c1 - c0;
    }
}

// joins the parts of pair (kv head x, sequence y); pairs that one CTA held are done
template <int HD, int GRP>
__global__ void __launch_bounds__(NT) k_paged_combine(const DecArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, nKv = a.kv.nKv;
    const Where w = locate(a, b, a.grid, 0);
    const int nc = chunks_of(a, b);
    float* out = a.out + (long long)b * a.nHq * HD + h * GRP * HD;
    if (nc == 0) {
        for (int i = tid; i < GRP * HD; i += NT) out[i] = 0.0f;
        return;
    }
    const long long all = w.total * nKv, per = (all + a.grid - 1) / a.grid;
    const long long u0 = w.below * nKv + (long long)h * nc, u1 = u0 + nc;
    const long long c0 = u0 / per, c1 = (u1 - 1) / per;
    if (c0 == c1) return;
    const long long s0 = 2 * c0 + (u0 == c0 * per ? 0 : 1);
    for (int i = tid; i < GRP * HD; i += NT) {
        const int g = i / HD, d = i % HD;
        float M = a.PML[s0 * GRP + g].x;
        for (long long c = c0 + 1; c <= c1; c++) M = fmaxf(M, a.PML[2 * c * GRP + g].x);
        float L = 0.0f, O = 0.0f;
        for (long long c = c0; c <= c1; c++) {
            const long long s = c == c0 ? s0 : 2 * c;
            const float2 ml = a.PML[s * GRP + g];
            const float e = exp2f(ml.x - M);
            L = fmaf(ml.y, e, L);
            O = fmaf(a.PO[(s * GRP + g) * HD + d], e, O);
        }
        out[i] = L > 0.0f ? O / L : 0.0f;
        if (d == 0 && a.ML) a.ML[(long long)b * a.nHq + h * GRP + g] = make_float2(M, L);
    }
}

// weights[b][h][j] += sum over the group of 2^(s - m) / l, for the keys seen
template <int GRP>
__global__ void __launch_bounds__(256) k_paged_weights(const DecArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int h = blockIdx.y, b = blockIdx.z, cap = a.kv.cap();
    const int n = a.kv.checked_len(__ldg(a.lens + b));
    const int j0 = blockIdx.x * 1024;
    if (j0 >= n) return;
    float m[GRP], r[GRP];
#pragma unroll
    for (int g = 0; g < GRP; g++) {
        const float2 ml = a.ML[(long long)b * a.nHq + h * GRP + g];
        m[g] = ml.x;
        r[g] = ml.y > 0.0f ? 1.0f / ml.y : 0.0f;
    }
    const long long at = ((long long)b * a.kv.nKv + h) * cap;
    for (int j = j0 + threadIdx.x; j < min(n, j0 + 1024); j += 256) {
        if (!key_seen(j, n - 1, a.window, a.sinks)) continue;
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < GRP; g++) s = fmaf(exp2f(a.SC[(at + j) * GRP + g] - m[g]), r[g], s);
        a.weights[at + j] += s;
    }
}

// device workspace: PO, PML, then (weights) ML and SC
struct DecWs {
    int grid;
    size_t po, pml, ml, sc;
    size_t bytes() const { return po + pml + ml + sc; }
};
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
DecWs dec_ws(const tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, bool weights)
{
    const int64_t cap = kv->max_pages * kv->page_rows, grp = nHq / kv->nKv;
    const int64_t chunks = kv->batch * kv->nKv * ((cap + KT * W - 1) / (KT * W));
    DecWs w{};
    w.grid = (int)std::min<int64_t>(chunks, 4LL * ctx->num_sms);
    w.po = up256((size_t)w.grid * 2 * grp * kv->hd * sizeof(float));
    w.pml = up256((size_t)w.grid * 2 * grp * sizeof(float2));
    if (weights) {
        w.ml = up256((size_t)kv->batch * nHq * sizeof(float2));
        w.sc = up256((size_t)kv->batch * nHq * cap * sizeof(float));
    }
    return w;
}

template <int HD, int GRP>
int launch_decode(tb_ctx* ctx, const DecArgs& a)
{
    cudaError_t e = tb_launch(ctx, k_paged_decode<HD, GRP>, dim3(a.grid), dim3(NT), 0, a);
    if (e == cudaSuccess) e = tb_launch(ctx, k_paged_combine<HD, GRP>, dim3(a.kv.nKv, a.kv.batch), dim3(NT), 0, a);
    if (e == cudaSuccess && a.weights)
        e = tb_launch(ctx, k_paged_weights<GRP>,
                      dim3(tb_cdiv((long long)a.kv.max_pages << a.kv.log_page, 1024), a.kv.nKv, a.kv.batch), dim3(256), 0, a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "attn_decode_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}

}  // namespace

extern "C" {

TB_API int tb_attn_decode_paged_ws(tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, int weights, size_t* bytes)
{
    if (!ctx || !bytes) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check_heads(ctx, kv, nHq);
    if (rc) return rc;
    *bytes = dec_ws(ctx, kv, nHq, weights != 0).bytes();
    return TB_OK;
}

TB_API int tb_attn_decode_paged_q8(tb_ctx* ctx, const tb_paged_kv* kv, float* out, const float* qr,
                                   const int32_t* lens, int64_t nHq, int64_t window, int64_t sinks, float* weights,
                                   void* ws, size_t ws_bytes)
{
    if (!ctx) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check_heads(ctx, kv, nHq);
    if (rc) return rc;
    TB_REQUIRE(ctx, out && qr && lens, "null pointer");
    TB_REQUIRE(ctx, TB_ALIGNED(out, 16) && TB_ALIGNED(qr, 16), "q and out must be 16-byte aligned");
    TB_REQUIRE(ctx, window >= 0 && sinks >= 0, "window and sinks must not be negative");
    DeviceGuard dev(ctx->device);
    const DecWs w = dec_ws(ctx, kv, nHq, weights != nullptr);
    if (!ws) {
        ws = tb_ctx_scratch(ctx, w.bytes());
        if (!ws) return TB_ERR_NOMEM;
    } else {
        TB_REQUIRE(ctx, TB_ALIGNED(ws, 256) && ws_bytes >= w.bytes(), "workspace: %zu bytes, 256-byte aligned, are needed",
                   w.bytes());
    }
    char* p = static_cast<char*>(ws);
    DecArgs a{};
    a.kv = paged_args(ctx, kv);
    a.q = qr;
    a.out = out;
    a.lens = lens;
    a.PO = reinterpret_cast<float*>(p);
    a.PML = reinterpret_cast<float2*>(p + w.po);
    if (weights) {
        a.ML = reinterpret_cast<float2*>(p + w.po + w.pml);
        a.SC = reinterpret_cast<float*>(p + w.po + w.pml + w.ml);
        a.weights = weights;
    }
    a.nHq = (int)nHq;
    a.window = (int)std::min<int64_t>(window, 1LL << 30);
    a.sinks = (int)std::min<int64_t>(sinks, 1LL << 30);
    a.grid = w.grid;
    a.qscale = 1.4426950408889634f / sqrtf((float)kv->hd);
    switch ((int)(kv->hd * 10 + nHq / kv->nKv)) {
    case 641: return launch_decode<64, 1>(ctx, a);
    case 642: return launch_decode<64, 2>(ctx, a);
    case 644: return launch_decode<64, 4>(ctx, a);
    case 648: return launch_decode<64, 8>(ctx, a);
    case 1281: return launch_decode<128, 1>(ctx, a);
    case 1282: return launch_decode<128, 2>(ctx, a);
    case 1284: return launch_decode<128, 4>(ctx, a);
    default: return launch_decode<128, 8>(ctx, a);
    }
}

}  // extern "C"
