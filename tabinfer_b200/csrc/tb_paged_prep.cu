// tb_paged_prep.cu -- new rows of the paged int8 KV cache: per head RMSNorm and
// rotary embedding of q and k, and k / v quantized into their pages.
//
//   y = x / sqrt(mean x^2 + eps) * w;  (y_i, y_{i+hd/2}) rotated by pos * theta^(-2i/hd)
//   per 32 elements m = max(1e-12, max|x|), byte = floor(0.5 + 127 * x / m)
//
// The q / k rows are formed in 64 bits and rounded to f32 once, so a byte of the
// cache does not depend on how a row's sum was split or in which call it was written
// (f32 sums put a byte one step off wherever they differ next to a rounding border);
// 64-bit FMAs run at half the f32 rate here and the kernel stays bound by its bytes.
#include "tb_paged.cuh"

namespace {

struct PrepArgs {
    PagedArgs kv;
    const float *q, *k, *v;
    const uint16_t *qw, *kw;
    float* qr;
    const int *seq, *slot, *pos;
    int nHq;
    double theta, eps;
};

// floor(0.5 + 127 x) of x clamped to [-1, 1] (pack4x8snorm)
__device__ __forceinline__ int8_t snorm8(float x)
{
    return (int8_t)floorf(__fadd_rn(0.5f, __fmul_rn(127.0f, fminf(1.0f, fmaxf(-1.0f, x)))));
}
__device__ __forceinline__ double warp_sum_f64(double v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One CTA a row; a warp takes whole heads (q, k, then v), lane l holding elements
// l + 32 i, so a rotary partner sits in the same lane hd/64 registers away.
template <int HD>
__global__ void __launch_bounds__(256) k_paged_prep(const PrepArgs a)
{
    __shared__ double cs[HD / 2], sn[HD / 2];
    tb_pdl_wait();
    tb_pdl_trigger();
    const int t = blockIdx.x, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
    constexpr int half = HD / 2, nw = HD / 32;
    const int b = a.seq[t], slot = a.slot[t];
    if (b < 0) return;                       // a padding row
    if (b >= a.kv.batch || slot < 0 || slot >= a.kv.cap()) {
        if (threadIdx.x == 0) atomicExch(a.kv.err, ERR_PAGED_LEN);
        return;
    }
    const int row = a.kv.row(b, slot);
    if (row < 0) return;
    for (int f = threadIdx.x; f < half; f += blockDim.x) {
        const double ang = (double)a.pos[t] * pow(a.theta, -2.0 * (double)f / (double)HD);
        sincos(ang, &sn[f], &cs[f]);
    }
    __syncthreads();
    const int nHq = a.nHq, nKv = a.kv.nKv;
    for (int role = wid; role < nHq + 2 * nKv; role += 8) {
        const bool isQ = role < nHq, isK = !isQ && role < nHq + nKv;
        const int head = isQ ? role : (isK ? role - nHq : role - nHq - nKv);
        const float* src = (isQ ? a.q + (long long)t * nHq * HD : (isK ? a.k : a.v) + (long long)t * nKv * HD) + head * HD;
        float x[nw];
#pragma unroll
        for (int i = 0; i < nw; i++) x[i] = src[32 * i + lane];
        if (isQ || isK) {
            const uint16_t* w16 = isQ ? a.qw : a.kw;
            double y[nw], ss = 0.0;
#pragma unroll
            for (int i = 0; i < nw; i++) {
                y[i] = (double)x[i];
                ss = fma(y[i], y[i], ss);
            }
            const double inv = 1.0 / sqrt(warp_sum_f64(ss) / (double)HD + a.eps);
#pragma unroll
            for (int i = 0; i < nw; i++) y[i] = y[i] * inv * (double)tb_h2f(w16[32 * i + lane]);
#pragma unroll
            for (int i = 0; i < nw / 2; i++) {
                const double c = cs[32 * i + lane], s = sn[32 * i + lane], lo = y[i], hi = y[i + nw / 2];
                x[i] = (float)(lo * c - hi * s);
                x[i + nw / 2] = (float)(hi * c + lo * s);
            }
            if (isQ) {
                float* dst = a.qr + (long long)t * nHq * HD + head * HD;
#pragma unroll
                for (int i = 0; i < nw; i++) dst[32 * i + lane] = x[i];
                continue;
            }
        }
        const long long at = (long long)row * nKv * HD + head * HD;
        int8_t* dq = (isK ? a.kv.Kq : a.kv.Vq) + at;
        float* ds = (isK ? a.kv.Ks : a.kv.Vs) + at / 32;
#pragma unroll
        for (int i = 0; i < nw; i++) {
            const float m = fmaxf(1e-12f, warp_max(fabsf(x[i])));
            dq[32 * i + lane] = snorm8(__fdiv_rn(x[i], m));
            if (lane == 0) ds[i] = m;
        }
    }
}

}  // namespace

extern "C" TB_API int tb_attn_prep_paged_q8(tb_ctx* ctx, const tb_paged_kv* kv, const float* q, const float* k,
                                            const float* v, const uint16_t* qw16, const uint16_t* kw16, float* qr,
                                            int64_t nHq, int64_t T, const int32_t* seq, const int32_t* slot,
                                            const int32_t* pos, float theta, float eps)
{
    if (!ctx) return TB_ERR_INVALID;
    int rc = paged_check(ctx, kv);
    if (rc) return rc;
    TB_REQUIRE(ctx, nHq > 0 && nHq <= 8192, "bad head count %lld", (long long)nHq);
    TB_REQUIRE(ctx, T >= 0 && T < (1LL << 31), "bad row count %lld", (long long)T);
    TB_REQUIRE(ctx, theta > 0.0f, "theta must be positive");
    if (T == 0) return TB_OK;
    TB_REQUIRE(ctx, q && k && v && qw16 && kw16 && qr && seq && slot && pos, "null pointer");
    DeviceGuard dev(ctx->device);
    PrepArgs a{paged_args(ctx, kv), q, k, v, qw16, kw16, qr, seq, slot, pos, (int)nHq, (double)theta, (double)eps};
    auto kern = kv->hd == 64 ? k_paged_prep<64> : k_paged_prep<128>;
    cudaError_t e = tb_launch(ctx, kern, dim3((unsigned)T), dim3(256), 0, a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "attn_prep_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}
