// tb_paged_prep.cu -- new rows of the paged int8 KV cache: per head RMSNorm and
// rotary embedding of q and k, and k / v quantized into their pages.
//
//   y = x / sqrt(mean x^2 + eps) * w;  (y_i, y_{i+hd/2}) rotated by pos * theta^(-2i/hd)
//   per 32 elements m = max(1e-12, max|x|), byte = floor(0.5 + 127 * x / m)
//
// The q / k rows are formed in 64 bits and rounded to f32 once: the bytes are then those of
// the definition, whatever the order of a sum (f32 sums put a byte one step off wherever they
// differ next to a rounding border).  That a byte does not depend on the call that wrote it
// comes from the fixed order of a head's sum, the same 32 lanes and tree for any R below.
// 64-bit arithmetic runs at half the f32 rate, so it is kept short: the norm weight goes
// into the rotation's coefficients (A = w_lo cos, B = w_hi sin, ...), formed once a row and
// warp, a head then costs 4 multiply-adds a pair and one multiplication by 1/rms an
// element, and the sums of four heads are reduced and inverted together.
//
// Four prompts of up to 2048 rows (16 / 8 heads of 128; 154 MB) take 46.9 us, 3.3 TB/s, against
// 23.5 us at a copy's rate: the 64-bit steps, the conversions to and from them (an element is
// converted for the sum and again for the rotation) and spills (32 bytes stored, 128 loaded at
// the 64 registers of four CTAs an SM) lie between; sums in two f32 terms, with the 64-bit step
// only beside a border, were not tried.  One row takes 5.7 us on the device, most of it the
// launch and the angles' sincos.
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

// floor(0.5 + 127 x / m), |x| <= m (pack4x8snorm of the rounded quotient).  The quotient by
// a reciprocal is off by less than 2^-21 of itself, so 127 times it by less than 7e-5: the
// division itself is needed only next to a border.
__device__ __forceinline__ int8_t snorm8(float x, float m, float inv)
{
    float v = __fadd_rn(0.5f, __fmul_rn(127.0f, x * inv));
    if (fabsf(v - rintf(v)) < 1e-4f || !(fabsf(v) < 200.0f) || m > 1e30f)
        v = __fadd_rn(0.5f, __fmul_rn(127.0f, fminf(1.0f, fmaxf(-1.0f, __fdiv_rn(x, m)))));
    return (int8_t)__float2int_rd(v);
}
__device__ __forceinline__ double shfl_xor_f64(double v, int m)
{
    return __hiloint2double(__shfl_xor_sync(0xffffffffu, __double2hiint(v), m),
                            __shfl_xor_sync(0xffffffffu, __double2loint(v), m));
}

// the warp's largest |x|, NaN where one of them is
__device__ __forceinline__ float redux_abs_nan(float x)
{
    float r;
    asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}
// x of one head (element l + 32 i in lane l) as snorm bytes with a scale a 32-group.  A NaN among
// the 32 makes the scale NaN, so that whoever reads the row meets it.
template <int NW>
__device__ __forceinline__ void store_q8(const float (&x)[NW], int8_t* dq, float* ds, int lane)
{
    float m[NW];
#pragma unroll
    for (int i = 0; i < NW; i++) {
        const float r = redux_abs_nan(x[i]);
        m[i] = r < 1e-12f ? 1e-12f : r;
    }
#pragma unroll
    for (int i = 0; i < NW; i++) dq[32 * i + lane] = snorm8(x[i], m[i], __fdividef(1.0f, m[i]));
    if (lane == 0) {
        if constexpr (NW == 4) *reinterpret_cast<float4*>(ds) = make_float4(m[0], m[1], m[2], m[3]);
        else *reinterpret_cast<float2*>(ds) = make_float2(m[0], m[1]);
    }
}

// R rows a CTA (8 warps): the angles of all of them first (one a thread at R = 4, hd 128), then
// 8 / R warps a row, each with every (8 / R)-th head, NB heads at a time: their loads are in
// flight together.  Lane l holds elements l + 32 i, a rotary partner hd / 64 registers away.
// One row a CTA where there are fewer than five rows a SM (latency): 5.2 us for one row against
// 9.3 at R = 4, 9.4 against 12.3 for 592 rows, 13.8 against 13.6 for 740, 52 against 37 for 4096
// (16 / 8 heads of 128, calls over 400 MB of inputs in turn).
constexpr int NB = 4;
template <int HD, int R>
__global__ void __launch_bounds__(256, 4) k_paged_prep(const PrepArgs a, int T)
{
    constexpr int HALF = HD / 2, NW = HD / 32, NP = NW / 2, WPR = 8 / R;
    __shared__ double cs[R][HALF], sn[R][HALF];
    tb_pdl_wait();
    tb_pdl_trigger();
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, t0 = blockIdx.x * R;
    if (R > 1) {                             // the powers once a CTA
        if (threadIdx.x < HALF) cs[0][threadIdx.x] = pow(a.theta, -2.0 * (double)threadIdx.x / (double)HD);
        __syncthreads();
    }
    {
        static_assert(R * HALF <= 256, "an angle a thread");
        const int r = threadIdx.x / HALF, f = threadIdx.x % HALF;
        const double p = R > 1 ? cs[0][f] : threadIdx.x < HALF ? pow(a.theta, -2.0 * (double)f / (double)HD) : 0.0;
        if (R > 1) __syncthreads();
        if (r < R && t0 + r < T) sincos((double)a.pos[t0 + r] * p, &sn[r][f], &cs[r][f]);
    }
    const int rr = wid / WPR, t = t0 + rr, part = wid % WPR;
    int row = -1;
    if (t < T) {
        const int b = a.seq[t], slot = a.slot[t];
        if (b >= a.kv.batch || (b >= 0 && (slot < 0 || slot >= a.kv.cap()))) {
            if (lane == 0) atomicExch(a.kv.err, ERR_PAGED_LEN);
        } else if (b >= 0) {                 // else a padding row
            row = a.kv.row(b, slot);
        }
    }
    __syncthreads();
    if (row < 0) return;
    const int nHq = a.nHq, nKv = a.kv.nKv;
#pragma unroll 1
    for (int type = 0; type < 2; type++) {   // q, then k
        const int heads = type ? nKv : nHq;
        const float* src = (type ? a.k : a.q) + (long long)t * heads * HD;
        const uint16_t* w16 = type ? a.kw : a.qw;
        double A[NP], B[NP], C[NP], D[NP];
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const double c = cs[rr][32 * i + lane], s = sn[rr][32 * i + lane];
            const double wl = (double)tb_h2f(w16[32 * i + lane]), wh = (double)tb_h2f(w16[HALF + 32 * i + lane]);
            A[i] = wl * c;
            B[i] = wh * s;
            C[i] = wh * c;
            D[i] = wl * s;
        }
#pragma unroll 1
        for (int h0 = part; h0 < heads; h0 += NB * WPR) {
            float x[NB][NW];
#pragma unroll
            for (int k = 0; k < NB; k++)
#pragma unroll
                for (int i = 0; i < NW; i++) {
                    const int h = h0 + k * WPR;
                    x[k][i] = h < heads ? __ldcs(src + h * HD + 32 * i + lane) : 0.0f;
                }
            double ss[NB];
#pragma unroll
            for (int k = 0; k < NB; k++) {
                ss[k] = 0.0;
#pragma unroll
                for (int i = 0; i < NW; i++) {
                    const double v = (double)x[k][i];
                    ss[k] = fma(v, v, ss[k]);
                }
            }
            // sums over the lanes: halves exchange halves of the heads, so a lane ends with the head of its
            // bits 4 and 3
#pragma unroll
            for (int w = NB / 2, m = 16; w >= 1; w >>= 1, m >>= 1)
#pragma unroll
                for (int k = 0; k < w; k++) {
                    const bool up = lane & m;
                    const double mine = up ? ss[k + w] : ss[k], other = up ? ss[k] : ss[k + w];
                    ss[k] = mine + shfl_xor_f64(other, m);
                }
            ss[0] += shfl_xor_f64(ss[0], 4);
            ss[0] += shfl_xor_f64(ss[0], 2);
            ss[0] += shfl_xor_f64(ss[0], 1);
            const double inv = 1.0 / sqrt(ss[0] * (1.0 / HD) + a.eps);
#pragma unroll
            for (int k = 0; k < NB; k++) {
                const int from = (k & 2 ? 16 : 0) | (k & 1 ? 8 : 0), h = h0 + k * WPR;
                const double n = __hiloint2double(__shfl_sync(0xffffffffu, __double2hiint(inv), from),
                                                  __shfl_sync(0xffffffffu, __double2loint(inv), from));
                if (h >= heads) break;
#pragma unroll
                for (int i = 0; i < NP; i++) {
                    const double lo = (double)x[k][i], hi = (double)x[k][i + NP];
                    x[k][i] = (float)(n * fma(lo, A[i], -(hi * B[i])));
                    x[k][i + NP] = (float)(n * fma(hi, C[i], lo * D[i]));
                }
                if (type == 0) {
                    float* dst = a.qr + ((long long)t * nHq + h) * HD;
#pragma unroll
                    for (int i = 0; i < NW; i++) dst[32 * i + lane] = x[k][i];
                } else {
                    const long long at = ((long long)row * nKv + h) * HD;
                    store_q8<NW>(x[k], a.kv.Kq + at, a.kv.Ks + at / 32, lane);
                }
            }
        }
    }
#pragma unroll 2
    for (int h = part; h < nKv; h += WPR) {
        float x[NW];
#pragma unroll
        for (int i = 0; i < NW; i++) x[i] = __ldcs(a.v + ((long long)t * nKv + h) * HD + 32 * i + lane);
        const long long at = ((long long)row * nKv + h) * HD;
        store_q8<NW>(x, a.kv.Vq + at, a.kv.Vs + at / 32, lane);
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
    const bool many = T >= 5LL * ctx->num_sms;
    auto kern = kv->hd == 64 ? (many ? k_paged_prep<64, 4> : k_paged_prep<64, 1>)
                             : (many ? k_paged_prep<128, 4> : k_paged_prep<128, 1>);
    cudaError_t e = tb_launch(ctx, kern, dim3((unsigned)(many ? (T + 3) / 4 : T)), dim3(256), 0, a, (int)T);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "attn_prep_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}
