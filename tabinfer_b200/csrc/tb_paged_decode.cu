// tb_paged_decode.cu -- attention of one new token a sequence over the paged int8 KV
// cache: ragged lengths, GQA, a sliding window with first tokens kept, and (optionally)
// the keys' attention weights added to an accumulator.
//
//   s_j = q . k_j / sqrt(hd) over the keys seen;  p = softmax(s);  out = sum_j p_j v_j
//   weights[b][kv head][j] += sum over the head's group of p_j
//
// The keys seen are a list of 32-key tiles.  The W warps of a CTA take HG neighbouring kv
// heads of W / HG consecutive tiles (a chunk), HG = 4, 2 or 1, the most that divides the
// heads: a cache row holds its heads side by side, so the CTA reads 512 contiguous bytes a
// row (one head a CTA left 128-byte pieces, and the 16-byte pieces of the scales, to CTAs
// that came by at other times: 505 MB from DRAM for a cache of 302 MB).  The chunks of all
// (sequence, head group) pairs in order are dealt out evenly to the CTAs, so ragged batches
// and long single sequences fill the machine alike.  A CTA whose range holds only a part of
// a pair's chunks writes (m, l, o) for it (at most two such parts a CTA: its first and its
// last pair); k_paged_combine joins a pair's parts in order, so results do not depend on
// timing.
#include "tb_paged.cuh"

namespace {

constexpr int W = 4, NT = 32 * W;
constexpr int CT = 512;    // threads of a joining CTA
constexpr float NEG_BIG = -3.0e38f;

struct DecArgs {
    CUtensorMap mk, mv;    // Kq / Vq as bytes [pool rows][nKv*HD], boxes of min(32, page_rows) rows x HD
    PagedArgs kv;
    const float* q;        // [B][nHq*HD]
    float* out;            // [B][nHq*HD]
    const int* lens;       // [B]
    float* PO;             // [grid][2][HG][GRP][HD]
    float2* PML;           // [grid][2][HG][GRP]
    float* SC;             // [B][nKv][cap][GRP] scores (log2), when weights are wanted
    float2* ML;            // [B][nHq] final (m, l), when weights are wanted
    float* weights;        // [B][nKv][cap]
    int nHq, window, sinks, grid;
    int log_hg;            // heads a group
    float qscale;          // log2(e) / (127 sqrt(HD))
};

__device__ __forceinline__ SeenTiles seen_of(const DecArgs& a, int n) { return SeenTiles(n - 1, n - 1, a.window, a.sinks); }
__device__ __forceinline__ int chunks_of(const DecArgs& a, int b)
{
    const int tw = W >> a.log_hg;      // tiles a chunk
    return (seen_of(a, a.kv.checked_len(__ldg(a.lens + b))).count + tw - 1) / tw;
}

// Where a unit stands.  A unit is a chunk of a (sequence, head group) pair; they are numbered
// by sequence, then group, then chunk (below 2^31 in all).
struct Where {
    int total;   // chunks of one group over all sequences
    int below;   // those of the sequences before b
    int b;
};
// The sequence find_b (when >= 0), else the one that holds unit cta * per, per = the units a
// CTA of `grid`.  Up to 32 sequences every warp finds it by itself; more take all threads and
// buf, (NT / 32 + 3) words of shared memory.
__device__ Where locate(const DecArgs& a, int find_b, int cta, int* buf)
{
    const int B = a.kv.batch, groups = a.kv.nKv >> a.log_hg;
    if (B == 1) return Where{chunks_of(a, 0), 0, 0};
    const int nt = B <= 32 ? 32 : (int)blockDim.x, tid = B <= 32 ? threadIdx.x & 31 : threadIdx.x;
    const int slice = (B + nt - 1) / nt, b0 = min(B, tid * slice), b1 = min(B, b0 + slice);
    int mine = 0;
    for (int b = b0; b < b1; b++) mine += chunks_of(a, b);
    int x = mine;                                   // inclusive sums over the threads
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, x, o);
        if ((tid & 31) >= o) x += v;
    }
    int total = __shfl_sync(0xffffffffu, x, 31);
    if (nt > 32) {
        if ((tid & 31) == 31) buf[tid >> 5] = x;
        __syncthreads();
        total = 0;
        for (int i = 0; i < nt / 32; i++) {
            if (i < (tid >> 5)) x += buf[i];
            total += buf[i];
        }
    }
    const int all = total * groups, at = cta * ((all + a.grid - 1) / a.grid);
    Where w{total, x - mine, b0};
    bool here;
    if (find_b >= 0) {
        here = b0 <= find_b && find_b < b1;
        if (here)
            for (; w.b < find_b; w.b++) w.below += chunks_of(a, w.b);
    } else {
        here = at < all && w.below * groups <= at && at < (w.below + mine) * groups;
        if (here)
            for (int n; at >= (w.below + (n = chunks_of(a, w.b))) * groups; w.b++) w.below += n;
    }
    if (nt == 32) {
        const int src = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
        w.below = __shfl_sync(0xffffffffu, w.below, max(src, 0));
        w.b = __shfl_sync(0xffffffffu, w.b, max(src, 0));
        return w;
    }
    int* out = buf + nt / 32;
    if (here) {
        out[0] = w.below;
        out[1] = w.b;
    }
    __syncthreads();
    w.below = out[0];                               // not read where no unit is left
    w.b = out[1];
    __syncthreads();                                // buf may be written again
    return w;
}

// Shared memory of a CTA: every warp has its own ring of NST tiles (K and V rows by TMA,
// swizzled; the keys' scales behind them) and words through which scores and weights pass
// between lanes, q's digits at a part's start and the outputs at its end.
template <int HD, int GRP>
struct RingLayout {
    static constexpr int NG = HD / 32, NN = (GRP * 4 + 7) / 8;   // 32-groups; 8-column tiles of (head, digit)
    static constexpr int ROWS = KT * HD, SCALES = KT * NG * 4;
    static constexpr int V = ROWS, KS = 2 * ROWS, VS = 2 * ROWS + SCALES;
    static constexpr int STAGE = 2 * ROWS + 2 * SCALES;          // 9216 or 4608: whole swizzle atoms
    // tiles in flight a warp (three: 131001 rows 67.3 us against 62.6)
    static constexpr int NST = 2;
    static constexpr int WORDS = GRP * HD * 4;                   // [GRP][NG][KT] words = [GRP][HD] floats
    static constexpr int OFF_WORDS = W * NST * STAGE;
    static constexpr int OFF_M = OFF_WORDS + W * WORDS;          // float [2][W][GRP] m and l
    static constexpr int OFF_BAR = OFF_M + 2 * W * GRP * 4;      // mbarriers, then the tiles' masks
    static constexpr int BYTES = OFF_BAR + W * NST * 12;
    // CTAs an SM: 232448 bytes of shared memory, 1 KB of them a CTA the system's
    // at most four, with 128 registers a thread; three for eight q heads a kv head, which take 168
    static constexpr int MOST = GRP == 8 ? 3 : 4;
    static constexpr int OCC = 232448 / (BYTES + 1024) < MOST ? 232448 / (BYTES + 1024) : MOST;
    static_assert(OCC >= 2, "two CTAs an SM");
    static_assert(GRP * 4 * HD <= WORDS, "q's digits fit in the words");
    static_assert(W * WORDS >= (W + 3) * 4, "the plan's sums fit in the words");
    static_assert(STAGE % (HD == 128 ? 1024 : 512) == 0 && OFF_BAR % 8 == 0, "alignment");
};

// A warp's walk over its tiles, pair after pair of the CTA's range of units.
struct Walk {
    int u, u1, base;           // first unit of the current part, end of the range, units below sequence b
    int b, grp, n, c0, c1, nc, i, t1;
    SeenTiles seen;

    __device__ Walk(const DecArgs& a, int u0, int u1_, int b_, int base_, int wid)
        : u(u0), u1(u1_), base(base_), b(b_), seen(-1, -1, 0, 0)
    {
        load(a);
        enter(a, wid);
    }
    __device__ void load(const DecArgs& a)
    {
        const int tw = W >> a.log_hg;
        n = a.kv.checked_len(__ldg(a.lens + b));
        seen = seen_of(a, n);
        nc = (seen.count + tw - 1) / tw;
    }
    __device__ void enter(const DecArgs& a, int wid)
    {
        if (u >= u1) return;
        const int groups = a.kv.nKv >> a.log_hg, tw = W >> a.log_hg;
        while (u >= base + nc * groups) {
            base += nc * groups;
            b++;
            load(a);
        }
        grp = (u - base) / nc;
        c0 = (u - base) - grp * nc;
        c1 = min(nc, c0 + (u1 - u));
        i = c0 * tw + (wid >> a.log_hg);
        t1 = min(seen.count, c1 * tw);
    }
    __device__ bool part() const { return u < u1; }
    __device__ bool tile() const { return i < t1; }
    __device__ int head(const DecArgs& a, int wid) const { return (grp << a.log_hg) + (wid & ((1 << a.log_hg) - 1)); }
    __device__ void next_part(const DecArgs& a, int wid)
    {
        u += c1 - c0;
        enter(a, wid);
    }
    // the warp's next tile, in this part or a later one
    __device__ void advance(const DecArgs& a, int wid)
    {
        i += W >> a.log_hg;
        settle(a, wid);
    }
    __device__ void settle(const DecArgs& a, int wid)
    {
        while (part() && !tile()) next_part(a, wid);
    }
};

__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return ffma2(a, b, make_float2(0.0f, 0.0f)); }

// What bounds it is HBM, so the arithmetic on each byte has to be short.  Both products run
// on the tensor cores with the cache's bytes as they are and exact int32 sums, 32 keys at a
// time (mma m16n8k32, one 32-group of q . k or 32 keys of p . v an instruction):
//   scores   A = K bytes (16 keys x 32 dims), B = q as four signed base-128 digits of one step
//            a head (|error| < 2^-28 of the largest |q|), columns (head, digit);
//   outputs  A = V bytes transposed (16 dims x 32 keys, ldmatrix.trans), B = the keys' weights
//            p * vscale as three unsigned base-256 digits of a power-of-two step that the tile's
//            largest weight sets (|error| <= 2^-22 of it), columns (head, digit).
// The int32 sums stay below 2^22, so they are seeded with 1.5 * 2^23 and read as floats.
// About 300 instructions a 32-key tile of 9.2 KB (hd 128, two q heads), against some 1600
// issue slots that the tile's share of the HBM rate leaves an SM; the form that converts V
// and K to f32 takes 1180.
// Measured with the join (bytes of the rows seen, their scales and the weights; 6.55 TB/s is
// what a copy reaches): 131001 rows of 8 heads of 128, 302 MB, 59 us (5.1 TB/s: memory, and
// a start of 6 us); 32 ragged sequences of 8192 rows and below with weights, 329 MB, 73.0 us
// (4.5 TB/s: three kernels, and the scores pass through memory); 16 windows of 4096 rows of 8
// heads of 64, 76 MB, 31.5 us (2.4 TB/s: a tile of half the bytes has as many steps behind one
// another, 2100 cycles and 1000 for the next one's copies; the 128 registers of four CTAs an SM
// hold no larger tile, and fewer CTAs with larger ones were not tried); one sequence of 4096
// rows 11.6 us, a chain of latencies: plan, page number, tile, products, join.
template <int HD, int GRP>
__global__ void __launch_bounds__(NT, RingLayout<HD, GRP>::OCC) k_paged_decode(const __grid_constant__ DecArgs a)
{
    using L = RingLayout<HD, GRP>;
    constexpr int NG = L::NG, NN = L::NN, NST = L::NST;
    constexpr float MAGIC = 12582912.0f;
    extern __shared__ __align__(1024) uint8_t smem[];
    const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, g8 = lane >> 2, t4 = lane & 3;
    uint8_t* ring = smem + wid * NST * L::STAGE;
    uint32_t* words = reinterpret_cast<uint32_t*>(smem + L::OFF_WORDS + wid * L::WORDS);
    int8_t* qd = reinterpret_cast<int8_t*>(words);                   // [GRP][4][HD]
    float* wo = reinterpret_cast<float*>(smem + L::OFF_WORDS);       // [W][GRP][HD]
    float* wm = reinterpret_cast<float*>(smem + L::OFF_M);
    float* wl = wm + W * GRP;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR) + wid * NST;
    uint32_t* okw = reinterpret_cast<uint32_t*>(smem + L::OFF_BAR + W * NST * 8) + wid * NST;
    if (lane == 0) {
        for (int s = 0; s < NST; s++) mbar_init(&full[s], 33);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    tb_pdl_wait();
    tb_pdl_trigger();
    const int nKv = a.kv.nKv, nHq = a.nHq, cta = blockIdx.x, hg = 1 << a.log_hg, tw = W >> a.log_hg;
    const Where w = locate(a, -1, cta, reinterpret_cast<int*>(smem + L::OFF_WORDS));
    const int all = w.total * (nKv >> a.log_hg), per = (all + a.grid - 1) / a.grid;
    const int u0 = cta * per, u1 = min(all, u0 + per);
    if (u0 >= u1) return;

    const int box = min(KT, 1 << a.kv.log_page);          // rows a copy
    // The tile at the walk's place: look() requests the lane's page number (a lane a key; a page is looked up
    // when one of its rows in this tile is seen), issue() sends the copies into ring stage s a tile's work
    // later, when the number is there.
    struct Look {
        int key, page, head;
        bool see, wanted;
    };
    auto look = [&](const Walk& p) {
        Look v;
        v.key = p.seen.tile(p.i) * KT + lane;
        v.head = p.head(a, wid);
        v.see = key_seen(v.key, p.n - 1, a.window, a.sinks);
        const unsigned any = __ballot_sync(0xffffffffu, v.see);
        v.wanted = box == KT || (any & (0xffffu << (lane & 16)));
        v.page = v.wanted ? __ldg(a.kv.table + (long long)p.b * a.kv.max_pages + (v.key >> a.kv.log_page)) : 0;
        return v;
    };
    auto issue = [&](const Look& v, int s) {
        const int ph = v.head;
        int row = -1;
        if (v.wanted) {
            if ((unsigned)v.page < (unsigned)a.kv.n_pages) row = (v.page << a.kv.log_page) | (v.key & ((1 << a.kv.log_page) - 1));
            else atomicExch(a.kv.err, ERR_PAGED_PAGE);
        }
        const int row0 = __shfl_sync(0xffffffffu, row, 0), row16 = __shfl_sync(0xffffffffu, row, 16);
        const bool see = v.see;
        const unsigned ok = __ballot_sync(0xffffffffu, see && row >= 0);
        uint8_t* st = ring + s * L::STAGE;
        if (lane == 0) okw[s] = ok;
        __syncwarp();          // before the arrival that releases it, which another lane may make
        const bool second = box < KT && row16 >= 0;
        mbar_expect_elect(&full[s], (uint32_t)(2 * HD * box * ((row0 >= 0) + second)));
        if (row0 >= 0) tma_2d_elect(st, &a.mk, st + L::V, &a.mv, ph * HD, row0, &full[s]);
        if (second) tma_2d_elect(st + 16 * HD, &a.mk, st + L::V + 16 * HD, &a.mv, ph * HD, row16, &full[s]);
        if (see && row >= 0) {
            const long long at = ((long long)row * nKv + ph) * NG;
            if constexpr (NG == 4) {
                cp_async16(st + L::KS + lane * 16, a.kv.Ks + at);
                cp_async16(st + L::VS + lane * 16, a.kv.Vs + at);
            } else {
                cp_async8(st + L::KS + lane * 8, a.kv.Ks + at);
                cp_async8(st + L::VS + lane * 8, a.kv.Vs + at);
            }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[s])) : "memory");
    };
    Walk c(a, u0, u1, w.b, w.below * (nKv >> a.log_hg), wid), p = c;
    p.settle(a, wid);
    int issued = 0, used = 0;
    bool alive = true;
    // the first part's q and the first tiles' page numbers are requested together
    float r[NG];
    auto load_q = [&](int g) {
        const float* src = a.q + (long long)c.b * nHq * HD + (c.head(a, wid) * GRP + g) * HD + lane;
#pragma unroll
        for (int i = 0; i < NG; i++) r[i] = __ldg(src + 32 * i);
    };
    load_q(0);
    {
        Look v[NST];
#pragma unroll
        for (int i = 0; i < NST; i++)
            if (p.part()) {
                v[i] = look(p);
                issued++;
                p.advance(a, wid);
            }
#pragma unroll
        for (int i = 0; i < NST; i++)
            if (i < issued) issue(v[i], i);
    }
    const float f1 = (t4 & 1) ? 0.0f : 256.0f, f2 = (t4 & 1) ? 65536.0f : 1.0f;
    const int lrow = (lane & 7) + (lane & 8), lchunk = lane >> 4;    // ldmatrix x4: 16 rows x two chunks
    auto swz = [](int row, int chunk) {
        return HD == 128 ? row * 128 + ((chunk ^ (row & 7)) << 4) : row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
    };

    for (bool first = true; c.part(); c.next_part(a, wid), first = false) {
        // ---- q of this warp's head: four signed digits, one step a q head
        const int h = c.head(a, wid);
        if (tw > 1) __syncthreads();       // the last part's merge has read the words
        float qf[GRP];
#pragma unroll
        for (int g = 0; g < GRP; g++) {
            if (g > 0 || !first) load_q(g);
            float mx = 0.0f;
            bool fine = true;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                mx = fmaxf(mx, fabsf(r[i]));
                fine = fine && fabsf(r[i]) <= 3.0e38f;
            }
            mx = redux_max(mx);
            fine = __all_sync(0xffffffffu, fine);
            float stp = mx > 1e-30f ? mx * (1.0f / 127.0f) : 1.0f;
            qf[g] = fine ? stp * a.qscale : __int_as_float(0x7fc00000);
            float inv = __frcp_rn(stp);
#pragma unroll
            for (int d = 0; d < 4; d++) {
#pragma unroll
                for (int i = 0; i < NG; i++) {
                    const int x = max(-127, min(127, __float2int_rn(r[i] * inv)));
                    r[i] = fmaf(-stp, (float)x, r[i]);
                    qd[(g * 4 + d) * HD + 32 * i + lane] = (int8_t)x;
                }
                stp *= 0.0078125f;
                inv *= 128.0f;
            }
        }
        __syncwarp();
        uint32_t qb[NN][NG][2];
        float qs[NN];
#pragma unroll
        for (int nt = 0; nt < NN; nt++) {
            const int col = 8 * nt + g8;
#pragma unroll
            for (int G = 0; G < NG; G++) {
                const int8_t* src = qd + col * HD + 32 * G + 4 * t4;
                qb[nt][G][0] = col < 4 * GRP ? *reinterpret_cast<const uint32_t*>(src) : 0u;
                qb[nt][G][1] = col < 4 * GRP ? *reinterpret_cast<const uint32_t*>(src + 16) : 0u;
            }
            qs[nt] = (2 * nt + 1 < GRP && (t4 >> 1) ? qf[(2 * nt + 1) % GRP] : qf[2 * nt]) * ((t4 & 1) ? 1.0f / 16384.0f : 1.0f);
        }
        __syncwarp();          // the digits are read: their words take scores and weights
        float m[GRP], l[GRP];
        float2 o[2 * NG][NN];      // (dims 16 mt + g8, + 8) of head 2 nt + t4 / 2, digits of this lane
#pragma unroll
        for (int g = 0; g < GRP; g++) {
            m[g] = NEG_BIG;
            l[g] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 2 * NG; i++)
#pragma unroll
            for (int nt = 0; nt < NN; nt++) o[i][nt] = make_float2(0.0f, 0.0f);

        for (; c.tile() && alive; c.i += tw, used++) {
            const int s = used % NST;
            Look v{};
            if (p.part()) v = look(p);
            if (!__all_sync(0xffffffffu, mbar_test(&full[s], (used / NST) & 1) || mbar_wait(&full[s], (used / NST) & 1))) {
                if (lane == 0) atomicExch(a.kv.err, ERR_PAGED_WAIT);
                alive = false;
                break;
            }
            const uint8_t* st = ring + s * L::STAGE;
            const uint32_t kb = smem_u32(st), vb = kb + L::V;
            const bool ok = (okw[s] >> lane) & 1;
            const float* ks = reinterpret_cast<const float*>(st + L::KS);
            float* scs = reinterpret_cast<float*>(words);
            // ---- scores
#pragma unroll
            for (int mt = 0; mt < 2; mt++) {
                float2 part[NN];
#pragma unroll
                for (int nt = 0; nt < NN; nt++) part[nt] = make_float2(0.0f, 0.0f);
                float k0[NG], k1[NG];
#pragma unroll
                for (int i = 0; i < NG; i += 2) {
                    *reinterpret_cast<float2*>(k0 + i) = *reinterpret_cast<const float2*>(ks + (16 * mt + g8) * NG + i);
                    *reinterpret_cast<float2*>(k1 + i) = *reinterpret_cast<const float2*>(ks + (16 * mt + g8 + 8) * NG + i);
                }
#pragma unroll
                for (int G = 0; G < NG; G++) {
                    uint32_t af[4];
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(af[0]), "=r"(af[1]), "=r"(af[2]), "=r"(af[3])
                                 : "r"(kb + swz(16 * mt + lrow, 2 * G + lchunk)));
#pragma unroll
                    for (int nt = 0; nt < NN; nt++) {
                        int d[4];
                        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                            "{%8,%9}, {%10,%10,%10,%10};"
                            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                            : "r"(af[0]), "r"(af[1]), "r"(af[2]), "r"(af[3]), "r"(qb[nt][G][0]), "r"(qb[nt][G][1]),
                              "r"(0x4B400000));
                        const float2 hi = fadd2(make_float2(__int_as_float(d[0]), __int_as_float(d[2])),
                                                make_float2(-MAGIC, -MAGIC));
                        const float2 lo = fadd2(make_float2(__int_as_float(d[1]), __int_as_float(d[3])),
                                                make_float2(-MAGIC, -MAGIC));
                        part[nt] = ffma2(ffma2(lo, make_float2(0.0078125f, 0.0078125f), hi), make_float2(k0[G], k1[G]),
                                         part[nt]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NN; nt++) {
                    float x = part[nt].x * qs[nt], y = part[nt].y * qs[nt];
                    x += __shfl_xor_sync(0xffffffffu, x, 1);
                    y += __shfl_xor_sync(0xffffffffu, y, 1);
                    const int hd_ = 2 * nt + (t4 >> 1);
                    if ((t4 & 1) == 0 && hd_ < GRP) {
                        scs[hd_ * KT + 16 * mt + g8] = x;
                        scs[hd_ * KT + 16 * mt + g8 + 8] = y;
                    }
                }
                __syncwarp();      // the lanes that wrote meet the others before the next ldmatrix
            }
            float pr[GRP], corr[GRP];
#pragma unroll
            for (int g = 0; g < GRP; g++) pr[g] = ok ? scs[g * KT + lane] : NEG_BIG;
            {   // a K scale without a number: inf times a group's exact sum has a sign that inf times its elements,
                // one by one, has not (a score of -inf would leave the key out)
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < NG; i += 2) {
                    const float2 x = *reinterpret_cast<const float2*>(ks + lane * NG + i);
                    z = fmaf(x.x, 0.0f, fmaf(x.y, 0.0f, z));
                }
                if (ok && z != 0.0f)
#pragma unroll
                    for (int g = 0; g < GRP; g++) pr[g] = z;
            }
            __syncwarp();
            if (a.SC) {
                const int key = c.seen.tile(c.i) * KT + lane;
                if (key < a.kv.cap()) {
                    float* dst = a.SC + (((long long)c.b * nKv + h) * a.kv.cap() + key) * GRP;
#pragma unroll
                    for (int g = 0; g < GRP; g++) dst[g] = ok ? pr[g] : -INFINITY;
                }
            }
            // ---- running maximum and sum (m the same in every lane, l per lane)
#pragma unroll
            for (int g = 0; g < GRP; g++) {
                const float mn = fmaxf(m[g], redux_max(pr[g]));
                corr[g] = exp2f(m[g] - mn);
                pr[g] = ok ? exp2f(pr[g] - mn) : 0.0f;
                l[g] = fmaf(l[g], corr[g], pr[g]);
                m[g] = mn;
            }
            // ---- the keys' weights a V group, as integers of a power-of-two step
            float sc[GRP][NG];
            {
                float vs[NG];
#pragma unroll
                for (int i = 0; i < NG; i += 2)
                    *reinterpret_cast<float2*>(vs + i) =
                        *reinterpret_cast<const float2*>(st + L::VS + (lane * NG + i) * 4);
#pragma unroll
                for (int G = 0; G < NG; G++)
#pragma unroll
                    for (int g = 0; g < GRP; g++) {
                        const float x = ok ? pr[g] * vs[G] : 0.0f;
                        const int e = max(24, (int)(__reduce_max_sync(0xffffffffu, __float_as_uint(x)) >> 23));
                        sc[g][G] = e > 250 ? __int_as_float(0x7fc00000) : __int_as_float((e - 21) << 23);   // 2^(e - 127 - 21)
                        words[(g * NG + G) * KT + lane] =
                            __float_as_uint(fmaf(x, __int_as_float((275 - min(e, 250)) << 23), 8388608.0f));
                    }
            }
            __syncwarp();
            // ---- outputs
#pragma unroll
            for (int nt = 0; nt < NN; nt++) {
                const int hb = 2 * nt + (g8 >> 2), sel = (g8 & 3) | ((4 + (g8 & 3)) << 4);
                // this lane's output columns belong to head 2 nt + t4 / 2
                const float cr = 2 * nt + 1 < GRP && (t4 >> 1) ? corr[(2 * nt + 1) % GRP] : corr[2 * nt];
                const float2 cr2 = make_float2(cr, cr);
#pragma unroll
                for (int G = 0; G < NG; G++) {
                    // columns of no head (GRP = 1) take a head's digits and are not written: no branch before ldmatrix
                    const uint32_t* src = words + ((GRP == 1 ? 0 : hb) * NG + G) * KT + 4 * t4;
                    const uint4 x = *reinterpret_cast<const uint4*>(src), y = *reinterpret_cast<const uint4*>(src + 16);
                    const uint32_t b0 = __byte_perm(__byte_perm(x.x, x.y, sel), __byte_perm(x.z, x.w, sel), 0x5410);
                    const uint32_t b1 = __byte_perm(__byte_perm(y.x, y.y, sel), __byte_perm(y.z, y.w, sel), 0x5410);
                    const float so = (2 * nt + 1 < GRP && (t4 >> 1) ? sc[(2 * nt + 1) % GRP][G] : sc[2 * nt][G]) * f2;
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int mt = 2 * G + k;
                        uint32_t af[4];
                        int d[4];
                        asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];"
                                     : "=r"(af[0]), "=r"(af[1]), "=r"(af[2]), "=r"(af[3]) : "r"(vb + swz(lane, mt)));
                        asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
                            "{%8,%9}, {%10,%10,%10,%10};"
                            : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                            : "r"(af[0]), "r"(af[1]), "r"(af[2]), "r"(af[3]), "r"(b0), "r"(b1), "r"(0x4B400000));
                        const float2 lo = fadd2(make_float2(__int_as_float(d[0]), __int_as_float(d[2])),
                                                make_float2(-MAGIC, -MAGIC));
                        const float2 hi = fadd2(make_float2(__int_as_float(d[1]), __int_as_float(d[3])),
                                                make_float2(-MAGIC, -MAGIC));
                        o[mt][nt] = ffma2(ffma2(hi, make_float2(f1, f1), lo), make_float2(so, so), mul2(o[mt][nt], cr2));
                    }
                }
            }
            __syncwarp();          // the stage and the words are read
            if (p.part()) {
                issue(v, s);
                issued++;
                p.advance(a, wid);
            }
        }
        // ---- the states of a head's warps meet
        __syncwarp();
#pragma unroll
        for (int g = 0; g < GRP; g++) {
            const float lt = warp_sum(l[g]);
            if (lane == 0) {
                wm[wid * GRP + g] = m[g];
                wl[wid * GRP + g] = lt;
            }
        }
#pragma unroll
        for (int nt = 0; nt < NN; nt++)
#pragma unroll
            for (int mt = 0; mt < 2 * NG; mt++) {
                const float x = o[mt][nt].x + __shfl_xor_sync(0xffffffffu, o[mt][nt].x, 1);
                const float y = o[mt][nt].y + __shfl_xor_sync(0xffffffffu, o[mt][nt].y, 1);
                const int hd_ = 2 * nt + (t4 >> 1);
                if ((t4 & 1) == 0 && hd_ < GRP) {
                    wo[(wid * GRP + hd_) * HD + 16 * mt + g8] = x;
                    wo[(wid * GRP + hd_) * HD + 16 * mt + g8 + 8] = y;
                }
            }
        if (tw > 1) __syncthreads();
        else __syncwarp();
        const bool whole = c.c0 == 0 && c.c1 == c.nc;
        const long long slot = ((2LL * cta + (c.u == u0 ? 0 : 1)) << a.log_hg) + (wid & (hg - 1));
        // the tw warps of a head share its outputs: a float4 a lane
        constexpr int QPH = HD / 4;
        const int k0 = wid & (hg - 1);
#pragma unroll
        for (int i = 0; i < (GRP * QPH + 31) / 32; i++) {
            if ((i & (tw - 1)) != wid >> a.log_hg) continue;
            const int at = 32 * i + lane, g = at / QPH, d = at % QPH * 4;
            if (GRP * QPH < 32 && at >= GRP * QPH) continue;
            float M = NEG_BIG, Ls = 0.0f;
            float4 O = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < W; k++)
                if ((k & (hg - 1)) == k0) M = fmaxf(M, wm[k * GRP + g]);
#pragma unroll
            for (int k = 0; k < W; k++)
                if ((k & (hg - 1)) == k0) {
                    const float e = exp2f(wm[k * GRP + g] - M);
                    const float4 x = *reinterpret_cast<const float4*>(wo + (k * GRP + g) * HD + d);
                    Ls = fmaf(wl[k * GRP + g], e, Ls);
                    O = make_float4(fmaf(x.x, e, O.x), fmaf(x.y, e, O.y), fmaf(x.z, e, O.z), fmaf(x.w, e, O.w));
                }
            const float f = whole ? (Ls > 0.0f || Ls != Ls ? 1.0f / (127.0f * Ls) : 0.0f) : 1.0f / 127.0f;
            O = make_float4(O.x * f, O.y * f, O.z * f, O.w * f);
            if (whole) {
                *reinterpret_cast<float4*>(a.out + (long long)c.b * nHq * HD + (h * GRP + g) * HD + d) = O;
                if (d == 0 && a.ML) a.ML[(long long)c.b * nHq + h * GRP + g] = make_float2(M, Ls);
            } else {
                *reinterpret_cast<float4*>(a.PO + (slot * GRP + g) * HD + d) = O;
                if (d == 0) a.PML[slot * GRP + g] = make_float2(M, Ls);
            }
        }
        __syncwarp();
    }
    // after a wait that gave up: no copy may land once the CTA has left
    if (!alive)
        for (int i = used; i < issued; i++) mbar_wait(&full[i % NST], (i / NST) & 1);
}

// Joins the parts of kv head x of sequence y; those that one CTA held are done.  The parts'
// (m, l) come first, all at once into shared memory, then each thread sums a float4 column of
// every CT-th part, eight loads in flight, and the CT sums are added in order.
template <int HD, int GRP>
__global__ void __launch_bounds__(CT) k_paged_combine(const __grid_constant__ DecArgs a)
{
    constexpr int COLS = GRP * HD / 4, P = CT / COLS;
    static_assert(CT % COLS == 0 && CT / 32 >= GRP, "whole columns, a warp a q head");
    extern __shared__ __align__(16) float2 ml[];     // [np][GRP]: m and l, then the factor 2^(m - M) for m
    __shared__ float4 part[P][COLS];
    __shared__ float sl[GRP];
    __shared__ int plan[CT / 32 + 3];
    tb_pdl_wait();
    tb_pdl_trigger();
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
    const Where w = locate(a, b, 0, plan);
    const int nc = chunks_of(a, b), groups = a.kv.nKv >> a.log_hg, hg = 1 << a.log_hg;
    float4* out = reinterpret_cast<float4*>(a.out + (long long)b * a.nHq * HD + h * GRP * HD);
    if (nc == 0) {
        if (tid < COLS) out[tid] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        return;
    }
    const int all = w.total * groups, per = (all + a.grid - 1) / a.grid;
    const int u0 = w.below * groups + (h >> a.log_hg) * nc, u1 = u0 + nc;
    const int c0 = u0 / per, c1 = (u1 - 1) / per;
    if (c0 == c1) return;
    // part k is CTA c0 + k's: its first part, but for a pair that starts inside CTA c0's range
    const int first = u0 == c0 * per ? 0 : 1, np = c1 - c0 + 1;
    auto slot = [&](int k) { return (size_t)((2 * (c0 + k) + (k == 0 ? first : 0)) * hg + (h & (hg - 1))) * GRP; };
    // every part's (m, l) at once, then a warp a q head over them in shared memory
    for (int i = tid; i < np * GRP; i += CT) {
        const int k = i / GRP;
        ml[i] = a.PML[slot(k) + i - k * GRP];
    }
    __syncthreads();
    if (wid < GRP) {
        float x = NEG_BIG;
        for (int k = lane; k < np; k += 32) x = fmaxf(x, ml[k * GRP + wid].x);
        x = warp_max(x);
        float l = 0.0f;
        for (int k = lane; k < np; k += 32) {
            const float e = exp2f(ml[k * GRP + wid].x - x);
            l = fmaf(ml[k * GRP + wid].y, e, l);
            ml[k * GRP + wid].x = e;
        }
        l = warp_sum(l);
        if (lane == 0) {
            sl[wid] = l;
            if (a.ML) a.ML[(long long)b * a.nHq + h * GRP + wid] = make_float2(x, l);
        }
    }
    __syncthreads();
    const int col = tid % COLS, pp = tid / COLS, g = col / (HD / 4);
    const float4* po = reinterpret_cast<const float4*>(a.PO) + col;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = pp; k < np; k += 8 * P) {
        float4 v[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k + i * P < np) v[i] = po[slot(k + i * P) * (HD / 4)];
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (k + i * P < np) {
                const float e = ml[(k + i * P) * GRP + g].x;
                o.x = fmaf(v[i].x, e, o.x);
                o.y = fmaf(v[i].y, e, o.y);
                o.z = fmaf(v[i].z, e, o.z);
                o.w = fmaf(v[i].w, e, o.w);
            }
    }
    part[pp][col] = o;
    __syncthreads();
    if (tid < COLS) {
        o = part[0][tid];
#pragma unroll
        for (int i = 1; i < P; i++) {
            const float4 v = part[i][tid];
            o.x += v.x;
            o.y += v.y;
            o.z += v.z;
            o.w += v.w;
        }
        const float l = sl[g];
        out[tid] = l > 0.0f || l != l ? make_float4(o.x / l, o.y / l, o.z / l, o.w / l) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
}

// weights[b][h][j] += sum over the group of 2^(s - m) / l, for the keys seen
constexpr int KEYS = 4;    // a thread
template <int GRP>
__global__ void __launch_bounds__(256) k_paged_weights(const __grid_constant__ DecArgs a)
{
    tb_pdl_wait();
    tb_pdl_trigger();
    const int h = blockIdx.y, b = blockIdx.z, cap = a.kv.cap();
    const int n = a.kv.checked_len(__ldg(a.lens + b));
    const int j0 = blockIdx.x * 256 * KEYS;
    if (j0 >= n) return;
    // every load before the first use
    const long long at = ((long long)b * a.kv.nKv + h) * cap;
    float sc[KEYS][GRP], old[KEYS];
    bool see[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        const int j = j0 + 256 * i + threadIdx.x;
        see[i] = j < n && key_seen(j, n - 1, a.window, a.sinks);
        if (!see[i]) continue;
        const float* src = a.SC + (at + j) * GRP;
#pragma unroll
        for (int g = 0; g < GRP; g++) sc[i][g] = __ldcg(src + g);
        old[i] = a.weights[at + j];
    }
    float m[GRP], r[GRP];
#pragma unroll
    for (int g = 0; g < GRP; g++) {
        const float2 ml = a.ML[(long long)b * a.nHq + h * GRP + g];
        m[g] = ml.x;
        r[g] = ml.y > 0.0f || ml.y != ml.y ? 1.0f / ml.y : 0.0f;     // a sum of no number leaves no weight one
    }
#pragma unroll
    for (int i = 0; i < KEYS; i++) {
        if (!see[i]) continue;
        float s = 0.0f;
#pragma unroll
        for (int g = 0; g < GRP; g++) s = fmaf(exp2f(sc[i][g] - m[g]), r[g], s);
        a.weights[at + j0 + 256 * i + threadIdx.x] = old[i] + s;
    }
}

// device workspace: PO, PML, then (weights) ML and SC
struct DecWs {
    int grid;
    size_t po, pml, ml, sc;
    size_t bytes() const { return po + pml + ml + sc; }
};
size_t up256(size_t x) { return (x + 255) & ~size_t(255); }
// heads a CTA reads side by side
int log_group(int64_t nKv) { return nKv % 4 == 0 ? 2 : (nKv % 2 == 0 ? 1 : 0); }
int dec_occ(int64_t hd, int64_t grp)
{
    if (hd == 64) return grp <= 2 ? (grp == 1 ? RingLayout<64, 1>::OCC : RingLayout<64, 2>::OCC)
                                  : (grp == 4 ? RingLayout<64, 4>::OCC : RingLayout<64, 8>::OCC);
    return grp <= 2 ? (grp == 1 ? RingLayout<128, 1>::OCC : RingLayout<128, 2>::OCC)
                    : (grp == 4 ? RingLayout<128, 4>::OCC : RingLayout<128, 8>::OCC);
}
DecWs dec_ws(const tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, bool weights)
{
    const int64_t cap = kv->max_pages * kv->page_rows, grp = nHq / kv->nKv;
    const int lhg = log_group(kv->nKv), tw = W >> lhg;
    const int64_t chunks = kv->batch * (kv->nKv >> lhg) * ((cap + KT * tw - 1) / (KT * tw));
    DecWs w{};
    w.grid = (int)std::min<int64_t>(chunks, (int64_t)dec_occ(kv->hd, grp) * ctx->num_sms);
    w.po = up256(((size_t)w.grid * 2 * grp * kv->hd * sizeof(float)) << lhg);
    w.pml = up256(((size_t)w.grid * 2 * grp * sizeof(float2)) << lhg);
    if (weights) {
        w.ml = up256((size_t)kv->batch * nHq * sizeof(float2));
        w.sc = up256((size_t)kv->batch * nHq * cap * sizeof(float));
    }
    return w;
}

template <int HD, int GRP>
int launch_decode(tb_ctx* ctx, const DecArgs& a)
{
    auto kern = k_paged_decode<HD, GRP>;
    constexpr int smem = RingLayout<HD, GRP>::BYTES;
    static bool attr_set[64] = {};   // per device and instantiation; setting it twice is harmless
    cudaError_t e = cudaSuccess;
    if (ctx->device >= 64 || !attr_set[ctx->device]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess && ctx->device < 64) attr_set[ctx->device] = true;
    }
    if (e == cudaSuccess) e = tb_launch(ctx, kern, dim3(a.grid), dim3(NT), (size_t)smem, a);
    if (e == cudaSuccess) e = tb_launch(ctx, k_paged_combine<HD, GRP>, dim3(a.kv.nKv, a.kv.batch), dim3(CT), (size_t)a.grid * GRP * sizeof(float2), a);
    if (e == cudaSuccess && a.weights)
        e = tb_launch(ctx, k_paged_weights<GRP>,
                      dim3(tb_cdiv((long long)a.kv.max_pages << a.kv.log_page, 256 * KEYS), a.kv.nKv, a.kv.batch), dim3(256), 0, a);
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
    TB_REQUIRE(ctx, kv->batch * kv->nKv * (kv->max_pages * kv->page_rows / KT + 1) < (1LL << 30),
               "batch x heads x rows too large");
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
    const int64_t cap = kv->max_pages * kv->page_rows;
    a.window = window < cap ? (int)window : 0;             // a window of every row is none
    a.sinks = (int)std::min<int64_t>(sinks, cap);
    a.grid = w.grid;
    a.log_hg = log_group(kv->nKv);
    a.qscale = 1.4426950408889634f / (127.0f * sqrtf((float)kv->hd));
    const int64_t cols = kv->nKv * kv->hd, rows = kv->n_pages * kv->page_rows;
    const int box = (int)std::min<int64_t>(KT, kv->page_rows);
    const CUtensorMapSwizzle swz = kv->hd == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    rc = tb_encode_2d(ctx, &a.mk, kv->Kq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, cols, rows, (int)kv->hd, box, swz);
    if (!rc) rc = tb_encode_2d(ctx, &a.mv, kv->Vq, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, cols, rows, (int)kv->hd, box, swz);
    if (rc) return rc;
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
