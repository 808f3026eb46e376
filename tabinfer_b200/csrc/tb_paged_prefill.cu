// tb_paged_prefill.cu -- attention of packed prompts or chunks of prompts over the paged
// int8 KV cache on the 5th-generation tensor cores: causal, GQA, a sliding window with
// first tokens kept.
//
// Rows cu[b] .. cu[b+1]-1 of q are the last t_b = cu[b+1]-cu[b] rows of sequence b; query i
// stands at row n_b - t_b + i.
//
// An item is 256 / GRP consecutive queries of a sequence and one kv head: with the group's
// q heads that is two 128-row tiles of S = Q K^T, so a dequantized K / V tile serves 256
// rows.  The 128-key tiles that an item's queries see are its work; items with more than
// their share (all tiles / SMs) are cut into parts, whose (m, l, O) a joining kernel merges
// in order.  k_prefill_plan (one CTA) lists the parts by length; the persistent CTAs (one an
// SM) take them in boustrophedon order.
//
// Warp roles of k_paged_prefill:
//   warps 0-3, 4-7   softmax of row tile 0 / 1, a thread a row: S from TMEM, P (f16) back
//                    over it; the reference maximum is raised (and O rescaled in TMEM) only
//                    when scores pass it by 2^2 to 2^8, so O is hardly ever touched; Q of the
//                    next part into shared memory, then the part's outputs
//   warps 8-11       K / V tiles: 16-byte copies ahead into thread-private shared memory, bytes
//                    -> f16 (one exact step, one multiplication by the group's scale) into
//                    swizzled tiles
//   warp 12          TMEM and the MMAs: S_t = Q_t K^T (both K-major), O_t += P_t V (P from
//                    TMEM, V MN-major as it lies in the cache), row tile 0 and 1 in turn so
//                    that one's softmax runs under the other's MMAs
// Roundings: Q, dequantized K and V (and their scales) and P to f16, relative 2^-11 each, and
// parts' outputs on their way through memory; S, the statistics and O in f32.  Q's rows, K and V
// of 32 keys, O and a part's outputs carry powers of two of their own (below), so this holds for
// numbers of any size and for weights down to 2^-22 of the reference (2^-33 of it is the error of
// those below): an element of K or V loses digits below 2^-25 of the largest one of its
// head in the same 32 rows (2^-36 of that one at most), one of Q below 2^-12 of its row's
// largest (2^-23).
//
// What bounds it.  Its operations at the bf16 rate a library product reaches (1679 TFLOP/s)
// would take 164 us at 8192 rows (16 / 8 heads of 128); it takes 310 alone (887 TFLOP/s;
// 349, 787, call after call over other inputs, at the power cap), 2048 rows 51 (337), three
// chunks of up to 2001 rows under a window of 1024 (32 / 8 heads of 64) 152 (276).  A half
// of 64 keys takes a softmax warp about 2200 cycles, two of them sharing a scheduler: 1100
// to 1500 for its 64 exponentials with their sums and conversions (1024 of the special
// function unit for both warps), the rest waits, TMEM loads and stores and the barriers;
// the tensor cores are busy half of the time, so 64-wide heads, with half the product for
// the same exponentials, come out at a third of the rate (their exponentials alone are a
// quarter of the time; the rest is the step's latency, and halves that no row of a tile
// sees are worked through).  Short chunks (77 rows behind 8192: 32 us) are the plan, the
// first tiles' latency and the join.  The powers of two, the lift and the marks cost 1 to
// 2.5 us a call, most of it instructions that a short call runs through once (8192 rows:
// nothing).
// Measured and not kept (times of their day, beside 314 to 320 at 8192 rows): 16 softmax
// warps of 16 columns (362 us at 8192 rows), whole tiles of 128 keys a softmax step (340),
// a quarter of the exponentials by polynomial (315), taking turns at the exponentials
// (352), the next half's scores fetched ahead of the weights' store (320), an MMA warp a
// row tile (323), raw bytes in registers (348).
// Every wait is bounded: one that gives up sets the error word and the CTA's abort flag, all
// roles leave, the MMA thread waits for its last commit and TMEM is freed.
#include <cuda_bf16.h>
#include <type_traits>

#include "tb_paged.cuh"
#include "tb_rounds.h"

namespace {

constexpr int PK = 128;                  // keys a tile
constexpr int ROWS = 256;                // rows an item: two tiles of 128
constexpr int THREADS = 512;               // 2 x 4 softmax and 4 producer warps, the MMA warp and three idle ones
constexpr int PROD = 128, W_MMA = 12;
constexpr int NC = 4;                      // 16-byte chunks a producer thread takes at a time
constexpr int KV_STAGES = 2;
constexpr int MAX_BATCH = 4096;          // sequences a call (the plan keeps their sums in shared memory)
// cycles by which row tile 1's softmax starts a part behind tile 0's (8192 rows 316 us with none, 318 with 450, 314
// with 900; three 2001-row chunks under a window 158, 153, 151.6; 2048 rows 50.2, 50.2, 49.5; short ones too: 700 rows
// 23.5, 23.2, 22.9, one row 12.6 with any)
constexpr int STAGGER = 900;
// Powers of two.  f16 holds 30 binades, so Q's rows and the K and V of 32 keys are brought to its upper end first:
// x = x' 2^(e - TOP), the largest |x'| of K and of V in [2^11, 2^15), e a multiple of 4, so that a group's powers are
// mostly the last one's.  K's and Q's powers go into the factor of the scores; a weight is multiplied by V's power over
// O's unit, the largest V's of the row so far, by an addition to the exponential's argument.
// The smallest e, a zero's too, leaves the factor of the scores a normal number: a score masked with -inf stays it.
constexpr int BIAS = 128, TOP = 15, E_MIN = -40;
constexpr int Q_E = 11, Q_MIN = -6;       // q whose rows' largest lie between 2^Q_MIN and 2^Q_E share e = Q_E
// A weight goes to f16 as 2^(score - reference + LIFT): one of the reference's size uses the upper part of f16's
// range, so weights down to 2^-22 of it keep 2^-11 of themselves, and those below lose 2^-33 of it at most (without
// the lift 2^-14 and 2^-25: many light keys beside a heavy one then came out wrong).
constexpr float LIFT = 8.0f;
// Sum of a half's weights that raises the reference: below it each of them fits f16, and with every score at or below
// the reference the 64 come to 2^14 at most.  (At 2^15 more halves are repeated: 77 rows 33.8 us instead of 33.1.)
constexpr float TOO_LARGE = 65504.0f;
constexpr float FAR = 1048576.0f;        // scores (log2) whose last bit, 2^-4, is felt in a weight

struct Part {
    int b, row0, nq, p0;                 // sequence, first packed row, queries, row of the first in the sequence
    int t0, t1;                          // its tiles in the item's list
    int slot;                            // partial slot, -1: the item whole
    int pad;
};
struct Item {
    int row0, nq, slot0, parts;
};

struct PrefillArgs {
    PagedArgs kv;
    const float* q;         // [T][nHq*HD]
    __nv_bfloat16* out;     // [T][nHq*HD]
    const int* cu;          // [B+1]
    const int* lens;        // [B]
    int* head;              // parts, items
    Part* parts;
    Item* items;
    // [slot][nKv][HD / 2][ROWS]: O / l as pairs of f16 (the operands' own rounding, half the bytes: as f32, 2048 rows
    // took 59 us instead of 53); a thread holds a row, so a warp writes 128 contiguous bytes
    uint32_t* PO;
    // [slot][nKv][ROWS] m and l, whose last 8 bits hold the unit of the part's outputs (a part's weight is then off by
    // 2^-16, far below the operands' 2^-11)
    float2* PML;
    int T, nHq, grp, window, sinks, sms;
    int max_items, max_parts, max_slots;   // what the workspace holds
    float sl2;              // log2(e) / sqrt(HD)
};

// ---- the plan: one CTA ---------------------------------------------------------------
constexpr int PT = 256, CLASS_BITS = 8;      // threads, and as many classes of part lengths
static_assert(PT == 1 << CLASS_BITS, "a thread a class");

__device__ int block_scan(int x, int* buf, int* total)      // inclusive; buf: PT / 32 words
{
    const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += v;
    }
    __syncthreads();
    if (lane == 31) buf[wid] = x;
    __syncthreads();
    int all = 0;
    for (int i = 0; i < PT / 32; i++) {
        if (i < wid) x += buf[i];
        all += buf[i];
    }
    *total = all;
    return x;
}

__global__ void __launch_bounds__(PT) k_prefill_plan(const PrefillArgs a)
{
    __shared__ int first[MAX_BATCH + 1];      // items below each sequence
    __shared__ int buf[PT / 32], hist[PT];
    __shared__ unsigned long long all_tiles;
    __shared__ int split;
    tb_pdl_wait();
    tb_pdl_trigger();
    const int tid = threadIdx.x, B = a.kv.batch, qb = ROWS / a.grp;
    int items = 0;
    for (int b0 = 0; b0 < B; b0 += PT) {
        const int b = b0 + tid;
        int n = 0;
        if (b < B) {
            const int c0 = a.cu[b], c1 = a.cu[b + 1];
            if (c0 >= 0 && c1 <= a.T && c1 >= c0) n = (c1 - c0 + qb - 1) / qb;
            else atomicExch(a.kv.err, ERR_PAGED_LEN);
        }
        int all;
        const int x = block_scan(n, buf, &all);
        if (b < B) first[b] = items + x - n;
        items += all;
    }
    if (tid == 0) first[B] = items;
    hist[tid] = 0;
    __syncthreads();
    if (items > a.max_items) {                // overlapping sequences: more rows than q has
        if (tid == 0) {
            a.head[0] = a.head[1] = 0;
            atomicExch(a.kv.err, ERR_PAGED_LEN);
        }
        return;
    }
    // the item's queries and tiles
    struct Shape {
        int b, row0, nq, p0, nt;
    };
    auto item = [&](int i) {
        Shape v;
        int lo = 0, hi = B;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= i) lo = mid;
            else hi = mid;
        }
        v.b = lo;
        const int c0 = a.cu[lo], rows = a.cu[lo + 1] - c0, at = (i - first[lo]) * qb;
        const int n = a.kv.checked_len(a.lens[lo]);
        v.row0 = c0 + at;
        v.nq = min(qb, rows - at);
        v.p0 = n - rows + at;
        v.nt = SeenTiles(max(v.p0, 0), v.p0 + v.nq - 1, a.window, a.sinks, PK).count;
        if (v.p0 < 0) atomicExch(a.kv.err, ERR_PAGED_LEN);
        return v;
    };
    // the thread's first item stays in registers
    const Shape own = tid < items ? item(tid) : Shape{0, 0, 0, 0, 0};
    unsigned long long tiles = own.nt;
    for (int i = tid + PT; i < items; i += PT) tiles += item(i).nt;
    if (tid == 0) {
        all_tiles = 0;
        split = 0;
    }
    __syncthreads();
    for (int o = 16; o > 0; o >>= 1) tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
    if ((tid & 31) == 0) atomicAdd(&all_tiles, tiles);
    __syncthreads();
    // the longest part: a CTA's share of all heads' tiles, down to one (77 rows behind 1000: 18.0 us, with two
    // tiles at least 19.5, with four 23.5)
    const int share = (int)min(1ull << 24, max(1ull, (all_tiles * a.kv.nKv + a.sms - 1) / a.sms));
    const int shift = max(0, 32 - __clz(share) - CLASS_BITS);  // part lengths as at most PT classes
    for (int i = tid; i < items; i += PT) {
        const int nt = i == tid ? own.nt : item(i).nt, np = max(1, (nt + share - 1) / share);
        for (int k = 0; k < np; k++)
            atomicAdd(&hist[((k + 1) * nt / np - k * nt / np) >> shift], 1);
    }
    __syncthreads();
    // places from the longest class down
    const int mine = hist[PT - 1 - tid];
    int parts;
    const int place = block_scan(mine, buf, &parts) - mine;
    __syncthreads();
    hist[PT - 1 - tid] = place;
    __syncthreads();
    int slots = 0;
    for (int i0 = 0; i0 < items; i0 += PT) {
        const int i = i0 + tid;
        Shape v = own;
        if (i0 > 0 && i < items) v = item(i);
        const int nt = v.nt, np = i < items ? max(1, (nt + share - 1) / share) : 0;
        int all;
        const int mine_slots = np > 1 ? np : 0;
        const int s0 = slots + block_scan(mine_slots, buf, &all) - mine_slots;
        slots += all;
        if (i >= items) continue;
        if (np > 1) a.items[atomicAdd(&split, 1)] = Item{v.row0, v.nq, s0, np};
        for (int k = 0; k < np; k++) {
            const int t0 = k * nt / np, t1 = (k + 1) * nt / np;
            const int at = atomicAdd(&hist[(t1 - t0) >> shift], 1);
            if (at < a.max_parts) a.parts[at] = Part{v.b, v.row0, v.nq, v.p0, t0, t1, np > 1 ? s0 + k : -1, 0};
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.head[0] = min(parts, a.max_parts);
        a.head[1] = split;                    // the items that were cut
    }
}

// ---- the products ---------------------------------------------------------------------
template <int HD>
struct PrefillLayout {
    static constexpr int HALF = 128 * 128;                     // 128 rows x 64 f16, 128-byte swizzle
    static constexpr int TILE = HALF * (HD / 64);
    static constexpr int OFF_Q = 0;                            // [2]
    static constexpr int OFF_K = 2 * TILE;                     // [KV_STAGES]
    static constexpr int OFF_V = OFF_K + KV_STAGES * TILE;
    static constexpr int OFF_ROW = OFF_V + KV_STAGES * TILE;   // int [3][PK] pool rows
    static constexpr int OFF_SC = OFF_ROW + 3 * PK * 4;        // f16 [3][2][PK][4] scales of K and V
    // uint4 [8][2]: of a half's two 32-key groups the keys of pages outside the pool, and marks: K's power of two in
    // byte 0, V's in byte 1 (both + BIAS; 0: no V but zero), bit 16 + G where some V has no number in its 32 dims G;
    // then, where there is such a bit, which keys: uint4 [8][PK / 32]
    static constexpr int OFF_MARK = OFF_SC + 3 * 2 * PK * 8, OFF_NAN = OFF_MARK + 8 * 2 * 16;
    // the producers' raw bytes: units of NC x 16 bytes a thread, thread-private (cp.async), NU in flight
    static constexpr int UNITS = HD / 64, NU = HD == 128 ? 3 : 2;
    static constexpr int OFF_RAW = OFF_NAN + 8 * PK / 32 * 16;
    static constexpr int OFF_BAR = OFF_RAW + NU * NC * 16 * PROD;
    static constexpr int BYTES = 1024 + OFF_BAR + 256;
    static_assert(BYTES <= 227 * 1024, "shared memory");
};
// byte offset of 16-byte chunk c (0..7) of row r in a half tile
__device__ __forceinline__ uint32_t sw128(int r, int c)
{
    return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((c ^ (r & 7)) << 4));
}
// K-major operand: 8-row atoms 1024 bytes apart
__device__ __forceinline__ uint64_t desc_k(uint32_t saddr)
{
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// MN-major operand: atoms of 64 columns x 8 keys, 1024 bytes apart along the keys and HALF
// bytes along the columns
__device__ __forceinline__ uint64_t desc_mn(uint32_t saddr)
{
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(16384 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}
// kind::f16: D f32, A and B f16; B MN-major at bit 16; N >> 3 at bit 17, M >> 4 at bit 24
constexpr uint32_t idesc(int n, bool bmn)
{
    return (1u << 4) | ((bmn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

#define TB_R32(r) \
    "=r"((r)[0]), "=r"((r)[1]), "=r"((r)[2]), "=r"((r)[3]), "=r"((r)[4]), "=r"((r)[5]), "=r"((r)[6]), "=r"((r)[7]), \
        "=r"((r)[8]), "=r"((r)[9]), "=r"((r)[10]), "=r"((r)[11]), "=r"((r)[12]), "=r"((r)[13]), "=r"((r)[14]), \
        "=r"((r)[15]), "=r"((r)[16]), "=r"((r)[17]), "=r"((r)[18]), "=r"((r)[19]), "=r"((r)[20]), "=r"((r)[21]), \
        "=r"((r)[22]), "=r"((r)[23]), "=r"((r)[24]), "=r"((r)[25]), "=r"((r)[26]), "=r"((r)[27]), "=r"((r)[28]), \
        "=r"((r)[29]), "=r"((r)[30]), "=r"((r)[31])
// 32 columns of this warp's 32 TMEM lanes
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
                 "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : TB_R32(r) : "r"(taddr));
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
                 "%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The MMA warp runs these with all lanes and warp-uniform operands and elects the issuing
// thread inside: addresses then stay in uniform registers and an MMA costs one instruction
// (issued from a branch on one lane, 128 x 128 x 16 took 115 cycles against 68 here).
__device__ __forceinline__ void tc_commit(uint64_t* bar)
{
    asm volatile("{\n .reg .pred e;\n elect.sync _|e, 0xffffffff;\n"
                 " @e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}"
                 ::"r"(smem_u32(bar)) : "memory");
}
// D (+)= A B^T over 64 k of f16: A and B K-major in shared memory, four steps of 32 bytes
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t da, uint64_t db, uint32_t id, uint32_t add)
{
#define TB_SS(i, pr)                                                                              \
    " add.u64 a, %1, " #i ";\n add.u64 b, %2, " #i ";\n"                                          \
    " @e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, " #pr ";\n"
    asm volatile("{\n .reg .pred e, p, t;\n .reg .b64 a, b;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
                 " elect.sync _|e, 0xffffffff;\n" TB_SS(0, p) TB_SS(2, t) TB_SS(4, t) TB_SS(6, t) "}"
                 ::"r"(d), "l"(da), "l"(db), "r"(id), "r"(add) : "memory");
#undef TB_SS
}
// D (+)= A B over 64 k: A f16 in TMEM (8 columns a step), B MN-major (2048 bytes a step)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t ta, uint64_t db, uint32_t id, uint32_t add)
{
#define TB_TS(i, j, pr)                                                                           \
    " add.u32 a, %1, " #i ";\n add.u64 b, %2, " #j ";\n"                                          \
    " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, " #pr ";\n"
    asm volatile("{\n .reg .pred e, p, t;\n .reg .b32 a;\n .reg .b64 b;\n setp.ne.b32 p, %4, 0;\n setp.eq.b32 t, 0, 0;\n"
                 " elect.sync _|e, 0xffffffff;\n" TB_TS(0, 0, p) TB_TS(8, 128, t) TB_TS(16, 256, t) TB_TS(24, 384, t) "}"
                 ::"r"(d), "r"(ta), "l"(db), "r"(id), "r"(add) : "memory");
#undef TB_TS
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi)
{
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// e with 2^(e-1) <= |x| < 2^e for the bits of |x|, at least E_MIN
__device__ __forceinline__ int size_of(uint32_t bits) { return max(E_MIN, (int)(bits >> 23) - 126); }
// bits 0 .. n - 1 (n clamped to 0 .. 32)
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }

// the k-th (part, head) of CTA c: rounds over the list, every other one backwards
__device__ __forceinline__ int nth(int k, int c, int grid) { return k * grid + ((k & 1) ? grid - 1 - c : c); }

template <int HD, int GRP>
__global__ void __launch_bounds__(THREADS, 1) k_paged_prefill(const __grid_constant__ PrefillArgs a)
{
    using L = PrefillLayout<HD>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
    uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);     // [2] Q of the part staged
    uint64_t* k_full = q_full + 2;                                          // [KV_STAGES]
    uint64_t* k_empty = k_full + KV_STAGES;
    uint64_t* v_full = k_empty + KV_STAGES;
    uint64_t* v_empty = v_full + KV_STAGES;
    uint64_t* s_full = v_empty + KV_STAGES;                                 // [2][2] a half of S written
    uint64_t* p_full = s_full + 4;                                          // [2][2] a half of P written, O rescaled
    uint64_t* o_done = p_full + 4;                                          // [2][2] O += P V of a half completed
    uint64_t* done = o_done + 4;                                            // every MMA completed
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(done + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(done + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, nKv = a.kv.nKv;
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&q_full[i], 4);
            mbar_init(&s_full[2 * i], 1);
            mbar_init(&s_full[2 * i + 1], 1);
            mbar_init(&p_full[2 * i], 4);
            mbar_init(&p_full[2 * i + 1], 4);
            mbar_init(&o_done[2 * i], 1);
            mbar_init(&o_done[2 * i + 1], 1);
        }
        for (int i = 0; i < KV_STAGES; i++) {
            mbar_init(&k_full[i], PROD / 32);
            mbar_init(&k_empty[i], 1);
            mbar_init(&v_full[i], PROD / 32);
            mbar_init(&v_empty[i], 1);
        }
        mbar_init(done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == W_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void*)tmem_slot)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_before();
    __syncthreads();
    tc_after();
    const uint32_t tmem = *tmem_slot;      // S 0, S 1 (128 columns each), O 0, O 1
    tb_pdl_wait();
    tb_pdl_trigger();
    const int total = a.head[0] * nKv, grid = gridDim.x, cta = blockIdx.x;
    auto give_up = [&]() {
        *abort_flag = 1;
        atomicExch(a.kv.err, ERR_PAGED_WAIT);
    };
    // one outcome for the warp: its lanes then run the .aligned instructions together
    auto wait_warp = [&](uint64_t* bar, uint32_t parity) {
        if (__all_sync(0xffffffffu, mbar_test(bar, parity))) return true;
        const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag));
        if (!ok && lane == 0) give_up();
        __syncwarp();
        return ok;
    };

    if (warp < 8) {
        // =============================== softmax ======================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;");      // 256 x 152 + 128 x 120 + 128 x 88 = 65536
        const int t = warp >> 2, wq = warp & 3, row = 32 * wq + lane;      // row of the tile
        const uint32_t ts = tmem + ((uint32_t)(32 * wq) << 16) + 128 * t;
        const uint32_t to = tmem + ((uint32_t)(32 * wq) << 16) + 256 + HD * t;
        uint8_t* qs = smem + L::OFF_Q + t * L::TILE;
        // Q rows of this warp: row r of the item = query r / GRP, head r % GRP.  Returns the factor of the scores that
        // belongs to the row of this lane.  As a rule a row goes in as 2^(TOP - Q_E) times itself; where that is too large
        // for f16 in one, or one has no element of 2^Q_MIN, the warp's rows go in again, each by its own power of two.
        auto load_q = [&](const Part& p, int h) {
            constexpr int C4 = HD / 4;                          // float4 columns a row
            auto load = [&](int i) {
                const int ir = 128 * t + 32 * wq + i / C4, qi = ir / GRP;
                const float* src = a.q + ((long long)(p.row0 + qi) * a.nHq + h * GRP + ir % GRP) * HD;
                return qi < p.nq ? __ldg(reinterpret_cast<const float4*>(src) + i % C4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            };
            auto store = [&](int i, float4 v, float f) {
                const int r = 32 * wq + i / C4, c = i % C4;
                *reinterpret_cast<uint2*>(qs + (c >> 4) * L::HALF + sw128(r, (c & 15) >> 1) + (c & 1) * 8) =
                    make_uint2(pack_h2(v.x * f, v.y * f), pack_h2(v.z * f, v.w * f));
            };
            auto large = [](float4 v) { return fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))); };
            int e = Q_E;
            constexpr int NL = 16;                              // loads in flight
            const int rows = p.nq * GRP - 128 * t - 32 * wq;    // the warp's rows that are there, and those behind them
            float most = 0.0f;
            bool fine = true;
#pragma unroll 1
            for (int i0 = lane; i0 < 32 * C4; i0 += 32 * NL) {
                float4 v[NL];
#pragma unroll
                for (int i = 0; i < NL; i++) v[i] = load(i0 + 32 * i);
                uint32_t has = 0;                               // bit i: load i has an element of 2^Q_MIN or more
#pragma unroll
                for (int i = 0; i < NL; i++) {
                    const float x = large(v[i]);
                    most = fmaxf(most, x);
                    if (x >= pow2(Q_MIN)) has |= 1u << i;
                    store(i0 + 32 * i, v[i], pow2(TOP - Q_E));
                }
                // of the row of load i; of the rows 2 i (bit i) and 2 i + 1 (bit 16 + i)
                has = __reduce_or_sync(0xffffffffu, C4 < 32 && lane >= 16 ? has << 16 : has);
                const uint32_t all = C4 == 32 ? below(min(16, rows - i0 / C4))
                                              : below(min(16, (rows + 1) / 2)) | below(min(16, rows / 2)) << 16;
                fine = fine && (has & all) == all;
            }
            if (!__all_sync(0xffffffffu, fine && most < pow2(Q_E))) {
#pragma unroll 1
                for (int i = lane; i < 32 * C4; i += 32) {
                    const float4 v = load(i);
                    float x = large(v);
#pragma unroll
                    for (int o = C4 / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
                    const int er = min(127, size_of(__float_as_uint(x)));        // of the row that this lane loads
                    const int mine = __shfl_sync(0xffffffffu, er, C4 == 32 ? 0 : (lane & 1) * 16);
                    if ((C4 == 32 ? lane : lane >> 1) == i / 32) e = mine;
                    store(i, v, pow2(TOP - er));
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[t]);
            return a.sl2 * pow2(e - TOP);
        };
        // the CTA's next part that has rows in this tile
        const uint4* mark = reinterpret_cast<const uint4*>(smem + L::OFF_MARK);
        const uint4* nans = reinterpret_cast<const uint4*>(smem + L::OFF_NAN);
        int tile = 0;                                            // tiles of the CTA so far (the masks' ring)
        auto find = [&](int k, Part& p, int& h) {
            for (;; k++) {
                if (k * grid >= total) return -1;
                const int i = nth(k, cta, grid);
                if (i >= total) continue;
                p = a.parts[i / nKv];
                h = i % nKv;
                if (p.t1 > p.t0 && (t == 0 || p.nq * GRP > 128)) return k;
                tile += p.t1 - p.t0;
                // a part that sees nothing: zeros (its rows lie before the sequence)
                if (p.t1 <= p.t0 && t == 0 && p.slot < 0)
                    for (int j = tid; j < p.nq * GRP * HD; j += 128)
                        a.out[((long long)(p.row0 + j / (GRP * HD)) * a.nHq + h * GRP) * HD + j % (GRP * HD)] =
                            __float2bfloat16_rn(0.0f);
            }
        };
        Part p;
        int h = 0, k = find(0, p, h), seq = 0;                   // seq: tiles of this row tile so far
        float sl = 0.0f;                                         // log2 of a weight a unit of S, before K's power
        if (k >= 0) sl = load_q(p, h);
        while (k >= 0) {
            const int qi = (128 * t + row) / GRP;
            const int pos = p.p0 + min(qi, p.nq - 1), pmin = max(p.p0, 0), pmax = p.p0 + p.nq - 1;
            const SeenTiles seen(pmin, pmax, a.window, a.sinks, PK);
            float m = -INFINITY, l = 0.0f;
            int unit = 0;                            // O's power of two + BIAS; 0: O is zero
            // the last half's marks (none is 0), its groups' factors of the scores, and how many binades d their V lies
            // below the unit, and b = 2^d
            uint32_t last0 = 0, last1 = 0;
            float sc0 = 0.0f, sc1 = 0.0f, d0 = 0.0f, d1 = 0.0f, b0 = 1.0f, b1 = 1.0f;
            uint32_t none = 0;                       // 32-groups of the row's output that have no number
            // tile 1 a little behind tile 0: its warps share their schedulers with tile 0's, and one's exponentials
            // then run under the other's loads, stores and waits
            bool ok = t == 0 || wait_warp(&s_full[2 * t], seq & 1);
            if (t == 1)
                for (const long long c0 = clock64(); clock64() - c0 < STAGGER;) {}
            for (int j = p.t0; ok && j < p.t1; j++, seq++, tile++) {
                const int k0 = seen.tile(j) * PK;
                const int hi = pos - k0, lo = a.window > 0 ? hi - a.window : -1, sk = a.sinks - k0;
                // In two halves of 64 keys: a half's P V and the next tile's Q K^T over its place run under the
                // other half's softmax, so scores are there when a thread comes for them.
                // One pass over a half's scores against the reference maximum as it stands: no maximum is
                // formed.  Where the sum tells that scores have passed it (one by 2^8, or all by 2^2), the maximum is
                // taken, O rescaled (every column, once the last product is in) and the pass repeated, once.  A
                // row's first reference is the maximum of the first half in which it sees a key.
#pragma unroll 1
                for (int hh = 0; hh < 2; hh++) {
                    const bool fresh = j == p.t0 && hh == 0;
                    const uint32_t th = ts + 64 * hh;
                    if (!(ok = wait_warp(&s_full[2 * t + hh], seq & 1))) break;
                    tc_after();
                    const uint4 mk = mark[2 * (tile & 7) + hh];
                    const int kh = k0 + 64 * hh;
                    // a half that some row sees only in part, or with keys on bad pages
                    const bool part = kh + 63 > pmin || (a.window > 0 && kh <= pmax - a.window && kh + 64 > a.sinks) ||
                                      (mk.x | mk.y);
                    // or with other marks than the last half's
                    const bool cut = part || mk.z != last0 || mk.w != last1;
                    // the half's keys that this row sees, as bits
                    uint32_t see0 = ~0u, see1 = ~0u;
                    float lower = 1.0f;                   // what a larger unit makes of O
                    if (cut) {
                        const int h0 = hi - 64 * hh, l0 = lo - 64 * hh, s0 = sk - 64 * hh;
                        see0 = below(h0 + 1) & (~below(l0 + 1) | below(s0)) & ~mk.x;
                        see1 = below(h0 - 31) & (~below(l0 - 31) | below(s0 - 32)) & ~mk.y;
                        auto told = [&](uint32_t w, uint32_t see, int g) {
                            if (!(w >> 16)) return;
                            const uint4 n = nans[4 * (tile & 7) + g];
                            none |= (n.x & see ? 1u : 0u) | (n.y & see ? 2u : 0u) | (n.z & see ? 4u : 0u) | (n.w & see ? 8u : 0u);
                        };
                        told(mk.z, see0, 2 * hh);
                        told(mk.w, see1, 2 * hh + 1);
                        // (marks with a key of no number are looked at in every half; a half seen in part may leave the
                        // row's unit below its V's, so the next one looks again)
                        last0 = part || (mk.z >> 16) ? 0u : mk.z;
                        last1 = part || (mk.w >> 16) ? 0u : mk.w;
                        sc0 = fminf(3.0e38f, sl * pow2((int)(mk.z & 255) - BIAS));
                        sc1 = fminf(3.0e38f, sl * pow2((int)(mk.w & 255) - BIAS));
                        // O's unit: the largest power of a V that the row sees
                        const int v0 = mk.z >> 8 & 255, v1 = mk.w >> 8 & 255, top = max(unit, max(see0 ? v0 : 0, see1 ? v1 : 0));
                        if (top > unit && unit > 0) lower = pow2(max(-126, unit - top));
                        unit = top;
                        // binades of a group's V below it; from 64 on its weights are zero in f16 whatever they are (the
                        // sums keep them in f32)
                        const int e0 = v0 ? max(0, min(64, unit - v0)) : 0, e1 = v1 ? max(0, min(64, unit - v1)) : 0;
                        d0 = (float)e0;
                        d1 = (float)e1;
                        b0 = pow2(e0);
                        b1 = pow2(e1);
                    }
                    auto mask = [&](float* s, uint32_t see) {
#pragma unroll
                        for (int c = 0; c < 32; c++)
                            if (!((see >> c) & 1)) s[c] = -INFINITY;
                    };
                    // the half's largest score, for the rows that need it
                    auto largest = [&] {
                        float t4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 2; c++) {
                            float s[32];
                            tmem_ld32(th + 32 * c, reinterpret_cast<uint32_t*>(s));
                            tmem_wait_ld();
                            if (cut) mask(s, c ? see1 : see0);
#pragma unroll
                            for (int i = 0; i < 32; i++) t4[2 * c + (i & 1)] = fmaxf(t4[2 * c + (i & 1)], s[i]);
                        }
                        return fmaxf(fmaxf(t4[0], t4[1]) * sc0, fmaxf(t4[2], t4[3]) * sc1);
                    };
                    if (__any_sync(0xffffffffu, m == -INFINITY)) {          // rows that have seen no key yet
                        const float mx = largest();
                        if (m == -INFINITY) m = mx;                         // O is zero, or not written
                    }
                    uint32_t pk[32];
                    float2 sum;                           // of either group
                    // The argument is x scale - m, of the product as it is (exact) or rounded as m was.  For the largest x the
                    // first is up to half an ulp of m from 0, which is nothing below FAR and past 2^24 any size, up or down;
                    // the second is 0 at most, and 0 for the largest x.
                    auto pass = [&](auto exact) {
                        const float off = m == -INFINITY ? 0.0f : -m, off0 = off + (LIFT - d0), off1 = off + (LIFT - d1);
                        float2 s2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                        float x[64];                      // all of the half at once: one wait, and the exponentials
                        tmem_ld32(th, reinterpret_cast<uint32_t*>(x));       // back to back (16 at a time took twice as long)
                        tmem_ld32(th + 32, reinterpret_cast<uint32_t*>(x) + 32);
                        tmem_wait_ld();
                        if (cut) {
                            mask(x, see0);
                            mask(x + 32, see1);
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) {
                            const float sc = i < 16 ? sc0 : sc1, of = i < 16 ? off0 : off1, d = i < 16 ? d0 : d1;
                            float2 y;
                            if (exact) y = ffma2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(sc, sc), make_float2(of, of));
                            else {                        // (the rounded product less m first: 0 for the largest)
                                y.x = __fadd_rn(__fadd_rn(__fmul_rn(x[2 * i], sc), off), LIFT - d);
                                y.y = __fadd_rn(__fadd_rn(__fmul_rn(x[2 * i + 1], sc), off), LIFT - d);
                            }
                            const float2 e = make_float2(ex2(y.x), ex2(y.y));
                            s2[i >> 4] = fadd2(s2[i >> 4], e);
                            pk[i] = pack_h2(e.x, e.y);
                        }
                        sum = make_float2(s2[0].x + s2[0].y, s2[1].x + s2[1].y);
                    };
                    pass(std::true_type());
                    // below it every weight fits f16; past it some score is above the reference
                    const bool far = fabsf(m) > FAR && m != -INFINITY;
                    if (__any_sync(0xffffffffu, sum.x + sum.y >= TOO_LARGE || lower < 1.0f || far)) {
                        const float mx = fmaxf(m, largest());
                        if (!fresh) {
                            // the half before: the last tile's second, or this tile's first
                            if (!(ok = wait_warp(&o_done[2 * t + (hh ^ 1)], (hh ? seq : seq - 1) & 1))) break;
                            tc_after();
                            const float f = mx > m ? ex2(m - mx) : 1.0f;
#pragma unroll
                            for (int c = 0; c < HD / 32; c++) {
                                uint32_t o[32];
                                tmem_ld32(to + 32 * c, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * (f * lower));
                                tmem_st32(to + 32 * c, o);
                            }
                            l *= f;
                        }
                        m = mx;
                        pass(std::false_type());          // once: no score of any row is above the reference now
                    }
                    tmem_st32(th, pk);                    // over scores that are read
                    l = fmaf(sum.x, b0, fmaf(sum.y, b1, l));
                    tmem_wait_st();
                    tc_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_full[2 * t + hh]);
                }
                if (!ok) break;
            }
            if (!ok) break;
            // the next part's Q goes in under this part's last product
            Part pn;
            int hn = 0;
            const int kn = find(k + 1, pn, hn);
            float sn = 0.0f;
            if (kn >= 0) sn = load_q(pn, hn);
            if (!wait_warp(&o_done[2 * t + 1], (seq - 1) & 1)) break;
            tc_after();
            const bool live = qi < p.nq;
            const long long slot = p.slot < 0 ? 0 : (long long)p.slot * nKv + h;
            if (p.slot >= 0)
                a.PML[slot * ROWS + 128 * t + row] = make_float2(m, __int_as_float((__float_as_int(l) & ~255) | unit));
            // (a part's outputs stay in the row's unit, so that they fit f16)
            const float rl = (l > 0.0f || l != l ? 1.0f / l : 0.0f) * (p.slot < 0 && unit ? pow2(unit - BIAS) : 1.0f);
#pragma unroll
            for (int c = 0; c < HD / 32; c++) {
                const float r = (none >> c) & 1 ? __int_as_float(0x7fc00000) : rl;
                uint32_t o[32];
                __syncwarp();                     // rows that are there meet those behind the last one
                tmem_ld32(to + 32 * c, o);
                tmem_wait_ld();
                if (p.slot >= 0) {
                    uint32_t* dst = a.PO + (slot * HD / 2 + 16 * c) * ROWS + 128 * t + row;
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        dst[i * ROWS] = pack_h2(__uint_as_float(o[2 * i]) * r, __uint_as_float(o[2 * i + 1]) * r);
                } else if (live) {
                    uint4* dst = reinterpret_cast<uint4*>(
                        a.out + ((long long)(p.row0 + qi) * a.nHq + h * GRP + (128 * t + row) % GRP) * HD + 32 * c);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        uint32_t w[4];
#pragma unroll
                        for (int x = 0; x < 4; x++) {
                            const __nv_bfloat162 v = __floats2bfloat162_rn(__uint_as_float(o[8 * i + 2 * x]) * r,
                                                                           __uint_as_float(o[8 * i + 2 * x + 1]) * r);
                            w[x] = *reinterpret_cast<const uint32_t*>(&v);
                        }
                        dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            __syncwarp();
            tc_before();       // O is read before the p_full that lets the next part's product write it
            p = pn;
            h = hn;
            k = kn;
            sl = sn;
        }
    } else if (warp < W_MMA) {
        // ============================ K / V tiles ======================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        const int pt = tid - 256;                                  // 0 .. 127: its key of a tile
        int* rows = reinterpret_cast<int*>(smem + L::OFF_ROW);
        uint2* scs = reinterpret_cast<uint2*>(smem + L::OFF_SC);    // [3][2][PK] four f16 scales
        constexpr int NG = HD / 32, CPR = HD / 16, RPU = NC * PROD / CPR;   // 16-byte chunks a row, rows a unit
        // the walk over the tiles of the CTA's parts
        int wk = -1, wj = 0, wt1 = 0, wb = 0, wh = 0, pmin = 0, pmax = 0, published = 0;
        uint32_t* marks = reinterpret_cast<uint32_t*>(smem + L::OFF_MARK);
        uint32_t* nans = reinterpret_cast<uint32_t*>(smem + L::OFF_NAN);
        SeenTiles seen(-1, -1, 0, 0, PK);
        // The thread's key of the next tile: its page number (requested here, looked at a tile later) and line;
        // a row that no query of the part sees is line -1 and stays zero.
        auto step = [&](int& page, int& line, int& hh) {
            while (wj >= wt1) {
                wk++;
                if (wk * grid >= total) return false;
                const int i = nth(wk, cta, grid);
                if (i >= total) continue;
                const Part p = a.parts[i / nKv];
                wh = i % nKv;
                wb = p.b;
                wj = p.t0;
                wt1 = p.t1;
                pmin = max(p.p0, 0);
                pmax = p.p0 + p.nq - 1;
                seen = SeenTiles(pmin, pmax, a.window, a.sinks, PK);
            }
            const int key = seen.tile(wj++) * PK + pt;
            const bool see = key <= pmax && (a.window <= 0 || key > pmin - a.window || key < a.sinks);
            page = see ? __ldg(a.kv.table + (long long)wb * a.kv.max_pages + (key >> a.kv.log_page)) : 0;
            line = see ? key & ((1 << a.kv.log_page) - 1) : -1;
            hh = wh;
            return true;
        };
        // the pool row: -1 not seen, -2 a page outside the pool
        auto finish = [&](int page, int line) {
            if (line < 0) return -1;
            if ((unsigned)page < (unsigned)a.kv.n_pages) return (page << a.kv.log_page) | line;
            atomicExch(a.kv.err, ERR_PAGED_PAGE);
            return -2;
        };
        auto load_scales = [&](int row, int hh, float (&ks)[4], float (&vs)[4]) {
#pragma unroll
            for (int i = 0; i < 4; i++) ks[i] = vs[i] = 0.0f;
            if (row >= 0) {
                const long long at = ((long long)row * nKv + hh) * NG;
                if constexpr (NG == 4) {
                    const float4 x = __ldg(reinterpret_cast<const float4*>(a.kv.Ks + at));
                    const float4 y = __ldg(reinterpret_cast<const float4*>(a.kv.Vs + at));
                    ks[0] = x.x; ks[1] = x.y; ks[2] = x.z; ks[3] = x.w;
                    vs[0] = y.x; vs[1] = y.y; vs[2] = y.z; vs[3] = y.w;
                } else {
                    const float2 x = __ldg(reinterpret_cast<const float2*>(a.kv.Ks + at));
                    const float2 y = __ldg(reinterpret_cast<const float2*>(a.kv.Vs + at));
                    ks[0] = x.x; ks[1] = x.y;
                    vs[0] = y.x; vs[1] = y.y;
                }
            }
        };
        // of the next tile to be published: the mark and the factors of the scales
        uint32_t mk = 0;
        float fk = 0.0f, fv = 0.0f;
        auto measure = [&](const float (&ks)[4], float (&vs)[4]) {
            constexpr float S = 128.0f / 127.0f;                    // bytes become q / 128
            // the warp's 32 keys: K's and V's powers of two from their largest scales (the bits of a scale that is not a
            // number are above those of every number)
            constexpr uint32_t INF = 0x7f800000u;
            auto bits = [](float x) { return __float_as_uint(fabsf(x)); };
            auto large = [&](const float (&x)[4]) {
                return max(max(bits(x[0]), bits(x[1])), max(bits(x[2]), bits(x[3])));
            };
            mk = 0;
            uint32_t kb = __reduce_max_sync(0xffffffffu, large(ks)), vb = __reduce_max_sync(0xffffffffu, large(vs));
            if (kb >= INF || vb >= INF) {
                // V without a number (an infinite scale, or NaN) goes in as zero: as it is, it would reach the rows that
                // do not see the key too, whose weight for it is zero (0 * inf).  The rows that see it are told.
                // (K's reaches its own column of scores only, and a score that is not seen is masked.)
                kb = vb = 0;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t who = __ballot_sync(0xffffffffu, bits(vs[i]) >= INF);
                    if (lane == 0) nans[4 * (4 * (published & 7) + (pt >> 5)) + i] = who;
                    if (who) mk |= 0x10000u << i;
                    if (bits(vs[i]) >= INF) vs[i] = 0.0f;
                    kb = max(kb, bits(ks[i]) < INF ? bits(ks[i]) : 0u);
                    vb = max(vb, bits(vs[i]));
                }
                kb = __reduce_max_sync(0xffffffffu, kb);
                vb = __reduce_max_sync(0xffffffffu, vb);
            }
            const int ke = (size_of(kb) + 3) & ~3, ve = (size_of(vb) + 3) & ~3;
            mk |= (uint32_t)(ke - TOP + BIAS) | (vb ? (uint32_t)(ve - TOP + BIAS) << 8 : 0u);
            fk = S * pow2(TOP - ke);
            fv = S * pow2(TOP - ve);
        };
        auto publish = [&](int buf, int row, const float (&ks)[4], float (&vs)[4]) {
            measure(ks, vs);
            // a row that is not there: any bytes, of scale zero
            rows[buf * PK + pt] = max(row, 0);
            // its key, on a page outside the pool, is left out by the softmax; of the eight masks the one
            // written here was last read seven tiles ago, four more than the stages hold
            const unsigned miss = __ballot_sync(0xffffffffu, row == -2);
            const int mat = (published & 7) * 8 + (pt >> 6) * 4 + ((pt >> 5) & 1);
            published++;
            if (lane == 0) {
                marks[mat] = miss;
                marks[mat + 2] = mk;
            }
            // (a scale goes in as f16, one rounding more an element: as f32 the three tiles' scales take 6 KB more than
            // the shared memory has left)
            scs[(2 * buf) * PK + pt] = make_uint2(pack_h2(ks[0] * fk, ks[1] * fk), pack_h2(ks[2] * fk, ks[3] * fk));
            scs[(2 * buf + 1) * PK + pt] = make_uint2(pack_h2(vs[0] * fv, vs[1] * fv), pack_h2(vs[2] * fv, vs[3] * fv));
        };
        const int ch = pt % CPR, r0 = pt / CPR;                     // chunk of a row; rows r0 + i * PROD / CPR
        uint4* raw = reinterpret_cast<uint4*>(smem + L::OFF_RAW) + pt;
        // unit x of a tile (K: 0 .. UNITS - 1, then V): this thread's chunk of four of its rows, into ring slot n
        auto load = [&](int x, int buf, int hh, int n) {
            const int8_t* pool = (x < L::UNITS ? a.kv.Kq : a.kv.Vq) + hh * HD + 16 * ch;
            const int* rr = rows + buf * PK + (x % L::UNITS) * RPU + r0;
            int at[NC];
#pragma unroll
            for (int i = 0; i < NC; i++) at[i] = rr[i * (PROD / CPR)];
#pragma unroll
            for (int i = 0; i < NC; i++) cp_async16(raw + (NC * n + i) * PROD, pool + (long long)at[i] * (nKv * HD));
        };
        auto store = [&](int x, uint8_t* tile, int buf, int n) {
            const __half* sc = reinterpret_cast<const __half*>(scs + (2 * buf + x / L::UNITS) * PK) + (ch >> 1);
            uint8_t* half = tile + (ch >> 2) * L::HALF;
            const int c0 = (ch & 3) * 2, swap = (ch >> 2) & 1;      // the halves' chunks go to other banks
            const int r = (x % L::UNITS) * RPU + r0;
            uint4 v[NC];                                            // all loads before the first store
            __half2 s2[NC];
#pragma unroll
            for (int i = 0; i < NC; i++) {
                v[i] = raw[(NC * n + i) * PROD];
                s2[i] = __half2half2(sc[4 * (r + i * (PROD / CPR))]);
            }
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const int ri = r + i * (PROD / CPR);
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                uint32_t o[8];
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    const uint32_t u = w[y] ^ 0x80808080u;          // byte + 128 -> 1024 + u -> (u - 128) / 128
                    const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
                    const __half2 k = __float2half2_rn(0.0078125f), m9 = __float2half2_rn(-9.0f);
                    const __half2 f0 = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&lo), k, m9), s2[i]);
                    const __half2 f1 = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&hi), k, m9), s2[i]);
                    o[2 * y] = *reinterpret_cast<const uint32_t*>(&f0);
                    o[2 * y + 1] = *reinterpret_cast<const uint32_t*>(&f1);
                }
                const uint4 lo4 = make_uint4(o[0], o[1], o[2], o[3]), hi4 = make_uint4(o[4], o[5], o[6], o[7]);
                *reinterpret_cast<uint4*>(half + sw128(ri, c0 + swap)) = swap ? hi4 : lo4;
                *reinterpret_cast<uint4*>(half + sw128(ri, c0 + 1 - swap)) = swap ? lo4 : hi4;
            }
        };
        // a barrier of the producers (the walks' tb_rounds.h); true when one of them has given up
        auto sync = [](bool dead) {
            uint32_t any;
            asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n"
                         " selp.u32 %0, 1, 0, q;\n}" : "=r"(any) : "r"((uint32_t)dead) : "memory");
            return any != 0;
        };
        // tile it is stored, it + 1's bytes are loaded, it + 2's scales and it + 3's page numbers requested
        int ring = 0, row = -1, page = 0, line = -1, h0 = 0, h1 = 0, h2 = 0, h3 = 0;
        float ks[4], vs[4];
        bool more0 = step(page, line, h0), more1 = false, more2 = false;
        if (more0) {
            row = finish(page, line);
            load_scales(row, h0, ks, vs);
            rows[pt] = max(row, 0);
            sync(false);
#pragma unroll
            for (int x = 0; x < L::NU; x++) {                       // the ring, from unit 0 on
                load(x, 0, h0, x);
                cp_async_commit();
            }
            publish(0, row, ks, vs);                                // seen after the loop's first barrier
            if ((more1 = step(page, line, h1))) {
                row = finish(page, line);
                load_scales(row, h1, ks, vs);
                more2 = step(page, line, h2);
            }
        }
        producer_rounds(
            more0, more1, more2,
            // rows and scales of the next tile (their buffer was last read two tiles ago)
            [&](int it) { publish(it % 3, row, ks, vs); }, sync,
            [&] {
                row = finish(page, line);
                load_scales(row, h2, ks, vs);
                return step(page, line, h3);
            },
            [&](int it, bool next) {
                const int s = it % KV_STAGES, buf = it % 3, nb = (it + 1) % 3;
                const uint32_t par = ((it / KV_STAGES) & 1) ^ 1;
#pragma unroll
                for (int x = 0; x < 2 * L::UNITS; x++) {
                    if (x == 0 || x == L::UNITS)
                        if (!wait_warp(x == 0 ? &k_empty[s] : &v_empty[s], par)) return false;
                    cp_async_wait<L::NU - 1>();                     // the thread's own copies of this unit
                    store(x, smem + (x < L::UNITS ? L::OFF_K : L::OFF_V) + s * L::TILE, buf, ring);
                    if (x == L::UNITS - 1 || x == 2 * L::UNITS - 1) {
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(x < L::UNITS ? &k_full[s] : &v_full[s]);
                    }
                    // the unit NU on: of this tile or the next
                    if (x + L::NU < 2 * L::UNITS) load(x + L::NU, buf, h0, ring);
                    else if (next) load(x + L::NU - 2 * L::UNITS, nb, h1, ring);
                    cp_async_commit();
                    ring = ring + 1 == L::NU ? 0 : ring + 1;
                }
                h0 = h1;
                h1 = h2;
                h2 = h3;
                return true;
            });
        cp_async_wait<0>();                                         // no copy in flight past here
    } else {
        // ================================ MMAs ==========================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        if (warp == W_MMA) {
            constexpr uint32_t I1 = idesc(PK / 2, false), I2 = idesc(HD, true);
            const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
            const uint64_t dq = desc_k(smem_u32(smem) + L::OFF_Q), dk = desc_k(smem_u32(smem) + L::OFF_K),
                           dv = desc_mn(smem_u32(smem) + L::OFF_V);
            uint32_t ph = 0;                               // parities of q_full (bits 0, 1) and p_full (2, 3)
            auto scores = [&](int t, int s, int c) {       // S_t = Q_t K^T over half c of the tile's keys
#pragma unroll
                for (int d = 0; d < HD / 64; d++)
                    mma_ss(tm + 128 * t + 64 * c, dq + (t * L::TILE + d * L::HALF) / 16,
                           dk + (s * L::TILE + d * L::HALF + c * 64 * 128) / 16, I1, d);
                tc_commit(&s_full[2 * t + c]);
            };
            auto output = [&](int t, int s, int c, bool add) {   // O_t (+)= P_t V over half c of the tile's keys
                mma_ts(tm + 256 + HD * t, tm + 128 * t + 64 * c, dv + (s * L::TILE + c * 64 * 128) / 16, I2, add ? 1u : 0u);
                tc_commit(&o_done[2 * t + c]);
            };
            int it = 0;
            bool ok = true;
            for (int k = 0; ok && k * grid < total; k++) {
                const int i = nth(k, cta, grid);
                if (i >= total) continue;
                const Part* p = a.parts + i / nKv;
                const int nt = p->t1 - p->t0, tiles = p->nq * GRP > 128 ? 2 : 1;
                if (nt <= 0) continue;
                if (!(ok = wait_warp(&k_full[it % KV_STAGES], (it / KV_STAGES) & 1))) break;
                for (int t = 0; t < tiles && ok; t++) {
                    if (!(ok = wait_warp(&q_full[t], (ph >> t) & 1))) break;
                    ph ^= 1u << t;
                    tc_after();
                    scores(t, it % KV_STAGES, 0);
                    scores(t, it % KV_STAGES, 1);
                }
                if (!ok) break;
                tc_commit(&k_empty[it % KV_STAGES]);
                for (int j = 0; j < nt && ok; j++, it++) {
                    const int s = it % KV_STAGES, sn = (it + 1) % KV_STAGES;
                    if (!(ok = wait_warp(&v_full[s], (it / KV_STAGES) & 1))) break;
                    if (j + 1 < nt && !(ok = wait_warp(&k_full[sn], ((it + 1) / KV_STAGES) & 1))) break;
                    for (int c = 0; c < 2 && ok; c++)
                        for (int t = 0; t < tiles; t++) {
                            if (!(ok = wait_warp(&p_full[2 * t + c], (ph >> (2 + t)) & 1))) break;
                            tc_after();
                            output(t, s, c, j > 0 || c > 0);
                            if (j + 1 < nt) scores(t, sn, c);
                        }
                    if (!ok) break;
                    ph ^= tiles == 2 ? 12u : 4u;
                    tc_commit(&v_empty[s]);
                    if (j + 1 < nt) tc_commit(&k_empty[sn]);
                }
            }
            tc_commit(done);
            if (!mbar_wait(done, 0) && lane == 0) give_up();            // no MMA in flight past here
            __syncwarp();
        }
    }
    tc_before();
    __syncthreads();
    if (warp == W_MMA) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Joins the parts of item x, kv head y, rows 32 z ..: lane = row, a warp takes CW columns.
// The parts' (m, l) come first (all at once, into shared memory), then eight parts' outputs
// at a time.
constexpr int JT = 512;
template <int HD, int GRP>
__global__ void __launch_bounds__(JT) k_prefill_join(const __grid_constant__ PrefillArgs a)
{
    constexpr int CW = HD / (JT / 32);
    extern __shared__ float2 ml[];            // [parts][32]: m and l
    tb_pdl_wait();
    tb_pdl_trigger();
    const int h = blockIdx.y, nKv = a.kv.nKv, lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c0 = wid * CW;
    const int row = 32 * blockIdx.z + lane, qi = row / GRP;
    const int split = a.head[1];
    for (int i = blockIdx.x; i < split; i += gridDim.x) {
        const Item it = a.items[i];
        if (32 * (int)blockIdx.z >= it.nq * GRP) continue;
        const float2* pml = a.PML + ((long long)it.slot0 * nKv + h) * ROWS + row;
        const uint32_t* po = a.PO + (((long long)it.slot0 * nKv + h) * HD / 2 + c0 / 2) * ROWS + row;
        __syncthreads();                      // the last item's are read
        for (int p = wid; p < it.parts; p += JT / 32) ml[p * 32 + lane] = pml[(long long)p * nKv * ROWS];
        __syncthreads();
        float M = -INFINITY;
        for (int p = 0; p < it.parts; p++) M = fmaxf(M, ml[p * 32 + lane].x);
        const float off = M == -INFINITY ? 0.0f : M;
        float l = 0.0f, o[CW];
#pragma unroll
        for (int c = 0; c < CW; c++) o[c] = 0.0f;
        for (int p0 = 0; p0 < it.parts; p0 += 8) {
            uint32_t v[8][CW / 2];
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int c = 0; c < CW / 2; c++)
                    if (p0 + k < it.parts) v[k][c] = po[((long long)(p0 + k) * nKv * HD / 2 + c) * ROWS];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                if (p0 + k >= it.parts) break;
                const float2 x = ml[(p0 + k) * 32 + lane];
                const int lu = __float_as_int(x.y), u = lu & 255;
                const float e = __int_as_float(lu & ~255) * exp2f(x.x - off), eu = u ? e * pow2(u - BIAS) : e;
                l += e;
#pragma unroll
                for (int c = 0; c < CW / 2; c++) {
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[k][c]));
                    o[2 * c] = fmaf(f.x, eu, o[2 * c]);
                    o[2 * c + 1] = fmaf(f.y, eu, o[2 * c + 1]);
                }
            }
        }
        if (qi >= it.nq) continue;
        const float r = l > 0.0f || l != l ? 1.0f / l : 0.0f;
        uint32_t w[CW / 2];
#pragma unroll
        for (int c = 0; c < CW / 2; c++) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(o[2 * c] * r, o[2 * c + 1] * r);
            w[c] = *reinterpret_cast<const uint32_t*>(&v);
        }
        __nv_bfloat16* dst = a.out + ((long long)(it.row0 + qi) * a.nHq + h * GRP + row % GRP) * HD + c0;
        if constexpr (CW == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
    }
}

// device workspace: head, parts, items, PML, PO
struct PrefillWs {
    int items, parts, slots;
    size_t o_parts, o_items, o_pml, o_po, bytes;
};
PrefillWs prefill_ws(const tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, int64_t T)
{
    const int64_t qb = ROWS / (nHq / kv->nKv), extra = ctx->num_sms / kv->nKv + 2;
    PrefillWs w{};
    // each sequence with rows has at most one item that is not full; an item of n tiles has at most
    // 1 + n / share parts, and all n / share add up to at most SMs / heads
    w.items = (int)(T / qb + std::min<int64_t>(kv->batch, T));
    w.parts = (int)(w.items + extra);
    w.slots = (int)(2 * extra);
    auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
    w.o_parts = 256;
    w.o_items = w.o_parts + up((size_t)w.parts * sizeof(Part));
    w.o_pml = w.o_items + up((size_t)w.items * sizeof(Item));
    w.o_po = w.o_pml + up((size_t)w.slots * kv->nKv * ROWS * sizeof(float2));
    w.bytes = w.o_po + up((size_t)w.slots * kv->nKv * ROWS * kv->hd * sizeof(uint16_t));
    return w;
}

template <int HD, int GRP>
int launch_prefill(tb_ctx* ctx, const PrefillArgs& a)
{
    auto kern = k_paged_prefill<HD, GRP>;
    constexpr int smem = PrefillLayout<HD>::BYTES;
    static bool attr_set[64] = {};   // per device and instantiation; setting it twice is harmless
    cudaError_t e = cudaSuccess;
    if (ctx->device >= 64 || !attr_set[ctx->device]) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess && ctx->device < 64) attr_set[ctx->device] = true;
    }
    if (e == cudaSuccess) e = tb_launch(ctx, k_prefill_plan, dim3(1), dim3(PT), 0, a);
    const int grid = (int)std::min<long long>(a.sms, (long long)a.max_parts * a.kv.nKv);
    if (e == cudaSuccess) e = tb_launch(ctx, kern, dim3(grid), dim3(THREADS), (size_t)smem, a);
    if (e == cudaSuccess) e = tb_launch(ctx, k_prefill_join<HD, GRP>, dim3(std::min(a.max_items, a.max_slots), a.kv.nKv, ROWS / 32),
                                           dim3(JT), (size_t)(a.max_slots / 2) * 32 * sizeof(float2), a);
    if (e != cudaSuccess) return tb_fail(ctx, TB_ERR_CUDA, "attn_prefill_paged launch: %s", cudaGetErrorString(e));
    return TB_OK;
}

int prefill_check(tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, int64_t T)
{
    int rc = paged_check(ctx, kv);
    if (!rc) rc = paged_check_heads(ctx, kv, nHq);
    if (rc) return rc;
    TB_REQUIRE(ctx, T >= 0 && T < (1LL << 24), "row count must be below 2^24 (got %lld)", (long long)T);
    TB_REQUIRE(ctx, kv->batch <= MAX_BATCH, "at most %d sequences a prefill (got %lld)", MAX_BATCH, (long long)kv->batch);
    return TB_OK;
}

}  // namespace

extern "C" {

TB_API int tb_attn_prefill_paged_ws(tb_ctx* ctx, const tb_paged_kv* kv, int64_t nHq, int64_t T, size_t* bytes)
{
    if (!ctx || !bytes) return TB_ERR_INVALID;
    const int rc = prefill_check(ctx, kv, nHq, T);
    if (rc) return rc;
    *bytes = T ? prefill_ws(ctx, kv, nHq, T).bytes : 0;
    return TB_OK;
}

TB_API int tb_attn_prefill_paged_q8(tb_ctx* ctx, const tb_paged_kv* kv, uint16_t* out_bf16, const float* q,
                                    const int32_t* cu, const int32_t* lens, int64_t nHq, int64_t T, int64_t window,
                                    int64_t sinks, void* ws, size_t ws_bytes)
{
    if (!ctx) return TB_ERR_INVALID;
    const int rc = prefill_check(ctx, kv, nHq, T);
    if (rc) return rc;
    TB_REQUIRE(ctx, window >= 0 && sinks >= 0, "window and sinks must not be negative");
    if (T == 0) return TB_OK;
    TB_REQUIRE(ctx, out_bf16 && q && cu && lens, "null pointer");
    TB_REQUIRE(ctx, TB_ALIGNED(out_bf16, 16) && TB_ALIGNED(q, 16), "q and out must be 16-byte aligned");
    DeviceGuard dev(ctx->device);
    const PrefillWs w = prefill_ws(ctx, kv, nHq, T);
    if (!ws) {
        ws = tb_ctx_scratch(ctx, w.bytes);
        if (!ws) return TB_ERR_NOMEM;
    } else {
        TB_REQUIRE(ctx, TB_ALIGNED(ws, 256) && ws_bytes >= w.bytes, "workspace: %zu bytes, 256-byte aligned, are needed",
                   w.bytes);
    }
    char* p = static_cast<char*>(ws);
    PrefillArgs a{};
    a.kv = paged_args(ctx, kv);
    a.q = q;
    a.out = reinterpret_cast<__nv_bfloat16*>(out_bf16);
    a.cu = cu;
    a.lens = lens;
    a.head = reinterpret_cast<int*>(p);
    a.parts = reinterpret_cast<Part*>(p + w.o_parts);
    a.items = reinterpret_cast<Item*>(p + w.o_items);
    a.PML = reinterpret_cast<float2*>(p + w.o_pml);
    a.PO = reinterpret_cast<uint32_t*>(p + w.o_po);
    a.T = (int)T;
    a.nHq = (int)nHq;
    a.grp = (int)(nHq / kv->nKv);
    const int64_t cap = kv->max_pages * kv->page_rows;
    a.window = window < cap ? (int)window : 0;             // a window of every row is none
    a.sinks = (int)std::min<int64_t>(sinks, cap);
    a.sms = ctx->num_sms;
    a.max_items = w.items;
    a.max_parts = w.parts;
    a.max_slots = w.slots;
    a.sl2 = 1.4426950408889634f / sqrtf((float)kv->hd);
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
