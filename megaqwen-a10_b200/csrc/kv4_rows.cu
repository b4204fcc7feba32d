// kv4_rows.cu -- attention of many query rows over the 4-bit KV cache (layout: kv4.cuh, work: kv4_plan.cuh): chunks of
// tokens, where the products and no longer the bytes bound it.
//
// An item has 128 query rows, the rows of tcgen05.mma (kind::f16, fp32 sums in TMEM).  For a tile of 64 positions the
// CTA brings K and V codes into shared memory, turns them into fp16 operands once for all 128 rows, and runs
//   S = Q K^T (128 x 64),  P = weights of S,  O += P V (128 x D).
// A thread has one row and half of the tile's columns.  The phases follow one another; two CTAs on an SM fill each
// other's waits.  Items cut between CTAs leave partials, which a second kernel joins (a partial is 128 rows, too much
// for one CTA to join at the end).
//
// Arithmetic.  A value code * scale has 3 + 8 significant bits.  Its operand is that value with the position's largest
// scale brought to [2^12, 2^13) by a power of two, which keeps 7 times it within fp16: exact for the groups whose scale is
// at least 2^-29 of the position's largest, rounded to 2^-37 of it below that (V: in single-token attention the product
// with the weight is rounded to 2^-32 of the row's largest; K: there each group's sum is in fp32).  The powers go to the
// scores (K) and into the weights' exponents (V).  q is fp16 with the row's largest element
// at 2^13, exact for fp16 and bf16 inputs down to 2^-27 of that element.  Weights are exp2 in fp32
// against a reference per row, rounded to fp16 for the product (11 bits down to 2^-21 of the largest), summed in fp32
// unrounded.  The reference moves (and O is scaled) when a weight exceeds 2^15.
//
// Measured: 4 sequences of 1000 to 6001 positions, 64 tokens each, 16 heads over 8 of 128 dims: 40 us with the joins
// (87 TFLOP/s; the products alone would take 2 us).  A tile takes a CTA 3.2 us, most of it turning codes into operands and
// scores into weights (46 % of the issue slots with two CTAs on an SM) between barriers; the queries 4 us at the start,
// the joins 5 at the end.
#include "kv4_plan.cuh"
#include "launch_lock.h"

namespace mq {
namespace kv4 {
namespace {

constexpr int ROWS = ROWS_BLOCK, TILE = 64, NTHR = 256, STAGES = 2;
constexpr int LIFT = 12;             // log2 of what a position's largest scale is brought to: 7 * 2^(LIFT + 1) < 65504
constexpr int QUP = 13;              // log2 of what a query row's largest element is brought to
constexpr unsigned WHOLE_UNITS = 8;  // units up to which one CTA takes a whole item
constexpr int TMEM_COLS = 256, O_COL = 128;

template <int D, int GS>
struct Geo {
    static constexpr int NG = D / 32, NS = D / GS;     // 32-dim blocks, scales of a row
    static constexpr int Q = ROWS * D * 2, K = TILE * D * 2, V = D * 128, PT = ROWS * 128;
    static constexpr int KC = TILE * D / 2;                            // codes
    static constexpr int SC = TILE * NS * 2;
    static constexpr int RAW = 2 * (KC + SC);                          // K codes, V codes, K scales, V scales
    static constexpr int TABLE = 3 * TILE * 4 + NS * TILE * 2;         // factors and fp16 V scales of a tile
    static constexpr int FIXED = Q + K + V + PT + STAGES * RAW + TABLE + ROWS * 8 + 2 * ROWS * 4 + TILE * 4;
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// Shared-memory matrix descriptor: K-major rows of 128 bytes in the 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::f16: fp16 A and B (both K-major), fp32 D, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_f16(int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
}
__device__ __forceinline__ void umma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 32 lanes x 32 consecutive fp32 columns of this warp's lane quadrant.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]),
          "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]),
          "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]),
          "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};\n\t"
        "tcgen05.wait::st.sync.aligned;" ::"f"(v[0]),
        "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]),
        "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]),
        "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]),
        "r"(taddr)
        : "memory");
}

// Joining: [items] first CTA and number of partials of an item that was cut, 0 partials where it was not.
struct RowsParams {
    AttendParams a;
    int2* table;
    int ctas;
};

template <int D, int GS>
__global__ void __launch_bounds__(NTHR, ROWS_CTAS) rows_kernel(const RowsParams R) {
    using G = Geo<D, GS>;
    constexpr int NG = G::NG, NS = G::NS;
    const AttendParams& P = R.a;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[STAGES], s_done, o_done;
    __shared__ uint32_t s_tmem;
    __shared__ unsigned s_max;
    __shared__ int s_holes;                    // the last tile with a V group that is not finite
    uint8_t* s_q = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* s_k = s_q + G::Q;
    uint8_t* s_v = s_k + G::K;
    uint8_t* s_p = s_v + G::V;
    uint8_t* raw = s_p + G::PT;
    float* kf = reinterpret_cast<float*>(raw + STAGES * G::RAW);   // [TILE] 2^(e - QUP): K is 2^e times its operand
    float* ve = kf + TILE;                                          // [TILE] e: V is 2^e times its operand
    float* vi = ve + TILE;                                          // [TILE] 2^-e
    __half* v16 = reinterpret_cast<__half*>(vi + TILE);             // [NS][TILE] V scales * 2^-e
    float* s_mul = reinterpret_cast<float*>(v16 + NS * TILE);       // [ROWS]
    int* s_lim = reinterpret_cast<int*>(s_mul + ROWS);              // [ROWS] positions that the row sees
    float* s_red = reinterpret_cast<float*>(s_lim + ROWS);          // [2][ROWS]
    unsigned* s_nan = reinterpret_cast<unsigned*>(s_red + 2 * ROWS); // [TILE] the position's V groups that are not finite
    unsigned* s_prefix = s_nan + TILE;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = tid & (ROWS - 1), half = tid >> 7;              // this thread's row and half of the columns

    if (tid == 0) {
        for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
        mbar_init(&s_done, 1);
        mbar_init(&o_done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Only now that this CTA has its TMEM: a later kernel of the stream that allocates some could otherwise take what a
    // CTA of this one still has to get, and wait for that CTA.
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0) {
        const unsigned most = scan_costs(P, s_prefix, lane);
        if (lane == 0) s_max = most;
    }
    __syncthreads();
    const uint32_t tmem = s_tmem, lanes = (uint32_t)(32 * (warp & 3)) << 16;
    Plan<1> plan{s_prefix, P.c.heads * P.blocks, P.blocks, 0, 0};
    const int per = plan.per, B = P.c.batch;
    const unsigned total = s_prefix[B] * (unsigned)per, items = (unsigned)B * (unsigned)per;
    const bool whole = s_max <= WHOLE_UNITS + OVER && items <= gridDim.x;
    unsigned Q = 1, f0, f1;
    if (whole) {
        f0 = f1 = 0;
        if (blockIdx.x < items) {
            const int b = (int)blockIdx.x / per, hr = (int)blockIdx.x % per;
            f0 = s_prefix[b] * (unsigned)per + (unsigned)hr * (unsigned)plan.cost(b);
            f1 = f0 + (unsigned)plan.cost(b);
        }
    } else {
        Q = max((total + gridDim.x - 1) / gridDim.x, (unsigned)(4 + OVER));
        f0 = min(total, blockIdx.x * Q);
        f1 = min(total, f0 + Q);
    }
    plan.f_end = f1;
    Segment cur;
    bool more = f0 < f1;
    if (more) plan.seek(cur, f0, B);
    while (more && cur.seg0 == cur.seg1) more = plan.next(cur);

    int nload = 0, nuse = 0, ns = 0, no = 0;   // tiles asked for and used, products of either kind waited for
    bool dead = false;                         // a wait ran out: the status says so, nothing more is issued
    // Bounded wait of every thread; false when it runs out.
    auto wait = [&](uint64_t* bar, int phase) {
        if (mbar_test(bar, phase & 1)) return true;
        const unsigned long long t0 = globaltimer();
        while (!mbar_test(bar, phase & 1))
            if (globaltimer() - t0 > WAIT_NS) {
                report(P.c, MQ_DEV_TIMEOUT_RING, blockIdx.x);
                return false;
            }
        return true;
    };
    // The last warp: the copies of positions [p0, p0 + 64) that lie before `end`, cut at the pages' ends; lane
    // 4 i + a has array a (K codes, V codes, K scales, V scales) of piece i.
    const int shift = P.c.page_shift, array = lane & 3;
    const uint8_t* src = array & 2 ? reinterpret_cast<const uint8_t*>(P.c.scales[array & 1]) : P.c.codes[array & 1];
    const int row_bytes = array & 2 ? NS * 2 : D / 2;
    const int dst = array & 2 ? 2 * G::KC + (array & 1) * G::SC : (array & 1) * G::KC;
    auto load = [&](int b, int h, int len, int p0, int end) {
        uint8_t* base = raw + (nload % STAGES) * G::RAW;
        uint64_t* bar = &full[nload % STAGES];
        ++nload;
        if (warp != NTHR / 32 - 1) return;
        const int n = max(0, min(TILE, min(end, len) - p0) + 7) / 8 * 8;      // whole 16-byte vectors of scales
        if (lane == 0) mbar_arrive_expect_tx(bar, (unsigned)(n * (G::RAW / TILE)));
        __syncwarp();
        const int page = (p0 >> shift) + (lane >> 2), from = max(p0, page << shift), to = min(p0 + n, (page + 1) << shift);
        if (from < to) {
            long long r = row_of(P.c, b, from, h);
            if (r < 0) r = 0;                  // no such page: reported, and read from page 0
            bulk_g2s(base + dst + (from - p0) * row_bytes, src + r * row_bytes, (to - from) * row_bytes, bar);
        }
    };
    auto open = [&](const Segment& c) {
        const int len = positions_of(P, c.b);
        for (int i = 0; i < STAGES && c.seg0 + 2 * i < c.seg1; ++i) load(c.b, c.h, len, (c.seg0 + 2 * i) * TP, c.seg1 * TP);
    };
    if (more) open(cur);

    while (more && !dead) {
        const Segment seg = cur;
        const int b = seg.b, h = seg.h, row0 = seg.rb * ROWS, nrows = min(ROWS, P.rows - row0), len = positions_of(P, b);
        const int count = P.counts ? min(max(P.counts[b], 0), P.tokens) : P.tokens;
        const int end = min(len, seg.seg1 * TP);         // of this segment's positions
        // ------------------------------------------------------------------ queries: 16 rows to a warp, 8 lanes to a row
        {
            constexpr int NCH = D / 64;                          // pieces of 8 dims of a lane
            const int l8 = lane & 7;
            const bool vec = ((reinterpret_cast<uintptr_t>(P.q) | (uintptr_t)(P.qb * 2) | (uintptr_t)(P.qt * 2) | (uintptr_t)(P.qh * 2)) & 15u) == 0;
            uint4 x[4][NCH];
            int t[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = warp * 16 + 4 * i + (lane >> 3);
                const bool real = r < nrows;
                t[i] = real ? (row0 + r) / P.share : 0;
                const int j = real ? row0 + r - t[i] * P.share : 0;
                const uint16_t* src = reinterpret_cast<const uint16_t*>(P.q) + (long long)b * P.qb + (long long)t[i] * P.qt +
                                      (long long)(h * P.share + j) * P.qh + 8 * NCH * l8;
                if (!real) t[i] = count;                         // no token
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    x[i][c] = make_uint4(0, 0, 0, 0);
                    if (real && vec) x[i][c] = *(reinterpret_cast<const uint4*>(src) + c);
                    if (real && !vec) {
                        const uint16_t* p = src + 8 * c;
                        x[i][c] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = warp * 16 + 4 * i + (lane >> 3);
                unsigned big = 0;
#pragma unroll
                for (int c = 0; c < NCH; ++c)
                    big = __vmaxu2(big, __vmaxu2(__vmaxu2(x[i][c].x & 0x7fff7fffu, x[i][c].y & 0x7fff7fffu),
                                                 __vmaxu2(x[i][c].z & 0x7fff7fffu, x[i][c].w & 0x7fff7fffu)));
#pragma unroll
                for (int o = 1; o < 8; o <<= 1) big = __vmaxu2(big, __shfl_xor_sync(0xffffffffu, big, o));
                big = max(big & 0xffffu, big >> 16);
                const unsigned bits = __float_as_uint(P.dtype == MQ_BF16 ? bf16_bits_to_f32(big) : __half2float(__ushort_as_half((unsigned short)big)));
                const int ex = min(max((int)(bits >> 23), QUP), 253);
                const float down = __uint_as_float((unsigned)(254 - ex + QUP) << 23) * (P.scale_log2 < 0.f ? -1.f : 1.f);
#pragma unroll
                for (int c = 0; c < NCH; ++c) {
                    const uint32_t w[4] = {x[i][c].x, x[i][c].y, x[i][c].z, x[i][c].w};
                    float f[8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        if (P.dtype == MQ_BF16) {
                            f[2 * k] = __uint_as_float(w[k] << 16);
                            f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
                        } else {
                            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
                            f[2 * k] = v.x; f[2 * k + 1] = v.y;
                        }
                    }
                    // pairs (0,4), (1,5), (2,6), (3,7), as the codes come out of their words
                    const int chunk = l8 * NCH + c;
                    *reinterpret_cast<uint4*>(s_q + (chunk >> 3) * (ROWS * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4)) =
                        make_uint4(pack_f16(f[0] * down, f[4] * down), pack_f16(f[1] * down, f[5] * down), pack_f16(f[2] * down, f[6] * down),
                                   pack_f16(f[3] * down, f[7] * down));
                }
                if (l8 == 0) {
                    s_mul[r] = __uint_as_float((unsigned)ex << 23) * fabsf(P.scale_log2);
                    // rows that are padding see everything and are written as zeros
                    s_lim[r] = t[i] < count ? max(0, len - count + t[i] + 1) : 0x7fffffff;
                }
            }
        }
        if (tid == 0) s_holes = -1;
        __syncthreads();
        int low = 0x7fffffff, high = 0;       // least and greatest limit of the rows
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int l = s_lim[lane + 32 * i];
            low = min(low, l);
            high = max(high, l == 0x7fffffff ? 0 : l);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        const float mul = s_mul[row];
        const int limit = min(s_lim[row], end);
        float ref = NEG_INF, sum = 0.f;
        bool any = false;                      // a product has gone into O
        unsigned spoilt = 0;                   // groups of the output that are NaN

        // ------------------------------------------------------------------ tiles
        for (int u = seg.seg0; u < seg.seg1; u += 2) {
            const int p0 = u * TP;
            uint8_t* base = raw + (nuse % STAGES) * G::RAW;
            bool ok = wait(&full[nuse % STAGES], nuse / STAGES);
            if (p0 < high) {
                // Scales: the position's power of two apart, the quotients are the operands'.  What lies beyond the sequence
                // may hold anything and counts as zero.
                auto scales = [&](int v, int p, float (&w)[NS], unsigned& nan) {
                    const uint16_t* sc = reinterpret_cast<const uint16_t*>(base + 2 * G::KC + v * G::SC) + p * NS;
                    unsigned e = 0, x[NS];
                    nan = 0;
#pragma unroll
                    for (int i = 0; i < NS; ++i) {
                        x[i] = p0 + p < end ? sc[i] : 0u;
                        if (x[i] < 0x7f80u) e = max(e, x[i]);
                        else nan |= 1u << i;
                    }
                    const int ex = min(max((int)(e >> 7), 67) - 127, 126) - LIFT;
                    const float down = __uint_as_float((unsigned)(127 - ex) << 23);
#pragma unroll
                    for (int i = 0; i < NS; ++i) w[i] = __uint_as_float(x[i] << 16) * down;
                    return ex;
                };
                if (tid < TILE) {
                    // V: a group that is not finite enters as zeros, as the product would carry a NaN into rows that do not
                    // see it, and is noted
                    float w[NS];
                    unsigned nan;
                    const int ex = scales(1, tid, w, nan);
#pragma unroll
                    for (int i = 0; i < NS; ++i) v16[i * TILE + tid] = __float2half_rn(nan >> i & 1u ? 0.f : w[i]);
                    ve[tid] = (float)ex;
                    vi[tid] = __uint_as_float((unsigned)(127 - ex) << 23);
                    s_nan[tid] = nan;
                    if (nan) s_holes = u;
                }
                // K operand: thread (position, block of 32 dims); D = 64 has work for half of the threads
                for (int i = tid; i < TILE * NG; i += NTHR) {
                    const int p = i / NG, g = i % NG;
                    float sc[NS];
                    unsigned nan;
                    const int ex = scales(0, p, sc, nan);
                    if (g == 0) kf[p] = __uint_as_float((unsigned)(127 + ex - QUP) << 23);
                    float mine = sc[0];
#pragma unroll
                    for (int k = 1; k < NS; ++k)
                        if (g * 32 / GS == k) mine = sc[k];
                    const __half2 s2 = __float2half2_rn(mine);
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t w[4];
                        codes_to_f16(*reinterpret_cast<const uint32_t*>(base + p * (D / 2) + c * (4 * NG) + g * 4), w);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&w[k]), s2);
                            w[k] = *reinterpret_cast<const uint32_t*>(&x);
                        }
                        const int chunk = g * 4 + c;
                        *reinterpret_cast<uint4*>(s_k + (chunk >> 3) * (TILE * 128) + p * 128 + (((chunk & 7) ^ (p & 7)) << 4)) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                fence_async();
                dead = __syncthreads_or(!ok) != 0;
                if (dead) break;
                if (s_holes == u)
                    for (int p = 0; p < TILE && p0 + p < limit; ++p) spoilt |= s_nan[p];
                if (tid == 0) {
                    tc_fence_after();
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        umma_f16(tmem, sdesc_sw128(smem_u32(s_q + (k >> 2) * (ROWS * 128))) + 2 * (k & 3),
                                 sdesc_sw128(smem_u32(s_k + (k >> 2) * (TILE * 128))) + 2 * (k & 3), idesc_f16(TILE), k > 0);
                    umma_commit(&s_done);
                }
                // V operand while S is summed: dims as rows, dim 32 g + 4 r + j in row 64 (g / 2) + 16 j + 8 (g % 2) + r (D = 64:
                // 32 g + 8 j + r), which keeps a warp's 32 rows in different banks; thread (lane r of the code order, block
                // of 32 dims, 8 positions)
                if (any) ok = wait(&o_done, no - 1);               // P, V and O are free again
                for (int i = tid; i < 64 * NG; i += NTHR) {
                    const int r = i & 7, g = (i >> 3) % NG, c = (i >> 3) / NG;
                    const uint8_t* src = base + G::KC + 8 * c * (D / 2) + r * (2 * NG) + g * 2;
                    const uint4 sc = *reinterpret_cast<const uint4*>(v16 + g * 32 / GS * TILE + 8 * c);
                    const uint32_t s2[4] = {sc.x, sc.y, sc.z, sc.w};
                    uint32_t o[4][4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t two = *reinterpret_cast<const uint16_t*>(src + 2 * k * (D / 2)) |
                                             (uint32_t)*reinterpret_cast<const uint16_t*>(src + (2 * k + 1) * (D / 2)) << 16;
                        uint32_t w[4];
                        codes_to_f16(two, w);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const __half2 x = __hmul2(*reinterpret_cast<__half2*>(&w[j]), *reinterpret_cast<const __half2*>(&s2[k]));
                            o[j][k] = *reinterpret_cast<const uint32_t*>(&x);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int n = NG == 4 ? 64 * (g >> 1) + 16 * j + 8 * (g & 1) + r : 32 * g + 8 * j + r;
                        *reinterpret_cast<uint4*>(s_v + n * 128 + ((c ^ r) << 4)) = make_uint4(o[j][0], o[j][1], o[j][2], o[j][3]);
                    }
                }
            } else {
                dead = __syncthreads_or(!ok) != 0;
                if (dead) break;
            }
            ++nuse;
            if (p0 >= high) {          // every thread has read the stage
                if (u + 2 * STAGES < seg.seg1) load(b, h, len, (u + 2 * STAGES) * TP, seg.seg1 * TP);
                continue;
            }

            ok = wait(&s_done, ns++) && ok;
            __syncwarp();                              // the waits of a warp's lanes end one by one; the loads take the whole warp
            tc_fence_after();
            float s[32];
            tmem_ld32(tmem + lanes + 32 * half, s);
            float m = NEG_INF;
            const bool edge = p0 + TILE > low || p0 + TILE > end;
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                const float4 k4 = *reinterpret_cast<const float4*>(kf + 32 * half + c);
                const float4 v4 = *reinterpret_cast<const float4*>(ve + 32 * half + c);
                s[c] = fmaf(s[c] * k4.x, mul, v4.x);
                s[c + 1] = fmaf(s[c + 1] * k4.y, mul, v4.y);
                s[c + 2] = fmaf(s[c + 2] * k4.z, mul, v4.z);
                s[c + 3] = fmaf(s[c + 3] * k4.w, mul, v4.w);
            }
            if (edge)
#pragma unroll
                for (int c = 0; c < 32; ++c)
                    if (p0 + 32 * half + c >= limit) s[c] = NEG_INF;
#pragma unroll
            for (int c = 0; c < 32; ++c) m = fmaxf(m, s[c]);
            s_red[half * ROWS + row] = m;
            named_bar(1 + (warp & 3), 64);             // the two warps of the row
            m = fmaxf(m, s_red[(half ^ 1) * ROWS + row]);
            const bool raise = m > ref + (BELOW + RAISE) || (ref == NEG_INF && m > NEG_INF);
            if (__any_sync(0xffffffffu, raise)) {      // the same in both warps of the row
                const float k = raise && ref != NEG_INF ? exp2_fast(ref - (m - BELOW)) : 1.f;
                if (raise) ref = m - BELOW;
                sum *= k;
                if (any)
#pragma unroll 1
                    for (int c = 0; c < D / 2; c += 32) {
                        float o[32];
                        const uint32_t at = tmem + lanes + O_COL + half * (D / 2) + c;
                        tmem_ld32(at, o);
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] *= k;
                        tmem_st32(at, o);
                    }
            }
            const float r = ref == NEG_INF ? 0.f : ref;
#pragma unroll
            for (int c = 0; c < 32; c += 8) {
                float w[8];
                const float4 a = *reinterpret_cast<const float4*>(vi + 32 * half + c), z = *reinterpret_cast<const float4*>(vi + 32 * half + c + 4);
                const float inv[8] = {a.x, a.y, a.z, a.w, z.x, z.y, z.z, z.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w[i] = exp2_fast(s[c + i] - r);
                    sum = fmaf(w[i], inv[i], sum);
                }
                *reinterpret_cast<uint4*>(s_p + row * 128 + (((4 * half + c / 8) ^ (row & 7)) << 4)) =
                    make_uint4(pack_f16(w[0], w[1]), pack_f16(w[2], w[3]), pack_f16(w[4], w[5]), pack_f16(w[6], w[7]));
            }
            tc_fence_before();
            fence_async();
            dead = __syncthreads_or(!ok) != 0;
            if (dead) break;
            if (tid == 0) {
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < TILE / 16; ++k)
                    umma_f16(tmem + O_COL, sdesc_sw128(smem_u32(s_p)) + 2 * k, sdesc_sw128(smem_u32(s_v)) + 2 * k, idesc_f16(D), any || k > 0);
                umma_commit(&o_done);
            }
            ++no;
            any = true;
            if (u + 2 * STAGES < seg.seg1) load(b, h, len, (u + 2 * STAGES) * TP, seg.seg1 * TP);   // the stage has been read
        }
        if (dead) break;
        do more = plan.next(cur);
        while (more && cur.seg0 == cur.seg1);
        if (more) open(cur);

        // ------------------------------------------------------------------ the segment's sums
        bool ok = !any || wait(&o_done, no - 1);
        s_red[half * ROWS + row] = sum;
        tc_fence_after();
        dead = __syncthreads_or(!ok) != 0;
        if (dead) break;
        const float L = sum + s_red[(half ^ 1) * ROWS + row];
        const int n = plan.units(b);
        const bool all = seg.seg0 == 0 && seg.seg1 == n;
        const size_t pstride = part_floats(ROWS, D);
        float* part = P.part + (2 * (size_t)blockIdx.x + (seg.seg0 == 0 ? 1 : 0)) * pstride;
        if (seg.seg0 == 0 && tid == 0) {
            const int c0 = (int)((seg.item_f + OVER) / Q), c1 = (int)((seg.item_f + OVER + (unsigned)n - 1) / Q);
            R.table[(unsigned)b * (unsigned)per + (unsigned)(seg.h * P.blocks + seg.rb)] = make_int2(c0, all ? 0 : c1 - c0 + 1);
        }
        if (!all && half == 0) *reinterpret_cast<float2*>(part + ROWS * D + 2 * row) = make_float2(ref, L);
        // this thread's columns are the dims from half * D / 2 on, in the V operand's order
#pragma unroll 1
        for (int e = 0; e < D / 64; ++e) {         // blocks of 32 dims
            float o[32];                           // [j][r]
            __syncwarp();                          // rows that do not exist skipped the stores
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float x[8];
                tmem_ld8(tmem + lanes + O_COL + half * (D / 2) + (NG == 4 ? 16 * j + 8 * e : 8 * j), x);
#pragma unroll
                for (int i = 0; i < 8; ++i) o[8 * j + i] = x[i];
            }
            const int d = half * (D / 2) + 32 * e;
            if (!any)
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.f;
            if (spoilt >> (d / GS) & 1u)
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = NAN;
            if (row < nrows) {
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    const float4 v = make_float4(o[r], o[8 + r], o[16 + r], o[24 + r]);
                    if (all) store_out(P, b, h, row0 + row, D, d + 4 * r, v, L);
                    else reinterpret_cast<float4*>(part)[(d / 4 + r) * ROWS + row] = v;
                }
            }
        }
        tc_fence_before();
        __syncthreads();     // O, the queries and the sums' exchange are free
        tc_fence_after();
    }
    // After a wait that ran out, copies and products may still be in flight: wait for them, with the same limit.
    if (dead && tid == 0) {
        for (int i = nuse; i < nload; ++i) wait(&full[i % STAGES], i / STAGES);
        wait(&s_done, ns);
        wait(&o_done, no);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

// Joins the partials of cut items ([4 dims][row] vectors, so that a warp's rows are neighbours): a lane has a row, a
// warp four dims of 32 rows.
template <int D>
__global__ void __launch_bounds__(256) join_kernel(const RowsParams R) {
    const AttendParams& P = R.a;
    pdl_launch_dependents();
    pdl_wait();
    constexpr int BLOCKS = D / 4 * (ROWS / 32) / 8;      // of an item, 8 warps each
    const unsigned item = blockIdx.x / BLOCKS;
    const int w = blockIdx.x % BLOCKS * 8 + (threadIdx.x >> 5), d4 = w / (ROWS / 32), row = w % (ROWS / 32) * 32 + (threadIdx.x & 31);
    const int2 cut = R.table[item];
    const int per = P.c.heads * P.blocks, b = item / per, hr = item % per, h = hr / P.blocks, row0 = (hr - h * P.blocks) * ROWS;
    // (bounds: the table is not written where a wait ran out)
    if (cut.y <= 0 || cut.x < 0 || cut.x + cut.y > R.ctas || row0 + row >= P.rows) return;
    const size_t pstride = part_floats(ROWS, D);
    float M = NEG_INF, L = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < cut.y; p += 4) {
        float2 ml[4];
        float4 a[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            ml[k] = make_float2(NEG_INF, 0.f);
            a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (p + k < cut.y) {
                const float* x = P.part + (2 * (size_t)(cut.x + p + k) + (p + k == 0 ? 1 : 0)) * pstride;
                ml[k] = *reinterpret_cast<const float2*>(x + ROWS * D + 2 * row);
                a[k] = reinterpret_cast<const float4*>(x)[d4 * ROWS + row];
            }
        }
        float m = M;
#pragma unroll
        for (int k = 0; k < 4; ++k) m = fmaxf(m, ml[k].x);
        const float was = L == 0.f ? 0.f : exp2_fast(M - m);
        M = m;
        L *= was;
        scale4(o, was);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float f = ml[k].y == 0.f ? 0.f : exp2_fast(ml[k].x - m);
            L = fmaf(ml[k].y, f, L);
            add4(o, a[k], f);
        }
    }
    store_out(P, b, h, row0 + row, D, 4 * d4, o, L);
}

constexpr int MAX_DEV = 64;

template <class Kern, class... Args>
int launch_pdl(Kern kern, unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, const Args&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, kern, args...);
}

template <int D, int GS>
int launch(const RowsParams& p, unsigned grid, cudaStream_t stream) {
    static bool set[MAX_DEV];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= MAX_DEV) return MQ_ERR_DEVICE;
    const size_t fixed = 1024 + Geo<D, GS>::FIXED;
    if (!set[dev]) {
        if ((e = cudaFuncSetAttribute(rows_kernel<D, GS>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(fixed + (MAX_BATCH + 1) * 4))) != cudaSuccess)
            return (int)e;
        set[dev] = true;
    }
    const LaunchLock lock(p.a.part);   // the join reads what this call's first kernel left
    const int rc = launch_pdl(rows_kernel<D, GS>, grid, NTHR, fixed + ((size_t)p.a.c.batch + 1) * 4, stream, p);
    if (rc != MQ_OK) return rc;
    const unsigned items = (unsigned)p.a.c.batch * p.a.c.heads * p.a.blocks;
    return launch_pdl(join_kernel<D>, items * (D / 4 * (ROWS / 32) / 8), 256, 0, stream, p);
}

}  // namespace

size_t rows_workspace(int D, unsigned grid, size_t items) {
    return 2 * (size_t)grid * part_floats(ROWS, D) * sizeof(float) + items * sizeof(int2);
}
int rows_attend(const AttendParams& a, int D, int GS, unsigned grid, cudaStream_t stream) {
    RowsParams p{a, reinterpret_cast<int2*>(a.part + 2 * (size_t)grid * part_floats(ROWS, D)), (int)grid};
    if (D == 128) return GS == 32 ? launch<128, 32>(p, grid, stream) : GS == 64 ? launch<128, 64>(p, grid, stream) : launch<128, 128>(p, grid, stream);
    return GS == 32 ? launch<64, 32>(p, grid, stream) : launch<64, 64>(p, grid, stream);
}

}  // namespace kv4
}  // namespace mq
