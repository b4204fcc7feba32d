// kv4_attend.cu -- attention over the 4-bit KV cache (layout: kv4.cuh), single tokens and chunks of tokens.
//
//   out[r] = sum_p w[r,p] v[p] / sum_p w[r,p],   w[r,p] = exp(scale q[r].k[p]),   p <= position of row r
//
// A row is a (token, query head); the rows of one KV head share its K and V.  Work is cut into items
// (sequence, KV head, block of 8 NB rows) of units of 32 positions; the items' units, laid end to end, are
// cut into equal ranges, one for each CTA, so that sequences of any mix of lengths load the SMs evenly.
// Within a CTA the part of an item in its range (a segment) is cut into one run of units for each warp; every
// warp streams its own tiles of 32 positions (K codes, K scales, V codes, V scales) through its own ring of
// bulk copies, which runs on across segments.  The warps of a segment meet in shared memory; an item that
// spans CTAs leaves partials in the workspace and the last of its CTAs to arrive joins them.
//
// Arithmetic.  Scores: S^T = K q^T by m16n8k16 fp16 products with fp32 sums; 16 positions are the rows of A,
// 8 query rows the columns (an A with the queries as rows would be half empty for up to 8 of them).  A K code
// enters as the fp16 subnormal nibble * 2^-24, which a mask alone makes (16 nibble * 2^-24 for every other one,
// against q / 16); the 8 that a code is above its value is taken off each group's fp32 sum as 8 sum q.  That leaves an
// error of about 2^-22 of 8 max|q| s, too much where a few elements of q are far above the others (more than half of
// them 2^-6 below the largest) and K is small in their dims.  The tiles of such a row block, and those at the end of what
// a row sees, take the codes as signed numbers instead (32 half2 sums more for 16 positions).  q enters as fp16 of
// q 2^(12-e), e the exponent of the row's largest element (exact for fp16 inputs down to 2^-22 and for bf16 inputs down
// to 2^-25 of that element, the dims that meet 16 nibble being 2^-4 smaller); the group's scale multiplies the group's
// sum.  Weights: exp2 in fp32 against a running reference per row.  Values: O^T = V^T (w s)^T; an 8 x 8 transpose within
// the warp brings the weights into place.  The product of weight and V scale is rounded once to fp16 (11 bits; bf16 would
// lose 3 more).  The reference follows the greatest (score + exponent of the position's largest V scale), so the products
// stay small and are rounded relative to the largest contribution, whatever the scales are (11 bits down to 2^-21 of it,
// 2^-32 of it below that, in the dims of a group whose scales are that far below the others' too).  V codes enter as
// nibble - 8 exactly (their offset, taken off a sum, would leave its rounding where a dim's large weights have code 0).  Sums of
// weights are fp32 and unrounded.  The reference moves only when a product exceeds 2^15 (a vote), so most tiles need no
// reduction across lanes.
//
// Where rows * groups <= 8, the groups of 32 to 128 dims have score columns of their own: q is zero in the other
// groups' columns, so one chain of products gives every group's sum, and a lane applies the scales of its own
// group only (2 rows, 4 groups: 641 warp instructions for a tile of 32 positions, 737 without).
//
// A segment's fixed costs are latency, and much of that is fetching instructions that run once, so the code around
// the tiles is written small: queries go through shared memory, joins take one output each.
//
// Measured, 16 heads over 8 of 128 dims, group 32: 64 sequences of 128 to 4096 (156 MB of codes and scales) 52 us,
// 3.0 TB/s -- 2.1 us of it the whole cache's products, the rest instructions (53 % of the issue slots; half of them run
// at half rate), about 6 us before the first tile and the spread of the CTAs' ends; one sequence of 32768 22.5 us, of which
// 7 are tiles; one of 200 7 us, which is latency.  Queries that ask for signed codes: 64 sequences 65 us.
#include <type_traits>
#include "kv4_plan.cuh"

namespace mq {
namespace kv4 {
namespace {

constexpr unsigned WHOLE_TILES = 2;   // tiles of a warp up to which one CTA takes a whole item
constexpr int NST = 2;               // ring stages of a warp
constexpr int QUP = 12;              // log2 of what a query row's largest element is brought to
constexpr float MOST = 32768.f;      // 2^(BELOW + RAISE): how large a product of weight and V scale may be before the reference moves
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The N scales of a row (bf16 at p) as floats.
template <int N>
__device__ __forceinline__ void load_scales(const uint8_t* p, float (&s)[N]) {
    if constexpr (N == 1) {
        s[0] = bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(p));
    } else {
        uint32_t w[N / 2];
        if constexpr (N == 4) {
            const uint2 v = *reinterpret_cast<const uint2*>(p);
            w[0] = v.x; w[1] = v.y;
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
}
// d = A B from zero.
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
// Pairs of nibbles (times F, in the low bits of either half) -> fp16 pairs F (nibble - 8): the nibble in the mantissa of 1024.
template <int F>
__device__ __forceinline__ uint32_t signed_codes(uint32_t v) {
    const uint32_t x = v | 0x64006400u;
    const __half2 y = __hadd2(*reinterpret_cast<const __half2*>(&x), __float2half2_rn(-(1024.f + 8.f * F)));
    return *reinterpret_cast<const uint32_t*>(&y);
}
// Transposes an 8 x 8 matrix of 16-bit elements, row lane / 4, columns 2 (lane % 4) and + 1 in each lane.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
template <int D, int GS>
struct Geo {
    static constexpr int NG = D / 32, NS = D / GS;      // 32-dim blocks, scales of a row
    static constexpr int CODES = TP * D / 2, SCALES = TP * NS * 2;
    static constexpr int STAGE = 2 * (CODES + SCALES);  // K codes, V codes, K scales, V scales
    static constexpr int QROW = 2 * D + 16;             // bytes of a staged query row, skewed over the banks
};

template <int D, int GS, int NB, int NW, bool REP>
__global__ void __launch_bounds__(NW * 32, NW > 4 ? 1 : NB == 1 ? 4 : 2) attend_kernel(const AttendParams P) {
    using G = Geo<D, GS>;
    constexpr int NG = G::NG, NS = G::NS, RB = 8 * NB, NTHR = NW * 32;
    constexpr int LDA = D + 4;                       // row of a warp's accumulators in shared memory
    constexpr int QROW = G::QROW;
    constexpr int CR = REP ? 8 / NS : 8;             // score columns of a group: rows of the block, once for each group
    static_assert(!REP || NB == 1, "the groups share the eight columns");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bars[NW][NST];
    __shared__ unsigned s_max, s_last, s_was[2];
    __shared__ Segment s_pend[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int quad = lane >> 2, cq = lane & 3;       // r and c of the fragment layouts
    const int B = P.c.batch;
    uint8_t* ring = smem + warp * (NST * G::STAGE);
    const int rmax = min(P.rows, RB);                // rows of a block that exist at most
    float* s_acc = reinterpret_cast<float*>(smem + NW * NST * G::STAGE);            // [warp][rmax][LDA]
    float* s_ref = s_acc + NW * max(rmax * LDA, 192);                                // [warp][RB]; 192: the joins need 6 words a thread
    float* s_sum = s_ref + NW * RB;                                                  // [warp][RB]
    float* s_off = s_sum + NW * RB;                                                  // [RB][NS] -8 sum q of a group
    float* s_mul = s_off + RB * NS;                                                  // [RB] q's factor
    int* s_lim = reinterpret_cast<int*>(s_mul + RB);                                 // [RB] positions that the row sees
    uint8_t* s_q = reinterpret_cast<uint8_t*>(s_lim + RB);                           // [RB][QROW] q as fp16, in fragment order
    unsigned* s_prefix = reinterpret_cast<unsigned*>(s_q + RB * QROW);               // [B + 1]

    if (REP && tid < RB) s_lim[tid] = 0x7fffffff;    // rows that the groups' columns leave no room for
    if (lane == 0) {
        for (int i = 0; i < NST; ++i) mbar_init(&bars[warp][i], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0) {
        const unsigned most = scan_costs(P, s_prefix, lane);
        if (lane == 0) s_max = most;
    }
    __syncthreads();
    Plan<NW> plan{s_prefix, P.c.heads * P.blocks, P.blocks, warp, 0};
    const int per = plan.per;
    const unsigned total = s_prefix[B] * (unsigned)per, items = (unsigned)B * (unsigned)per;
    // Short contexts: one CTA for each item, no joining across CTAs.  Otherwise equal ranges.
    const bool whole = s_max <= WHOLE_TILES * NW + OVER && items <= gridDim.x;
    unsigned Q = 1, f0, f1;
    if (whole) {
        f0 = f1 = 0;
        if (blockIdx.x < items) {
            const int b = (int)blockIdx.x / per, hr = (int)blockIdx.x % per;
            f0 = s_prefix[b] * (unsigned)per + (unsigned)hr * (unsigned)plan.cost(b);
            f1 = f0 + (unsigned)plan.cost(b);
        }
    } else {
        Q = max((total + gridDim.x - 1) / gridDim.x, (unsigned)(NW + OVER));
        f0 = min(total, blockIdx.x * Q);
        f1 = min(total, f0 + Q);
    }
    plan.f_end = f1;
    if (f0 >= f1) return;

    int nuse = 0, nload = 0;          // tiles used and asked for; a tile's stage is its number modulo NST
    bool dead = false;                // a wait ran out: no further copies, the status says so
    int pages = 0, page0 = 0;         // page ids page0 .. page0 + 31 of the segment's sequence, one in each lane

    // Issues the copies of unit u of (b, h) into the next stage: lanes 0..3 have K codes, V codes, K scales, V scales.
    const uint8_t* src = lane & 2 ? reinterpret_cast<const uint8_t*>(P.c.scales[lane & 1]) : P.c.codes[lane & 1];
    const uint32_t row_bytes = lane & 2 ? NS * 2 : D / 2;
    const uint32_t dst = (lane & 2 ? 2 * G::CODES + (lane & 1) * G::SCALES : (lane & 1) * G::CODES);
    const int shift = P.c.page_shift, rows = min(TP, 1 << shift);        // of one page
    auto load = [&](int b, int h, int len, int u) {
        const int p0 = u * TP, st = nload % NST;
        ++nload;
        uint64_t* bar = &bars[warp][st];
        const int first = p0 >> shift;
        if (P.c.table && first + 1 >= page0 + 32) {
            page0 = first;
            pages = page0 + lane < P.c.pages_per_seq ? P.c.table[(long long)b * P.c.pages_per_seq + page0 + lane] : 0;
        }
        const bool second = rows < TP && p0 + rows < len;                // two pages of 16 in a tile
        if (lane == 0) mbar_arrive_expect_tx(bar, (unsigned)(p0 < len ? rows * (second ? 2 : 1) * (G::STAGE / TP) : 0));
        __syncwarp();
#pragma unroll 1
        for (int o = 0; o <= (int)second && p0 < len; ++o) {
            const int i = first + o;
            int page = P.c.table ? __shfl_sync(0xffffffffu, pages, i - page0) : b * P.c.pages_per_seq + i;
            if ((unsigned)page >= (unsigned)P.c.num_pages) {   // reported, and read from page 0
                if (lane == 0) report(P.c, MQ_DEV_BAD_PAGE, b);
                page = 0;
            }
            const long long row = (((long long)page * P.c.heads + h) << shift) + (o ? 0 : p0 & ((1 << shift) - 1));
            if (lane < 4) bulk_g2s(ring + st * G::STAGE + dst + o * 16 * row_bytes, src + row * row_bytes, rows * row_bytes, bar);
        }
    };
    // First copies of a segment.
    auto open = [&](const Segment& c) {
        if (dead || c.u >= c.u1) return;
        const int len = positions_of(P, c.b);
        if (P.c.table) {
            page0 = (c.u * TP) >> P.c.page_shift;
            pages = page0 + lane < P.c.pages_per_seq ? P.c.table[(long long)c.b * P.c.pages_per_seq + page0 + lane] : 0;
        }
        for (int i = 0; i < NST && c.u + i < c.u1; ++i) load(c.b, c.h, len, c.u + i);
    };
    // Stages a segment's query rows, a row for a warp: fp16 of q 2^(QUP - e) in the order of the fragments (block of 8 dims:
    // pairs (0,4), (1,5) / 16, (2,6), (3,7) / 16), the groups' sums, the factor that undoes it all, the row's limit.
    auto stage_q = [&](const Segment& c) {
        const int row0 = c.rb * RB, nrows = min(RB, P.rows - row0);
        const int len = positions_of(P, c.b);
        const int count = P.counts ? min(max(P.counts[c.b], 0), P.tokens) : P.tokens;
        constexpr int V = D / 32;     // dims of a lane
#pragma unroll 1
        for (int r = warp; r < (REP ? CR : RB); r += NW) {
            const int t = r < nrows ? (row0 + r) / P.share : 0;
            const bool real = r < nrows && t < count;          // else no row, or padding: zeros that nothing depends on
            const int j = real ? row0 + r - t * P.share : 0;
            const uint16_t* src = reinterpret_cast<const uint16_t*>(P.q) + (long long)c.b * P.qb + (long long)t * P.qt +
                                  (long long)(c.h * P.share + j) * P.qh + V * lane;
            uint16_t raw[V];
#pragma unroll
            for (int i = 0; i < V; ++i) raw[i] = real ? src[i] : (uint16_t)0;
            float f[V];
            unsigned big = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                f[i] = P.dtype == MQ_BF16 ? bf16_bits_to_f32(raw[i]) : __half2float(__ushort_as_half(raw[i]));
                big = max(big, __float_as_uint(f[i]) & 0x7fffffffu);
            }
            big = __reduce_max_sync(0xffffffffu, big);
            int small = 0;
#pragma unroll
            for (int i = 0; i < V; ++i) small += fabsf(f[i]) < __uint_as_float(big) * 0x1p-6f;
            const bool peaked = __reduce_add_sync(0xffffffffu, small) > D / 2;
            const int ex = min(max((int)(big >> 23), QUP), 253);
            // 2^(QUP - (ex - 127)), with the sign of the scale so that a larger sum is a larger score
            const float down = __uint_as_float((unsigned)(254 - ex + QUP) << 23) * (P.scale_log2 < 0.f ? -1.f : 1.f);
            float part = 0.f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int d = V * lane + i, k = d & 3;
                const __half x = __float2half_rn(f[i] * down * (k & 1 ? 0.0625f : 1.f));
                *reinterpret_cast<__half*>(s_q + r * QROW + (d >> 3) * 16 + k * 4 + ((d >> 2) & 1) * 2) = x;
                part = fmaf(__half2float(x), k & 1 ? 16.f : 1.f, part);
            }
#pragma unroll
            for (int o = 1; o < GS / V; o <<= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
            if (lane % (GS / V) == 0) s_off[r * NS + lane / (GS / V)] = part * (-8.f / 16777216.f);
            if (lane == 0) {
                // 2^24: codes are subnormals; the sign says that the row's largest elements are far above the others
                s_mul[r] = __uint_as_float((unsigned)ex << 23) * fabsf(P.scale_log2) * (16777216.f / (1 << QUP)) * (peaked ? -1.f : 1.f);
                s_lim[r] = real ? max(0, len - count + t + 1) : 0x7fffffff;   // else: as the row that sees most (below)
            }
        }
    };
    int npend = 0;                    // partials that wait to be joined
    Segment cur;
    plan.seek(cur, f0, B);
    bool more = true;
    while (more && cur.seg0 == cur.seg1) more = plan.next(cur);
    if (!more) return;
    open(cur);
    stage_q(cur);
    __syncthreads();

    while (more) {
        // ------------------------------------------------------------------ one segment
        const int b = cur.b, h = cur.h;
        const int row0 = cur.rb * RB, nrows = min(RB, P.rows - row0);
        const int len = positions_of(P, b);
        float acc[NB][NG][2][4];
        // of this lane's score columns 2c + i (row (2c + i) % CR of block nb, group (2c + i) / CR where the groups have
        // columns of their own): reference, sum of weights, q's factor, -8 sum q of the groups
        float ref[NB][2], sum[NB][2], mul[NB][2];
        float off[NB][2][REP ? 1 : NS];
        int limit[NB][2];
        uint32_t qf[NB][NG][4];
        const int lim = lane < RB ? s_lim[lane] : 0x7fffffff;
        int low = __reduce_min_sync(0xffffffffu, lim);                                     // least and greatest limit of
        const int high = __reduce_max_sync(0xffffffffu, lim == 0x7fffffff ? 0 : lim);      // the block's rows
        if (__any_sync(0xffffffffu, lane < CR * NB && signbit(s_mul[lane]))) low = 0;      // every tile takes signed codes
        const int cg = REP ? 2 * cq / CR : 0;            // the group of this lane's columns
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint4 v = *reinterpret_cast<const uint4*>(s_q + (8 * nb + quad % CR) * QROW + (g * 4 + cq) * 16);
                if (REP && g * 32 / GS != quad / CR) v = make_uint4(0, 0, 0, 0);
                qf[nb][g][0] = v.x; qf[nb][g][1] = v.y; qf[nb][g][2] = v.z; qf[nb][g][3] = v.w;
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 8 * nb + (2 * cq + i) % CR;
                mul[nb][i] = fabsf(s_mul[r]);
                limit[nb][i] = min(s_lim[r], high);   // a row without a token must not weigh what was never loaded: its
                                                      // votes move the references of the others
                ref[nb][i] = NEG_INF; sum[nb][i] = 0.f;
#pragma unroll
                for (int gs = 0; gs < (REP ? 1 : NS); ++gs) off[nb][i][gs] = s_off[r * NS + (REP ? cg : gs)];
            }
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[nb][g][m][i] = 0.f;
        }

        // One tile of 32 positions; EDGE: some row does not see all of it, or a row asks for signed codes.
        auto tile = [&](auto edge, const uint8_t* base, int p0) {
            constexpr bool EDGE = decltype(edge)::value;
            constexpr int SETS = REP ? 1 : NS;           // weight fragments: one, or one for each group's scales
            const uint8_t* kscale = base + 2 * G::CODES;
            const uint8_t* vscale = kscale + G::SCALES;
            float s[2][NB][4];           // positions 16x + r, + 8 of this lane's columns
            uint32_t pb[2][NB][SETS][2]; // their products with the V scales, as fragments
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t w[2][NG];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const uint8_t* kr = base + (16 * x + 8 * k + quad) * (D / 2) + cq * (4 * NG);
                    if constexpr (NG == 4) {
                        const uint4 v = *reinterpret_cast<const uint4*>(kr);
                        w[k][0] = v.x; w[k][1] = v.y; w[k][2] = v.z; w[k][3] = v.w;
                    } else {
                        const uint2 v = *reinterpret_cast<const uint2*>(kr);
                        w[k][0] = v.x; w[k][1] = v.y;
                    }
                }
                float ks[2][SETS];
#pragma unroll
                for (int k = 0; k < 2; ++k) load_scales<SETS>(kscale + ((16 * x + 8 * k + quad) * NS + cg) * 2, ks[k]);
                float d[NB][4];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t v0 = w[0][g] >> 8, v1 = w[1][g] >> 8;
                    uint32_t a0 = w[0][g] & 0x000f000fu, a1 = w[1][g] & 0x000f000fu, a2 = w[0][g] & 0x00f000f0u, a3 = w[1][g] & 0x00f000f0u;
                    uint32_t b0 = v0 & 0x000f000fu, b1 = v1 & 0x000f000fu, b2 = v0 & 0x00f000f0u, b3 = v1 & 0x00f000f0u;
                    if constexpr (EDGE) {
                        a0 = signed_codes<1>(a0); a1 = signed_codes<1>(a1); a2 = signed_codes<16>(a2); a3 = signed_codes<16>(a3);
                        b0 = signed_codes<1>(b0); b1 = signed_codes<1>(b1); b2 = signed_codes<16>(b2); b3 = signed_codes<16>(b3);
                    }
                    const bool starts = REP ? g == 0 : g * 32 % GS == 0, ends = REP ? g == NG - 1 : (g + 1) * 32 % GS == 0;
                    const int gs = REP ? 0 : g * 32 / GS;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        if (starts) mma_f16_first(d[nb], a0, a1, a2, a3, qf[nb][g][0], qf[nb][g][1]);
                        else mma_f16(d[nb], a0, a1, a2, a3, qf[nb][g][0], qf[nb][g][1]);
                        mma_f16(d[nb], b0, b1, b2, b3, qf[nb][g][2], qf[nb][g][3]);
                        if (ends)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float z = EDGE ? d[nb][i] * 0x1p-24f : d[nb][i] + off[nb][i & 1][gs];
                                s[x][nb][i] = gs == 0 ? ks[i >> 1][gs] * z : fmaf(ks[i >> 1][gs], z, s[x][nb][i]);
                            }
                    }
                }
                if constexpr (REP && NS > 1) {           // the groups of a row are in neighbouring lanes
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[x][0][i] += __shfl_xor_sync(0xffffffffu, s[x][0][i], 2);
                        if (NS == 4) s[x][0][i] += __shfl_xor_sync(0xffffffffu, s[x][0][i], 1);
                    }
                }
                if constexpr (EDGE)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (p0 + 16 * x + 8 * (i >> 1) + quad >= limit[nb][i & 1]) s[x][nb][i] = NEG_INF;
            }
            // New references: the greatest score + exponent of the largest V scale (NaN ones do not count).
            auto raise = [&]() {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float r = NEG_INF;
#pragma unroll 1
                        for (int x = 0; x < 2; ++x)
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint8_t* p = vscale + (16 * x + 8 * k + quad) * NS * 2;
                                unsigned e = 0;
#pragma unroll
                                for (int gs = 0; gs < NS; ++gs) {
                                    const unsigned v = reinterpret_cast<const uint16_t*>(p)[gs];
                                    if (v < 0x7f80u) e = max(e, v);
                                }
                                const float v = x ? s[1][nb][2 * k + i] : s[0][nb][2 * k + i];
                                if (v != NEG_INF) r = fmaxf(r, fmaf(v, mul[nb][i], (float)max((int)(e >> 7), 67) - 127.f));
                            }
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) r = fmaxf(r, __shfl_xor_sync(0xffffffffu, r, o));
                        r = fmaxf(ref[nb][i], r - BELOW);
                        const float k = ref[nb][i] == NEG_INF ? 1.f : exp2_fast(ref[nb][i] - r);
                        ref[nb][i] = r;
                        sum[nb][i] *= k;
#pragma unroll
                        for (int g = 0; g < NG; ++g)
#pragma unroll
                            for (int mt = 0; mt < 2; ++mt) {
                                acc[nb][g][mt][i] *= k;
                                acc[nb][g][mt][2 + i] *= k;
                            }
                    }
            };
            // Weights and products against the present reference; where one comes out too large (or there is no
            // reference yet) it is raised, and they are taken again.
            float part[NB][2];
            auto weigh = [&]() {
                float most = 0.f;
                bool bad = false;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        part[nb][i] = 0.f;
                        bad = bad || ref[nb][i] == NEG_INF;
                    }
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        float vs[SETS];
                        load_scales<SETS>(vscale + ((16 * x + 8 * k + quad) * NS + cg) * 2, vs);
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            float w[2];
                            bool seen[2];
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                const float v = s[x][nb][2 * k + i], r = ref[nb][i] == NEG_INF ? 0.f : ref[nb][i];
                                seen[i] = !EDGE || p0 + 16 * x + 8 * k + quad < limit[nb][i];
                                w[i] = EDGE && v == NEG_INF ? 0.f : exp2_fast(fmaf(v, mul[nb][i], -r));
                                part[nb][i] += w[i];
                            }
#pragma unroll
                            for (int gs = 0; gs < SETS; ++gs) {
                                // a masked position adds nothing, whatever its values are
                                const float a = seen[0] ? w[0] * vs[gs] : 0.f, c = seen[1] ? w[1] * vs[gs] : 0.f;
                                most = fmaxf(most, fmaxf(a, c));
                                pb[x][nb][gs][k] = pack_f16(a, c);
                            }
                        }
                    }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 2; ++i) bad = bad || part[nb][i] > 0x1p90f;
                return bad || most > MOST;
            };
            if (__any_sync(0xffffffffu, weigh())) {
                raise();
                weigh();
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
                for (int i = 0; i < 2; ++i) sum[nb][i] += part[nb][i];
#pragma unroll
                for (int x = 0; x < 2; ++x)
#pragma unroll
                    for (int gs = 0; gs < SETS; ++gs)
#pragma unroll
                        for (int k = 0; k < 2; ++k) pb[x][nb][gs][k] = transpose8x8(pb[x][nb][gs][k]);
            }
            // V words: the two rows of a pair are read in an order that spreads them over the banks (odd c the
            // other way round) and put in order by the permute's selector
            const int pa = 2 * cq + (cq & 1), pz = 2 * cq + 1 - (cq & 1);
            const uint32_t sel0 = cq & 1 ? 0x1054u : 0x5410u, sel1 = cq & 1 ? 0x3276u : 0x7632u;
            uint32_t w[2][2][2][NG / 2];
#pragma unroll
            for (int y = 0; y < 2; ++y)                          // 16 positions at a time
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint8_t* p = base + G::CODES + (16 * y + 8 * k + (i ? pz : pa)) * (D / 2) + quad * (2 * NG);
                        if constexpr (NG == 4) {
                            const uint2 v = *reinterpret_cast<const uint2*>(p);
                            w[y][k][i][0] = v.x; w[y][k][i][1] = v.y;
                        } else {
                            w[y][k][i][0] = *reinterpret_cast<const uint32_t*>(p);
                        }
                    }
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const int gs = REP ? 0 : g * 32 / GS;
                    uint32_t a[2][4];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        codes_to_f16(__byte_perm(w[y][k][0][g / 2], w[y][k][1][g / 2], g & 1 ? sel1 : sel0), a[k]);
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
                            mma_f16(acc[nb][g][mt], a[0][2 * mt], a[0][2 * mt + 1], a[1][2 * mt], a[1][2 * mt + 1], pb[y][nb][gs][0],
                                    pb[y][nb][gs][1]);
                }
        };

        for (int u = cur.u; u < cur.u1 && !dead; ++u) {
            const int p0 = u * TP, st = nuse % NST;
            bool late = false;
            if (!mbar_test(&bars[warp][st], (nuse / NST) & 1)) {
                const unsigned long long t0 = globaltimer();
                while (!mbar_test(&bars[warp][st], (nuse / NST) & 1))
                    if (globaltimer() - t0 > WAIT_NS) { late = true; break; }
            }
            dead = __any_sync(0xffffffffu, late);
            if (dead) {              // this tile and those after it are not counted as used: the end waits for their copies
                if (lane == 0) report(P.c, MQ_DEV_TIMEOUT_RING, blockIdx.x);
                break;
            }
            const uint8_t* base = ring + st * G::STAGE;
            if (p0 < high) {         // low: the greatest number where every row is padding
                if (p0 + TP <= low) tile(std::false_type{}, base, p0);
                else tile(std::true_type{}, base, p0);
            }
            ++nuse;
            __syncwarp();        // every lane has read the stage before it is filled again
            if (u + NST < cur.u1) load(b, h, len, u + NST);
        }
        // the next segment's copies and queries are under way while this one's warps meet
        const Segment seg = cur;
        do more = plan.next(cur);
        while (more && cur.seg0 == cur.seg1);
        if (more) open(cur);

        // ------------------------------------------------------------------ the warps of the segment meet
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum[nb][i] += __shfl_xor_sync(0xffffffffu, sum[nb][i], o);
                const int r = 8 * nb + (2 * cq + i) % CR;
                if (quad == 0 && cg == 0) { s_ref[warp * RB + r] = ref[nb][i]; s_sum[warp * RB + r] = sum[nb][i]; }
                if (r < nrows) {
                    float* dst = s_acc + (warp * rmax + r) * LDA + 4 * quad;
#pragma unroll
                    for (int g = 0; g < NG; ++g)
                        if (!REP || g * 32 / GS == cg)
                            *reinterpret_cast<float4*>(dst + 32 * g) =
                                make_float4(acc[nb][g][0][i], acc[nb][g][0][2 + i], acc[nb][g][1][i], acc[nb][g][1][2 + i]);
                }
            }
        __syncthreads();
        if (more) stage_q(cur);
        const int n = plan.units(b);
        const bool all = seg.seg0 == 0 && seg.seg1 == n;
        const size_t pstride = part_floats(rmax, D);
        // an item's first CTA has it as its last segment, the others as their first
        float* part = P.part + (2 * (size_t)blockIdx.x + (seg.seg0 == 0 ? 1 : 0)) * pstride;
#pragma unroll 1
        for (int i = tid; i < nrows * (D / 4); i += NTHR) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float M = NEG_INF, L = 0.f;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < NW; ++w) M = fmaxf(M, s_ref[w * RB + r]);
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float l = s_sum[w * RB + r];       // 0: nothing added, and the sums are zeros (a NaN goes on)
                const float k = l == 0.f ? 0.f : exp2_fast(s_ref[w * RB + r] - M);
                L = fmaf(l, k, L);
                add4(o, *reinterpret_cast<const float4*>(s_acc + (w * rmax + r) * LDA + d), k);
            }
            if (all) {
                store_out(P, b, h, row0 + r, D, d, o, L);
            } else {
                *reinterpret_cast<float4*>(part + r * D + d) = o;
                if (d == 0) *reinterpret_cast<float2*>(part + rmax * D + 2 * r) = make_float2(M, L);
            }
        }
        // Partial: the arrival at the item's counter is under way while the next segment runs (a CTA has two at most,
        // its first segment and its last).
        if (!all) {
            __syncthreads();
            if (tid == 0) {
                s_pend[npend] = seg;
                __threadfence();
                s_was[npend] = atomicAdd(&P.counters[(unsigned)b * (unsigned)per + (unsigned)(seg.h * P.blocks + seg.rb)], 1u);
            }
            ++npend;
        }
        __syncthreads();         // shared memory of the meeting is free, and the next queries are in place
    }
    // ------------------------------------------------------------------ joins
    // The last of an item's CTAs to arrive joins the partials, in a fixed order: each thread has four outputs and every
    // `splits`-th partial.
#pragma unroll 1
    for (int i = 0; i < npend; ++i) {
        const Segment seg = s_pend[i];
        const int b = seg.b, h = seg.h, row0 = seg.rb * RB, nrows = min(RB, P.rows - row0), n = plan.units(b);
        const size_t pstride = part_floats(rmax, D);
        const int c0 = (int)((seg.item_f + OVER) / Q), np = (int)((seg.item_f + OVER + (unsigned)n - 1) / Q) - c0 + 1;
        if (tid == 0) {
            s_last = s_was[i] == (unsigned)np - 1;
            if (s_last) P.counters[(unsigned)b * (unsigned)per + (unsigned)(seg.h * P.blocks + seg.rb)] = 0;
        }
        __syncthreads();
        if (s_last) {
            __threadfence();
            const int tasks = nrows * (D / 4);
            int splits = 1;
            while (splits < 8 && tasks * splits * 2 <= NTHR && splits * 4 <= np) splits *= 2;
            const int width = NTHR / splits, s0 = tid / width;
#pragma unroll 1
            for (int i0 = 0; i0 < tasks; i0 += width) {
                const int i = min(i0 + tid - s0 * width, tasks - 1), r = i / (D / 4);
                float M = NEG_INF, L = 0.f;
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
                for (int p = s0; p < np; p += 8 * splits) {
                    float2 ml[8];
                    float4 a[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int q = p + k * splits;
                        const float* x = P.part + (2 * (size_t)(c0 + q) + (q == 0 ? 1 : 0)) * pstride;
                        ml[k] = make_float2(NEG_INF, 0.f);
                        a[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (q < np) {
                            ml[k] = __ldcg(reinterpret_cast<const float2*>(x + rmax * D + 2 * r));
                            a[k] = __ldcg(reinterpret_cast<const float4*>(x) + i);
                        }
                    }
                    float m = M;
#pragma unroll
                    for (int k = 0; k < 8; ++k) m = fmaxf(m, ml[k].x);
                    const float was = L == 0.f ? 0.f : exp2_fast(M - m);
                    M = m;
                    L *= was;
                    scale4(o, was);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float f = ml[k].y == 0.f ? 0.f : exp2_fast(ml[k].x - m);
                        L = fmaf(ml[k].y, f, L);
                        add4(o, a[k], f);
                    }
                }
                if (splits > 1) {
                    // [split][width] of (M, L) and of the sums; tasks * splits <= NTHR, so this is the only round
                    float* s_ml = s_acc + 4 * NTHR;
                    *reinterpret_cast<float4*>(s_acc + 4 * tid) = o;
                    s_ml[tid] = M;
                    s_ml[NTHR + tid] = L;
                    __syncthreads();
                    if (s0 == 0) {
                        float m = M;
                        for (int k = 1; k < splits; ++k) m = fmaxf(m, s_ml[k * width + tid]);
                        const float was = L == 0.f ? 0.f : exp2_fast(M - m);
                        L *= was;
                        scale4(o, was);
                        for (int k = 1; k < splits; ++k) {
                            const float l = s_ml[NTHR + k * width + tid];
                            const float f = l == 0.f ? 0.f : exp2_fast(s_ml[k * width + tid] - m);
                            L = fmaf(l, f, L);
                            add4(o, *reinterpret_cast<const float4*>(s_acc + 4 * (k * width + tid)), f);
                        }
                    }
                }
                if (s0 == 0 && i0 + tid < tasks) store_out(P, b, h, row0 + r, D, i % (D / 4) * 4, o, L);
            }
        }
        __syncthreads();
    }
    // after a wait that ran out, copies may still be in flight: wait for them, with the same limit
    if (dead && lane == 0)
        for (; nuse < nload; ++nuse) {
            const unsigned long long t0 = globaltimer();
            while (!mbar_test(&bars[warp][nuse % NST], (nuse / NST) & 1))
                if (globaltimer() - t0 > WAIT_NS) break;
        }
}

size_t smem_bytes(int D, int GS, int stage, int NB, int NW, int rows, int batch) {
    const int rb = 8 * NB, rmax = rows < rb ? rows : rb;
    const int acc = rmax * (D + 4) > 192 ? rmax * (D + 4) : 192;
    return (size_t)NW * (NST * stage + acc * 4 + 2 * rb * 4) + rb * (D / GS + 2) * 4 + rb * (2 * D + 16) + ((size_t)batch + 1) * 4;
}
// Warps of a CTA: few items take one CTA of 8 an SM, so that an item has few partials to join (one sequence of 32768
// positions, 8 KV heads: 20.8 us; 6, 10, 12, 14, 16 warps: 24.7, 22.7, 21.7, 23.9, 24.4); many take CTAs of 4, whose
// warps share a segment with less rounding, as many as the registers allow (4 for 8 rows, 2 for 16).
constexpr int FEW_WARPS = 8, MANY_WARPS = 4;
constexpr int many_ctas(int NB) { return NB == 1 ? 4 : 2; }
constexpr int FEW_BATCH = 1024;      // sequences a large CTA's shared memory has room for
constexpr int MAX_DEV = 64;
int g_sm_count[MAX_DEV];

// Query rows of an item: 8 or 16 here, 128 (kv4_rows.cu) for more than 32.  16 heads over 8, us, blocks of 16 against 128:
//   rows                                  16           32           48           64
//   4 sequences of 6000                   29.5  46.6   40.8  47.1   51.0  47.9   60.8  48.1
//   32 sequences of 128 to 4096                        115   118    173   119    228   120
//   1 sequence of 3000                                 21.9  23.6   18.1  24.1   23.7  24.1
// The rule looks at the rows alone: one short sequence with 33 to 64 rows would be up to 6 us quicker in blocks of 16.
int block_rows(int rows) { return rows <= 8 ? 8 : rows <= 32 ? 16 : ROWS_BLOCK; }

int sm_count(int& n) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= MAX_DEV) return MQ_ERR_DEVICE;
    if (!g_sm_count[dev] && (e = cudaDeviceGetAttribute(&g_sm_count[dev], cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return (int)e;
    n = g_sm_count[dev];
    return MQ_OK;
}

template <int D, int GS, int NB, int NW, bool REP>
int launch(const AttendParams& p, unsigned grid, cudaStream_t stream) {
    static bool set[MAX_DEV];
    const size_t smem = smem_bytes(D, GS, Geo<D, GS>::STAGE, NB, NW, p.rows, p.c.batch);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (!set[dev]) {
        const size_t most = smem_bytes(D, GS, Geo<D, GS>::STAGE, NB, NW, 8 * NB, NW == MANY_WARPS ? MAX_BATCH : FEW_BATCH);
        if ((e = cudaFuncSetAttribute(attend_kernel<D, GS, NB, NW, REP>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most)) != cudaSuccess)
            return (int)e;
        set[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(NW * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, attend_kernel<D, GS, NB, NW, REP>, p);
}
template <int D, int GS, int NB, bool REP>
int launch_nw(const AttendParams& p, int nw, unsigned grid, cudaStream_t stream) {
    return nw == FEW_WARPS ? launch<D, GS, NB, FEW_WARPS, REP>(p, grid, stream)
                               : launch<D, GS, NB, MANY_WARPS, REP>(p, grid, stream);
}
template <int D, int GS>
int launch_nb(const AttendParams& p, int nw, unsigned grid, cudaStream_t stream) {
    if (block_rows(p.rows) > 8) return launch_nw<D, GS, 2, false>(p, nw, grid, stream);
    if (GS == D || p.rows * (D / GS) <= 8) return launch_nw<D, GS, 1, true>(p, nw, grid, stream);
    if constexpr (GS < D) return launch_nw<D, GS, 1, false>(p, nw, grid, stream);
    return MQ_ERR_ARG;
}

// Sizes of one call; MQ_OK or an error.
int plan_call(const MQKV4Cache* c, int tokens, int qheads, int& rows, int& blocks, int& nw, unsigned& grid) {
    if (tokens < 1 || qheads < 1 || qheads % c->num_kv_heads != 0) return MQ_ERR_ARG;
    if (c->batch > MAX_BATCH) return MQ_ERR_SIZE;
    const long long r = (long long)tokens * (qheads / c->num_kv_heads);
    if (r > (1 << 24)) return MQ_ERR_SIZE;
    rows = (int)r;
    const int rb = block_rows(rows);
    blocks = (rows + rb - 1) / rb;
    const double items = (double)c->batch * c->num_kv_heads * blocks;
    const double units = items * ((c->max_seq_len + TP - 1) / TP + OVER);
    if (units >= 2147483648.0 || items >= 134217728.0) return MQ_ERR_SIZE;      // flattened units, grids
    int sms = 0;
    const int rc = sm_count(sms);
    if (rc != MQ_OK) return rc;
    nw = items < 2.0 * sms && c->batch <= FEW_BATCH ? FEW_WARPS : MANY_WARPS;
    const double most = (double)sms * (rb == ROWS_BLOCK ? ROWS_CTAS : nw == FEW_WARPS ? 1 : many_ctas(rb / 8));
    grid = (unsigned)(units < most ? units : most);
    return MQ_OK;
}
bool aligned(const void* p, int a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }

}  // namespace
}  // namespace kv4
}  // namespace mq

using namespace mq;
using namespace mq::kv4;

extern "C" int mq_kv4_attend_workspace(const MQKV4Cache* cache, int tokens, int num_q_heads, size_t* bytes, size_t* counters) {
    View v;
    int rc = make_view(cache, v);
    if (rc != MQ_OK) return rc;
    if (!bytes || !counters) return MQ_ERR_ARG;
    int rows = 0, blocks = 0, nw = 0;
    unsigned grid = 0;
    if ((rc = plan_call(cache, tokens, num_q_heads, rows, blocks, nw, grid)) != MQ_OK) return rc;
    const int rb = block_rows(rows);
    const size_t items = (size_t)cache->batch * cache->num_kv_heads * blocks;
    *bytes = rb == ROWS_BLOCK ? rows_workspace(cache->head_dim, grid, items)
                              : (size_t)2 * grid * part_floats(rows < rb ? rows : rb, cache->head_dim) * sizeof(float);
    *counters = items;
    return MQ_OK;
}

extern "C" int mq_kv4_attend(const MQKV4Cache* cache, int dtype, const void* q, const int64_t* q_strides, void* out,
                             const int* lengths, const int* counts, int tokens, int num_q_heads, float scale,
                             void* workspace, size_t workspace_bytes, int* counters, size_t num_counters, cudaStream_t stream) {
    AttendParams p{};
    int rc = make_view(cache, p.c);
    if (rc != MQ_OK) return rc;
    if (tokens < 0) return MQ_ERR_ARG;
    if (tokens == 0) return MQ_OK;
    if ((dtype != MQ_BF16 && dtype != MQ_FP16) || !q || !q_strides || !out || !lengths || !workspace || !counters) return MQ_ERR_ARG;
    if (!aligned(q, 2) || !aligned(out, 16) || !aligned(lengths, 4) || !aligned(counts, 4) || !aligned(workspace, 16) ||
        !aligned(counters, 4))
        return MQ_ERR_ARG;
    unsigned grid = 0;
    int nw = 0;
    if ((rc = plan_call(cache, tokens, num_q_heads, p.rows, p.blocks, nw, grid)) != MQ_OK) return rc;
    size_t need = 0, cnt = 0;
    mq_kv4_attend_workspace(cache, tokens, num_q_heads, &need, &cnt);
    if (workspace_bytes < need || num_counters < cnt) return MQ_ERR_SIZE;
    p.q = q; p.qb = q_strides[0]; p.qt = q_strides[1]; p.qh = q_strides[2];
    p.out = out; p.lengths = lengths; p.counts = counts; p.dtype = dtype; p.tokens = tokens;
    p.qheads = num_q_heads; p.share = num_q_heads / cache->num_kv_heads;
    p.scale_log2 = scale * 1.4426950408889634f;
    p.counters = (unsigned*)counters; p.part = (float*)workspace;
    const int D = cache->head_dim, G = cache->group;
    if (block_rows(p.rows) == ROWS_BLOCK) return rows_attend(p, D, G, grid, stream);
    if (D == 128) {
        if (G == 32) return launch_nb<128, 32>(p, nw, grid, stream);
        if (G == 64) return launch_nb<128, 64>(p, nw, grid, stream);
        return launch_nb<128, 128>(p, nw, grid, stream);
    }
    if (G == 32) return launch_nb<64, 32>(p, nw, grid, stream);
    return launch_nb<64, 64>(p, nw, grid, stream);
}
