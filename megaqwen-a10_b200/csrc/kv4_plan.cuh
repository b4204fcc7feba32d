// kv4_plan.cuh -- what the two attention kernels over the 4-bit cache share: their arguments, the division of the
// work among CTAs, and small arithmetic.
//
// Work is counted in units of 32 positions of an item (sequence, KV head, block of query rows).  The items' units,
// each item led by OVER units that stand for what starting and ending it costs, are laid end to end and cut into
// equal ranges, one for each CTA.  The part of an item in a CTA's range is a segment.
#pragma once
#include "kv4.cuh"

namespace mq {
namespace kv4 {

constexpr int TP = 32;               // positions of a tile, and of a unit of work
constexpr int OVER = 8;    // what starting and ending a segment costs, in units: added to an item's length in the split
constexpr int MAX_BATCH = 4096;      // its prefix sums lie in shared memory
// A new reference lies this far (log2) below the largest contribution: weights start at 2^7, may grow by 2^8 before
// the reference moves, and keep fp16's 11 bits down to 2^-21 of the largest.
constexpr float BELOW = 7.f, RAISE = 8.f;
constexpr float NEG_INF = -INFINITY;
constexpr unsigned long long WAIT_NS = 2000000000ull;

struct AttendParams {
    View c;
    const void* q;
    long long qb, qt, qh;            // strides in elements
    void* out;                       // [batch][tokens][q heads][D]
    const int* lengths;
    const int* counts;
    int dtype, tokens, qheads, share, rows, blocks;   // share: q heads of a KV head; rows = tokens * share
    float scale_log2;
    unsigned* counters;              // [items], zero between calls
    float* part;                     // [2 * CTAs][part_floats]
};

// Floats of one partial: rows x D sums, then (reference, sum of weights) of each row; whole 16-byte vectors.
__host__ __device__ constexpr size_t part_floats(int rows, int D) { return (size_t)rows * D + ((2 * rows + 3) / 4) * 4; }

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Nibbles k and k + 4 of w (k = 0..3, as out[k]) -> fp16 pairs nibble - 8: the nibble in the mantissa of 1024
// (16 nibble for every other one), then the offset off.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t (&out)[4]) {
    const __half2 m8 = __floats2half2_rn(-1032.f, -1032.f);       // 1024 + 8
    const __half2 inv = __floats2half2_rn(0.0625f, 0.0625f);
    const __half2 m72 = __floats2half2_rn(-72.f, -72.f);          // (1024 + 16 * 8) / 16
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = i ? w >> 8 : w;
        uint32_t lo, hi;
        asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(lo) : "r"(v));   // (v & mask) | 1024
        asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(hi) : "r"(v));   // 1024 + 16 nibble
        const __half2 a = __hadd2(*reinterpret_cast<__half2*>(&lo), m8);
        const __half2 b = __hfma2(*reinterpret_cast<__half2*>(&hi), inv, m72);
        out[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
        out[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
}
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void scale4(float4& v, float k) { v.x *= k; v.y *= k; v.z *= k; v.w *= k; }
__device__ __forceinline__ void add4(float4& v, const float4& a, float k) {
    v.x = fmaf(a.x, k, v.x); v.y = fmaf(a.y, k, v.y); v.z = fmaf(a.z, k, v.z); v.w = fmaf(a.w, k, v.w);
}
// Positions of sequence b that its rows can see: none where no row of the call is its token, and then nothing of the
// sequence is needed, whatever its length says.
__device__ __forceinline__ int positions_of(const AttendParams& P, int b) {
    const int len = P.lengths[b], count = P.counts ? P.counts[b] : 1;      // two loads at once
    return count > 0 ? min(max(len, 0), P.c.max_seq) : 0;
}
// Four dims of an output row from the sum of weights L (0: the row saw nothing).
__device__ __forceinline__ void store_out(const AttendParams& P, int b, int h, int row, int D, int d, float4 o, float L) {
    const int t = row / P.share, j = row - t * P.share;
    if (L == 0.f || (P.counts && t >= P.counts[b])) o = make_float4(0.f, 0.f, 0.f, 0.f);
    else scale4(o, 1.f / L);
    const long long at = (((long long)b * P.tokens + t) * P.qheads + h * P.share + j) * D + d;
    uint2 v;
    if (P.dtype == MQ_BF16) {
        v.x = f32_to_bf16_bits(o.x) | f32_to_bf16_bits(o.y) << 16;
        v.y = f32_to_bf16_bits(o.z) | f32_to_bf16_bits(o.w) << 16;
    } else {
        v.x = pack_f16(o.x, o.y); v.y = pack_f16(o.z, o.w);
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(P.out) + at) = v;
}

// The part of an item in a CTA's range, and one warp's units of it.
struct Segment {
    int b, h, rb;           // item: sequence, KV head and row block
    unsigned item_f;        // flattened start of the item
    unsigned end;           // flattened end of the segment
    int seg0, seg1;         // the segment's units within the item (none: only its overhead fell into this range)
    int u, u1;              // this warp's units
};

template <int NW>
struct Plan {
    const unsigned* prefix;   // [batch + 1] costs of one (head, block) of the sequences before b
    int per, blocks;          // heads * blocks
    int warp;
    unsigned f_end;           // end of the CTA's range
    // units of sequence b's items, with the overhead and without
    __device__ __forceinline__ int cost(int b) const { return (int)(prefix[b + 1] - prefix[b]); }
    __device__ __forceinline__ int units(int b) const { return cost(b) - OVER; }
    __device__ __forceinline__ void cut(Segment& c, unsigned f) const {
        const int n = cost(c.b);
        c.item_f = prefix[c.b] * (unsigned)per + (unsigned)(c.h * blocks + c.rb) * (unsigned)n;
        c.end = min(f_end, c.item_f + (unsigned)n);
        c.seg0 = max(0, (int)(f - c.item_f) - OVER);
        c.seg1 = max(0, (int)(c.end - c.item_f) - OVER);
        const int len = c.seg1 - c.seg0;
        c.u = c.seg0 + split_lo(len, NW, warp);
        c.u1 = c.seg0 + split_lo(len, NW, warp + 1);
    }
    // Segment at flattened unit f < f_end.
    __device__ __forceinline__ void seek(Segment& c, unsigned f, int batch) const {
        int lo = 0, hi = batch - 1;   // last b with prefix[b] * per <= f (every sequence has a unit)
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (prefix[mid] * (unsigned)per <= f) lo = mid; else hi = mid - 1;
        }
        c.b = lo;
        const int hr = (int)((f - prefix[lo] * (unsigned)per) / (unsigned)cost(lo));
        c.h = blocks == 1 ? hr : hr / blocks;
        c.rb = hr - c.h * blocks;
        cut(c, f);
    }
    __device__ __forceinline__ bool next(Segment& c) const {
        const unsigned f = c.end;
        if (f >= f_end) return false;
        if (++c.rb == blocks) {
            c.rb = 0;
            if (++c.h * blocks == per) { c.h = 0; ++c.b; }
        }
        cut(c, f);
        return true;
    }
};

// Prefix sums of the sequences' costs into prefix[0 .. batch], by one warp; returns the greatest cost.  Lengths
// outside [0, max_seq_len] are reported, and cut off.
__device__ __forceinline__ unsigned scan_costs(const AttendParams& P, unsigned* prefix, int lane) {
    unsigned carry = 0, most = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < P.c.batch; b0 += 32) {
        const int b = b0 + lane;
        unsigned n = 0;
        if (b < P.c.batch) {
            const int len = P.lengths[b];
            if (len < 0 || len > P.c.max_seq) report(P.c, MQ_DEV_BAD_POSITION, b);
            n = (unsigned)(max(1, (positions_of(P, b) + TP - 1) / TP) + OVER);
        }
        most = max(most, n);
        unsigned x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        if (b < P.c.batch) prefix[b + 1] = carry + x;
        carry += __shfl_sync(0xffffffffu, x, 31);
    }
    if (lane == 0) prefix[0] = 0;
    return __reduce_max_sync(0xffffffffu, most);
}

// Many rows (kv4_rows.cu): workspace of a call, and the call.
constexpr int ROWS_BLOCK = 128, ROWS_CTAS = 2;      // query rows of an item, CTAs of an SM
size_t rows_workspace(int D, unsigned grid, size_t items);
int rows_attend(const AttendParams& a, int D, int GS, unsigned grid, cudaStream_t stream);

}  // namespace kv4
}  // namespace mq
