// linear8.cu -- matrix product in 8-bit integers with a scale for each token and each output channel.
//
//   s_x[m] = max(fp32(max_k |x[m,k]| / 127), 1e-12),   c[m,k] = round_half_even(x[m,k] / s_x[m])
//   y[m,n] = (sum_k c[m,k] W[n,k]) * (s_x[m] * s_w[n])
//
// The sum is exact (int32: K * 127 * 128 < 2^31 for K <= 131072); the quotient is an IEEE fp32 division.  A token
// with an infinity or a NaN gets the scale NaN and the codes 0, so its whole row of y is NaN.
//
// Three ways, chosen by the number of tokens M:
//   * up to four tokens of a small layer (few_tokens): one kernel, bound by its latency; every CTA quantises the tokens
//     for itself into shared memory while its first weights are on their way, and the warps take four rows of W at a
//     time with dp4a (1 token, 4096 channels of 1024: 2.7 us).
//   * else a kernel that quantises the tokens (bound by reading x) and the tensor-core product (tcgen05.mma kind::i8,
//     s32 sums in TMEM); operands come by TMA in 128-byte slabs of K.  The product starts to load W while the
//     quantiser still runs: by then everything before the quantiser has finished.  With tiles enough for the SMs the
//     128 rows of the MMA are tokens and its columns 256 channels, and the outputs leave by TMA; else the rows are
//     channels and the columns 16 to 256 tokens, so that few tokens waste no tensor work.
//   * Where the tiles are too few for the SMs, a cluster of 2, 4 or 8 CTAs shares a tile along K; the partial sums
//     meet through distributed shared memory, in integers, so the result does not depend on the split.
// Measured with the quantiser: 64 tokens x 151936 channels x K 1024 to fp32 (195 MB) 35.6 us, 5.5 TB/s, bound by the
// memory; 37 x 1024 x 3072 8.2 us, two launches' latency and 24 slabs over 8 CTAs; 8192 x 6144 x 1024 57 us (1.8
// Pop/s), of which 43 us are slabs (0.48 us for 32 KB of operands in each SM, 2.4 Pop/s, also at larger K) and the rest the
// quantiser and the tiles' ends (gemm_pair_kernel).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>
#include "common.cuh"
#include "launch_lock.h"

namespace mq {
namespace lin8 {
namespace {

constexpr int MAX_DEV = 64;
constexpr unsigned long long WAIT_NS = 2000000000ull;

// Words of eight 16-bit or fp32 neighbours as floats.
template <int DT>
__device__ __forceinline__ void unpack8(const uint32_t* w, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        if constexpr (DT == MQ_FP32) x[j] = __uint_as_float(w[j]);
        else if constexpr (DT == MQ_BF16) x[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        else x[j] = __half2float(__ushort_as_half((unsigned short)(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu)));
    }
}
template <int DT>
constexpr int WORDS = DT == MQ_FP32 ? 8 : 4;   // of eight neighbours
// The words of eight neighbours from element i on, of which n exist (the others are 0).  VEC: 16-byte aligned; else the
// aligned vectors around them are read and the elements cut out.  Only vectors that hold an element of the row are read
// (with n <= 0 the row's last, if any), and such a vector ends in no other page than its element.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* p, long long i, int n, uint32_t (&w)[WORDS<DT>]) {
    constexpr int W = WORDS<DT>, ES = W / 2;                              // bytes of an element
    const uintptr_t at = reinterpret_cast<uintptr_t>(p) + (uintptr_t)(i * ES);
    if (VEC && n >= 8) {
#pragma unroll
        for (int v = 0; v < W / 4; ++v) {
            const uint4 a = reinterpret_cast<const uint4*>(at)[v];
            w[4 * v] = a.x; w[4 * v + 1] = a.y; w[4 * v + 2] = a.z; w[4 * v + 3] = a.w;
        }
        return;
    }
    const uint4* base = reinterpret_cast<const uint4*>(at & ~(uintptr_t)15);
    const int off = (int)(at & 15), end = off + min(n, 8) * ES;           // bytes within the vectors
    uint32_t a[W + 4], c[W + 1];
#pragma unroll
    for (int v = 0; v < W / 4 + 1; ++v) {
        const uint4 q = 16 * v < end ? base[v] : make_uint4(0, 0, 0, 0);
        a[4 * v] = q.x; a[4 * v + 1] = q.y; a[4 * v + 2] = q.z; a[4 * v + 3] = q.w;
    }
#pragma unroll
    for (int j = 0; j < W + 1; ++j) {
        const uint32_t w0 = off & 4 ? a[min(j + 1, W + 3)] : a[j], w2 = off & 4 ? a[min(j + 3, W + 3)] : a[min(j + 2, W + 3)];
        c[j] = off & 8 ? w2 : w0;
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
        w[j] = ES == 2 && (off & 2) ? __funnelshift_r(c[j], c[j + 1], 16) : c[j];
        if (n < 8) {
            const int k = n - (ES == 2 ? 2 : 1) * j;                      // elements from this word on
            if (k <= 0) w[j] = 0;
            else if (ES == 2 && k == 1) w[j] &= 0xffffu;
        }
    }
}
__device__ __forceinline__ void store_elem(void* p, long long i, int dtype, float v) {
    if (dtype == MQ_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
    else if (dtype == MQ_FP16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<float*>(p)[i] = v;
}
// The larger of a and the words' |elements|, as bits that order like them: an fp32's, or two 16-bit ones side by side.
template <int DT>
__device__ __forceinline__ unsigned max_bits(unsigned a, const uint32_t (&w)[WORDS<DT>]) {
#pragma unroll
    for (int j = 0; j < WORDS<DT>; ++j) a = DT == MQ_FP32 ? max(a, w[j] & 0x7fffffffu) : __vmaxu2(a, w[j] & 0x7fff7fffu);
    return a;
}
// The fp32 bits of the largest (infinities and NaN stay on top).
template <int DT>
__device__ __forceinline__ unsigned max_float(unsigned a) {
    if (DT == MQ_FP32) return a;
    a = max(a & 0xffffu, a >> 16);
    return DT == MQ_BF16 ? a << 16 : __float_as_uint(__half2float(__ushort_as_half((unsigned short)a)));
}
// Scale of a token whose largest |x| has the bits a (infinities and NaN on top).
__device__ __forceinline__ float token_scale(unsigned a) {
    return a < 0x7f800000u ? fmaxf(__fdiv_rn(__uint_as_float(a), 127.f), 1e-12f) : __uint_as_float(0x7fc00000u);
}
// Codes of eight neighbours.  x * (1 / s) is within 2^-16 of the fp32 quotient (which is at most 127), so its
// rounding is the quotient's unless it lies that near to a half; then (rarely) the quotient itself decides.
// Adding 1.5 * 2^23 rounds to a whole number, half to even, whose low byte is the code.
template <int DT>
__device__ __forceinline__ uint2 pack8(const uint32_t (&e)[WORDS<DT>], float s, float inv, bool finite) {
    if (!finite) return make_uint2(0u, 0u);
    const float magic = 12582912.f;
    float x[8], t[8], far = 0.f;
    unpack8<DT>(e, x);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        t[j] = fmaf(x[j], inv, magic);
        far = fmaxf(far, fabsf(fmaf(x[j], inv, magic - t[j])));
    }
    if (far > 0.5f - 0x1p-14f)
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = __fdiv_rn(x[j], s) + magic;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t lo = __byte_perm(__float_as_uint(t[4 * i]), __float_as_uint(t[4 * i + 1]), 0x0040);
        const uint32_t hi = __byte_perm(__float_as_uint(t[4 * i + 2]), __float_as_uint(t[4 * i + 3]), 0x0040);
        w[i] = __byte_perm(lo, hi, 0x5410);
    }
    return make_uint2(w[0], w[1]);
}

// ------------------------------------------------------------------ tokens -> codes
struct QuantParams {
    const void* x;
    long long ldx;       // elements
    int dtype, vec;
    int M, K, ldq;       // ldq: bytes of a code row, a multiple of 16
    int8_t* q;
    float* scale;
};
// tpr threads for each row (a power of two >= 32), up to CH chunks of 8 elements each in registers, in x's own type; what
// is longer is read twice.  Bound by the memory once the rows are many: 4764 x K 6656 in bf16, 95 MB in and out, in 29 us
// (3.3 TB/s); few rows by the latency of one load, the reduction and one store.
template <int DT, bool VEC, int CH>
__global__ void __launch_bounds__(1024) quantize_tokens_kernel(const QuantParams P, int tpr) {
    pdl_wait();
    pdl_launch_dependents();     // after the wait: see gemm_kernel
    __shared__ unsigned s_max[32];
    const int sub = threadIdx.x / tpr, t = threadIdx.x & (tpr - 1);
    const long long m = (long long)blockIdx.x * (blockDim.x / tpr) + sub;
    const bool in = m < P.M;
    const int chunks = in ? (P.K + 7) / 8 : 0;
    uint32_t x[CH][WORDS<DT>];
    unsigned a = 0;
    auto fetch = [&](int c, uint32_t (&v)[WORDS<DT>]) { load8<DT, VEC>(P.x, m * P.ldx + 8 * c, P.K - 8 * c, v); };
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        if (t + i * tpr < chunks) {
            fetch(t + i * tpr, x[i]);
        } else {
#pragma unroll
            for (int j = 0; j < WORDS<DT>; ++j) x[i][j] = 0;
        }
    }
#pragma unroll
    for (int i = 0; i < CH; ++i) a = max_bits<DT>(a, x[i]);
    for (int c = t + CH * tpr; c < chunks; c += tpr) {
        uint32_t v[WORDS<DT>];
        fetch(c, v);
        a = max_bits<DT>(a, v);
    }
    a = max_float<DT>(a);
    a = __reduce_max_sync(0xffffffffu, a);
    if (tpr > 32) {
        const int per = tpr >> 5;
        if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = a;
        __syncthreads();
        for (int i = 0; i < per; ++i) a = max(a, s_max[sub * per + i]);
    }
    if (!in) return;
    const float s = token_scale(a), inv = 1.f / s;
    const bool finite = a < 0x7f800000u;
    if (t == 0) P.scale[m] = s;
    int8_t* row = P.q + m * P.ldq;
#pragma unroll
    for (int i = 0; i < CH; ++i) {
        const int c = t + i * tpr;
        if (8 * c < P.ldq) *reinterpret_cast<uint2*>(row + 8 * c) = pack8<DT>(x[i], s, inv, finite);
    }
    for (int c = t + CH * tpr; 8 * c < P.ldq; c += tpr) {
        uint32_t v[WORDS<DT>];
#pragma unroll
        for (int j = 0; j < WORDS<DT>; ++j) v[j] = 0;
        if (c < chunks) fetch(c, v);
        *reinterpret_cast<uint2*>(row + 8 * c) = pack8<DT>(v, s, inv, finite);
    }
}

// ------------------------------------------------------------------ few tokens
struct GemvParams {
    const void* x;
    long long ldx;
    int dtype, vec, out_dtype;
    int M, N, K;
    const int8_t* w;
    long long ldw;
    const float* ws;
    void* out;
};
constexpr int GV_WARPS = 8, GV_ROWS = 4;

__device__ __forceinline__ uint4 load_stream(const int8_t* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

template <int MT, int DT, bool VEC>
__global__ void __launch_bounds__(GV_WARPS * 32) gemv_kernel(const GemvParams P) {
    extern __shared__ __align__(16) uint8_t smem[];   // codes [MT][units * 16]
    __shared__ unsigned s_max[MT][GV_WARPS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int units = (P.K + 15) / 16;
    pdl_launch_dependents();
    pdl_wait();
    int n0 = (blockIdx.x * GV_WARPS + warp) * GV_ROWS;
    const int step = gridDim.x * GV_WARPS * GV_ROWS;
    // the first weights are on their way while the tokens are quantised
    uint4 first[GV_ROWS];
    auto row = [&](int r) { return P.w + (long long)min(n0 + r, P.N - 1) * P.ldw; };
#pragma unroll
    for (int r = 0; r < GV_ROWS; ++r) first[r] = lane < units && n0 < P.N ? load_stream(row(r) + 16 * lane) : make_uint4(0, 0, 0, 0);
    unsigned a[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        a[t] = 0;
        if (t < P.M)
            for (int c = tid; c < units * 2; c += GV_WARPS * 32) {
                uint32_t v[WORDS<DT>];
                load8<DT, VEC>(P.x, t * P.ldx + 8 * c, P.K - 8 * c, v);
                a[t] = max_bits<DT>(a[t], v);
            }
        a[t] = max_float<DT>(a[t]);
        a[t] = __reduce_max_sync(0xffffffffu, a[t]);
        if (lane == 0) s_max[t][warp] = a[t];
    }
    __syncthreads();
    float sx[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int w = 0; w < GV_WARPS; ++w) a[t] = max(a[t], s_max[t][w]);
        sx[t] = token_scale(a[t]);
        const float inv = 1.f / sx[t];
        for (int c = tid; c < units * 2; c += GV_WARPS * 32) {
            uint32_t v[WORDS<DT>];
            load8<DT, VEC>(P.x, t < P.M ? t * P.ldx + 8 * c : 0, t < P.M ? P.K - 8 * c : 0, v);
            *reinterpret_cast<uint2*>(smem + (size_t)t * units * 16 + 8 * c) = pack8<DT>(v, sx[t], inv, a[t] < 0x7f800000u);
        }
    }
    __syncthreads();
    for (bool again = false; n0 < P.N; n0 += step, again = true) {
        int acc[GV_ROWS][MT];
#pragma unroll
        for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = 0;
        auto use = [&](const uint4 (&w)[GV_ROWS], int u) {
#pragma unroll
            for (int t = 0; t < MT; ++t) {
                const int4 x = *reinterpret_cast<const int4*>(smem + (size_t)t * units * 16 + 16 * u);
#pragma unroll
                for (int r = 0; r < GV_ROWS; ++r) {
                    acc[r][t] = __dp4a((int)w[r].x, x.x, acc[r][t]);
                    acc[r][t] = __dp4a((int)w[r].y, x.y, acc[r][t]);
                    acc[r][t] = __dp4a((int)w[r].z, x.z, acc[r][t]);
                    acc[r][t] = __dp4a((int)w[r].w, x.w, acc[r][t]);
                }
            }
        };
        int u = lane;
        if (!again) {
            if (u < units) use(first, u);
            u += 32;
        }
#pragma unroll 2
        for (; u < units; u += 32) {
            uint4 w[GV_ROWS];
#pragma unroll
            for (int r = 0; r < GV_ROWS; ++r) w[r] = load_stream(row(r) + 16 * (long long)u);
            use(w, u);
        }
#pragma unroll
        for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t) acc[r][t] = __reduce_add_sync(0xffffffffu, acc[r][t]);
        // lane r * MT + t writes row r of token t
        int v = 0;
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < GV_ROWS; ++r)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                if (lane == r * MT + t) { v = acc[r][t]; s = sx[t]; }
        const int r = lane / MT, t = lane % MT;
        if (lane < GV_ROWS * MT && n0 + r < P.N && t < P.M)
            store_elem(P.out, (long long)t * P.N + n0 + r, P.out_dtype, (float)v * (s * P.ws[n0 + r]));
    }
}

// ------------------------------------------------------------------ tensor-core product
struct GemmParams {
    const float* xs;
    const float* ws;
    void* out;
    int* status;
    int out_dtype, M, N, K, ntok;   // ntok: token tiles
    int tiles, splits, tma_out;
    int rows;                       // channels of a tile, up to 128 (gemm_kernel)
};

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// Shared-memory matrix descriptor: K-major rows of 128 bytes in the 128-byte swizzle, 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t sdesc_sw128(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | (1ull << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// Instruction descriptor, kind::i8: signed 8-bit A and B (both K-major), s32 D, M = 128.
__device__ __forceinline__ constexpr uint32_t idesc_i8(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}
__device__ __forceinline__ void umma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// 32 lanes x 16 consecutive s32 columns (this warp's lane quadrant); waits for the load.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}

// A tile has 128 channels (the rows) and BN tokens.
template <int BN>
struct Gemm {
    static constexpr int A = 128 * 128, B = BN * 128, STAGE = A + B;
    static constexpr int NST = STAGE > 40960 ? 4 : STAGE > 30000 ? 6 : 8;
    static constexpr int RING = NST * STAGE;                     // also holds a split's [BN][128] partial sums
    static constexpr int EPI = 4;                                // epilogue warps, one for each quadrant of lanes
    static constexpr int THREADS = 64 + 32 * EPI;
    static constexpr int SCALES = BN * 4;                        // the tokens' scales
    static constexpr int SMEM = RING + SCALES + 1024;            // aligned to 1024 by hand
    static constexpr int ACC = BN < 32 ? 32 : BN;                // TMEM columns of an accumulator
    static constexpr int COLS = 2 * ACC;                         // two accumulators
};
// 16 bytes of outputs from 4 or 8 sums.
template <class T> __device__ __forceinline__ uint4 pack16(const float* v);
template <> __device__ __forceinline__ uint4 pack16<float>(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <> __device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float* v) {
    union { __nv_bfloat162 h[4]; uint4 u; } w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    return w.u;
}
template <> __device__ __forceinline__ uint4 pack16<__half>(const float* v) {
    union { __half2 h[4]; uint4 u; } w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w.h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    return w.u;
}
template <class T> __device__ __forceinline__ T out_of(float v);
template <> __device__ __forceinline__ __nv_bfloat16 out_of(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half out_of(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float out_of(float v) { return v; }

// Takes one accumulator of channels x tokens out: a lane has one channel, neighbouring lanes store neighbours.
template <class T, int BN>
__device__ __forceinline__ void epilogue_channels(const GemmParams& P, uint32_t at, int ch, int t0, const float* sx) {
    const float sw = ch < P.N ? P.ws[ch] : 0.f;
    T* p = reinterpret_cast<T*>(P.out) + (long long)t0 * P.N + ch;
#pragma unroll 1
    for (int j = 0; j < BN && t0 + j < P.M; j += 16) {
        int v[16];
        __syncwarp();            // the lanes without a channel skipped the stores
        tmem_ld16(at + j, v);
        const int n = min(16, P.M - t0 - j);
        if (ch < P.N) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 s = *reinterpret_cast<const float4*>(sx + j + i);
                const float k[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (i + u < n) *p = out_of<T>((float)v[i + u] * (k[u] * sw));
                    p += P.N;
                }
            }
        }
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]),
          "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]),
          "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr)
        : "memory");
}
// All loads so far have arrived; the registers pass through so that nothing reads them earlier.
__device__ __forceinline__ void tmem_wait32(int (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]),
                   "+r"(v[9]), "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]),
                   "+r"(v[17]), "+r"(v[18]), "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]),
                   "+r"(v[25]), "+r"(v[26]), "+r"(v[27]), "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tma_store_2d(const void* tmap, const void* src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(tmap), "r"(x), "r"(y),
                 "r"(smem_u32(src))
                 : "memory");
}
// Puts 128 channels of 32 tokens out: a lane has one token, v its sums, k the channels' scales.  Boxes of 32 tokens x
// 128 bytes are put together in shared memory in the 128-byte swizzle (no two lanes meet in a bank) and leave by TMA,
// which also leaves out what lies beyond the matrix; where its rows are not 16-byte aligned the warp stores them.
template <class T>
__device__ __forceinline__ void store_tokens(const GemmParams& P, const CUtensorMap* mo, const int (&v)[4][32], float sx, const float* k,
                                             uint8_t* box, int ch0, int t0, int lane) {
    constexpr int CH = 128 / sizeof(T), E = 16 / sizeof(T);    // channels of a box and of a 16-byte vector
#pragma unroll
    for (int b = 0; b < 128 / CH; ++b) {
        if (P.tma_out) {                                       // the box's last store has been read
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
        }
#pragma unroll
        for (int c = 0; c < 8; ++c) {
            float y[E];
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const int ch = b * CH + c * E + i;
                const float4 s = *reinterpret_cast<const float4*>(k + ch);
                y[i] = (float)v[ch / 32][ch % 32] * (sx * s.x);
                y[i + 1] = (float)v[ch / 32][ch % 32 + 1] * (sx * s.y);
                y[i + 2] = (float)v[ch / 32][ch % 32 + 2] * (sx * s.z);
                y[i + 3] = (float)v[ch / 32][ch % 32 + 3] * (sx * s.w);
            }
            *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) * 16)) = pack16<T>(y);
        }
        if (P.tma_out) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0 && t0 < P.M && ch0 + b * CH < P.N) {
                tma_store_2d(mo, box, ch0 + b * CH, t0);
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            __syncwarp();
            T* p = reinterpret_cast<T*>(P.out) + (long long)t0 * P.N + ch0 + b * CH;
            const bool whole = t0 + 32 <= P.M && ch0 + b * CH + CH <= P.N;
            if (whole && (sizeof(T) == 4 || (P.N % 2 == 0 && (reinterpret_cast<uintptr_t>(P.out) & 3u) == 0))) {
                // a row's 128 bytes, four to a lane
#pragma unroll 8
                for (int r = 0; r < 32; ++r, p += P.N)
                    reinterpret_cast<uint32_t*>(p)[lane] = *reinterpret_cast<const uint32_t*>(box + r * 128 + ((4 * lane) ^ ((r & 7) << 4)));
            } else {
                constexpr int S = (int)sizeof(T);
#pragma unroll 4
                for (int r = 0; r < 32; ++r, p += P.N) {
                    if (t0 + r >= P.M) break;
#pragma unroll
                    for (int e = 0; e < CH; e += 32)
                        if (whole || ch0 + b * CH + e + lane < P.N)
                            p[e + lane] = *reinterpret_cast<const T*>(box + r * 128 + ((S * (e + lane)) ^ ((r & 7) << 4)));
                }
            }
            __syncwarp();
        }
    }
}

// Roles: warp 0 loads, warp 1 issues the MMAs, the others take the accumulators out while the next tile is summed.
template <int BN>
__global__ void __launch_bounds__(Gemm<BN>::THREADS, 1) gemm_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx,
                                                                      const GemmParams P) {
    using G = Gemm<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[G::NST], empty[G::NST], acc_full[2], acc_empty[2];
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* s_scale = reinterpret_cast<float*>(ring + G::RING);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = P.splits, rank = S > 1 ? (int)(blockIdx.x % S) : 0;
    const int first = S > 1 ? (int)blockIdx.x / S : (int)blockIdx.x, step = S > 1 ? P.tiles : (int)gridDim.x;
    const int slabs = (P.K + 127) / 128;
    const int k0 = split_lo(slabs, S, rank), k1 = split_lo(slabs, S, rank + 1);
    if (tid == 0) {
        for (int i = 0; i < G::NST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], G::EPI); }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(G::COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();

    // Bounded wait; false (and the status) when it runs out or another role has given up.
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_test(bar, parity)) return true;
        const unsigned long long t0 = globaltimer();
        while (!mbar_test(bar, parity)) {
            if (s_abort) return false;
            if (globaltimer() - t0 > WAIT_NS) {
                s_abort = 1;
                P.status[1] = (int)blockIdx.x;
                P.status[0] = MQ_DEV_TIMEOUT_RING;
                return false;
            }
        }
        return true;
    };

    if (warp == 0) {
        if (lane == 0) {
            // W may be read before the quantiser has finished (it has passed its own wait, so what came before it is
            // complete); the codes only after the wait.
            int it = 0, pre = 0;
            bool ok = true;
            auto load_w = [&](int tile, int kb, int st) {
                mbar_arrive_expect_tx(&full[st], (uint32_t)(P.rows * 128 + G::B));
                tma_load_2d(ring + st * G::STAGE, &mw, kb * 128, (tile / P.ntok) * P.rows, &full[st]);
            };
            for (; pre < G::NST && pre < k1 - k0 && first < P.tiles; ++pre) load_w(first, k0 + pre, pre);
            pdl_wait();
            for (int tile = first; tile < P.tiles && ok; tile += step)
                for (int kb = k0; kb < k1 && ok; ++kb, ++it) {
                    const int st = it % G::NST;
                    if (it >= G::NST) ok = wait(&empty[st], ((it / G::NST) & 1) ^ 1);
                    if (!ok) break;
                    if (it >= pre) load_w(tile, kb, st);
                    tma_load_2d(ring + st * G::STAGE + G::A, &mx, kb * 128, (tile % P.ntok) * BN, &full[st]);
                }
            if (!ok) {   // copies in flight land before the CTA leaves; a stage whose second copy was not issued is left out
                for (int i = max(0, it - G::NST); i < it; ++i) {
                    const unsigned long long t0 = globaltimer();
                    while (!mbar_test(&full[i % G::NST], (i / G::NST) & 1))
                        if (globaltimer() - t0 > WAIT_NS) break;
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int it = 0, n = 0;
            bool ok = true;
            for (int tile = first; tile < P.tiles && ok; tile += step, ++n) {
                const int buf = n & 1;
                if (n >= 2) ok = wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1);
                tc_fence_after();
                for (int kb = k0; kb < k1 && ok; ++kb, ++it) {
                    const int st = it % G::NST;
                    ok = wait(&full[st], (it / G::NST) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t base = smem_u32(ring + st * G::STAGE);
                    const uint64_t da = sdesc_sw128(base), db = sdesc_sw128(base + G::A);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        umma_i8(tmem + buf * G::ACC, da + 2 * i, db + 2 * i, idesc_i8(BN), kb > k0 || i > 0);
                    umma_commit(&empty[st]);
                }
                if (ok) umma_commit(&acc_full[buf]);
            }
            // the last commits have arrived before TMEM is freed: the epilogue waits for acc_full; after a failure, here
            if (!ok && it > 0) {
                const unsigned long long t0 = globaltimer();
                while (!mbar_test(&empty[(it - 1) % G::NST], ((it - 1) / G::NST) & 1))
                    if (globaltimer() - t0 > WAIT_NS) break;
            }
        }
    } else {
        pdl_wait();
        const int quadrant = warp & 3, c = 32 * quadrant + lane;
        int n = 0;
        for (int tile = first; tile < P.tiles; tile += step, ++n) {
            const int buf = n & 1;
            const int wrow = (tile / P.ntok) * P.rows, xrow = (tile % P.ntok) * BN;
            const int ch = c < P.rows ? wrow + c : P.N;      // no channel: the tile ends before
            named_bar(1, 32 * G::EPI);   // the last tile's have been read
            for (int i = tid - 64; i < BN; i += 32 * G::EPI)
                s_scale[i] = xrow + i < P.M ? P.xs[xrow + i] : 0.f;
            named_bar(1, 32 * G::EPI);
            const bool ok = __all_sync(0xffffffffu, wait(&acc_full[buf], (n >> 1) & 1));
            tc_fence_after();
            const uint32_t at = tmem + buf * G::ACC + ((uint32_t)(32 * quadrant) << 16);
            if (!ok) {
                // given up: every warp still takes part in the tiles' barriers above
            } else if (S > 1) {
                int* part = reinterpret_cast<int*>(ring);        // [BN][128]; all of this CTA's MMAs have read the ring
#pragma unroll 1
                for (int j = 0; j < BN; j += 16) {
                    int v[16];
                    tmem_ld16(at + j, v);
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(j + i) * 128 + c] = v[i];
                }
            } else {
                if (P.out_dtype == MQ_BF16) epilogue_channels<__nv_bfloat16, BN>(P, at, ch, xrow, s_scale);
                else if (P.out_dtype == MQ_FP16) epilogue_channels<__half, BN>(P, at, ch, xrow, s_scale);
                else epilogue_channels<float, BN>(P, at, ch, xrow, s_scale);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
            __syncwarp();        // before the next tile's barrier
        }
    }
    if (S > 1) {
        __syncwarp();            // one lane ran the roles of warps 0 and 1: the aligned barriers below take whole warps
        // every CTA of the cluster adds up its share of the tokens
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (!s_abort) {
            pdl_wait();
            const int n0 = (first / P.ntok) * P.rows, t0 = (first % P.ntok) * BN;
            const int j0 = split_lo(BN, S, rank), j1 = split_lo(BN, S, rank + 1);
            const uint32_t local = smem_u32(ring);
            for (int i = tid; i < (j1 - j0) * 32; i += G::THREADS) {
                const int j = j0 + i / 32, c4 = (i % 32) * 4;
                if (t0 + j >= P.M) break;
                int4 sum = make_int4(0, 0, 0, 0);
                for (int r = 0; r < S; ++r) {
                    uint32_t peer;
                    int4 v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(local + (uint32_t)(j * 128 + c4) * 4), "r"(r));
                    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(peer));
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                const float sx = P.xs[t0 + j];
                const int v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (n0 + c4 + k < P.N)
                        store_elem(P.out, (long long)(t0 + j) * P.N + n0 + c4 + k, P.out_dtype, (float)v[k] * (sx * P.ws[n0 + c4 + k]));
            }
        }
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(G::COLS) : "memory");
    }
}

// ------------------------------------------------------------------ pairs of CTAs
// Two CTAs of a cluster share a tile of 256 tokens x 256 channels (tcgen05.mma cta_group::2, M = 256): each brings
// its own 128 tokens of x and half of the channels of W, and has its tokens' sums in its own TMEM.  The operands of
// a tile cross from L2 once for both: 32 KB a slab and CTA instead of 48 (8192 tokens x 6144 channels x K 1024, with the quantiser: 61 -> 58 us).
__device__ __forceinline__ uint32_t peer_addr(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
    return a;
}
// Load into this CTA's shared memory that reports to a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_2d_pair(void* dst, const void* tmap, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            smem_u32(dst)),
        "l"(tmap), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accum)
        : "memory");
}
// Arrives at the same barrier of both CTAs when the products so far are done.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
                 "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

struct Pair {
    static constexpr int BN = 256, HALF = 128 * 128, STAGE = 2 * HALF, NST = 5, RING = NST * STAGE;
    static constexpr int EPI = 8, THREADS = 64 + 32 * EPI;     // epilogue warps: two for each quadrant of lanes, 128 channels each
    static constexpr int OUT = EPI * 4096, SCALES = EPI * 512; // for each a box of 32 rows x 128 bytes, and its channels' scales
    static constexpr int SMEM = RING + OUT + SCALES + 1024;    // aligned to 1024 by hand
};

__global__ void __launch_bounds__(Pair::THREADS, 1) gemm_pair_kernel(const __grid_constant__ CUtensorMap mw, const __grid_constant__ CUtensorMap mx,
                                                                      const __grid_constant__ CUtensorMap mo, const GemmParams P) {
    using G = Pair;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t full[G::NST], empty[G::NST], acc_full[2], acc_empty[2];   // full and acc_empty: the first CTA's are used
    __shared__ uint32_t s_tmem;
    __shared__ volatile int s_abort;
    uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* s_out = ring + G::RING;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)blockIdx.x & 1, first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;
    const int slabs = (P.K + 127) / 128;
    if (tid == 0) {
        for (int i = 0; i < G::NST; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 2 * G::EPI); }
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();              // the other CTA's barriers exist
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();

    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_test(bar, parity)) return true;
        const unsigned long long t0 = globaltimer();
        while (!mbar_test(bar, parity)) {
            if (s_abort) return false;
            if (globaltimer() - t0 > WAIT_NS) {
                s_abort = 1;
                P.status[1] = (int)blockIdx.x;
                P.status[0] = MQ_DEV_TIMEOUT_RING;
                return false;
            }
        }
        return true;
    };

    if (warp == 0) {
        if (lane == 0) {
            int it = 0, pre = 0;
            bool ok = true;
            auto load_w = [&](int tile, int kb, int st) {      // before the quantiser has finished: see gemm_kernel
                if (rank == 0) mbar_arrive_expect_tx(&full[st], 2 * G::STAGE);
                tma_load_2d_pair(ring + st * G::STAGE + G::HALF, &mw, kb * 128, (tile / P.ntok) * 256 + rank * 128, peer_addr(&full[st], 0));
            };
            for (; pre < G::NST && pre < slabs && first < P.tiles; ++pre) load_w(first, pre, pre);
            pdl_wait();
            for (int tile = first; tile < P.tiles && ok; tile += step)
                for (int kb = 0; kb < slabs && ok; ++kb, ++it) {
                    const int st = it % G::NST;
                    if (it >= G::NST) ok = wait(&empty[st], ((it / G::NST) & 1) ^ 1);
                    if (!ok) break;
                    if (it >= pre) load_w(tile, kb, st);
                    tma_load_2d_pair(ring + st * G::STAGE, &mx, kb * 128, (tile % P.ntok) * 256 + rank * 128, peer_addr(&full[st], 0));
                }
            if (!ok && rank == 0)    // copies in flight land before the CTAs leave
                for (int i = max(0, it - G::NST); i < it; ++i) {
                    const unsigned long long t0 = globaltimer();
                    while (!mbar_test(&full[i % G::NST], (i / G::NST) & 1))
                        if (globaltimer() - t0 > WAIT_NS) break;
                }
        }
    } else if (warp == 1) {
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(256 >> 3) << 17) | ((uint32_t)(256 >> 4) << 24);
            int it = 0, n = 0;
            bool ok = true;
            for (int tile = first; tile < P.tiles && ok; tile += step, ++n) {
                const int buf = n & 1;
                if (n >= 2) ok = wait(&acc_empty[buf], ((n >> 1) & 1) ^ 1);
                tc_fence_after();
                for (int kb = 0; kb < slabs && ok; ++kb, ++it) {
                    const int st = it % G::NST;
                    ok = wait(&full[st], (it / G::NST) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    const uint32_t base = smem_u32(ring + st * G::STAGE);
                    const uint64_t da = sdesc_sw128(base), db = sdesc_sw128(base + G::HALF);
#pragma unroll
                    for (int i = 0; i < 4; ++i) umma_i8_pair(tmem + buf * G::BN, da + 2 * i, db + 2 * i, idesc, kb > 0 || i > 0);
                    umma_commit_pair(&empty[st]);
                }
                if (ok) umma_commit_pair(&acc_full[buf]);
            }
            if (!ok && it > 0) {
                const unsigned long long t0 = globaltimer();
                while (!mbar_test(&empty[(it - 1) % G::NST], ((it - 1) / G::NST) & 1))
                    if (globaltimer() - t0 > WAIT_NS) break;
            }
        }
    } else {
        pdl_wait();
        const int quadrant = warp & 3, c0 = ((warp - 2) >> 2) * 128;
        uint8_t* box = s_out + (warp - 2) * 4096;
        float* k = reinterpret_cast<float*>(s_out + G::OUT) + (warp - 2) * 128;
        // the scales of a tile's tokens and channels, asked for a tile ahead
        float sx = 0.f, kn[4];
        auto scales = [&](int tile) {
            const int ch0 = (tile / P.ntok) * 256 + c0 + lane, t = (tile % P.ntok) * 256 + rank * 128 + 32 * quadrant + lane;
            sx = tile < P.tiles && t < P.M ? P.xs[t] : 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) kn[i] = tile < P.tiles && ch0 + 32 * i < P.N ? P.ws[ch0 + 32 * i] : 0.f;
        };
        scales(first);
        int n = 0;
        for (int tile = first; tile < P.tiles; tile += step, ++n) {
            const int buf = n & 1;
            const int ch0 = (tile / P.ntok) * 256 + c0, t0 = (tile % P.ntok) * 256 + rank * 128 + 32 * quadrant;
            __syncwarp();                            // the last tile's scales have been read
#pragma unroll
            for (int i = 0; i < 4; ++i) k[lane + 32 * i] = kn[i];
            const float s = sx;
            scales(tile + step);
            __syncwarp();
            const bool ok = __all_sync(0xffffffffu, wait(&acc_full[buf], (n >> 1) & 1));
            tc_fence_after();
            const uint32_t at = tmem + buf * G::BN + c0 + ((uint32_t)(32 * quadrant) << 16);
            int v[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_ld32(at + 32 * i, v[i]);
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_wait32(v[i]);
            tc_fence_before();
            __syncwarp();
            if (lane == 0)                           // the sums are in registers: the accumulator is free
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(peer_addr(&acc_empty[buf], 0)) : "memory");
            if (ok) {
                if (P.out_dtype == MQ_BF16) store_tokens<__nv_bfloat16>(P, &mo, v, s, k, box, ch0, t0, lane);
                else if (P.out_dtype == MQ_FP16) store_tokens<__half>(P, &mo, v, s, k, box, ch0, t0, lane);
                else store_tokens<float>(P, &mo, v, s, k, box, ch0, t0, lane);
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync();              // nothing of the pair is in use any more
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ------------------------------------------------------------------ host
int sm_count(int& dev, int& n) {
    static int known[MAX_DEV];
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= MAX_DEV) return MQ_ERR_DEVICE;
    if (!known[dev] && (e = cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev)) != cudaSuccess) return (int)e;
    n = known[dev];
    return MQ_OK;
}
bool aligned(const void* p, int a) { return ((uintptr_t)p & (uintptr_t)(a - 1)) == 0; }
size_t round_up(size_t n, size_t a) { return (n + a - 1) / a * a; }
// Where one kernel that quantises in every CTA and multiplies with dp4a is faster than the quantiser and the tensor
// cores, which take 5.3 us at least but read W faster and quantise once (us, one kernel and two): 1 token x 4096 x
// K 1024 2.7 and 5.9, x 16384 x 2048 9.9 and 10.3, x 16384 x 4096 20 and 18, x 4096 x 8192 18 and 12; 2 x 4096 x 4096
// 7.1 and 8.2; 4 x 4096 x 1024 5.2 and 5.9, x 16384 x 512 8.4 and 5.4, x 1024 x 4096 8.1 and 6.9.
bool few_tokens(int M, int N, int K) {
    return M <= 4 && (long long)M * K <= 8192 && (long long)M * N * K <= (M <= 2 ? 1 << 25 : 1 << 24);
}

// Matrix [rows][cols] of `dtype` (-1: bytes) with a row stride in bytes, boxes of 128 bytes x box rows in the 128-byte swizzle.
int encode_map(CUtensorMap* map, const void* base, int rows, int cols, long long stride, int box, int dtype = -1) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
    if (!encode) {
        cudaDriverEntryPointQueryResult q;
        void* fn = nullptr;
        const cudaError_t e = cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q);
        if (e != cudaSuccess) return (int)e;
        if (q != cudaDriverEntryPointSuccess || !fn) return (int)cudaErrorNotSupported;
        encode = (PFN_cuTensorMapEncodeTiled_v12000)fn;
    }
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride};
    const cuuint32_t boxes[2] = {dtype < 0 ? 128u : dtype == MQ_FP32 ? 32u : 64u, (cuuint32_t)box};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = encode(map, dtype < 0 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : dtype == MQ_FP32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 :
                              dtype == MQ_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, boxes, estr,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? MQ_OK : (int)cudaErrorInvalidValue;
}

void pdl_attr(cudaLaunchAttribute& at) {
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
}

int launch_quantize(const QuantParams& p, cudaStream_t stream) {
    const int chunks = p.ldq / 8;
    int tpr = 32;
    // four chunks for each thread where there are rows enough to fill the SMs, else one (whole call, four and one: 4764
    // tokens x K 6656 45 and 106 us, 600 x 8192 12.2 and 19.5, 128 x 4096 8.6 and 8.0)
    const int each = p.M >= 512 ? 4 : 1;
    while (tpr < 1024 && tpr * each < chunks) tpr *= 2;
    const int rows = tpr >= 256 ? 1 : 256 / tpr;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((p.M + rows - 1) / rows));
    cfg.blockDim = dim3((unsigned)(tpr * rows));
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    pdl_attr(at[0]);
    cfg.attrs = at;
    cfg.numAttrs = 1;
    if (p.vec) {
        if (p.dtype == MQ_BF16) return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_BF16, true, 4>, p, tpr);
        if (p.dtype == MQ_FP16) return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_FP16, true, 4>, p, tpr);
        return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_FP32, true, 4>, p, tpr);
    }
    if (p.dtype == MQ_BF16) return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_BF16, false, 4>, p, tpr);
    if (p.dtype == MQ_FP16) return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_FP16, false, 4>, p, tpr);
    return (int)cudaLaunchKernelEx(&cfg, quantize_tokens_kernel<MQ_FP32, false, 4>, p, tpr);
}

template <int MT, int DT, bool VEC>
int launch_gemv_as(const GemvParams& p, int sms, cudaStream_t stream) {
    const size_t smem = (size_t)MT * ((p.K + 15) / 16) * 16;              // 11 KB at most
    const long long blocks = ((long long)p.N + GV_WARPS * GV_ROWS - 1) / (GV_WARPS * GV_ROWS);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(blocks < 4LL * sms ? blocks : 4LL * sms));
    cfg.blockDim = dim3(GV_WARPS * 32);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute at[1];
    pdl_attr(at[0]);
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&cfg, gemv_kernel<MT, DT, VEC>, p);
}
template <int MT>
int launch_gemv(const GemvParams& p, int sms, cudaStream_t stream) {
    if (p.vec) {
        if (p.dtype == MQ_BF16) return launch_gemv_as<MT, MQ_BF16, true>(p, sms, stream);
        if (p.dtype == MQ_FP16) return launch_gemv_as<MT, MQ_FP16, true>(p, sms, stream);
        return launch_gemv_as<MT, MQ_FP32, true>(p, sms, stream);
    }
    if (p.dtype == MQ_BF16) return launch_gemv_as<MT, MQ_BF16, false>(p, sms, stream);
    if (p.dtype == MQ_FP16) return launch_gemv_as<MT, MQ_FP16, false>(p, sms, stream);
    return launch_gemv_as<MT, MQ_FP32, false>(p, sms, stream);
}

// CTAs that share a tile along K: 1, 2, 4 or 8, as far as there are SMs and slabs.
int splits_of(long long tiles, int K, int sms) {
    int s = 1;
    while (s < 8 && tiles * s * 2 <= sms && s * 2 <= (K + 127) / 128) s *= 2;
    return s;
}

template <int BN>
int launch_gemm(GemmParams p, const int8_t* w, long long ldw, const int8_t* xq, int ldq, int sms, cudaStream_t stream) {
    using G = Gemm<BN>;
    static bool set[MAX_DEV];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (!set[dev]) {
        if ((e = cudaFuncSetAttribute(gemm_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::SMEM)) != cudaSuccess) return (int)e;
        set[dev] = true;
    }
    p.ntok = (p.M + BN - 1) / BN;
    long long tiles = (long long)((p.N + 127) / 128) * p.ntok;
    p.rows = 128;
    if (tiles > sms) {
        // as many rounds of tiles as before, but of a height that fills the last one (151936 channels: 9 rounds of 116
        // instead of 8 of 128 and one that 3 SMs have work in; 64 tokens 36.6 -> 35.0 us)
        const long long rounds = (tiles + sms - 1) / sms, across = rounds * sms / p.ntok;
        const long long rows = ((p.N + across - 1) / across + 3) / 4 * 4;
        if (rows < 128) p.rows = (int)rows;
        tiles = ((long long)p.N + p.rows - 1) / p.rows * p.ntok;
    }
    if (tiles > 0x7fffffff / 8) return MQ_ERR_SIZE;
    p.tiles = (int)tiles;
    CUtensorMap mw, mx;
    int rc = encode_map(&mw, w, p.N, p.K, ldw, p.rows);
    if (rc == MQ_OK) rc = encode_map(&mx, xq, p.M, p.K, ldq, BN);
    if (rc != MQ_OK) return rc;
    p.splits = splits_of(tiles, p.K, sms);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(p.splits > 1 ? p.tiles * p.splits : (tiles < sms ? (int)tiles : sms)));
    cfg.blockDim = dim3(G::THREADS);
    cfg.dynamicSmemBytes = G::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    pdl_attr(at[0]);
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)p.splits;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, gemm_kernel<BN>, mw, mx, p);
}

int launch_pair(GemmParams p, const int8_t* w, long long ldw, const int8_t* xq, int ldq, int sms, cudaStream_t stream) {
    static bool set[MAX_DEV];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (!set[dev]) {
        if ((e = cudaFuncSetAttribute(gemm_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Pair::SMEM)) != cudaSuccess) return (int)e;
        set[dev] = true;
    }
    const int os = p.out_dtype == MQ_FP32 ? 4 : 2;
    CUtensorMap mw, mx, mo{};
    int rc = encode_map(&mw, w, p.N, p.K, ldw, 128);
    if (rc == MQ_OK) rc = encode_map(&mx, xq, p.M, p.K, ldq, 128);
    p.tma_out = aligned(p.out, 16) && (long long)p.N * os % 16 == 0;
    if (rc == MQ_OK && p.tma_out) rc = encode_map(&mo, p.out, p.M, p.N, (long long)p.N * os, 32, p.out_dtype);
    if (rc != MQ_OK) return rc;
    p.ntok = (p.M + 255) / 256;
    const long long tiles = (long long)((p.N + 255) / 256) * p.ntok;
    if (tiles > 0x7fffffff / 8) return MQ_ERR_SIZE;
    p.tiles = (int)tiles;
    const int pairs = tiles < sms / 2 ? (int)tiles : sms / 2;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(Pair::THREADS);
    cfg.dynamicSmemBytes = Pair::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute at[2];
    pdl_attr(at[0]);
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = 2;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, gemm_pair_kernel, mw, mx, mo, p);
}

}  // namespace
}  // namespace lin8
}  // namespace mq

using namespace mq;
using namespace mq::lin8;

extern "C" int mq_linear8_workspace_bytes(int M, int K, size_t* bytes) {
    if (!bytes || M < 0 || K < 1) return MQ_ERR_ARG;
    *bytes = round_up((size_t)M * round_up(K, 16), 256) + round_up((size_t)M * 4, 16);
    return MQ_OK;
}

extern "C" int mq_linear8(const void* x, int dtype, int64_t x_stride, const int8_t* w, int64_t w_stride, const float* w_scale,
                          void* out, int out_dtype, int M, int N, int K, void* workspace, size_t workspace_bytes, int* status,
                          cudaStream_t stream) {
    if (dtype < MQ_BF16 || dtype > MQ_FP32 || out_dtype < MQ_BF16 || out_dtype > MQ_FP32 || M < 0 || N < 1 || K < 1) return MQ_ERR_ARG;
    if (M == 0) return MQ_OK;
    if (!x || !w || !w_scale || !out || !status) return MQ_ERR_ARG;
    if (K > 131072) return MQ_ERR_SIZE;                   // the int32 sum
    if (N > 0x7fffff00 || M > 0x7fffff00) return MQ_ERR_SIZE;
    const int es = dtype == MQ_FP32 ? 4 : 2, os = out_dtype == MQ_FP32 ? 4 : 2;
    if (x_stride < 0 || w_stride < (int64_t)round_up(K, 16) || w_stride % 16 != 0) return MQ_ERR_ARG;
    if (!aligned(x, es) || !aligned(out, os) || !aligned(w, 16) || !aligned(w_scale, 4) || !aligned(status, 4)) return MQ_ERR_ARG;
    int dev = 0, sms = 0;
    int rc = sm_count(dev, sms);
    if (rc != MQ_OK) return rc;
    const int vec = aligned(x, 16) && (x_stride * es) % 16 == 0;
    if (few_tokens(M, N, K)) {
        GemvParams g{x, x_stride, dtype, vec, out_dtype, M, N, K, w, w_stride, w_scale, out};
        return M == 1 ? launch_gemv<1>(g, sms, stream) : M == 2 ? launch_gemv<2>(g, sms, stream) : launch_gemv<4>(g, sms, stream);
    }
    const int ldq = (int)round_up(K, 16);
    const size_t codes = round_up((size_t)M * ldq, 256);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < codes + (size_t)M * 4) return MQ_ERR_SIZE;
    QuantParams q{x, x_stride, dtype, vec, M, K, ldq, (int8_t*)workspace, (float*)((uint8_t*)workspace + codes)};
    const LaunchLock lock(workspace);   // the product reads the codes of this call's quantiser
    if ((rc = launch_quantize(q, stream)) != MQ_OK) return rc;
    GemmParams p{q.scale, w_scale, out, status, out_dtype, M, N, K, 0, 0, 1, 0, 128};
    // Pairs of CTAs where there is a tile for every pair.
    if (M > 128 && (long long)((M + 255) / 256) * ((N + 255) / 256) >= sms / 2) return launch_pair(p, w, w_stride, q.q, ldq, sms, stream);
    if (M <= 16) return launch_gemm<16>(p, w, w_stride, q.q, ldq, sms, stream);
    if (M <= 32) return launch_gemm<32>(p, w, w_stride, q.q, ldq, sms, stream);
    // The width that a model of the kernel calls fastest: an SM takes operands in at about 64 GB/s (2 ns for a row of a
    // slab), the rounds follow one another, the last accumulator is put out at 30 ns a token, a split costs 1 us.
    // (136 tokens x 451 x K 185: 17.3 us with 256 tokens a tile, 9.7 with 64; 599 x 2138 x 4818: 28 and 33.)
    double best = 0.;
    int width = 0;
    for (int bn = 64; bn <= 256; bn *= 2) {
        const long long tiles = (long long)((N + 127) / 128) * ((M + bn - 1) / bn);
        const int s = splits_of(tiles, K, sms);
        const double t = (double)((tiles * s + sms - 1) / sms) * ((K + 128 * s - 1) / (128 * s)) * (128 + bn) * 0.002 + 0.03 * bn + (s > 1 ? 1. : 0.);
        if (!width || t < best) { best = t; width = bn; }
    }
    if (width == 64) return launch_gemm<64>(p, w, w_stride, q.q, ldq, sms, stream);
    if (width == 128) return launch_gemm<128>(p, w, w_stride, q.q, ldq, sms, stream);
    return launch_gemm<256>(p, w, w_stride, q.q, ldq, sms, stream);
}
