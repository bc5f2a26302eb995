// Rows of 8-bit codes with one scale a row, for products in 8-bit integers (linear_int8.cuh): of activations or weights as they are, and
// of their root-mean-square norm with the shortcut's addition in front.
//
//   quantize   a = max_c |x_c|            scale = a / 127                                  q_c = 127 x_c / a, nearest, ties to even
//   norm       h = x + residual in x's type, u_c = h_c w_c in 32 bits, a = max_c |u_c|
//              scale = a / 127 / sqrt(mean_c h_c^2 + eps)                                  q_c = 127 u_c / a, likewise
//
// The norm is a factor of the whole row, so the codes do not depend on it: only the scale does, and codes come out the same whatever
// the order in which the squares were added.  h is rounded to x's type before anything else looks at it, so that the norm is that of
// the tensor that is handed on; u is held in 32 bits; the quotient 127 u / a is rounded as in exact arithmetic (code_words).  A row
// whose a is below 2^-119, where a / 127 leaves the normal numbers, has scale 0 and codes 0.  A row with a NaN or an infinity (or one
// whose u is beyond 32 bits) has scale NaN and codes 0, so that it stays NaN through a product.
//
// Bound by the bytes for long batches.  A row is read once, 16 bytes a load, and stays in registers between its maximum and its codes; what
// kept these kernels from memory's rate at first was the number of instructions a value takes (25 to 75; now 14 to 20), most of them
// addresses and what a thread does once per row, so that a thread has 16 to 64 values.  Measured: 16384 x 4096 bf16 with a shortcut 84 us =
// 5.6 TB/s of 6.55; 200704 x 64 float with a shortcut 29 us = 5.8; 256 x 64 x 56 x 56 float NCHW 47.5 us = 5.5; 7777 x 1001 half 8.3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "wg_common.cuh"

namespace wg {

constexpr float kTinyRow = 0x1p-119f;
constexpr float kRound = 12582912.f;        // 1.5 * 2^23: a sum with it is rounded to a whole number (ties to even), in its low bits
constexpr float kNearTie = 0.49999f;        // see code_words

enum { kQuantize = 0, kNorm = 1, kNormRes = 2 };

struct RowsParams {
    const void *X, *R;          // x; the shortcut (kNormRes)
    void *H;                    // x + shortcut (kNormRes); may lie exactly over X or R
    const void *Wt;             // the norm's weights, C of them
    signed char *Q;
    float *scale;
    long long ldx, ldr, ldh, ldq, rows;
    int C, HW;                  // HW: pixels of a plane (NCHW)
    int group;                  // threads of a row, where a block has several rows; NCHW: warps of 32 pixels
    int w_f32, relu;
    unsigned inv;               // NCHW: ceil(2^32 / pieces of a row of codes), see there
    float eps;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// max(a, |b|) for a that is not negative; NaN stays
__device__ __forceinline__ float mag_max(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}
// max(x, low), low = 0 for a ReLU (NaN stays) and -infinity for none
__device__ __forceinline__ float at_least(float x, float low)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
    return r;
}

// 16 bytes, and the N = 4 or 8 values that they are.  Sums are rounded once to the type: the same as through 32 bits, which hold 2 p + 2
// bits of both types' p.
struct Pack { unsigned w[4]; };
__device__ __forceinline__ Pack pack_at(const void *p)
{
    const uint4 v = *static_cast<const uint4 *>(p);
    return Pack{{v.x, v.y, v.z, v.w}};
}
template <typename T> struct Types;
template <> struct Types<float> {
    static __device__ __forceinline__ void open(const Pack &k, float (&f)[4])
    {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = __uint_as_float(k.w[j]);
    }
    static __device__ __forceinline__ Pack sum(const Pack &a, const Pack &b)
    {
        Pack k;
#pragma unroll
        for (int j = 0; j < 4; ++j) k.w[j] = __float_as_uint(__fadd_rn(__uint_as_float(a.w[j]), __uint_as_float(b.w[j])));
        return k;
    }
    static __device__ __forceinline__ unsigned bits(float v) { return __float_as_uint(v); }
    static __device__ __forceinline__ float value(unsigned b) { return __uint_as_float(b); }
};
template <> struct Types<__half> {
    static __device__ __forceinline__ void open(const Pack &k, float (&f)[8])
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __half2float(__ushort_as_half((unsigned short)(k.w[j >> 1] >> (16 * (j & 1)))));
    }
    static __device__ __forceinline__ Pack sum(const Pack &a, const Pack &b)
    {
        Pack k;
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("add.rn.f16x2 %0, %1, %2;" : "=r"(k.w[j]) : "r"(a.w[j]), "r"(b.w[j]));
        return k;
    }
    static __device__ __forceinline__ unsigned bits(__half v) { return __half_as_ushort(v); }
    static __device__ __forceinline__ __half value(unsigned b) { return __ushort_as_half((unsigned short)b); }
};
template <> struct Types<__nv_bfloat16> {
    static __device__ __forceinline__ void open(const Pack &k, float (&f)[8])
    {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(j & 1 ? k.w[j >> 1] & 0xffff0000u : k.w[j >> 1] << 16);
    }
    static __device__ __forceinline__ Pack sum(const Pack &a, const Pack &b)
    {
        Pack k;
#pragma unroll
        for (int j = 0; j < 4; ++j) asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(k.w[j]) : "r"(a.w[j]), "r"(b.w[j]));
        return k;
    }
    static __device__ __forceinline__ unsigned bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }
    static __device__ __forceinline__ __nv_bfloat16 value(unsigned b) { return __ushort_as_bfloat16((unsigned short)b); }
};

// The values c0 .. c0 + N - 1 of a row of C.  (Plain loads: H may lie over the tensor that is read, which the read-only path must not be
// used for.)  ODD: a row need not begin or end on 16 bytes, p + c0 does; a piece that reaches beyond the row is read whole where it lies
// within the tensor [lo, hi), else value by value.
template <typename T, int N, bool ODD>
__device__ __forceinline__ Pack load_pack(const T *p, int c0, int C, const T *lo, const T *hi)
{
    Pack r = {{0, 0, 0, 0}};
    if (c0 < C) {
        if (!ODD || (p + c0 >= lo && p + c0 + N <= hi)) {
            r = pack_at(p + c0);
        } else {
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (c0 + j >= 0 && c0 + j < C) r.w[j * 4 / N] |= Types<T>::bits(p[c0 + j]) << (N == 8 ? 16 * (j & 1) : 0);
        }
    }
    return r;
}
// The same on its way to shared memory (dst, and `at`, its address there); nothing for c0 >= C.  safe: all of it lies within the tensor.
template <typename T, int N>
__device__ __forceinline__ void fetch_pack(uint4 *dst, uint32_t at, const T *p, int c0, int C, bool safe, const T *lo, const T *hi)
{
    if (c0 >= C) return;
    if (safe || (p + c0 >= lo && p + c0 + N <= hi)) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(p + c0) : "memory");
    } else {
        const Pack r = load_pack<T, N, true>(p, c0, C, lo, hi);
        *dst = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    }
}
// What lies behind a row's end becomes zero
template <typename T, int N>
__device__ __forceinline__ void clear_outside(Pack &r, int c0, int C)
{
    if (c0 + N > C) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c0 + j >= C) r.w[j * 4 / N] &= N == 8 ? (j & 1 ? 0x0000ffffu : 0xffff0000u) : 0u;
    }
}
template <typename T, int N, bool ODD>
__device__ __forceinline__ void store_pack(T *p, int c0, int C, const Pack &r)
{
    if ((!ODD || c0 >= 0) && c0 + N <= C) {
        *reinterpret_cast<uint4 *>(p + c0) = make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
    } else if (ODD) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c0 + j >= 0 && c0 + j < C) p[c0 + j] = Types<T>::value(r.w[j * 4 / N] >> (N == 8 ? 16 * (j & 1) : 0));
    }
}
__device__ __forceinline__ float weight_at(const RowsParams &p, const float *, int c) { return static_cast<const float *>(p.Wt)[c]; }
template <typename T>
__device__ __forceinline__ float weight_at(const RowsParams &p, const T *, int c)
{
    return p.w_f32 ? static_cast<const float *>(p.Wt)[c] : to_f(static_cast<const T *>(p.Wt)[c]);
}
// N weights from channel c0 on
template <typename T, int N>
__device__ __forceinline__ void load_weights(const RowsParams &p, int c0, float (&w)[N])
{
    const bool f32 = sizeof(T) == 4 || p.w_f32;
    const char *at = static_cast<const char *>(p.Wt) + (long long)c0 * (f32 ? 4 : 2);
    if (c0 >= 0 && c0 + N <= p.C && (reinterpret_cast<uintptr_t>(at) & 15u) == 0) {
        if (f32) {
#pragma unroll
            for (int j = 0; j < N; j += 4) {
                const float4 t = reinterpret_cast<const float4 *>(at)[j / 4];
                w[j] = t.x; w[j + 1] = t.y; w[j + 2] = t.z; w[j + 3] = t.w;
            }
        } else {
            Types<T>::open(pack_at(at), w);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = c0 + j >= 0 && c0 + j < p.C ? weight_at(p, (const T *)nullptr, c0 + j) : 0.f;
    }
}

// The code of u beyond doubt: the half way point next to u inv (which is within 7.6e-6 of 127 u / a) is compared with 127 u / a, or rather
// 127 u with that many a, as sums of two 32-bit numbers each.  Where they are close the high parts lie within a factor of two of each
// other and the low ones have 8 bits, so that every difference is exact.  `scale` moves both to where nothing overflows or is denormal.
__device__ __forceinline__ unsigned sure_code(float u, float inv, float a, float scale)
{
    const float r = __fsub_rn(fmaf(u, inv, kRound), kRound), e = fmaf(u, inv, -r), half = r + (e >= 0.f ? 0.5f : -0.5f);
    const float v = u * scale, p = __fmul_rn(127.f, v), q = __fmul_rn(half, a);
    const float d = __fadd_rn(__fsub_rn(p, q), __fsub_rn(fmaf(127.f, v, -p), fmaf(half, a, -q)));
    const unsigned below = __float_as_uint((half - 0.5f) + kRound);
    return below + (d > 0.f || (d == 0.f && (below & 1u)) ? 1u : 0u);
}
__device__ __noinline__ unsigned sure_word(float u0, float u1, float u2, float u3, float inv, float a)
{
    const float s = a >= 2.f ? 0x1p-64f : 0x1p64f, b = a * s;
    return __byte_perm(__byte_perm(sure_code(u0, inv, b, s), sure_code(u1, inv, b, s), 0x0040),
                       __byte_perm(sure_code(u2, inv, b, s), sure_code(u3, inv, b, s), 0x0040), 0x5410);
}

// Codes of N values, four a word.  inv = 127 / a rounded, so |u inv - 127 u / a| <= 127 * 2^-24 = 7.6e-6.  m holds the whole number
// nearest to u inv, which the fused multiply-add rounds once; d, its distance, is exact to 3e-8.  Wherever |d| <= 0.49999 that number is
// also the one nearest to 127 u / a; elsewhere sure_word says.  a below kTinyRow or not finite: inv = 0, and the caller clears the codes.
//
// Values of 16-bit types (COARSE) are half way between two codes in nearly every row (u = a / 2; every second value where a's mantissa is a
// multiple of 127), but never close to it without being there: for u, a of at most 11 bits 254 u / ((2 k + 1) a) is a quotient of whole
// numbers below 2^19, so it is 1 or differs from it by 2^-19.  u inv, rounded twice, is within 2^-23 of 127 u / a, two units of its last
// place (four below 1/2): rounded to a multiple of eight of them it is k + 1/2 where that is the case, and on its own side of it where not.
template <int N, bool COARSE>
__device__ __forceinline__ float fast_codes(const float (&u)[N], float inv, unsigned (&w)[N / 4], float off = 0.f)      // -> the largest |d|
{
#pragma unroll
    for (int g = 0; g < N / 4; ++g) {
        unsigned r[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float x = u[4 * g + j];
            float m;
            if (COARSE) {
                m = __fadd_rn(__uint_as_float((__float_as_uint(__fmul_rn(x, inv)) + 4u) & ~7u), kRound);
            } else {
                m = fmaf(x, inv, kRound);
                off = fmaxf(off, fabsf(fmaf(x, inv, -__fsub_rn(m, kRound))));
            }
            r[j] = __float_as_uint(m);
        }
        w[g] = __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
    }
    return off;
}
template <int N>
__device__ __forceinline__ void mend_codes(const float (&u)[N], float inv, float a, unsigned (&w)[N / 4])
{
#pragma unroll
    for (int g = 0; g < N / 4; ++g) w[g] = sure_word(u[4 * g], u[4 * g + 1], u[4 * g + 2], u[4 * g + 3], inv, a);
}
template <int N, bool COARSE>
__device__ __forceinline__ void code_words(const float (&u)[N], float inv, float a, unsigned (&w)[N / 4])
{
    if (fast_codes<N, COARSE>(u, inv, w) > kNearTie) mend_codes<N>(u, inv, a, w);
}

struct RowCodes {
    float inv, a;
    unsigned live;                // all ones, or zero where the codes are 0 whatever u
};
constexpr float kDown = 0x1p-100f;     // for a row whose squares leave 32 bits: some |h| is above 2^64 / sqrt(C), all are below 2^128
__device__ __forceinline__ RowCodes row_codes(float a)
{
    RowCodes k;
    k.a = a;
    const bool ok = a >= kTinyRow && a <= 3.402823466e38f;
    k.live = ok ? 0xffffffffu : 0u;
    k.inv = ok ? __fdiv_rn(127.f, a) : 0.f;
    return k;
}
__device__ __forceinline__ float row_scale(const RowCodes &k)
{
    return k.live ? __fdiv_rn(k.a, 127.f) : (k.a < kTinyRow ? 0.f : __uint_as_float(0x7fffffffu));
}
// scale / sqrt(mean square + eps); ss: the sum of the squares of h, or of kDown * h
__device__ __forceinline__ float norm_scale(const RowCodes &k, float ss, int C, float eps, bool down)
{
    const float scale = row_scale(k);
    if (!k.live) return scale;
    const float mean = __fdiv_rn(ss, (float)C);
    if (down) {
        const float root = __fsqrt_rn(mean + eps * kDown * kDown);
        return scale > 1.f ? __fdiv_rn(scale * kDown, root) : __fdiv_rn(scale, root) * kDown;
    }
    return __fdiv_rn(scale, 2.f * __fsqrt_rn(fmaf(0.25f, mean, 0.25f * eps)));         // (of a quarter: the sum of both can leave 32 bits)
}

// The largest magnitude and the sum over `width` lanes (2 to 32).  By shuffles: the warp's own reduction (__reduce_max_sync), behind the ends
// of a row that some lanes handle apart, left out what those lanes had.
template <bool SUM>
__device__ __forceinline__ void reduce_lanes(float &a, float &ss, int width)
{
    for (int o = width >> 1; o; o >>= 1) a = mag_max(a, __shfl_xor_sync(0xffffffffu, a, o));
    if (SUM)
        for (int o = width >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
}
// Over the block; every thread has the result, from the same order of additions.  `part`: 32 of them, not those of the call before (whose
// values other warps may still be reading).
template <bool SUM>
__device__ __forceinline__ void reduce_block(float &a, float &ss, float2 *part)
{
    reduce_lanes<SUM>(a, ss, 32);
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    if (lane == 0) part[threadIdx.x >> 5] = make_float2(a, ss);
    __syncthreads();
    a = ss = 0.f;
    if (warps <= 8) {
        for (int w = 0; w < warps; ++w) {
            const float2 v = part[w];
            a = mag_max(a, v.x);
            ss += v.y;
        }
    } else {
        if (lane < warps) { a = part[lane].x; ss = part[lane].y; }
        reduce_lanes<SUM>(a, ss, 32);
    }
}

// Rows in registers: V loads of 16 bytes a thread and tensor.  BLOCK: a row per block, else blockDim.x / group rows.  A warp has
// neighbouring pieces of a row, V times 32 of them (or V times 2 to 16, where it has several rows).
// AHEAD: a block has several rows (or blocks of rows) in turn, and the loads of the next AHEAD of them are on their way to shared memory
// while it works on one.  Every thread fetches the pieces that it uses itself (but for ODD), so nothing waits for other threads.  (16384 x 4096 bf16 with
// a shortcut: AHEAD = 1 and V = 4 85 us, AHEAD = 2 90, V = 2 100; the next row in registers instead 130.)
// ODD: rows that do not begin on 16 bytes, or whose length is not a multiple; x, shortcut and sum have the same offset to a 16-byte
// boundary in every row.  The aligned pieces that a row touches come to shared memory; there the shortcut is added to them, and every
// thread then reads its N channels at the offset that the row has.  A row can touch a piece more than its length has; the thread of its first
// channels fetches that one too (a load slot for it left half of the slots empty
// where the length is just below a power of two: 65536 x 255 float 40 us, now 24, 8192 x 4095 with a shortcut 117, 88).
template <typename T, int MODE, int V, bool BLOCK, bool ODD, int AHEAD>
__global__ void __launch_bounds__(BLOCK ? (V == 1 || (V == 4 && AHEAD == 0) ? 1024 : 512) : 256, !BLOCK && V == 4 ? 3 : 1) rows_kernel(const RowsParams p)
{
    constexpr int N = 16 / sizeof(T), WORDS = N / 4, STAGES = AHEAD + 1;
    constexpr bool SUM = MODE != kQuantize;
    // [STAGES][x, shortcut][V][thread], ODD: [STAGES][x, shortcut][row][V * threads of a row + 1]; then the weights of the thread's channels
    extern __shared__ uint4 ring[];
    __shared__ float2 part[BLOCK ? 3 * 32 : 1];
    constexpr bool W_AT_HAND = SUM && AHEAD;
    wait_for_previous_kernel(kNumSMs);
    const int lane = threadIdx.x & 31;
    const int width = BLOCK ? 32 : p.group, at = lane & (width - 1);
    const int i0 = BLOCK ? (threadIdx.x >> 5) * (32 * V) + lane : at;           // the thread's pieces: i0 + v * width
    const int per_block = BLOCK ? 1 : blockDim.x / p.group, mine = BLOCK ? 0 : threadIdx.x / p.group;
    const long long stride = (long long)gridDim.x * per_block, first = (long long)blockIdx.x * per_block;
    const float low = p.relu ? 0.f : __uint_as_float(0xff800000u);
    const T *X = static_cast<const T *>(p.X), *R = static_cast<const T *>(p.R);
    const T *x_end = X + (p.rows - 1) * p.ldx + p.C, *r_end = R + (p.rows - 1) * p.ldr + p.C;
    auto offset = [&](const T *x) { return ODD ? (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)) : 0; };

    // The block's rows first + mine, + stride, ...: tensors at the row in work, and at the one to be fetched
    const T *x = X + (first + mine) * p.ldx, *r = R + (first + mine) * p.ldr, *xf = x, *rf = r;
    T *h = static_cast<T *>(p.H) + (first + mine) * p.ldh;
    signed char *q = p.Q + (first + mine) * p.ldq;
    const long long x_step = stride * p.ldx, r_step = stride * p.ldr, h_step = stride * p.ldh, q_step = stride * p.ldq;
    // piece v of the thread, of stage s: ring[s * stage + v * slot + mine_in], the shortcut's at + half
    const int in_row = (BLOCK ? (int)blockDim.x : p.group) * V;
    const int slot = ODD ? width : blockDim.x, mine_in = ODD ? mine * (in_row + 1) + i0 : threadIdx.x;
    const int half = ODD ? per_block * (in_row + 1) : V * blockDim.x, stage = MODE == kNormRes ? 2 * half : half;
    const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
    long long next = first;
    int put = 0, get = 0, turn = 0;
    auto fetch = [&] {                  // the loads of the block's row `next`, to stage `put`
        if (next < p.rows && (BLOCK || next + mine < p.rows)) {
            const int mis = offset(xf), at0 = put * stage + mine_in;
            // (whether every piece of the row lies within the tensors)
            const bool safe = !ODD || (xf - N >= X && xf + p.C + N <= x_end && (MODE != kNormRes || (rf - N >= R && rf + p.C + N <= r_end)));
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int c0 = (i0 + v * width) * N - mis, o = at0 + v * slot;
                fetch_pack<T, N>(ring + o, ring_at + 16u * o, xf, c0, p.C, safe, X, x_end);
                if (MODE == kNormRes) fetch_pack<T, N>(ring + o + half, ring_at + 16u * (o + half), rf, c0, p.C, safe, R, r_end);
            }
            if (ODD && i0 == 0) {
                const int c0 = in_row * N - mis, o = at0 + in_row;
                fetch_pack<T, N>(ring + o, ring_at + 16u * o, xf, c0, p.C, safe, X, x_end);
                if (MODE == kNormRes) fetch_pack<T, N>(ring + o + half, ring_at + 16u * (o + half), rf, c0, p.C, safe, R, r_end);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        next += stride;
        xf += x_step;
        if (MODE == kNormRes) rf += r_step;
        put = put + 1 < STAGES ? put + 1 : 0;
    };
    float4 *const weights = reinterpret_cast<float4 *>(ring + STAGES * stage) + threadIdx.x;
    if (AHEAD) {
        for (int s = 0; s < AHEAD; ++s) fetch();
        if (W_AT_HAND)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float w[N];
                load_weights<T, N>(p, (i0 + v * width) * N, w);
#pragma unroll
                for (int j = 0; j < N; j += 4) weights[(v * N + j) / 4 * blockDim.x] = make_float4(w[j], w[j + 1], w[j + 2], w[j + 3]);
            }
    }
    for (long long base = first; base < p.rows; base += stride) {
        const long long row = base + mine;
        const bool have = BLOCK || row < p.rows;
        const int C = have ? p.C : -N;                  // (nothing of a row that is not there)
        const int mis = offset(x);
        float u[V][N];
        if (ODD && !BLOCK) __syncwarp();                // the stage that is fetched into has been read by all lanes
        if (AHEAD || ODD) {
            fetch();
            asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
        }
        uint4 *const got = ring + get * stage + mine_in;
        if (ODD) {
            if (MODE == kNormRes) {
                auto add = [&](uint4 *piece, int c0) {
                    if (c0 >= C) return;
                    const Pack sum = Types<T>::sum(pack_at(piece), pack_at(piece + half));
                    store_pack<T, N, true>(h, c0, C, sum);
                    *piece = make_uint4(sum.w[0], sum.w[1], sum.w[2], sum.w[3]);
                };
#pragma unroll
                for (int v = 0; v < V; ++v) add(got + v * slot, (i0 + v * width) * N - mis);
                if (i0 == 0) add(got + in_row, in_row * N - mis);
            }
            if (BLOCK) __syncthreads();
            else __syncwarp();
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c0 = (i0 + v * width) * N;
            Pack a = {{0, 0, 0, 0}};
            if (ODD) {
                if (c0 < C) {
                    // (two loads of 16 bytes and selects: word by word, four lanes at a time met in the same banks)
                    const Pack s0 = pack_at(got + v * slot), s1 = pack_at(got + v * slot + 1);
                    const bool one = mis * (int)sizeof(T) & 4, two = mis * (int)sizeof(T) & 8;
                    unsigned r[7], t[5];
#pragma unroll
                    for (int j = 0; j < 7; ++j) {
                        const unsigned here = j < 4 ? s0.w[j & 3] : s1.w[j & 3], next = j < 3 ? s0.w[(j + 1) & 3] : s1.w[(j + 1) & 3];
                        r[j] = one ? next : here;
                    }
#pragma unroll
                    for (int j = 0; j < 5; ++j) t[j] = two ? r[j + 2] : r[j];
#pragma unroll
                    for (int j = 0; j < 4; ++j) a.w[j] = N == 8 ? __funnelshift_r(t[j], t[j + 1], 16 * (mis & 1)) : t[j];
                }
                clear_outside<T, N>(a, c0, C);
            } else {
                Pack b = a;
                if (AHEAD) {
                    if (c0 < C) {
                        a = pack_at(got + v * slot);
                        if (MODE == kNormRes) b = pack_at(got + v * slot + half);
                    }
                } else {
                    a = load_pack<T, N, false>(x, c0, C, X, x_end);
                    if (MODE == kNormRes) b = load_pack<T, N, false>(r, c0, C, R, r_end);
                }
                if (MODE == kNormRes) {
                    a = Types<T>::sum(a, b);
                    store_pack<T, N, false>(h, c0, C, a);
                }
            }
            Types<T>::open(a, u[v]);
        }
        get = get + 1 < STAGES ? get + 1 : 0;
        float amax = 0.f, ss = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (MODE != kQuantize) {
                float w[N];
                if (W_AT_HAND) {
#pragma unroll
                    for (int j = 0; j < N; j += 4) {
                        const float4 t = weights[(v * N + j) / 4 * blockDim.x];
                        w[j] = t.x; w[j + 1] = t.y; w[j + 2] = t.z; w[j + 3] = t.w;
                    }
                } else {
                    load_weights<T, N>(p, (i0 + v * width) * N, w);
                }
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    ss = fmaf(u[v][j], u[v][j], ss);
                    u[v][j] = __fmul_rn(u[v][j], w[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j) u[v][j] = at_least(u[v][j], low);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) amax = mag_max(amax, u[v][j]);
        }
        if (BLOCK) reduce_block<SUM>(amax, ss, part + 32 * turn);
        else reduce_lanes<SUM>(amax, ss, width);
        turn ^= 1;
        RowCodes k = row_codes(amax);
        if (MODE != kQuantize) {
            const bool down = k.live && !(ss <= 3.402823466e38f);
            if (BLOCK ? down : __any_sync(0xffffffffu, down)) {        // the squares of a row of large values: once more, scaled (h as it was stored)
                float s2 = 0.f, none = 0.f;
#pragma unroll 1
                for (int v = 0; v < V; ++v)
                    for (int j = 0; j < N; ++j) {
                        const int c = (i0 + v * width) * N + j;
                        if (c >= C) continue;
                        const float f = to_f(MODE == kNormRes ? h[c] : x[c]) * kDown;
                        s2 = fmaf(f, f, s2);
                    }
                if (BLOCK) {
                    reduce_block<true>(none, s2, part + 64);
                    __syncthreads();
                } else {
                    reduce_lanes<true>(none, s2, width);
                }
                if (down) ss = s2;
            }
            if (have && i0 == 0) p.scale[row] = norm_scale(k, ss, p.C, p.eps, down);
        } else if (have && i0 == 0) {
            p.scale[row] = row_scale(k);
        }

        unsigned w[V][WORDS];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            code_words<N, MODE == kQuantize && N == 8>(u[v], k.inv, k.a, w[v]);
#pragma unroll
            for (int g = 0; g < WORDS; ++g) w[v][g] &= k.live;
        }
        const bool whole = !ODD || (reinterpret_cast<uintptr_t>(q) & (N - 1)) == 0;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c0 = (i0 + v * width) * N;
            if (ODD ? c0 + N <= C && whole : c0 < C) {
                if (WORDS == 2) *reinterpret_cast<uint2 *>(q + c0) = make_uint2(w[v][0], w[v][WORDS - 1]);
                else *reinterpret_cast<unsigned *>(q + c0) = w[v][0];
            } else if (ODD && c0 < C) {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (c0 + j < C) q[c0 + j] = (signed char)(w[v][j >> 2] >> (8 * (j & 3)));
            }
        }
        x += x_step;
        if (MODE == kNormRes) { r += r_step; h += h_step; }
        q += q_step;
    }
}

// Rows of any length and alignment, value by value; read a second time for the codes (from L2): what rows_kernel does not hold, and, with
// NCHW, images of more channels than nchw_kernel's shared memory takes codes of (some 6000).
template <typename T, int MODE, bool NCHW>
__global__ void __launch_bounds__(512) rows_any_kernel(const RowsParams p)
{
    __shared__ float2 part[2 * 32];
    wait_for_previous_kernel(kNumSMs);
    const long long row = blockIdx.x, step = NCHW ? p.HW : 1, pixel = NCHW ? row / p.HW * p.C * p.HW + row % p.HW : 0;
    const T *x = static_cast<const T *>(p.X) + (NCHW ? pixel : row * p.ldx);
    const T *res = MODE == kNormRes ? static_cast<const T *>(p.R) + (NCHW ? pixel : row * p.ldr) : nullptr;
    T *h = MODE == kNormRes ? static_cast<T *>(p.H) + (NCHW ? pixel : row * p.ldh) : nullptr;
    const T *again = MODE == kNormRes ? h : x;
    auto value = [&](int c) {
        const float v = to_f(again[c * step]);
        return MODE != kQuantize ? __fmul_rn(v, weight_at(p, (const T *)nullptr, c)) : p.relu ? relu_nan(v) : v;
    };
    float amax = 0.f, ss = 0.f;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        if (MODE == kNormRes) h[c * step] = from_f<T>(__fadd_rn(to_f(x[c * step]), to_f(res[c * step])));
        const float v = to_f(again[c * step]);
        ss = fmaf(v, v, ss);
        amax = mag_max(amax, value(c));
    }
    reduce_block<true>(amax, ss, part);
    RowCodes k = row_codes(amax);
    if (MODE != kQuantize && k.live) {
        const bool down = !(ss <= 3.402823466e38f);
        if (down) {
            float none = 0.f;
            ss = 0.f;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                const float f = to_f(again[c * step]) * kDown;
                ss = fmaf(f, f, ss);
            }
            reduce_block<true>(none, ss, part + 32);
        }
        if (threadIdx.x == 0) p.scale[row] = norm_scale(k, ss, p.C, p.eps, down);
    } else if (threadIdx.x == 0) {
        p.scale[row] = row_scale(k);
    }
    signed char *q = p.Q + row * p.ldq;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        const float u[4] = {value(c), 0.f, 0.f, 0.f};
        unsigned w[1];
        code_words<4, MODE == kQuantize && sizeof(T) == 2>(u, k.inv, k.a, w);
        q[c] = (signed char)(w[0] & k.live);
    }
}

// NCHW: lane = pixel (of any images), so that a load is 32 consecutive values of a plane.  p.group warps share a tile of 32 pixels, each
// with groups of four neighbouring channels, whose codes are a word: NQ groups a thread (0: any number, read a second time).  As many as
// registers allow, because a thread has costs of its own per pixel (its image, the divisions, the meeting of its warps).  With a shortcut, sixteen groups
// a thread (more than 512 channels) are a few more than that: 12 to 68 bytes of a thread are spilled where all groups exist, 160 to 216
// elsewhere, and still faster than reading twice (us: 64 x 1024 x 14 x 14 half 40 / 80, float 42 / 53, 128 x 600 x 7 x 7 bf16 24.9 / 26.4).  The words are
// turned through shared memory and leave as pieces of rows.
template <typename T, int MODE, int NQ, bool FULL>
__global__ void __launch_bounds__(512) nchw_kernel(const RowsParams p)
{
    extern __shared__ __align__(16) unsigned turned_all[];        // [tile of the block][32][pitch], then the weights
    __shared__ float2 part[2][16][32];
    constexpr bool SUM = MODE != kQuantize, COARSE = MODE == kQuantize && sizeof(T) == 2;
    wait_for_previous_kernel(kNumSMs);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = p.group;
    const int tile = warp / share, wi = warp - tile * share, tiles = (blockDim.x >> 5) / share;
    const long long row0 = ((long long)blockIdx.x * tiles + tile) * 32, row = row0 + lane;
    const bool have = row < p.rows;
    const long long src = have ? row : p.rows - 1;          // (a lane without a pixel reads the last one, and stores nothing)
    long long base;
    if (p.rows <= 0x7fffffffLL) {
        const unsigned b = (unsigned)src / (unsigned)p.HW;
        base = (long long)b * p.C * p.HW + ((unsigned)src - b * (unsigned)p.HW);
    } else {
        const long long b = src / p.HW;
        base = b * p.C * p.HW + (src - b * p.HW);
    }
    const T *x = static_cast<const T *>(p.X) + base;
    const T *res = MODE == kNormRes ? static_cast<const T *>(p.R) + base : nullptr;
    T *h = MODE == kNormRes ? static_cast<T *>(p.H) + base : nullptr;
    const int C = p.C, words = (C + 3) >> 2, pitch = words | 1;
    const long long HW = p.HW;
    const float low = p.relu ? 0.f : __uint_as_float(0xff800000u);
    float *weights = reinterpret_cast<float *>(turned_all) + tiles * 32 * pitch;
    auto stage_weights = [&] {          // (behind the pixels' loads where those are all at hand)
        for (int c = threadIdx.x; c < 4 * words; c += blockDim.x) weights[c] = c < C ? weight_at(p, (const T *)nullptr, c) : 0.f;
        __syncthreads();
    };
    if (SUM && !NQ) stage_weights();

    constexpr int KEEP = NQ ? NQ : 1, LOOP = 4;
    float u[KEEP][4];
    float amax = 0.f, ss = 0.f;
    if (NQ) {
        // The thread's groups of four channels: wi, wi + share, ...  FULL: all of them exist.  Else those from `whole` on are read like the
        // last whole one, which costs nothing beside loads behind conditions, and replaced: by the up to three channels that are left, which
        // are read apart, and by zeros.
        const long long step = 4 * share * HW;
        const int whole = C >> 2;
        auto load = [&](const T *base, float (&v)[4], int g) {
            const T *t = base + (FULL ? g * step + 4 * wi * HW : 4LL * min(wi + g * share, whole - 1) * HW);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = to_f(t[j * HW]);
        };
        auto load_rest = [&](const T *base, float (&v)[4]) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = 4 * whole + j < C ? to_f(base[(4LL * whole + j) * HW]) : 0.f;
        };
        auto replace = [&](float (&v)[4], const float (&rest)[4], int g) {
            const int q = wi + g * share;
            if (FULL || q < whole) return;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = q == whole ? rest[j] : 0.f;
        };
        float rest[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int g = 0; g < KEEP; ++g) load(x, u[g], g);
        if (!FULL && (C & 3)) load_rest(x, rest);
#pragma unroll
        for (int g = 0; g < KEEP; ++g) replace(u[g], rest, g);
        if (SUM) stage_weights();
        if (MODE == kNormRes) {
            constexpr int HALF = KEEP > 8 ? 8 : KEEP;
#pragma unroll
            for (int g0 = 0; g0 < KEEP; g0 += HALF) {
                float r[HALF][4];
#pragma unroll
                for (int g = 0; g < HALF; ++g) load(res, r[g], g0 + g);
                if (!FULL && (C & 3)) load_rest(res, rest);
#pragma unroll
                for (int g = 0; g < HALF; ++g) {
                    replace(r[g], rest, g0 + g);
                    const int left = have ? C - 4 * (wi + (g0 + g) * share) : 0;
                    T *o = h + 4LL * (wi + (g0 + g) * share) * HW;
                    T s[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        s[j] = from_f<T>(__fadd_rn(u[g0 + g][j], r[g][j]));
                        u[g0 + g][j] = to_f(s[j]);
                    }
                    if (FULL ? have : left >= 4) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j * HW] = s[j];
                    } else if (!FULL && left > 0) {
#pragma unroll
                        for (int j = 0; j < 3; ++j)
                            if (j < left) o[j * HW] = s[j];
                    }
                }
            }
        }
#pragma unroll
        for (int g = 0; g < KEEP; ++g) {
            if (SUM) {
                const int q = wi + g * share;
                const float4 w4 = FULL || q < words ? *reinterpret_cast<const float4 *>(weights + 4 * q) : make_float4(0.f, 0.f, 0.f, 0.f);
                const float w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    ss = fmaf(u[g][j], u[g][j], ss);
                    u[g][j] = __fmul_rn(u[g][j], w[j]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) u[g][j] = at_least(u[g][j], low);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) amax = mag_max(amax, u[g][j]);
        }
    } else {
        for (int q0 = wi; q0 < words; q0 += LOOP * share) {
            float v[LOOP][4], r[LOOP][4], some = 0.f;         // some: these squares (one by one, a thread's would be up to 750 additions on one sum)
#pragma unroll
            for (int g = 0; g < LOOP; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 4 * (q0 + g * share) + j;
                    v[g][j] = c < C ? to_f(x[c * HW]) : 0.f;
                    if (MODE == kNormRes) r[g][j] = c < C ? to_f(res[c * HW]) : 0.f;
                }
#pragma unroll
            for (int g = 0; g < LOOP; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 4 * (q0 + g * share) + j;
                    if (MODE == kNormRes) {
                        const T s = from_f<T>(__fadd_rn(v[g][j], r[g][j]));
                        if (have && c < C) h[c * HW] = s;
                        v[g][j] = to_f(s);
                    }
                    if (SUM) some = fmaf(v[g][j], v[g][j], some);
                    amax = mag_max(amax, SUM ? (c < C ? __fmul_rn(v[g][j], weights[c]) : 0.f) : at_least(v[g][j], low));
                }
            ss += some;
        }
    }
    // a pixel's maximum and sum over the warps that share it; each of them adds in the same order
    auto over_warps = [&](float &m, float &s, int turn) {
        if (share == 1) return;
        part[turn][warp][lane] = make_float2(m, s);
        __syncthreads();
        m = s = 0.f;
        for (int w = 0; w < share; ++w) {
            const float2 v = part[turn][tile * share + w][lane];
            m = mag_max(m, v.x);
            s += v.y;
        }
    };
    over_warps(amax, ss, 0);
    RowCodes k = row_codes(amax);
    if (MODE != kQuantize) {
        const bool down = k.live && !(ss <= 3.402823466e38f);
        const bool any = share == 1 ? __any_sync(0xffffffffu, down) : __syncthreads_or(down);
        if (any) {
            const T *again = MODE == kNormRes ? h : x;          // (h as any of these warps stored it: there has been a barrier)
            float s2 = 0.f, none = 0.f;
            for (int c = wi; c < C; c += share) {
                const float f = to_f(again[c * HW]) * kDown;
                s2 = fmaf(f, f, s2);
            }
            over_warps(none, s2, 1);
            if (down) ss = s2;
        }
        if (wi == 0 && have) p.scale[row] = norm_scale(k, ss, p.C, p.eps, down);
    } else if (wi == 0 && have) {
        p.scale[row] = row_scale(k);
    }
    unsigned *turned = turned_all + tile * 32 * pitch;
    if (NQ) {
        unsigned w[KEEP][1];
        float off = 0.f;
#pragma unroll
        for (int g = 0; g < KEEP; ++g) off = fast_codes<4, COARSE>(u[g], k.inv, w[g], off);
        if (off > kNearTie) {
#pragma unroll
            for (int g = 0; g < KEEP; ++g) code_words<4, COARSE>(u[g], k.inv, k.a, w[g]);       // (each word with a look of its own)
        }
#pragma unroll
        for (int g = 0; g < KEEP; ++g) {
            const int q = wi + g * share;
            if (FULL || q < words) turned[lane * pitch + q] = w[g][0] & k.live;
        }
    } else {
        const T *again = MODE == kNormRes ? h : x;          // (what this thread itself has read or stored)
        for (int q0 = wi; q0 < words; q0 += LOOP * share) {
            float v[LOOP][4];
#pragma unroll
            for (int g = 0; g < LOOP; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 4 * (q0 + g * share) + j;
                    v[g][j] = c < C ? to_f(again[c * HW]) : 0.f;
                }
#pragma unroll
            for (int g = 0; g < LOOP; ++g) {
                const int q = q0 + g * share;
#pragma unroll
                for (int j = 0; j < 4; ++j) v[g][j] = SUM ? (4 * q + j < C ? __fmul_rn(v[g][j], weights[4 * q + j]) : 0.f) : at_least(v[g][j], low);
                unsigned w[1];
                code_words<4, COARSE>(v[g], k.inv, k.a, w);
                if (q < words) turned[lane * pitch + q] = w[0] & k.live;
            }
        }
    }
    {
        if (share == 1) __syncwarp();
        else __syncthreads();
        const int n = row0 < p.rows ? (int)min(32LL, p.rows - row0) : 0;
        signed char *rows = p.Q + row0 * p.ldq;
        const unsigned align = (unsigned)reinterpret_cast<uintptr_t>(p.Q) | (unsigned)p.ldq;
        // pieces of 16 bytes, and what is left of a row by the lane of its number; else words, the last one byte by byte.  i / pieces = the
        // high word of i * inv
        const bool by16 = (align & 15u) == 0;
        const int pieces = by16 ? C >> 4 : words;
        for (int i = 32 * wi + lane; i < n * pieces; i += 32 * share) {
            const int r = pieces == 1 ? i : (int)__umulhi((unsigned)i, p.inv), q = i - r * pieces;
            const unsigned *src = turned + r * pitch + (by16 ? 4 * q : q);
            signed char *dst = rows + r * p.ldq + (by16 ? 16 * q : 4 * q);
            if (by16) {
                *reinterpret_cast<uint4 *>(dst) = make_uint4(src[0], src[1], src[2], src[3]);
            } else if ((align & 3u) == 0 && 4 * q + 4 <= C) {
                *reinterpret_cast<unsigned *>(dst) = *src;
            } else {
                const unsigned w = *src;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * q + j < C) dst[j] = (signed char)(w >> (8 * j));
            }
        }
        if (by16 && (C & 15) && wi == share - 1 && lane < n) {
            const unsigned *src = turned + lane * pitch;
            signed char *dst = rows + lane * p.ldq;
            int q = pieces * 4;
            for (; 4 * q + 4 <= C; ++q) *reinterpret_cast<unsigned *>(dst + 4 * q) = src[q];
            for (int c = 4 * q; c < C; ++c) dst[c] = (signed char)(src[q] >> (8 * (c & 3)));
        }
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
// AHEAD = 0: as many blocks as there are rows (or blocks of rows); else at most as many as run at once
template <typename T, int MODE, int V, bool BLOCK, bool ODD, int AHEAD>
static int launch_rows(int threads, const RowsParams &p, cudaStream_t st)
{
    auto *kernel = rows_kernel<T, MODE, V, BLOCK, ODD, AHEAD>;
    const int tensors = MODE == kNormRes ? 2 : 1, pieces = ODD ? V * threads + (BLOCK ? 1 : threads / p.group) : V * threads;
    const size_t smem = (AHEAD || ODD ? (size_t)(AHEAD + 1) * tensors * pieces * 16 : 0) + (AHEAD && MODE != kQuantize ? (size_t)V * (16 / sizeof(T)) * 4 * threads : 0);
    long long blocks = cdivll(p.rows, BLOCK ? 1 : threads / p.group);
    if (AHEAD) {
        static const int regs = [&] {
            cudaFuncAttributes a;
            return cudaFuncGetAttributes(&a, reinterpret_cast<const void *>(kernel)) == cudaSuccess && a.numRegs > 0 ? (a.numRegs + 7) / 8 * 8 : 128;
        }();
        // (a quarter of the SM's registers for every fourth warp: five blocks of three warps with 112 registers, not six, the last of which
        // would begin when others have ended)
        const int warps = threads / 32, by_regs = 16384 / (regs * 32) * 4 / warps;
        const long long at_once = std::max(1, std::min({64 / warps, by_regs, (int)(228 * 1024 / (smem + 2048))}));
        blocks = std::min(blocks, kNumSMs * at_once);
    }
    return launch(kernel, dim3((unsigned)blocks), threads, smem, st, p);
}
template <typename T, int MODE, int V, bool BLOCK, int AHEAD>
static int launch_rows(bool odd, int threads, const RowsParams &p, cudaStream_t st)
{
    return odd ? launch_rows<T, MODE, V, BLOCK, true, AHEAD>(threads, p, st) : launch_rows<T, MODE, V, BLOCK, false, AHEAD>(threads, p, st);
}

template <typename T, int MODE>
static int rows_int8(RowsParams p, cudaStream_t st)
{
    constexpr int N = 16 / (int)sizeof(T);
    if (p.rows > 0x7fffffffLL) return WG2X2_ERR_UNSUPPORTED;
    auto offset = [](const void *q, long long ld) { return (unsigned)((reinterpret_cast<uintptr_t>(q) & 15u) | ((ld * (long long)sizeof(T)) & 15) << 4); };
    const unsigned ox = offset(p.X, p.ldx);
    const bool same = MODE != kNormRes || (offset(p.R, p.ldr) == ox && offset(p.H, p.ldh) == ox);
    const bool odd = ox || p.C % N || p.ldq % N || (reinterpret_cast<uintptr_t>(p.Q) & (N - 1));
    const long long nv = cdivll(p.C, N);
    if (!same || nv > 4096) return launch(rows_any_kernel<T, MODE, false>, dim3((unsigned)p.rows), 512, 0, st, p);
    // Rows that fit the GPU at once with a thread for every load (1024 threads an SM) are taken so: norm with a shortcut, us in a graph,
    // 300 x 1024 bf16 2.4, the other way 4.4; beyond the bound 2000 x 1283 bf16 10.6 and 8.9, 600 x 1283 float 6.9 and 4.5.  Else a row in a
    // warp or a part of one up to 128 loads, and four or eight loads a thread.
    const bool little = p.rows * nv <= 1024LL * kNumSMs;
    if (little && nv > 32 && nv <= 1024) return launch_rows<T, MODE, 1, true, 0>(odd, (int)(cdivll(nv, 32) * 32), p, st);
    if (nv <= 128) {
        const int V = little ? 1 : nv >= 8 ? 4 : nv >= 4 ? 2 : 1;
        for (p.group = 2; p.group < 32 && p.group * V < nv;) p.group *= 2;
        if (p.group * V >= nv) {
            if (little) return launch_rows<T, MODE, 1, false, 0>(odd, 256, p, st);
            if (V == 1) return launch_rows<T, MODE, 1, false, 3>(odd, 256, p, st);
            if (V == 2) return launch_rows<T, MODE, 2, false, 2>(odd, 256, p, st);
        }
        p.group = 32;
        while (p.group > 2 && p.group * 2 >= nv) p.group /= 2;
        return launch_rows<T, MODE, 4, false, 1>(odd, 256, p, st);
    }
    if (nv <= 2048) return launch_rows<T, MODE, 4, true, 1>(odd, (int)(cdivll(nv, 128) * 32), p, st);
    // (the longest rows: with a shortcut in 32 bits four loads a thread and tensor, which leave registers for twice the threads: 7000 x 10656
    // 258 us, eight 366; without one four 105, eight 63)
    constexpr int MOST = N == 4 && MODE == kNormRes ? 4 : 8;
    return launch_rows<T, MODE, MOST, true, 0>(odd, (int)(cdivll(nv, 32 * MOST) * 32), p, st);
}

template <typename T, int MODE>
static int nchw_int8(RowsParams p, cudaStream_t st)
{
    const int words = cdiv(p.C, 4), most = MODE == kNormRes && words <= 128 ? 8 : 16;
    const long long tiles = cdivll(p.rows, 32);
    // warps that share 32 pixels: as few as the registers allow, more where the pixels are few; blocks of two warps (256 x 64 x 56 x 56: 46.4
    // us; of eight, which wait for the last of them, 50.7; two warps to a tile 48.3)
    int share = std::min(16, cdiv(words, most));
    while (share < 9 && words >= 4 * share && tiles * share < 8 * kNumSMs) share = std::min(16, 2 * share);
    const bool loop = words > share * most || p.C < 4;          // (128 x 512 x 14 x 14 bf16 so: 27 us, in registers 12)
    if (loop) share = 8;
    p.group = share;
    const int per_block = share == 1 ? 2 : 1, warps = share * per_block;
    const long long blocks = cdivll(tiles, per_block);
    if (blocks > 0x7fffffffLL) return WG2X2_ERR_UNSUPPORTED;
    const bool by16 = p.ldq % 16 == 0 && (reinterpret_cast<uintptr_t>(p.Q) & 15u) == 0;
    const int pieces = by16 ? p.C / 16 : words;
    p.inv = pieces > 1 ? (unsigned)((0x100000000ull + pieces - 1) / pieces) : 0;       // i / pieces exact for i * pieces < 2^32
    const size_t smem = (size_t)per_block * 32 * (words | 1) * 4 + (MODE != kQuantize ? (size_t)16 * words : 0);
    if (smem > 216 * 1024)
        return p.rows > 0x7fffffffLL ? WG2X2_ERR_UNSUPPORTED : launch(rows_any_kernel<T, MODE, true>, dim3((unsigned)p.rows), 512, 0, st, p);
    const int nq = loop ? 0 : cdiv(words, share) <= 2 ? 2 : cdiv(words, share) <= 4 ? 4 : cdiv(words, share) <= 8 ? 8 : 16;
    const bool full = p.C == 4 * nq * share;
#define WG_NCHW(NQ)                                                                                                          \
    (full ? launch(nchw_kernel<T, MODE, NQ, (NQ) != 0>, dim3((unsigned)blocks), 32 * warps, smem, st, p)                      \
          : launch(nchw_kernel<T, MODE, NQ, false>, dim3((unsigned)blocks), 32 * warps, smem, st, p))
    return nq == 0 ? WG_NCHW(0) : nq == 2 ? WG_NCHW(2) : nq == 4 ? WG_NCHW(4) : nq == 8 ? WG_NCHW(8) : WG_NCHW(16);
#undef WG_NCHW
}

static int codes_int8(int mode, int type, RowsParams &p, long long B, int HW, int C, int layout, cudaStream_t st)
{
    if (type < WG2X2_F32 || type > WG2X2_BF16 || (layout != WG2X2_NHWC && layout != WG2X2_NCHW)) return WG2X2_ERR_BAD_ARG;
    if (B < 0 || HW <= 0 || C <= 0 || B > 0x7fffffffffffLL / HW) return WG2X2_ERR_BAD_ARG;
    p.rows = B * HW;
    p.C = C;
    p.HW = HW;
    if (!p.rows) return WG2X2_OK;
    if (C > 1 << 30 || p.rows > 1LL << 36 || p.ldx >= 1LL << 40 || p.ldr >= 1LL << 40 || p.ldh >= 1LL << 40 || p.ldq >= 1LL << 40)
        return WG2X2_ERR_UNSUPPORTED;          // (a channel's index and a step beyond it fit 32 bits; see also the kernels' launchers)
    const int e = type == WG2X2_F32 ? 4 : 2;
    const bool nchw = layout == WG2X2_NCHW;
    if (!p.X || !p.Q || !p.scale || (mode != kQuantize && !p.Wt) || (mode == kNormRes && (!p.R || !p.H))) return WG2X2_ERR_BAD_ARG;
    if (p.ldq < C || (!nchw && (p.ldx < C || (mode == kNormRes && (p.ldr < C || p.ldh < C))))) return WG2X2_ERR_BAD_ARG;
    auto off = [](const void *q, int size) { return (reinterpret_cast<uintptr_t>(q) & (unsigned)(size - 1)) != 0; };
    if (off(p.X, e) || off(p.R, e) || off(p.H, e) || off(p.scale, 4) || (p.Wt && off(p.Wt, p.w_f32 ? 4 : e))) return WG2X2_ERR_BAD_ARG;
    // the tensors as rows of bytes (an NCHW one: a single row)
    struct Span { const void *at; long long ld, n; };
    if (nchw && p.rows > (1LL << 60) / C) return WG2X2_ERR_UNSUPPORTED;
    auto image = [&](const void *q, long long ld) { return nchw ? Span{q, 0, p.rows * C * e} : Span{q, ld * e, (long long)C * e}; };
    auto meet = [&](const Span &a, const Span &b) { return a.at && b.at && rows_overlap(a.at, a.ld, a.n, a.ld ? p.rows : 1, b.at, b.ld, b.n, b.ld ? p.rows : 1); };
    const Span q{p.Q, p.ldq, C}, s{p.scale, 0, 4 * p.rows}, x = image(p.X, p.ldx), r = image(p.R, p.ldr), h = image(p.H, p.ldh);
    const Span w{p.Wt, 0, (long long)C * (p.w_f32 ? 4 : e)};
    if (meet(q, s) || meet(q, x) || meet(q, r) || meet(q, h) || meet(q, w) || meet(s, x) || meet(s, r) || meet(s, h) || meet(s, w)) return WG2X2_ERR_BAD_ARG;
    // the sum may lie exactly over what it adds
    auto apart = [&](const Span &a) { return (h.at == a.at && h.ld == a.ld) || !meet(h, a); };
    if (mode == kNormRes && (!apart(x) || !apart(r) || meet(h, w))) return WG2X2_ERR_BAD_ARG;
#define WG_CODES(T)                                                                                                             \
    (nchw ? (mode == kQuantize ? nchw_int8<T, kQuantize>(p, st) : mode == kNorm ? nchw_int8<T, kNorm>(p, st) : nchw_int8<T, kNormRes>(p, st)) \
          : (mode == kQuantize ? rows_int8<T, kQuantize>(p, st) : mode == kNorm ? rows_int8<T, kNorm>(p, st) : rows_int8<T, kNormRes>(p, st)))
    if (type == WG2X2_F32) return WG_CODES(float);
    if (type == WG2X2_F16) return WG_CODES(__half);
    return WG_CODES(__nv_bfloat16);
#undef WG_CODES
}

}  // namespace wg

extern "C" int wg2x2_quantize_int8(const void *X, int type, long long ldx, void *Q, long long ldq, float *scale, long long B, int HW, int C,
                                   int layout, int relu, void *stream)
{
    wg::RowsParams p = {};
    p.X = X; p.ldx = ldx; p.Q = static_cast<signed char *>(Q); p.ldq = ldq; p.scale = scale; p.relu = relu != 0;
    return wg::codes_int8(wg::kQuantize, type, p, B, HW, C, layout, (cudaStream_t)stream);
}

extern "C" int wg2x2_rms_norm_int8(const void *X, long long ldx, const void *residual, long long ldr, void *residual_out, long long ldo,
                                   const void *weight, int weight_f32, float eps, int type, void *Q, long long ldq, float *scale, long long B,
                                   int HW, int C, int layout, void *stream)
{
    if (!(eps >= 1e-30f) || !(eps <= 3.402823466e38f) || (residual == nullptr) != (residual_out == nullptr)) return WG2X2_ERR_BAD_ARG;
    wg::RowsParams p = {};
    p.X = X; p.ldx = ldx; p.R = residual; p.ldr = ldr; p.H = residual_out; p.ldh = ldo; p.Wt = weight; p.w_f32 = type == WG2X2_F32 || weight_f32;
    p.eps = eps; p.Q = static_cast<signed char *>(Q); p.ldq = ldq; p.scale = scale;
    return wg::codes_int8(residual ? wg::kNormRes : wg::kNorm, type, p, B, HW, C, layout, (cudaStream_t)stream);
}
