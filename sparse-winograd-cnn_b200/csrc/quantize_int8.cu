// Rows of 8-bit codes with one scale a row, for products in 8-bit integers (linear_int8.cuh): of activations or weights as they are, and
// of their root-mean-square norm with the shortcut's addition in front.
//
//   quantize   a = max_c |x_c|            scale = a / 127                                  q_c = 127 x_c / a, nearest, ties to even
//   norm       h = x + residual in x's type, u_c = h_c w_c in 32 bits, a = max_c |u_c|
//              scale = a / 127 / sqrt(mean_c h_c^2 + eps)                                  q_c = 127 u_c / a, likewise
//
// The norm is a factor of the whole row, so the codes do not depend on it: only the scale does, and codes come out the same whatever
// the order in which the squares were added.  h is rounded to x's type before anything else looks at it, so that the norm is that of
// the tensor that is handed on; u is held in 32 bits; the quotient 127 u / a is rounded as in exact arithmetic (code_word).  A row
// whose a is below 2^-119, where a / 127 leaves the normal numbers, has scale 0 and codes 0.  A row with a NaN or an infinity (or one
// whose u is beyond 32 bits) has scale NaN and codes 0, so that it stays NaN through a product.
//
// Bound by the bytes.  A row is read once, 16 bytes a load, and stays in registers between its maximum and its codes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "wg_common.cuh"

namespace wg {

constexpr float kTinyRow = 0x1p-119f;
constexpr float kRound = 12582912.f;        // 1.5 * 2^23: adding it leaves the nearest whole number (ties to even) in the low bits
constexpr float kNearTie = 0.49998f;        // see code_word

enum { kQuantize = 0, kNorm = 1, kNormRes = 2 };

struct RowsParams {
    const void *X, *R;          // x; the shortcut (kNormRes)
    void *H;                    // x + shortcut (kNormRes); may lie exactly over X or R
    const void *Wt;             // the norm's weights, C of them
    signed char *Q;
    float *scale;
    long long ldx, ldr, ldh, ldq, rows;
    int C, HW;                  // HW: pixels of a plane (NCHW)
    int group;                  // threads of a row, where a block has several rows
    int w_f32, relu;
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

// 16 bytes as values
template <typename T> struct alignas(16) Pack { T v[16 / sizeof(T)]; };

// (plain loads: H may lie over the tensor that is read, which the read-only path must not be used for)
template <typename T, int N>
__device__ __forceinline__ Pack<T> load_pack(const T *p, int c0, int C)
{
    Pack<T> r;
    if (c0 >= 0 && c0 + N <= C) {
        *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(p + c0);
    } else {                                            // the ends of a row that does not begin or end on 16 bytes
#pragma unroll
        for (int j = 0; j < N; ++j) r.v[j] = c0 + j >= 0 && c0 + j < C ? p[c0 + j] : from_f<T>(0.f);
    }
    return r;
}
template <typename T, int N>
__device__ __forceinline__ void store_pack(T *p, int c0, int C, const Pack<T> &r)
{
    if (c0 >= 0 && c0 + N <= C) {
        *reinterpret_cast<uint4 *>(p + c0) = *reinterpret_cast<const uint4 *>(&r);
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (c0 + j >= 0 && c0 + j < C) p[c0 + j] = r.v[j];
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
            for (int j = 0; j < N; j += 4) *reinterpret_cast<float4 *>(w + j) = reinterpret_cast<const float4 *>(at)[j / 4];
        } else {
            Pack<T> r;
            *reinterpret_cast<uint4 *>(&r) = *reinterpret_cast<const uint4 *>(at);
#pragma unroll
            for (int j = 0; j < N; ++j) w[j] = to_f(r.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) w[j] = c0 + j >= 0 && c0 + j < p.C ? weight_at(p, (const T *)nullptr, c0 + j) : 0.f;
    }
}

__device__ __noinline__ unsigned exact_code(float u, float a) { return (unsigned)__double2int_rn((double)u * 127.0 / (double)a); }

// Four codes as a word.  inv = 127 / a rounded, t = u inv rounded: |t - 127 u / a| < 127 * 2^-23 * 1.01 = 1.53e-5, so wherever t is
// further than 2e-5 from half way between two whole numbers its nearest is that of 127 u / a.  Elsewhere (u = a / 2 is common in
// 16-bit types) the quotient is taken in 64 bits: 127 u is exact there, and a quotient that is not half way differs from it by more
// than 2^-33.  a below kTinyRow or not finite: inv = 0, and the caller clears the codes.
__device__ __forceinline__ unsigned code_word(const float *u, float inv, float a)
{
    unsigned r[4];
    float off = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float t = __fmul_rn(u[j], inv), m = __fadd_rn(t, kRound);
        off = fmaxf(off, fabsf(__fsub_rn(t, __fsub_rn(m, kRound))));
        r[j] = __float_as_uint(m);
    }
    if (off > kNearTie) {
#pragma unroll 1
        for (int j = 0; j < 4; ++j) r[j] = exact_code(j == 0 ? u[0] : j == 1 ? u[1] : j == 2 ? u[2] : u[3], a);
    }
    return __byte_perm(__byte_perm(r[0], r[1], 0x0040), __byte_perm(r[2], r[3], 0x0040), 0x5410);
}

// A row's largest magnitude, as the bits of |u|: NaN above infinity above everything else
__device__ __forceinline__ unsigned mag(float u) { return __float_as_uint(u) & 0x7fffffffu; }

struct RowCodes {
    float inv, a, scale;
    unsigned live;                // all ones, or zero where the codes are 0 whatever u
};
constexpr float kDown = 0x1p-100f;     // for a row whose squares leave 32 bits: some |h| is above 2^64 / sqrt(C), all are below 2^128
__device__ __forceinline__ RowCodes row_codes(unsigned amax)
{
    RowCodes k;
    k.a = __uint_as_float(amax);
    const bool ok = k.a >= kTinyRow && amax < 0x7f800000u;
    k.live = ok ? 0xffffffffu : 0u;
    k.inv = ok ? __fdiv_rn(127.f, k.a) : 0.f;
    k.scale = ok ? __fdiv_rn(k.a, 127.f) : (k.a < kTinyRow ? 0.f : __uint_as_float(0x7fffffffu));
    return k;
}
// scale / sqrt(mean square + eps); ss: the sum of the squares of h, or of kDown * h (where eps counts for nothing)
__device__ __forceinline__ float norm_scale(float scale, float ss, int C, float eps, bool down)
{
    const float mean = __fdiv_rn(ss, (float)C);
    if (down) return scale > 1.f ? __fdiv_rn(scale * kDown, __fsqrt_rn(mean)) : __fdiv_rn(scale, __fsqrt_rn(mean)) * kDown;
    return __fdiv_rn(scale, __fsqrt_rn(mean + eps));
}

__device__ __forceinline__ void reduce_group(unsigned &amax, float &ss, int width)
{
    for (int o = width >> 1; o; o >>= 1) {
        amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
}
// Over the block; every thread has the result, in the same order of additions
__device__ __forceinline__ void reduce_block(unsigned &amax, float &ss, uint2 *part)
{
    reduce_group(amax, ss, 32);
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_uint2(amax, __float_as_uint(ss));
    __syncthreads();
    amax = 0;
    ss = 0.f;
    for (int w = 0; w < warps; ++w) {
        const uint2 v = part[w];
        amax = max(amax, v.x);
        ss += __uint_as_float(v.y);
    }
    __syncthreads();          // (part may be used again)
}

// Rows in registers: V loads of 16 bytes a thread.  BLOCK: a row per block, else blockDim.x / group rows.  ODD: rows that do not begin
// on 16 bytes, or whose length is not a multiple; x, shortcut and sum have the same offset to a 16-byte boundary in every row.  Loads
// are then of the aligned pieces that a row touches (its ends value by value), and codes reach their own 4 or 8 bytes by a shift with
// the next lane's.
template <typename T, int MODE, int V, bool BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) rows_kernel(const RowsParams p)
{
    constexpr int N = 16 / sizeof(T), WORDS = N / 4;
    __shared__ uint2 part[BLOCK ? 32 : 1];
    wait_for_previous_kernel(kNumSMs);
    const int lane = threadIdx.x & 31;
    const long long row = BLOCK ? (long long)blockIdx.x : (long long)blockIdx.x * (blockDim.x / p.group) + threadIdx.x / p.group;
    const int i0 = BLOCK ? threadIdx.x : threadIdx.x & (p.group - 1), step = BLOCK ? blockDim.x : p.group;
    const bool have = BLOCK || row < p.rows;
    const int C = have ? p.C : 0;                  // (no element is then loaded or stored)
    const T *x = static_cast<const T *>(p.X) + (have ? row : 0) * p.ldx;
    const T *res = MODE == kNormRes ? static_cast<const T *>(p.R) + (have ? row : 0) * p.ldr : nullptr;
    T *h = MODE == kNormRes ? static_cast<T *>(p.H) + (have ? row : 0) * p.ldh : nullptr;
    const int mis = ODD ? (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T)) : 0;

    float u[V][N];
    {
        Pack<T> a[V], b[V];
#pragma unroll
        for (int v = 0; v < V; ++v) a[v] = load_pack<T, N>(x, (i0 + v * step) * N - mis, C);
        if (MODE == kNormRes) {
#pragma unroll
            for (int v = 0; v < V; ++v) b[v] = load_pack<T, N>(res, (i0 + v * step) * N - mis, C);
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int j = 0; j < N; ++j) a[v].v[j] = from_f<T>(__fadd_rn(to_f(a[v].v[j]), to_f(b[v].v[j])));
                store_pack<T, N>(h, (i0 + v * step) * N - mis, C, a[v]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int j = 0; j < N; ++j) u[v][j] = to_f(a[v].v[j]);
    }
    unsigned amax = 0;
    float ss = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (MODE != kQuantize) {
            float w[N];
            load_weights<T, N>(p, C ? (i0 + v * step) * N - mis : p.C, w);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                ss = fmaf(u[v][j], u[v][j], ss);
                u[v][j] = __fmul_rn(u[v][j], w[j]);
            }
        } else if (p.relu) {
#pragma unroll
            for (int j = 0; j < N; ++j) u[v][j] = relu_nan(u[v][j]);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) amax = max(amax, mag(u[v][j]));
    }
    if (BLOCK) reduce_block(amax, ss, part);
    else reduce_group(amax, ss, p.group);
    RowCodes k = row_codes(amax);
    if (MODE != kQuantize) {
        bool down = k.live && !(ss <= 3.402823466e38f);
        if (BLOCK ? down : __any_sync(0xffffffffu, down)) {        // the squares of a row of large values: once more, scaled (h as it was stored)
            float s2 = 0.f;
            unsigned none = 0;
#pragma unroll 1
            for (int v = 0; v < V; ++v)
                for (int j = 0; j < N; ++j) {
                    const int c = (i0 + v * step) * N - mis + j;
                    if (c < 0 || c >= C) continue;
                    const float f = to_f(MODE == kNormRes ? h[c] : x[c]) * kDown;
                    s2 = fmaf(f, f, s2);
                }
            if (BLOCK) reduce_block(none, s2, part);
            else reduce_group(none, s2, p.group);
            if (down) ss = s2;
        }
        k.scale = k.live ? norm_scale(k.scale, ss, p.C, p.eps, down) : k.scale;
    }
    if (have && i0 == 0) p.scale[row] = k.scale;

    signed char *q = p.Q + (have ? row : 0) * p.ldq;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int i = i0 + v * step, c0 = i * N;
        unsigned w[2 * WORDS];
#pragma unroll
        for (int g = 0; g < WORDS; ++g) w[g] = code_word(u[v] + 4 * g, k.inv, k.a) & k.live;
        if (!ODD) {
            if (c0 < C) {
                if (WORDS == 2) *reinterpret_cast<uint2 *>(q + c0) = make_uint2(w[0], w[WORDS - 1]);
                else *reinterpret_cast<unsigned *>(q + c0) = w[0];
            }
        } else {
            // codes of channels c0 - mis .. c0 - mis + N - 1 here, the next N in the next lane (not behind the last lane of a warp or
            // of a row's group).  A lane with a next one stores channels c0 .. c0 + N - 1, else what it has of them; the first lane also
            // what lies in front of c0.
#pragma unroll
            for (int g = 0; g < WORDS; ++g) w[WORDS + g] = __shfl_down_sync(0xffffffffu, w[g], 1);
            const int width = BLOCK ? 32 : p.group, at = BLOCK ? lane : i0;
            const bool next = at < width - 1;
            const int own = N - mis, count = min(next ? N : own, C - c0);
            if (at == 0)
                for (int j = 0; j < mis; ++j)
                    if (c0 - mis + j >= 0 && c0 - mis + j < C) q[c0 - mis + j] = (signed char)(w[j >> 2] >> (8 * (j & 3)));
            unsigned o[WORDS];
#pragma unroll
            for (int g = 0; g < WORDS; ++g) {
                unsigned lo = w[g], hi = w[g + 1];
                if (WORDS == 2 && (mis & 4)) { lo = hi; hi = w[min(g + 2, 2 * WORDS - 1)]; }
                o[g] = __funnelshift_r(lo, hi, 8 * (mis & 3));
            }
            if (count == N && (reinterpret_cast<uintptr_t>(q) & (N - 1)) == 0) {
                if (WORDS == 2) *reinterpret_cast<uint2 *>(q + c0) = make_uint2(o[0], o[WORDS - 1]);
                else *reinterpret_cast<unsigned *>(q + c0) = o[0];
            } else {
#pragma unroll
                for (int j = 0; j < N; ++j)
                    if (j < count) q[c0 + j] = (signed char)(o[j >> 2] >> (8 * (j & 3)));
            }
        }
    }
}

// Rows of any length and alignment, value by value; read a second time for the codes (from L2): what rows_kernel does not hold.
template <typename T, int MODE>
__global__ void __launch_bounds__(512) rows_any_kernel(const RowsParams p)
{
    __shared__ uint2 part[32];
    wait_for_previous_kernel(kNumSMs);
    const long long row = blockIdx.x;
    const T *x = static_cast<const T *>(p.X) + row * p.ldx;
    const T *res = MODE == kNormRes ? static_cast<const T *>(p.R) + row * p.ldr : nullptr;
    T *h = MODE == kNormRes ? static_cast<T *>(p.H) + row * p.ldh : nullptr;
    const T *again = MODE == kNormRes ? h : x;
    auto value = [&](int c) {
        const float v = to_f(again[c]);
        return MODE != kQuantize ? __fmul_rn(v, weight_at(p, (const T *)nullptr, c)) : p.relu ? relu_nan(v) : v;
    };
    unsigned amax = 0;
    float ss = 0.f;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        if (MODE == kNormRes) h[c] = from_f<T>(__fadd_rn(to_f(x[c]), to_f(res[c])));
        const float v = to_f(again[c]);
        ss = fmaf(v, v, ss);
        amax = max(amax, mag(value(c)));
    }
    reduce_block(amax, ss, part);
    RowCodes k = row_codes(amax);
    if (MODE != kQuantize && k.live) {
        const bool down = !(ss <= 3.402823466e38f);
        if (down) {
            unsigned none = 0;
            ss = 0.f;
            for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
                const float f = to_f(again[c]) * kDown;
                ss = fmaf(f, f, ss);
            }
            reduce_block(none, ss, part);
        }
        k.scale = norm_scale(k.scale, ss, p.C, p.eps, down);
    }
    if (threadIdx.x == 0) p.scale[row] = k.scale;
    signed char *q = p.Q + row * p.ldq;
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
        const float u[4] = {value(c), 0.f, 0.f, 0.f};
        q[c] = (signed char)(code_word(u, k.inv, k.a) & k.live);
    }
}

// NCHW: 32 pixels a block, lane = pixel (of any images), so that a load is 32 consecutive values of a plane; a warp takes four
// neighbouring channels at a time, whose codes are a word.  NQ: groups of four channels that a thread keeps (0: any number, read a
// second time).  The words are turned through shared memory and leave as rows.
template <typename T, int MODE, int NQ>
__global__ void __launch_bounds__(512) nchw_kernel(const RowsParams p)
{
    extern __shared__ unsigned turned[];            // [32][pitch]
    __shared__ uint2 part[16][32];
    wait_for_previous_kernel(kNumSMs);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const long long row0 = (long long)blockIdx.x * 32, row = row0 + lane;
    const bool have = row < p.rows;
    const long long b = have ? row / p.HW : 0, base = b * p.C * p.HW + (have ? row - b * p.HW : 0);
    const T *x = static_cast<const T *>(p.X) + base;
    const T *res = MODE == kNormRes ? static_cast<const T *>(p.R) + base : nullptr;
    T *h = MODE == kNormRes ? static_cast<T *>(p.H) + base : nullptr;
    const int words = (p.C + 3) >> 2, pitch = words | 1;
    const long long HW = p.HW;
    auto value = [&](float v, int c) { return MODE != kQuantize ? __fmul_rn(v, weight_at(p, (const T *)nullptr, c)) : p.relu ? relu_nan(v) : v; };

    constexpr int KEEP = NQ ? NQ : 1;
    float u[KEEP][4];
    unsigned amax = 0;
    float ss = 0.f;
    if (NQ) {
#pragma unroll
        for (int g = 0; g < KEEP; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = 4 * (warp + g * warps) + j;
                u[g][j] = have && c < p.C ? to_f(x[c * HW]) : 0.f;
            }
        if (MODE == kNormRes) {
#pragma unroll
            for (int g = 0; g < KEEP; ++g)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int c = 4 * (warp + g * warps) + j;
                    if (!have || c >= p.C) continue;
                    const T s = from_f<T>(__fadd_rn(u[g][j], to_f(res[c * HW])));
                    h[c * HW] = s;
                    u[g][j] = to_f(s);
                }
        }
#pragma unroll
        for (int g = 0; g < KEEP; ++g)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = 4 * (warp + g * warps) + j;
                ss = fmaf(u[g][j], u[g][j], ss);
                u[g][j] = c < p.C ? value(u[g][j], c) : 0.f;
                amax = max(amax, mag(u[g][j]));
            }
    } else {
        for (int c = warp; have && c < p.C; c += warps) {
            float v = to_f(x[c * HW]);
            if (MODE == kNormRes) {
                const T s = from_f<T>(__fadd_rn(v, to_f(res[c * HW])));
                h[c * HW] = s;
                v = to_f(s);
            }
            ss = fmaf(v, v, ss);
            amax = max(amax, mag(value(v, c)));
        }
    }
    // a pixel's maximum and sum over the warps; every warp adds in the same order
    auto over_warps = [&](unsigned &m, float &s) {
        part[warp][lane] = make_uint2(m, __float_as_uint(s));
        __syncthreads();
        m = 0;
        s = 0.f;
        for (int w = 0; w < warps; ++w) {
            const uint2 v = part[w][lane];
            m = max(m, v.x);
            s += __uint_as_float(v.y);
        }
        __syncthreads();
    };
    over_warps(amax, ss);
    RowCodes k = row_codes(amax);
    if (MODE != kQuantize) {
        const bool down = k.live && !(ss <= 3.402823466e38f);
        if (__any_sync(0xffffffffu, down)) {       // (the same in every warp: all have the same sums)
            const T *again = MODE == kNormRes ? h : x;
            float s2 = 0.f;
            unsigned none = 0;
            for (int c = warp; have && c < p.C; c += warps) {
                const float f = to_f(again[c * HW]) * kDown;
                s2 = fmaf(f, f, s2);
            }
            over_warps(none, s2);
            if (down) ss = s2;
        }
        k.scale = k.live ? norm_scale(k.scale, ss, p.C, p.eps, down) : k.scale;
    }
    if (warp == 0 && have) p.scale[row] = k.scale;
    if (NQ) {
#pragma unroll
        for (int g = 0; g < KEEP; ++g) {
            const int q = warp + g * warps;
            if (q < words) turned[lane * pitch + q] = code_word(u[g], k.inv, k.a) & k.live;
        }
        __syncthreads();
        const int n = (int)min(32LL, p.rows - row0);
        const bool whole = (p.ldq & 3) == 0 && (reinterpret_cast<uintptr_t>(p.Q) & 3u) == 0;
        for (int i = threadIdx.x; i < n * words; i += blockDim.x) {
            const int r = i / words, q = i - r * words;
            const unsigned w = turned[r * pitch + q];
            signed char *dst = p.Q + (row0 + r) * p.ldq + 4 * q;
            if (whole && 4 * q + 4 <= p.C) {
                *reinterpret_cast<unsigned *>(dst) = w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * q + j < p.C) dst[j] = (signed char)(w >> (8 * j));
            }
        }
    } else {
        // (h as any warp stored it: over_warps is a barrier)
        for (int q = warp; have && q < words; q += warps) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int c = 4 * q + j;
                v[j] = c < p.C ? value(to_f((MODE == kNormRes ? h : x)[c * HW]), c) : 0.f;
            }
            const unsigned w = code_word(v, k.inv, k.a) & k.live;
            signed char *dst = p.Q + row * p.ldq + 4 * q;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (4 * q + j < p.C) dst[j] = (signed char)(w >> (8 * j));
        }
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
template <typename T, int MODE, int V, bool BLOCK>
static int launch_rows(bool odd, unsigned blocks, int threads, const RowsParams &p, cudaStream_t st)
{
    return odd ? launch(rows_kernel<T, MODE, V, BLOCK, true>, dim3(blocks), threads, 0, st, p)
               : launch(rows_kernel<T, MODE, V, BLOCK, false>, dim3(blocks), threads, 0, st, p);
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
    const long long nv = odd ? cdivll((long long)p.C + N - 1, N) : p.C / N;
    if (!same || nv > 4096) return launch(rows_any_kernel<T, MODE>, dim3((unsigned)p.rows), 512, 0, st, p);
    // A few rows: as many threads a row as it has loads.  Many: a row in a warp or a part of one up to 128 loads.
    const bool few = p.rows < 2 * kNumSMs;
    if (nv <= 32 || (nv <= 128 && !few)) {
        p.group = 32;
        while (p.group > 8 && p.group / 2 >= nv) p.group /= 2;
        const unsigned blocks = (unsigned)cdivll(p.rows, 256 / p.group);
        if (nv <= 32) return launch_rows<T, MODE, 1, false>(odd, blocks, 256, p, st);
        if (nv <= 64) return launch_rows<T, MODE, 2, false>(odd, blocks, 256, p, st);
        return launch_rows<T, MODE, 4, false>(odd, blocks, 256, p, st);
    }
    const int V = few && nv <= 1024 ? 1 : nv <= 2048 ? 2 : 4;
    const int threads = (int)(cdivll(cdivll(nv, V), 32) * 32);
    if (V == 1) return launch_rows<T, MODE, 1, true>(odd, (unsigned)p.rows, threads, p, st);
    if (V == 2) return launch_rows<T, MODE, 2, true>(odd, (unsigned)p.rows, threads, p, st);
    return launch_rows<T, MODE, 4, true>(odd, (unsigned)p.rows, threads, p, st);
}

template <typename T, int MODE>
static int nchw_int8(const RowsParams &p, cudaStream_t st)
{
    const long long blocks = cdivll(p.rows, 32);
    if (blocks > 0x7fffffffLL) return WG2X2_ERR_UNSUPPORTED;
    const int words = cdiv(p.C, 4);
    const size_t smem = (size_t)32 * (words | 1) * 4;
    if (words <= 16) return launch(nchw_kernel<T, MODE, 2>, dim3((unsigned)blocks), 256, smem, st, p);
    if (words <= 32) return launch(nchw_kernel<T, MODE, 4>, dim3((unsigned)blocks), 256, smem, st, p);
    if (words <= 64) return launch(nchw_kernel<T, MODE, 8>, dim3((unsigned)blocks), 256, smem, st, p);
    if (words <= 128) return launch(nchw_kernel<T, MODE, 8>, dim3((unsigned)blocks), 512, smem, st, p);
    if (words <= 256) return launch(nchw_kernel<T, MODE, 16>, dim3((unsigned)blocks), 512, smem, st, p);
    return launch(nchw_kernel<T, MODE, 0>, dim3((unsigned)blocks), 512, 0, st, p);
}

static int codes_int8(int mode, int type, RowsParams &p, long long B, int HW, int C, int layout, cudaStream_t st)
{
    if (type < WG2X2_F32 || type > WG2X2_BF16 || (layout != WG2X2_NHWC && layout != WG2X2_NCHW)) return WG2X2_ERR_BAD_ARG;
    if (B < 0 || HW <= 0 || C <= 0 || B > 0x7fffffffffffLL / HW) return WG2X2_ERR_BAD_ARG;
    p.rows = B * HW;
    p.C = C;
    p.HW = HW;
    if (!p.rows) return WG2X2_OK;
    const int e = type == WG2X2_F32 ? 4 : 2;
    const bool nchw = layout == WG2X2_NCHW;
    if (!p.X || !p.Q || !p.scale || (mode != kQuantize && !p.Wt) || (mode == kNormRes && (!p.R || !p.H))) return WG2X2_ERR_BAD_ARG;
    if (p.ldq < C || (!nchw && (p.ldx < C || (mode == kNormRes && (p.ldr < C || p.ldh < C))))) return WG2X2_ERR_BAD_ARG;
    auto off = [](const void *q, int size) { return (reinterpret_cast<uintptr_t>(q) & (unsigned)(size - 1)) != 0; };
    if (off(p.X, e) || off(p.R, e) || off(p.H, e) || off(p.scale, 4) || (p.Wt && off(p.Wt, p.w_f32 ? 4 : e))) return WG2X2_ERR_BAD_ARG;
    // the tensors as rows of bytes (an NCHW one: a single row)
    struct Span { const void *at; long long ld, n; };
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
