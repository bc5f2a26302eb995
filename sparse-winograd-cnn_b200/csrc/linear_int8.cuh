// Products in 8-bit integers with a scale for each row of either operand (a token or pixel; an output channel):
//
//   Y[r][k] = (sum_c q[r][c] w[k][c]) * w_scale[k] * q_scale[r] (+ bias[k])        optionally through a ReLU, in 32 or 16 bits
//
// The sums are exact: 32-bit integers in tensor memory (tcgen05 kind::i8), C at most 131071, so 128^2 C < 2^31.  The rest is 32-bit
// floating point.  Included by conv_tc.cu.
//
// Which operand has the 128 lanes of tensor memory goes by the result's layout, so that a warp's store of one column is of consecutive
// elements: channels last, lanes = output channels (A = the weights, columns = rows of q); NCHW, lanes = pixels (A = q, columns =
// output channels).  A tile is 128 lanes x N columns; a CTA walks its tiles with two accumulators, so that one is stored while the next
// is computed.  Where the tiles are too few for the GPU, a cluster of S CTAs shares a tile: each takes a share of the contraction, and
// the shares (whole numbers, so the order does not matter) meet through distributed shared memory, every CTA finishing N / S columns.
#pragma once

constexpr int kLiEpiWarps = 16;               // two sets of eight, one for each accumulator: a product with few channels is all epilogue
constexpr int kLiThreads = 32 * (2 + kLiEpiWarps);       // producer, MMA issuer, epilogue
constexpr int kLiChunk = 128;                 // bytes of the contraction a stage
constexpr int kLiMaxStages = 12;
constexpr int kLiSmem = 232448;               // all that a CTA can have
constexpr int kLiAhead = 2;
constexpr int kLiCorner = 128;                // columns of a tile that an epilogue warp finishes, at most
constexpr int kLiCtrl = 512 + kLiEpiWarps * 2 * kLiCorner * 4;     // barriers; the scales and biases of those columns, for each epilogue warp
constexpr int kLiMaxC = 131071;

struct LiParams {
    void *Y;
    const float *lane_scale, *col_scale, *bias;     // bias: of the output channels
    long long ldy;                                  // channels last: elements from row to row
    int lanes, cols;                                // rows of A and of B
    int K, HW;                                      // NCHW: channels and pixels of Y's images
    int N, stages, chunks;                          // columns of a tile; stages of operands; chunks of the contraction
    int lane_tiles, col_tiles, splits, pair, relu;
    uint32_t spin_limit;
    int drop_load;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
// D[tmem] (+)= A[smem] * B[smem], M=128, K=32, signed 8-bit operands, 32-bit integer accumulator
__device__ __forceinline__ void umma_i8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// Instruction descriptor: D = s32, A = B = s8, both K-major
__host__ __device__ constexpr uint32_t make_idesc_i8(int M, int N)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, int (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld8i(uint32_t taddr, int (&r)[8])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}

// The registers of the loads above pass through the wait, so that nothing that reads them can be moved in front of it
__device__ __forceinline__ void tmem_wait32(int (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 ::"memory");
}
__device__ __forceinline__ void tmem_wait8(int (&r)[8])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) ::"memory");
}

template <typename T> __device__ __forceinline__ T li_out(float v);
template <> __device__ __forceinline__ float li_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __half li_out<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 li_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// (The weights' scale first: of the two it is the one of ordinary size.  Without a bias the sum is with -0, which changes nothing; low = 0
// for a ReLU, which keeps NaN, and -infinity for none.)
__device__ __forceinline__ float li_value(int acc, float w_scale, float q_scale, float bias, float low)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fmaf(__fmul_rn((float)acc, w_scale), q_scale, bias)), "f"(low));
    return r;
}

// 16 lane tiles x all column tiles at a time, so that the CTAs that run together share operands in L2
__device__ __forceinline__ void li_decode(const LiParams &p, int u, int &lt, int &ct)
{
    if (p.col_tiles == 1) {
        lt = u;
        ct = 0;
        return;
    }
    const int group = u / (16 * p.col_tiles), r = u - group * 16 * p.col_tiles, size = min(16, p.lane_tiles - 16 * group);
    ct = r / size;
    lt = 16 * group + r - ct * size;
}

// An epilogue thread's share of a tile: its lane (row of A) with all of the warp's columns
struct LiScale { float scale, bias; };          // of a lane; the bias where lanes are output channels
template <bool NCHW>
__device__ __forceinline__ LiScale li_lane_scale(const LiParams &p, int lane_row)
{
    const int r = min(lane_row, p.lanes - 1);
    return {p.lane_scale[r], !NCHW && p.bias ? p.bias[r] : -0.f};
}
template <bool NCHW, typename T>
struct LiLane {
    T *dst;                     // Y at column 0
    long long step;             // elements from column to column
    float scale, bias, low;
    bool live;
    __device__ __forceinline__ LiLane(const LiParams &p, int lane_row, const LiScale &s) : scale(s.scale), bias(s.bias)
    {
        live = lane_row < p.lanes;
        const unsigned r = live ? lane_row : 0;
        low = p.relu ? 0.f : __uint_as_float(0xff800000u);
        if (NCHW) {
            const unsigned b = r / (unsigned)p.HW;
            dst = static_cast<T *>(p.Y) + (long long)b * p.K * p.HW + (r - b * p.HW);
            step = p.HW;
        } else {
            dst = static_cast<T *>(p.Y) + r;
            step = p.ldy;
        }
    }
};
// Scales (and biases) of a warp's columns, 32 a time one a lane: asked for while the tile before is stored, then put where all lanes read them
template <bool NCHW>
struct LiColumns {
    float scale[kLiCorner / 32], bias[kLiCorner / 32];
    __device__ __forceinline__ void load(const LiParams &p, int col0, int ncols, int lane)
    {
#pragma unroll
        for (int k = 0; k < kLiCorner / 32; ++k) {
            const int c = col0 + 32 * k + lane;
            const bool ok = 32 * k < ncols && c < p.cols;
            scale[k] = ok ? p.col_scale[c] : 0.f;
            bias[k] = NCHW && ok && p.bias ? p.bias[c] : -0.f;
        }
    }
    __device__ __forceinline__ void put(float *corner, int lane) const
    {
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kLiCorner / 32; ++k) {
            corner[32 * k + lane] = scale[k];
            if (NCHW) corner[kLiCorner + 32 * k + lane] = bias[k];
        }
        __syncwarp();
    }
};
template <bool NCHW, typename T, bool WHOLE>
__device__ __forceinline__ void li_store32(const LiLane<NCHW, T> &me, const int (&r)[32], const float *corner, T *dst, int n)
{
#pragma unroll
    for (int x4 = 0; x4 < 8; ++x4) {
        const float4 cs4 = *reinterpret_cast<const float4 *>(corner + 4 * x4);
        const float4 cb4 = NCHW ? *reinterpret_cast<const float4 *>(corner + kLiCorner + 4 * x4) : make_float4(0.f, 0.f, 0.f, 0.f);
        const float cs[4] = {cs4.x, cs4.y, cs4.z, cs4.w}, cb[4] = {cb4.x, cb4.y, cb4.z, cb4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int x = 4 * x4 + j;
            const float v = NCHW ? li_value(r[x], cs[j], me.scale, cb[j], me.low) : li_value(r[x], me.scale, cs[j], me.bias, me.low);
            if (WHOLE || (me.live && x < n)) *dst = li_out<T>(v);
            dst += me.step;
        }
    }
}
// ncols columns (at most kLiCorner) from tensor memory at taddr, the first being column col0 of the result
template <bool NCHW, typename T>
__device__ __forceinline__ void li_store(const LiParams &p, const LiLane<NCHW, T> &me, uint32_t taddr, const float *corner, int col0, int ncols)
{
    const int have = min(ncols, p.cols - col0);
    const bool live = __all_sync(0xffffffffu, me.live);
    T *dst = me.dst + col0 * me.step;
    for (int c = 0; c < have; c += 32) {
        int r[32];
        tmem_ld32(taddr + (uint32_t)c, r);
        tmem_wait32(r);
        if (live && have - c >= 32) li_store32<NCHW, T, true>(me, r, corner + c, dst, 32);
        else li_store32<NCHW, T, false>(me, r, corner + c, dst, have - c);
        dst += 32 * me.step;
    }
}

// What epilogue warp 0 .. 15 (the CTA's warps from 2 on) does with its tiles of first, first + step, ..., of `lanes_tile` lanes; the CTA's
// begin at lane0 of them.  Every second tile is in the second accumulator, and warps 8 .. 15's, so that one set waits for its tile, or for
// tensor memory, while the other computes and stores.  accf, acce: barriers of the first accumulator, those of the second 8 bytes further;
// `release` hands an accumulator back.  False: gave up waiting.
// Bound, where the contraction is short, by the result's way to memory: 200704 x 64 -> 128, NCHW in 32 bits, 25.5 us, 15.4 without its stores
// (103 MB, which a plain fill writes in 18); two stores of half as many instructions each, or eight warps in all, measured the same.
template <bool NCHW, typename T, typename Release>
__device__ __forceinline__ bool li_epilogue(const LiParams &prm, int first, int step, int lanes_tile, int lane0, int warp, int lane, float *corner,
                                            uint32_t tmem, uint32_t accf, uint32_t acce, volatile int *abort_flag, Release release)
{
    const int set = warp >> 3, part = (warp >> 2) & 1, q = (warp + 2) & 3;      // (a warp reads the lanes 32 (its number in the CTA & 3) on)
    const int units = prm.lane_tiles * prm.col_tiles, width = max(32, prm.N / 2);
    const int c_tile = part * width, ncols = min(width, prm.N - c_tile);         // the warp's columns of a tile (none: ncols <= 0)
    // A tile with a short contraction takes less time than a load from memory: the lanes' scales are asked for kLiAhead tiles ahead
    LiScale ahead[kLiAhead];
    int lt, ct, col_now = -1;
    uint32_t use = 0;
    auto at = [&](int u, int k) { return (int)min((long long)units - 1, u + 2LL * k * step); };
    first += set * step;
#pragma unroll
    for (int k = 0; k < kLiAhead; ++k) {
        li_decode(prm, at(first, k), lt, ct);
        ahead[k] = li_lane_scale<NCHW>(prm, lt * lanes_tile + lane0 + q * 32 + lane);
    }
    LiColumns<NCHW> columns;
    for (int u = first; u < units; u += 2 * step) {
        li_decode(prm, u, lt, ct);
        const LiLane<NCHW, T> me(prm, lt * lanes_tile + lane0 + q * 32 + lane, ahead[0]);
        const int col0 = ct * prm.N + c_tile;
#pragma unroll
        for (int k = 0; k + 1 < kLiAhead; ++k) ahead[k] = ahead[k + 1];
        if (col0 != col_now) {
            columns.load(prm, col0, ncols, lane);
            columns.put(corner, lane);
            col_now = col0;
        }
        li_decode(prm, at(u, kLiAhead), lt, ct);
        ahead[kLiAhead - 1] = li_lane_scale<NCHW>(prm, lt * lanes_tile + lane0 + q * 32 + lane);
        if (!mbar_wait_warp(accf + 8u * set, use & 1u, abort_flag, 0x1F00u | set, prm.spin_limit)) return false;
        tc_fence_after();
        li_store<NCHW, T>(prm, me, tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(set * 256 + c_tile), corner, col0, ncols);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) release(acce + 8u * set);
        ++use;
    }
    return true;
}

// SPLIT: one tile per cluster of `splits` CTAs, else the CTA's tiles in turn
template <bool NCHW, typename T, bool SPLIT>
__global__ void __launch_bounds__(kLiThreads, 1)
linear_int8_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const LiParams prm)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *gen_base = smem_raw + (base - raw);
    const int stage_bytes = (kBlockM + prm.N) * kLiChunk;
    const uint32_t ctrl = base + prm.stages * stage_bytes;
    uint8_t *ctrl_gen = gen_base + prm.stages * stage_bytes;
    auto full_bar = [&](int s) { return ctrl + 8u * s; };
    auto empty_bar = [&](int s) { return ctrl + 8u * (kLiMaxStages + s); };
    auto accf_bar = [&](int b) { return ctrl + 8u * (2 * kLiMaxStages + b); };
    auto acce_bar = [&](int b) { return ctrl + 8u * (2 * kLiMaxStages + 2 + b); };
    volatile uint32_t *tmem_ptr_slot = reinterpret_cast<volatile uint32_t *>(ctrl_gen + 8 * (2 * kLiMaxStages + 4));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(ctrl_gen + 8 * (2 * kLiMaxStages + 5));
    static_assert(8 * (2 * kLiMaxStages + 6) <= 512, "control block");
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = SPLIT ? (int)cluster_ctarank() : 0;
    const int first = SPLIT ? blockIdx.x / prm.splits : blockIdx.x, step = SPLIT ? 1 << 30 : (int)gridDim.x;
    const int units = prm.lane_tiles * prm.col_tiles;
    // (at least one chunk for every CTA: splits <= chunks)
    const int kbeg = SPLIT ? rank * prm.chunks / prm.splits : 0, kend = SPLIT ? (rank + 1) * prm.chunks / prm.splits : prm.chunks;
    auto load = [&](int s, int lt, int ct, int kc) {
        mbar_expect_tx(full_bar(s), (uint32_t)stage_bytes);
        const uint32_t dst = base + s * stage_bytes;
        tma_load_2d(dst, &mapA, full_bar(s), kc * kLiChunk, lt * kBlockM);
        tma_load_2d(dst + kBlockM * kLiChunk, &mapB, full_bar(s), kc * kLiChunk, ct * prm.N);
    };
    // The first tile's loads, as many as there are stages, go out before the rest of the set-up.  (The next kernel is let in by
    // warp 1, as soon as every CTA has its tensor memory.)
    if (threadIdx.x == 32 || threadIdx.x == 64)
        asm volatile("prefetch.tensormap [%0];" ::"l"(threadIdx.x == 32 ? &mapA : &mapB) : "memory");
    const int early = prm.drop_load >= 0 ? 0 : min(prm.stages, kend - kbeg);
    if (threadIdx.x == 0) {
        for (int s = 0; s < prm.stages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(accf_bar(b), 1); mbar_init(acce_bar(b), kLiEpiWarps / 2); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        int lt, ct;
        li_decode(prm, first, lt, ct);
        wait_for_previous_results();
        for (int s = 0; s < early; ++s) load(s, lt, ct, kbeg + s);
    }
    __syncwarp();
    if (warp == 1) {
        tmem_alloc(smem_u32((const void *)tmem_ptr_slot), kTmemCols);
        tmem_relinquish();
        let_next_kernel_in(kNumSMs);
    }
    tc_fence_before();
    __syncthreads();
    if (SPLIT) cluster_sync_all();                  // (a CTA's shared memory is written by others only once it runs)
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr_slot, 0);
    if (threadIdx.x != 0) wait_for_previous_results();
    bool ok = true;
    // SPLIT: an epilogue thread's lane of the tile, and of its columns (part, part + 4, ... of the CTA's) the lane-th; asked for while the
    // products run
    int lt, ct;
    LiScale lane_scale = {};
    float col_scale = 0.f, col_bias = -0.f;

    if (warp == 0) {
        if (lane == 0) {
            int s = early % prm.stages, loads = 0;
            uint32_t ph = early == prm.stages ? 1 : 0;
            for (int u = first; u < units && ok; u += step) {
                int lt, ct;
                li_decode(prm, u, lt, ct);
                for (int kc = kbeg + (u == first ? early : 0); kc < kend; ++kc) {
                    if (loads++ == prm.drop_load && blockIdx.x == 0) { ok = false; break; }
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, 0x1C00u | s, prm.spin_limit)) { ok = false; break; }
                    load(s, lt, ct, kc);
                    if (++s == prm.stages) { s = 0; ph ^= 1u; }
                }
                if (step == 1 << 30) break;
            }
            if (!ok) let_them_land();
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t idesc = make_idesc_i8(kBlockM, prm.N);
        int s = 0, buf = 0;
        uint32_t ph = 0, use = 0;                   // use: rounds of the two accumulators
        for (int u = first; u < units && ok; u += step) {
            if (!mbar_wait_warp(acce_bar(buf), (use & 1u) ^ 1u, abort_flag, 0x1D00u | buf, prm.spin_limit)) { ok = false; break; }
            tc_fence_after();
            const uint32_t d_tmem = tmem_base + (uint32_t)(buf * 256);
            for (int kc = kbeg; kc < kend; ++kc) {
                if (!mbar_wait_warp(full_bar(s), ph, abort_flag, 0x1E00u | s, prm.spin_limit)) { ok = false; break; }
                tc_fence_after();
                const uint32_t at = base + s * stage_bytes;
                const uint64_t ad = make_desc_k_sw128(at), bd = make_desc_k_sw128(at + kBlockM * kLiChunk);
                if (leader) {
#pragma unroll
                    for (int kk = 0; kk < kLiChunk / 32; ++kk) umma_i8(d_tmem, ad + 2u * kk, bd + 2u * kk, idesc, kc > kbeg || kk > 0 ? 1u : 0u);
                    umma_commit(empty_bar(s));
                }
                __syncwarp();
                if (++s == prm.stages) { s = 0; ph ^= 1u; }
            }
            if (ok && leader) umma_commit(accf_bar(buf));
            __syncwarp();
            buf ^= 1;
            if (buf == 0) ++use;
            if (step == 1 << 30) break;
        }
        if (!ok) let_them_land();
    } else {
        const int q = warp & 3, part = (warp - 2) >> 2;
        float *corner = reinterpret_cast<float *>(ctrl_gen + 512) + (warp - 2) * 2 * kLiCorner;
        const uint32_t quarter = (uint32_t)(q * 32) << 16;
        if (!SPLIT) {
            ok = li_epilogue<NCHW, T>(prm, first, step, kBlockM, 0, warp - 2, lane, corner, tmem_base, accf_bar(0), acce_bar(0), abort_flag,
                                      [](uint32_t bar) { mbar_arrive(bar); });
        } else {
            // this CTA's share of the sums to the CTAs that finish them: [share][column][lane]
            li_decode(prm, first, lt, ct);
            lane_scale = li_lane_scale<NCHW>(prm, lt * kBlockM + q * 32 + lane);
            const int c = part + 4 * lane, col = ct * prm.N + rank * (prm.N / prm.splits) + c;
            if (c < prm.N / prm.splits && col < prm.cols) {
                col_scale = prm.col_scale[col];
                if (NCHW && prm.bias) col_bias = prm.bias[col];
            }
            ok = mbar_wait_warp(accf_bar(0), 0, abort_flag, 0x1F00u, prm.spin_limit);
            tc_fence_after();
            if (ok) {
                const int mine = prm.N / prm.splits;
                const uint32_t sums = ctrl + kLiCtrl;
                for (int c8 = part * 8; c8 < prm.N; c8 += 32) {
                    int r[8];
                    tmem_ld8i(tmem_base + quarter + (uint32_t)c8, r);
                    tmem_wait8(r);
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        const int c = c8 + x, to = c / mine;
                        const uint32_t at = mapa_rank(sums + (uint32_t)(((rank * mine + c - to * mine) * kBlockM + q * 32 + lane) * 4), (uint32_t)to);
                        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(at), "r"(r[x]) : "memory");
                    }
                }
            }
        }
    }
    tc_fence_before();
    if (SPLIT) {
        __syncwarp();
        cluster_sync_all();                         // every thread of every CTA, whatever came before
        if (warp >= 2) {
            const int q = warp & 3, part = (warp - 2) >> 2, mine = prm.N / prm.splits;
            const LiLane<NCHW, T> me(prm, lt * kBlockM + q * 32 + lane, lane_scale);
            const int *sums = reinterpret_cast<const int *>(ctrl_gen + kLiCtrl) + q * 32 + lane;
            for (int c = part; c < mine; c += 4) {
                const int col = ct * prm.N + rank * mine + c;
                if (col >= prm.cols) break;
                int acc = 0;
                for (int s = 0; s < prm.splits; ++s) acc += sums[(s * mine + c) * kBlockM];
                const float cs = __shfl_sync(0xffffffffu, col_scale, c >> 2), cb = NCHW ? __shfl_sync(0xffffffffu, col_bias, c >> 2) : me.bias;
                const float v = NCHW ? li_value(acc, cs, me.scale, cb, me.low) : li_value(acc, me.scale, cs, cb, me.low);
                if (me.live) me.dst[col * me.step] = li_out<T>(v);
            }
        }
    }
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// The same on pairs of SMs (tcgen05 cta_group::2) for tiles of 256 lanes x N columns: each CTA of a cluster of two has 128 of the lanes and
// brings half of B, which the tensor cores exchange, so that 256 columns take 32 KB of operands a chunk and SM instead of 48: at one CTA a
// tile it is the operands' way from L2 that the products wait for.  8192 x 4096 x 4096: 89.8 us = 3060 T/s at full clock, tensor pipe busy
// 78 % of the time, operands at 47 bytes a clock and SM (one CTA a tile: 95 us; back to back for seconds, under the power limit: 103 and
// 112).  Barriers as in conv_tc_gemm2.cuh: `full` in the leader counts both
// CTAs' bytes, `empty` and `accf` are committed to both, `acce` in the leader counts the epilogue warps of both.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t cluster_bar, int c0, int c1)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void umma_i8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
template <bool NCHW, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kLiThreads, 1)
linear_int8_pair_kernel(const __grid_constant__ CUtensorMap mapA, const __grid_constant__ CUtensorMap mapB, const LiParams prm)
{
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    const int stage_bytes = (kBlockM + prm.N / 2) * kLiChunk;             // of one CTA
    const uint32_t ctrl = base + prm.stages * stage_bytes;
    uint8_t *ctrl_gen = smem_raw + (ctrl - raw);
    auto full_bar = [&](int s) { return ctrl + 8u * s; };
    auto empty_bar = [&](int s) { return ctrl + 8u * (kLiMaxStages + s); };
    auto accf_bar = [&](int b) { return ctrl + 8u * (2 * kLiMaxStages + b); };
    auto acce_bar = [&](int b) { return ctrl + 8u * (2 * kLiMaxStages + 2 + b); };
    volatile uint32_t *tmem_ptr_slot = reinterpret_cast<volatile uint32_t *>(ctrl_gen + 8 * (2 * kLiMaxStages + 4));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(ctrl_gen + 8 * (2 * kLiMaxStages + 5));
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    if (threadIdx.x == 0) {
        for (int s = 0; s < prm.stages; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < 2; ++b) { mbar_init(accf_bar(b), 1); mbar_init(acce_bar(b), kLiEpiWarps); }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {       // the same warp of both CTAs, the same slot address
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void *)tmem_ptr_slot)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();    // the partner's barriers exist before anything is signalled into them
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_ptr_slot, 0);
    wait_for_previous_kernel(kNumSMs);

    const int first = blockIdx.x >> 1, step = gridDim.x >> 1, units = prm.lane_tiles * prm.col_tiles;
    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            int s = 0, loads = 0;
            uint32_t ph = 0;
            for (int u = first; u < units && ok; u += step) {
                int lt, ct;
                li_decode(prm, u, lt, ct);
                const int row = lt * 256 + (int)rank * kBlockM, col = ct * prm.N + (int)rank * (prm.N / 2);
                for (int kc = 0; kc < prm.chunks; ++kc) {
                    if (loads++ == prm.drop_load && blockIdx.x == 0) { ok = false; break; }
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, 0x1C00u | s, prm.spin_limit)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(full_bar(s), 2u * stage_bytes);      // both CTAs' tiles land on the leader's barrier
                    const uint32_t dst = base + s * stage_bytes, bar = mapa_rank0(full_bar(s));
                    tma_load_2d_pair(dst, &mapA, bar, kc * kLiChunk, row);
                    tma_load_2d_pair(dst + kBlockM * kLiChunk, &mapB, bar, kc * kLiChunk, col);
                    if (++s == prm.stages) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok) let_them_land();
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0) {
            const bool leader = elect_one();
            const uint32_t idesc = make_idesc_i8(256, prm.N);
            int s = 0, buf = 0;
            uint32_t ph = 0, use = 0;
            for (int u = first; u < units && ok; u += step) {
                if (!mbar_wait_warp(acce_bar(buf), (use & 1u) ^ 1u, abort_flag, 0x1D00u | buf, prm.spin_limit)) { ok = false; break; }
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + (uint32_t)(buf * 256);
                for (int kc = 0; kc < prm.chunks; ++kc) {
                    if (!mbar_wait_warp(full_bar(s), ph, abort_flag, 0x1E00u | s, prm.spin_limit)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at = base + s * stage_bytes;
                    const uint64_t ad = make_desc_k_sw128(at), bd = make_desc_k_sw128(at + kBlockM * kLiChunk);
                    if (leader) {
#pragma unroll
                        for (int kk = 0; kk < kLiChunk / 32; ++kk) umma_i8_pair(d_tmem, ad + 2u * kk, bd + 2u * kk, idesc, kc > 0 || kk > 0 ? 1u : 0u);
                        umma_commit_pair(empty_bar(s));
                    }
                    __syncwarp();
                    if (++s == prm.stages) { s = 0; ph ^= 1u; }
                }
                if (ok && leader) umma_commit_pair(accf_bar(buf));
                __syncwarp();
                buf ^= 1;
                if (buf == 0) ++use;
            }
            if (!ok) let_them_land();
        }
    } else {
        float *corner = reinterpret_cast<float *>(ctrl_gen + 512) + (warp - 2) * 2 * kLiCorner;
        li_epilogue<NCHW, T>(prm, first, step, 256, (int)rank * kBlockM, warp - 2, lane, corner, tmem_base, accf_bar(0), acce_bar(0), abort_flag, [](uint32_t bar) { mbar_arrive_cluster(mapa_rank0(bar)); });
    }
    // Neither CTA may leave, or free its tensor memory, while the other can still read its shared memory through an MMA or signal one of its
    // barriers
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols) : "memory");
    }
}

// The next two kernels are for products so small that the set-up of those above (tensor memory, barriers, a cluster's exchange) takes longer
// than their work.
struct LiSmallParams {
    const signed char *Q, *W;
    const float *q_scale, *w_scale, *bias;
    void *Y;
    long long ldq, ldw, ldy;
    int rows, C, K, HW, group, relu;        // HW: 0, or an NCHW result's pixels
};

// One row of codes: nothing but the weights' bytes counts.  `group` lanes have a row of weights, 16 bytes a load and eight loads on their way,
// and multiply four codes an instruction.  In a graph, against the kernel for a small product below: 4096 x 4096 (16.8 MB, 2.6 us of memory)
// 5.1 us / 5.6, 4096 x 1000 2.6 / 3.2, 8192 x 4096 8.0 / 9.6.  Several rows are the other kernel's from two on (4096 x 4096: 7.4 / 5.6).
template <typename T>
__global__ void __launch_bounds__(128) linear_int8_row_kernel(const LiSmallParams p)
{
    constexpr int AT_ONCE = 8;
    wait_for_previous_kernel(8 * kNumSMs);
    const int at = threadIdx.x & (p.group - 1), k = (int)(((long long)blockIdx.x * 128 + threadIdx.x) / p.group);
    const signed char *w = p.W + min(k, p.K - 1) * p.ldw;
    int acc = 0;
    const int pieces = p.C >> 4;
    for (int i0 = at; i0 < pieces; i0 += AT_ONCE * p.group) {
        int4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int i = i0 + j * p.group;
            v[j] = i < pieces ? *reinterpret_cast<const int4 *>(w + 16LL * i) : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
            const int4 x = *reinterpret_cast<const int4 *>(p.Q + 16LL * min(i0 + j * p.group, pieces - 1));
            acc = __dp4a(v[j].x, x.x, __dp4a(v[j].y, x.y, __dp4a(v[j].z, x.z, __dp4a(v[j].w, x.w, acc))));
        }
    }
    for (int c = 16 * pieces + at; c < p.C; c += p.group) acc += (int)w[c] * (int)p.Q[c];
    for (int o = p.group >> 1; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (at || k >= p.K) return;
    static_cast<T *>(p.Y)[k] = li_out<T>(li_value(acc, p.w_scale[k], p.q_scale[0], p.bias ? p.bias[k] : -0.f, p.relu ? 0.f : __uint_as_float(0xff800000u)));
}

// A small product: straight from registers with the warps' matrix instruction (16 x 8 rows, 32 bytes of both).  A CTA has 16 TILES rows of
// codes and 8 of weights (CODES16), or 8 TILES of codes and 16 of weights.  Its eight warps take every eighth 64 bytes of the contraction
// each, AT_ONCE such pieces loaded at once, and meet in shared memory.  Four lanes have 64 bytes of a row, 16 each; which four of those bytes
// an instruction calls its k-th is the same for both operands, so that no bytes change places.  li_small has the rule and what it measured.
__device__ __forceinline__ void mma_s8(int (&d)[4], int a0, int a1, int a2, int a3, int b0, int b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes of a row of C from c on, zeros behind its end
__device__ __forceinline__ int4 li_piece(const signed char *row, int c, int C)
{
    if (c + 16 <= C) return *reinterpret_cast<const int4 *>(row + c);
    int w[4] = {0, 0, 0, 0};
    if (c < C)
#pragma unroll
        for (int j = 0; j < 15; ++j)
            if (c + j < C) w[j >> 2] |= (int)(unsigned char)row[c + j] << (8 * (j & 3));
    return make_int4(w[0], w[1], w[2], w[3]);
}
template <bool CODES16, int TILES, int AT_ONCE, int RESIDENT, typename T>
__global__ void __launch_bounds__(256, RESIDENT) linear_int8_small_kernel(const LiSmallParams p)
{
    constexpr int MT = CODES16 ? TILES : 1, NT = CODES16 ? 1 : TILES, ROWS = CODES16 ? 16 * MT : 8 * NT, COLS = CODES16 ? 8 : 16;
    __shared__ int sums[8][ROWS][COLS + 1];
    wait_for_previous_kernel(RESIDENT * kNumSMs);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * COLS, row0 = blockIdx.y * ROWS, rows = min(p.rows - row0, ROWS);
    auto codes = [&](int i) { return p.Q + (row0 + min(i + g, rows - 1)) * p.ldq; };
    auto weights = [&](int i) { return p.W + min(n0 + i + g, p.K - 1) * p.ldw; };
    const signed char *pa[MT][2], *pb[NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) pa[m][h] = CODES16 ? codes(16 * m + 8 * h) : weights(16 * m + 8 * h);
#pragma unroll
    for (int n = 0; n < NT; ++n) pb[n] = CODES16 ? weights(8 * n) : codes(8 * n);
    int acc[MT][NT][4];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[m][n][j] = 0;
    for (int c0 = 64 * warp; c0 < p.C; c0 += AT_ONCE * 512) {
        int4 a[AT_ONCE][MT][2], b[AT_ONCE][NT];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const int c = c0 + 512 * i + 16 * t;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) a[i][m][h] = li_piece(pa[m][h], c, p.C);
#pragma unroll
            for (int n = 0; n < NT; ++n) b[i][n] = li_piece(pb[n], c, p.C);
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int4 x = a[i][m][0], y = a[i][m][1], z = b[i][n];
                    mma_s8(acc[m][n], x.x, y.x, x.y, y.y, z.x, z.y);
                    mma_s8(acc[m][n], x.z, y.z, x.w, y.w, z.z, z.w);
                }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int ia = 16 * m + 8 * (j >> 1) + g, ib = 8 * n + 2 * t + (j & 1);
                sums[warp][CODES16 ? ia : ib][CODES16 ? ib : ia] = acc[m][n][j];
            }
    const int col = threadIdx.x % COLS, k = n0 + col;
    const bool have = k < p.K;
    const float ws = have ? p.w_scale[k] : 0.f, bias = have && p.bias ? p.bias[k] : -0.f, low = p.relu ? 0.f : __uint_as_float(0xff800000u);
    __syncthreads();
    for (int i = threadIdx.x / COLS; i < rows; i += 256 / COLS) {
        const int r = row0 + i;
        int sum = 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) sum += sums[u][i][col];
        const long long to = p.HW ? (long long)(r / p.HW) * p.K * p.HW + r % p.HW + (long long)k * p.HW : r * p.ldy + k;
        if (have) static_cast<T *>(p.Y)[to] = li_out<T>(li_value(sum, ws, p.q_scale[r], bias, low));
    }
}
template <bool CODES16, int TILES, int AT_ONCE, int RESIDENT, typename T>
static bool li_small_launch(const LiSmallParams &p, cudaStream_t st, int *rc)
{
    const long long across = cdiv(p.K, CODES16 ? 8 : 16), down = cdiv(p.rows, CODES16 ? 16 * TILES : 8 * TILES);
    if (across * down > RESIDENT * kNumSMs) return false;
    *rc = launch(linear_int8_small_kernel<CODES16, TILES, AT_ONCE, RESIDENT, T>, dim3((unsigned)across, (unsigned)down), 256, 0, st, p);
    return true;
}
// Launches a product that is small enough for one of the two, or says that it is not.  The CTAs of the second all run at once (in two waves
// they would load their codes twice over and lose), and the contraction is short enough for the loads of eight warps.  Against the kernels
// with tensor memory, us in a graph, rows x C x K (weights in turn, 250 MB of them or 16 sets):
//    up to 8 rows: the instruction's narrow side, half as many loads of codes.  8 x 512 x 1000 1.9 / 3.7, 8 x 1024 x 4096 2.3 / 4.9, 8 x 2048 x
//       8191 5.4 / 7.0, 8 x 4096 x 4096 5.8 / 8.1, 8 x 8192 x 4096 9.9 / 10.6; behind the rule 8 x 4096 x 12000 12.3 / 10.9.  Four pieces at
//       once where there are that many: 8 x 4096 x 4096 6.5 with two
//    9 to 16: 16 x 512 x 1000 2.1 / 3.7, 16 x 1024 x 4096 2.7 / 4.9, 16 x 4096 x 4096 6.6 / 8.1; behind it 16 x 6100 x 1000 7.8 / 6.7, 16 x 4096
//       x 12000 13.0 / 10.9.  With more than 740 CTAs of eight rows of weights, sixteen: 16 x 2048 x 8191 6.4 / 7.0
//    more: 32 x 64 x 100 2.1 / 3.9, 32 x 512 x 4096 3.3 / 4.4, 32 x 4096 x 4096 8.5 / 9.6, 128 x 2048 x 1000 4.8 / 6.8, 128 x 4096 x 1000 7.7 /
//       8.0; behind it 32 x 2048 x 8191 8.8 / 7.5, 256 x 512 x 1000 5.0 / 4.4.  32 x 16 rows a CTA where that is one for nearly every SM, else 32
//       x 8: 32 x 512 x 1000 2.6 / 2.8 with the wide ones, 32 x 2048 x 4096 5.7 / 6.3 with the narrow
//    (four pieces at once with eight rows, and two with 32, spill 20 to 36 bytes a thread for the blocks that then run at once; measured so)
//    one row: see above; in short rows of weights the second kernel is the faster too (1 x 512 x 8191 2.4 / 4.4, 1 x 1024 x 4096 2.3 / 2.8)
template <typename T>
static bool li_small(LiSmallParams p, long long rows, cudaStream_t st, int *rc)
{
    const int C = p.C;
    if (rows > 32 * 4 * kNumSMs) return false;
    p.rows = (int)rows;
    if (rows == 1 && C > 1024) {
    } else if (rows <= 8) {
        if (C <= 1024 && li_small_launch<false, 1, 2, 5, T>(p, st, rc)) return true;
        if (C > 1024 && C <= 8192 && li_small_launch<false, 1, 4, 4, T>(p, st, rc)) return true;
    } else if (rows <= 16) {
        if (C <= 4096 && (li_small_launch<true, 1, 2, 5, T>(p, st, rc) || li_small_launch<false, 2, 2, 4, T>(p, st, rc))) return true;
    } else if (C <= 4096) {
        return cdivll(rows, 32) * cdiv(p.K, 16) < 128 ? li_small_launch<true, 2, 2, 4, T>(p, st, rc) : li_small_launch<false, 4, 2, 2, T>(p, st, rc);
    }
    if (rows > 1) return false;
    for (p.group = 4; p.group < 32 && p.group * 16 < C;) p.group *= 2;
    *rc = launch(linear_int8_row_kernel<T>, dim3((unsigned)cdivll(p.K, 128 / p.group)), 128, 0, st, p);
    return true;
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
// A (rows, C) tensor of bytes, rows `ld` bytes apart; bytes outside it read as zero
static bool make_map_codes(CUtensorMap *map, const void *ptr, int C, long long rows, long long ld, int box_rows)
{
    EncodeTiledFn fn = encode_fn_raw();
    if (!fn) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)C, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)kLiChunk, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    auto encode = [&] {
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if ((r == CUDA_ERROR_INVALID_CONTEXT || r == CUDA_ERROR_NOT_INITIALIZED) && cudaFree(nullptr) == cudaSuccess) r = encode();
    return r == CUDA_SUCCESS;
}

// Clusters of 2, 4 and 8 CTAs that run at once ([1], [2], [3]; of kernels that need a whole SM)
struct LiClusters { int n[4]; };
static LiClusters li_clusters()
{
    static std::atomic<unsigned long long> known[64];           // 0: not asked yet, else 1 and the three numbers, 16 bits each
    LiClusters c = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return c;
    unsigned long long v = known[dev].load();
    if (!v) {
        v = 1;
        auto *kernel = linear_int8_kernel<false, float, true>;
        for (int i = 1; i < 4 && grant_smem(reinterpret_cast<const void *>(kernel), kLiSmem); ++i) {
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = 1u << i;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(8 * kNumSMs);
            cfg.blockDim = dim3(kLiThreads);
            cfg.dynamicSmemBytes = kLiSmem;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) { n = 0; (void)cudaGetLastError(); }
            v |= (unsigned long long)(n & 0xffff) << (16 * i);
        }
        known[dev].store(v);
    }
    for (int i = 1; i < 4; ++i) c.n[i] = (int)((v >> (16 * i)) & 0xffff);
    return c;
}

// Columns of a tile, CTAs that share one, and whether pairs of SMs do, by an estimate in clocks, fitted to 338 products with every plan measured
// (weights from memory in turn; the plan taken costs 1.0 % more than the fastest on average, over 5 % in 23 of them, at most 20; of 331 others the same).  Operands
// reach an SM at 59 bytes a clock, one of a pair at 45, all SMs together at 8600 (4350 from memory): more than the products themselves take;
// the first of them after 1100.  A column of 128 lanes is finished in about 14 clocks and a tile in 680 more, beside the next tile's products
// where there is one.  CTAs come in at 13 clocks each.  CTAs that share a tile: two cluster barriers, and the sums' way between SMs, which
// is narrow.  Measured in a graph, us, rows x C x K, (N, S) taken / next best / a worse one:
//   24 x 2048 x 8191 (32, 1) 7.2 / (16, 1) 7.6 / (32, 2) 9.2          64 x 512 x 8000 (64, 1) 4.1 / (32, 1) 4.5 / (16, 1) 5.9
//   256 x 4096 x 4096 (64, 1) 10.4 / (128, 1) 11.4 / (256, 1) 15.1    100 x 8192 x 1024 (32, 4) 9.7 / (64, 4) 10.8 / (16, 2) 12.0
//   16 x 8192 x 1024 (16, 8) 7.2 / (16, 4) 8.6 / (16, 1) 16.0         2000 x 2048 x 2048 (256, 1) 10.1 / pairs 11.5 / (128, 1) 11.8
//   8192 x 1024 x 1024 (256, 1) 10.8 / pairs 12.3 / (128, 1) 13.2     8192 x 4096 x 4096 pairs 89.2 / (256, 1) 96.0 / (128, 1) 120.7
static void li_choose(LiParams &p, const LiClusters &clusters)
{
    double best = 1e300;
    const int lanes = p.lanes;
    const double from_memory = 128.0 * p.chunks * ((double)lanes + p.cols) / 4350;
    for (int N = 16; N <= 256; N *= 2) {
        const long long cols = cdiv(p.cols, N), tiles = cols * cdiv(lanes, kBlockM);
        const double bytes = std::max(from_memory, 128.0 * p.chunks * (double)tiles * (kBlockM + N) / 8600), column = 680 + 14.0 * N;
        for (int i = 0; i < 4; ++i) {
            const int S = 1 << i;
            if (S > 1 && (N > 128 || S > p.chunks || tiles > clusters.n[i])) break;
            const double main = 1100 + (double)cdiv(p.chunks, S) * 128 * (kBlockM + N) / 59, store = column / S;
            const double t = std::max(bytes, (double)cdivll(tiles * S, kNumSMs) * std::max(main, store)) + std::min(main, store) +
                             13.0 * (double)std::min<long long>(tiles * S, kNumSMs) + (S > 1 ? 3500 + 57 * N : 0);
            if (t < best * 0.999) { best = t; p.N = N; p.splits = S; p.pair = 0; }
        }
        if (N == 256 && clusters.n[1] > 0) {          // (pairs with 128 columns: never the fastest by more than measurements differ)
            const long long pairs = cols * cdiv(lanes, 256);
            const double main = 1100 + (double)p.chunks * 128 * (kBlockM + N / 2) / 45, two = std::max(from_memory, 128.0 * p.chunks * (double)pairs * (256 + N) / 8600);
            const double t = std::max(two, (double)cdivll(pairs, clusters.n[1]) * std::max(main, column)) + std::min(main, column) +
                             13.0 * (double)std::min<long long>(2 * pairs, kNumSMs) + 1800;
            if (t < best * 0.999) { best = t; p.N = N; p.splits = 1; p.pair = 1; }
        }
    }
    p.lane_tiles = cdiv(lanes, p.pair ? 256 : kBlockM);
    p.col_tiles = cdiv(p.cols, p.N);
}

static void li_sides(LiParams &p, bool nchw, long long rows, int C, int K)
{
    p.lanes = nchw ? (int)rows : K;
    p.cols = nchw ? K : (int)rows;
    p.chunks = cdiv(C, kLiChunk);
}
// The choice as a test sees it, on a GPU that holds at_once[0], [1], [2] clusters of 2, 4 and 8 CTAs: {columns of a tile, CTAs that share one, pairs}
int linear_int8_plan(long long rows, int C, int K, int layout, const int *at_once, int *plan)
{
    if (rows < 1 || rows > 0x7fffffffLL - 256 || C < 1 || C > kLiMaxC || K < 1 || K > 0x7fffffff - 256 || (layout != WG2X2_NHWC && layout != WG2X2_NCHW) || !at_once || !plan)
        return WG2X2_ERR_BAD_ARG;
    LiParams p = {};
    li_sides(p, layout == WG2X2_NCHW, rows, C, K);
    li_choose(p, LiClusters{{0, at_once[0], at_once[1], at_once[2]}});
    plan[0] = p.N; plan[1] = p.splits; plan[2] = p.pair;
    return WG2X2_OK;
}

template <bool NCHW, typename T, bool SPLIT>
static int li_launch(const CUtensorMap &mapA, const CUtensorMap &mapB, const LiParams &p, size_t smem, cudaStream_t st)
{
    const long long tiles = (long long)p.lane_tiles * p.col_tiles;
    if (!SPLIT) return launch(linear_int8_kernel<NCHW, T, false>, dim3((unsigned)std::min<long long>(tiles, kNumSMs)), kLiThreads, smem, st, mapA, mapB, p);
    return launch_cluster(linear_int8_kernel<NCHW, T, true>, dim3((unsigned)(tiles * p.splits)), p.splits, kLiThreads, smem, st, mapA, mapB, p);
}
template <bool NCHW, typename T>
static int li_launch(const CUtensorMap &mapA, const CUtensorMap &mapB, const LiParams &p, int pairs, size_t smem, cudaStream_t st)
{
    if (p.pair)
        return launch(linear_int8_pair_kernel<NCHW, T>, dim3(2 * (unsigned)std::min<long long>((long long)p.lane_tiles * p.col_tiles, pairs)), kLiThreads, smem, st, mapA, mapB, p);
    return p.splits > 1 ? li_launch<NCHW, T, true>(mapA, mapB, p, smem, st) : li_launch<NCHW, T, false>(mapA, mapB, p, smem, st);
}

int linear_int8(const void *Q, long long ldq, const float *q_scale, const void *W, long long ldw, const float *w_scale, const float *bias, int relu,
                void *Y, int type, long long ldy, long long B, int HW, int C, int K, int layout, cudaStream_t st)
{
    if (type < WG2X2_F32 || type > WG2X2_BF16 || (layout != WG2X2_NHWC && layout != WG2X2_NCHW)) return WG2X2_ERR_BAD_ARG;
    if (B < 0 || HW <= 0 || C <= 0 || K <= 0 || B > 0x7fffffffffffLL / HW) return WG2X2_ERR_BAD_ARG;
    const long long rows = B * HW;
    if (!rows) return WG2X2_OK;
    const bool nchw = layout == WG2X2_NCHW;
    const int e = type == WG2X2_F32 ? 4 : 2;
    if (!Q || !q_scale || !W || !w_scale || !Y || ldq < C || ldw < C || (!nchw && ldy < K)) return WG2X2_ERR_BAD_ARG;
    auto off = [](const void *q, unsigned size) { return (reinterpret_cast<uintptr_t>(q) & (size - 1)) != 0; };
    if (off(Q, 16) || off(W, 16) || ldq % 16 || ldw % 16 || off(q_scale, 4) || off(w_scale, 4) || off(bias, 4) || off(Y, e)) return WG2X2_ERR_BAD_ARG;
    if (C > kLiMaxC || rows > 0x7fffffffLL - 256 || K > 0x7fffffff - 256 || ldq >= 1LL << 40 || ldw >= 1LL << 40 || ldy >= 1LL << 40 ||
        rows > (1LL << 60) / K)
        return WG2X2_ERR_UNSUPPORTED;
    const long long ybytes = nchw ? rows * K * e : (long long)K * e, ypitch = nchw ? 0 : ldy * e, ny = nchw ? 1 : rows;
    auto meets = [&](const void *p, long long ld, long long n, long long count) { return p && rows_overlap(Y, ypitch, ybytes, ny, p, ld, n, count); };
    if (meets(Q, ldq, C, rows) || meets(W, ldw, C, K) || meets(q_scale, 0, 4 * rows, 1) || meets(w_scale, 0, 4LL * K, 1) || meets(bias, 0, 4LL * K, 1))
        return WG2X2_ERR_BAD_ARG;
    LiSmallParams f = {};
    f.Q = static_cast<const signed char *>(Q); f.W = static_cast<const signed char *>(W);
    f.q_scale = q_scale; f.w_scale = w_scale; f.bias = bias; f.Y = Y; f.ldq = ldq; f.ldw = ldw; f.ldy = ldy;
    f.C = C; f.K = K; f.HW = nchw ? HW : 0; f.relu = relu != 0;
    const int drop_load = take_drop_load();         // (also by a product whose kernel has no such load: the hook is of the next call, not of a later one)
    int rc;
    if (type == WG2X2_F32 ? li_small<float>(f, rows, st, &rc) : type == WG2X2_F16 ? li_small<__half>(f, rows, st, &rc) : li_small<__nv_bfloat16>(f, rows, st, &rc)) return rc;
    LiParams p = {};
    p.Y = Y; p.ldy = ldy; p.bias = bias; p.K = K; p.HW = HW; p.relu = relu != 0;
    p.lane_scale = nchw ? q_scale : w_scale;
    p.col_scale = nchw ? w_scale : q_scale;
    li_sides(p, nchw, rows, C, K);
    const LiClusters clusters = li_clusters();
    li_choose(p, clusters);
    const int pairs = clusters.n[1];
    if ((long long)p.lane_tiles * p.col_tiles > 0x3fffffffLL || p.col_tiles > 0x3ffffff) return WG2X2_ERR_UNSUPPORTED;
    const int b_rows = p.pair ? p.N / 2 : p.N, stage = (kBlockM + b_rows) * kLiChunk, other = 1024 + kLiCtrl + (p.splits > 1 ? p.N * kBlockM * 4 : 0);
    p.stages = std::min({kLiMaxStages, (kLiSmem - other) / stage, std::max(2, p.splits > 1 ? cdiv(p.chunks, p.splits) : kLiMaxStages)});
    p.spin_limit = wait_limit();
    p.drop_load = drop_load;
    CUtensorMap mapA, mapB;
    const void *A = nchw ? Q : W, *Bop = nchw ? W : Q;
    const long long lda = nchw ? ldq : ldw, ldb = nchw ? ldw : ldq;
    if (!make_map_codes(&mapA, A, C, p.lanes, lda, kBlockM) || !make_map_codes(&mapB, Bop, C, p.cols, ldb, b_rows)) return WG2X2_ERR_LAUNCH;
    // CTAs that wait for one another take all of an SM's shared memory, whatever the tile: sharing an SM with another kernel's or cluster's CTA
    // that holds tensor memory, and waits in turn for a CTA on an SM where this cluster holds some, they could wait without an end
    const size_t smem = p.splits > 1 || p.pair ? (size_t)kLiSmem : (size_t)other + (size_t)p.stages * stage;
    if (type == WG2X2_F32) return nchw ? li_launch<true, float>(mapA, mapB, p, pairs, smem, st) : li_launch<false, float>(mapA, mapB, p, pairs, smem, st);
    if (type == WG2X2_F16) return nchw ? li_launch<true, __half>(mapA, mapB, p, pairs, smem, st) : li_launch<false, __half>(mapA, mapB, p, pairs, smem, st);
    return nchw ? li_launch<true, __nv_bfloat16>(mapA, mapB, p, pairs, smem, st) : li_launch<false, __nv_bfloat16>(mapA, mapB, p, pairs, smem, st);
}
