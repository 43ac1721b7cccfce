// Dense algebra in 8-bit floating point with an fp32 scale for each block of 128 values along the reduction: quantisation of a
// tensor in both of its directions, and the product of two quantised matrices on the tensor cores.
#include <type_traits>
#include <cuda_fp8.h>
#include "tc_ptx.cuh"

namespace {

using namespace eb;

constexpr int kBlk = 128;
constexpr int kMaxSide = 0x7fffff00;            // indexes within the last tile of a side stay in 32 bits

// ---- quantisation ------------------------------------------------------------------------------------------------------------
// One block per 128 x 128 tile, one read of it for both directions; bound by memory (4 bytes read, 1 or 2 written a value).  A warp
// takes eight rows, a lane four columns of each, so a row's 128 values are one 512-byte access and their largest magnitude one warp
// reduction; the columns' come from the warps' through shared memory.  A scale is worked out by one lane (of a row) or thread (of a
// column) and handed to the others: a division a value would cost more than the copy.  The transpose goes through a 16 KB byte tile (8-byte
// pieces, swizzled so that neither side has bank conflicts to speak of) and leaves in 128-byte lines.
struct QuantArgs {
    const float *a;
    uint8_t *q, *qt;
    float *scale, *scale_t;
    size_t ldq, ldqt;
    int rows, cols, tiles_x;
    int pow2;
};

struct Scale { float scale, factor; };
template <int FORMAT>
__device__ __forceinline__ Scale scale_of(unsigned peak_bits, int pow2) {
    constexpr float largest = FORMAT == EDDLB200_E4M3 ? 448.f : 57344.f;
    constexpr unsigned least = 27u << 23;                              // 2^-100
    const float peak = __uint_as_float(max(peak_bits, least));
    if (peak_bits >= 0x7f800000u) return Scale{__uint_as_float(0x7f800000u), 0.f};
    if (!pow2) return Scale{__fdiv_rn(peak, largest), __fdiv_rn(largest, peak)};
    // both formats' largest number is 1.75 2^E: the power is the peak's own, one more where its mantissa is past 1.75
    constexpr int E = FORMAT == EDDLB200_E4M3 ? 8 : 15;
    const unsigned bits = __float_as_uint(peak);
    const int power = (int)(bits >> 23) - 127 - E + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    return Scale{__uint_as_float((unsigned)(power + 127) << 23), __uint_as_float((unsigned)(127 - power) << 23)};
}
template <int FORMAT>
__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
    constexpr __nv_fp8_interpretation_t kind = FORMAT == EDDLB200_E4M3 ? __NV_E4M3 : __NV_E5M2;
    const unsigned lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
    return lo | hi << 16;
}
template <int FORMAT, bool TILE, bool VEC>
__global__ void __launch_bounds__(512, 2) fp8_quantize_kernel(const QuantArgs a) {
    EB_GRID_WAIT();
    constexpr int WARPS = 16, ROWS = kBlk / WARPS;
    __shared__ float col_peak[WARPS][kBlk], col_factor[kBlk];
    __shared__ __align__(16) uint8_t turned[kBlk * kBlk];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int tx = blockIdx.x % a.tiles_x, ty = blockIdx.x / a.tiles_x;
    const int r0 = ty * kBlk + warp * ROWS, c0 = tx * kBlk + lane * 4;
    float v[ROWS][4];
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float *src = a.a + (size_t)(r0 + i) * a.cols + c0;
        const bool row = r0 + i < a.rows;
        if (VEC) {
            const float4 q = row && c0 < a.cols ? ld_stream4(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            v[i][0] = q.x; v[i][1] = q.y; v[i][2] = q.z; v[i][3] = q.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[i][j] = row && c0 + j < a.cols ? src[j] : 0.f;
        }
    }
    // largest magnitudes; fmaxf leaves a NaN out
    if (TILE || a.qt) {
        float mine[4] = {0.f, 0.f, 0.f, 0.f};                          // of the lane's columns over the warp's rows
#pragma unroll
        for (int i = 0; i < ROWS; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) mine[j] = fmaxf(mine[j], fabsf(v[i][j]));
        *reinterpret_cast<float4 *>(&col_peak[warp][lane * 4]) = make_float4(mine[0], mine[1], mine[2], mine[3]);
        __syncthreads();
    }
    Scale tile{0.f, 0.f};
    if (TILE) {
        // every warp looks through the columns of all
        float peak = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) {
            const float4 p = *reinterpret_cast<const float4 *>(&col_peak[w][lane * 4]);
            peak = fmaxf(peak, fmaxf(fmaxf(p.x, p.y), fmaxf(p.z, p.w)));
        }
        tile = scale_of<FORMAT>(__reduce_max_sync(0xffffffffu, __float_as_uint(peak)), a.pow2);
        if (threadIdx.x == 0) {
            const int row_blocks = (a.rows + kBlk - 1) / kBlk;
            if (a.q) a.scale[(size_t)tx * row_blocks + ty] = tile.scale;
            if (a.qt) a.scale_t[(size_t)ty * a.tiles_x + tx] = tile.scale;
        }
    } else if (a.qt && threadIdx.x < kBlk) {
        float peak = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; w++) peak = fmaxf(peak, col_peak[w][threadIdx.x]);
        const Scale s = scale_of<FORMAT>(__float_as_uint(peak), a.pow2);
        col_factor[threadIdx.x] = s.factor;
        if (tx * kBlk + (int)threadIdx.x < a.cols) a.scale_t[(size_t)ty * a.cols + tx * kBlk + threadIdx.x] = s.scale;
    }
    if (a.q) {
        Scale own = tile;                                              // of row `lane`
        if (!TILE) {
            unsigned peak = 0;
#pragma unroll
            for (int i = 0; i < ROWS; i++) {
                const unsigned of_row = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fmaxf(fmaxf(0.f, fabsf(v[i][0])), fabsf(v[i][1])), fmaxf(fabsf(v[i][2]), fabsf(v[i][3])))));
                if (lane == i) peak = of_row;
            }
            own = scale_of<FORMAT>(peak, a.pow2);
            if (lane < ROWS && r0 + lane < a.rows) a.scale[(size_t)tx * a.rows + r0 + lane] = own.scale;
        }
#pragma unroll
        for (int i = 0; i < ROWS; i++) {
            const float f = TILE ? tile.factor : __shfl_sync(0xffffffffu, own.factor, i);
            if (r0 + i >= a.rows || c0 >= a.cols) continue;
            const unsigned bytes = pack4<FORMAT>(__fmul_rn(v[i][0], f), __fmul_rn(v[i][1], f), __fmul_rn(v[i][2], f), __fmul_rn(v[i][3], f));
            uint8_t *dst = a.q + (size_t)(r0 + i) * a.ldq + c0;
            if (VEC || c0 + 4 <= a.cols) *reinterpret_cast<unsigned *>(dst) = bytes;
            else for (int j = 0; c0 + j < a.cols; j++) dst[j] = (uint8_t)(bytes >> 8 * j);
        }
    }
    if (!a.qt) return;
    float4 factor = make_float4(tile.factor, tile.factor, tile.factor, tile.factor);
    if (!TILE) {
        __syncthreads();
        factor = *reinterpret_cast<const float4 *>(&col_factor[lane * 4]);
    }
    const float each[4] = {factor.x, factor.y, factor.z, factor.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        unsigned b[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
            b[i] = pack4<FORMAT>(__fmul_rn(v[4 * i][j], each[j]), __fmul_rn(v[4 * i + 1][j], each[j]), __fmul_rn(v[4 * i + 2][j], each[j]), __fmul_rn(v[4 * i + 3][j], each[j]));
        // row lane * 4 + j of the turned tile, bytes warp * 8 ..: 16-byte piece warp / 2 lies at piece (warp / 2) ^ (lane & 7)
        *reinterpret_cast<uint2 *>(turned + (lane * 4 + j) * kBlk + (((warp >> 1) ^ lane) & 7) * 16 + (warp & 1) * 8) = make_uint2(b[0], b[1]);
    }
    __syncthreads();
    const int at = (threadIdx.x & 7) * 16, left = a.rows - ty * kBlk - at;            // bytes of this piece that are there
    if (left <= 0) return;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int col = (int)(threadIdx.x >> 3) + 64 * i, gc = tx * kBlk + col;
        if (gc >= a.cols) break;
        const uint8_t *src = turned + col * kBlk + (((threadIdx.x & 7) ^ (col >> 2)) & 7) * 16;
        uint8_t *dst = a.qt + (size_t)gc * a.ldqt + (size_t)ty * kBlk + at;
        if (left >= 16) *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src);
        else for (int j = 0; j < left; j++) dst[j] = src[j];
    }
}

template <int FORMAT>
auto quantize_kernel(bool tile, bool vec) {
    return tile ? (vec ? fp8_quantize_kernel<FORMAT, true, true> : fp8_quantize_kernel<FORMAT, true, false>)
                : (vec ? fp8_quantize_kernel<FORMAT, false, true> : fp8_quantize_kernel<FORMAT, false, false>);
}

// ---- product -----------------------------------------------------------------------------------------------------------------
// D[i][j] = sum over blocks b: s_i[b] s_j[b] sum_k P[i][k] Q[j][k].  The tensor core's M side (128 lanes of tensor memory) is the matrix whose rows are
// C's COLUMNS, so that the lanes of a warp store to neighbouring addresses, and its N side the one whose rows are C's rows: BN of
// them, as few as 16 for a single token.  Every K-block of 128 is one accumulation of four instructions into tensor memory; the
// epilogue warps take it out, scale it and add it to fp32 sums in registers while the next K-block runs into the other buffer.
// Where the tiles do not fill the GPU a cluster of up to eight blocks shares the K-blocks of a tile and adds its partial
// tiles in rank order through distributed shared memory: one launch, no partial sums in memory.
struct ProdParams {
    CUtensorMap map_p, map_q;
    const float *scale_p, *scale_q;
    float *c;
    volatile int *status;                    // site of a wait that gave up | warp << 8 | 6 or 7 << 16
    int p_rows, q_rows, kblocks;             // p_rows: columns of C, q_rows: rows of C
    int p_shift, q_shift, p_scales, q_scales;   // rows of a scale (log2) and scales of a K-block
    int tiles_p, splits, inc, tail;          // tail: the kernel on pairs halves that many tiles, the last ones
    unsigned idesc;
};

// Up to 64 rows of Q two blocks share an SM: the chain copy -> MMA -> epilogue of one K-block is long and its work short, so what counts is how many
// K-blocks are on their way (tensor memory holds BUFS of them a block).
template <int BN>
struct ProdShape {
    static constexpr int EPI = BN >= 64 ? 8 : 4, THREADS = 64 + EPI * 32, COLS = BN / (EPI / 4), PER_SM = BN <= 64 ? 2 : 1;
    static constexpr int STAGE = 128 * kBlk + BN * kBlk, STAGES = BN == 16 ? 6 : BN == 32 ? 5 : BN == 64 ? 4 : BN == 128 ? 6 : 4;
    static constexpr int BUFS = BN <= 32 ? 8 : BN == 256 ? 2 : 4, TMEM = BUFS * BN;
    static constexpr int PER_LANE = (COLS + 31) / 32;
    static constexpr int SCALES = EPI * 2 * PER_LANE * 32 * 4;
    static constexpr int SMEM = 1024 + STAGES * STAGE + SCALES;
    static_assert(STAGES * STAGE >= BN * 512, "the partial tile of a split takes the place of the operands");
    static_assert(PER_SM * TMEM <= 512 && PER_SM * (SMEM + 2048) <= 228 * 1024, "blocks of one SM");
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst_smem, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst_smem), "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// the copy engine's look at a map, ahead of its first copy
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory"); }
__device__ __forceinline__ void umma_fp8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// four values at this address in the shared memory of the cluster's block `rank`
__device__ __forceinline__ float4 lds4_of(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(map_to_rank(addr, rank)) : "memory");
    return v;
}
// fp32 sums, both operands K-major; formats: 0 = e4m3, 1 = e5m2
constexpr unsigned fp8_idesc(int format_a, int format_b, int m, int n) {
    return (1u << 4) | (unsigned)format_a << 7 | (unsigned)format_b << 10 | (unsigned)(n >> 3) << 17 | (unsigned)(m >> 4) << 24;
}

template <int BN>
__global__ void __launch_bounds__(ProdShape<BN>::THREADS, ProdShape<BN>::PER_SM) fp8_product_kernel(const __grid_constant__ ProdParams P) {
    using S = ProdShape<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float *scales = (float *)(ring + S::STAGES * S::STAGE);
    __shared__ __align__(8) uint64_t bars[2 * S::STAGES + 2 * S::BUFS];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * S::STAGES, bar_acc_full = bar_empty + 8 * S::STAGES, bar_acc_empty = bar_acc_full + 8 * S::BUFS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int split = (int)(blockIdx.x % P.splits), tile = (int)(blockIdx.x / P.splits);
    const int p0 = (tile % P.tiles_p) * 128, q0 = (tile / P.tiles_p) * BN;
    const int kb0 = (int)((long long)P.kblocks * split / P.splits), kb1 = (int)((long long)P.kblocks * (split + 1) / P.splits);
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; s++) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int s = 0; s < S::BUFS; s++) { mbar_init(bar_acc_full + 8 * s, 1); mbar_init(bar_acc_empty + 8 * s, S::EPI); }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&P.map_p); prefetch_map(&P.map_q);
    }
    if (warp == 1) tmem_alloc(smem_u32(&tmem_slot), S::TMEM);
    EB_GRID_WAIT();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    int fail = 0;
    float acc[S::COLS];
#pragma unroll
    for (int i = 0; i < S::COLS; i++) acc[i] = 0.f;
    const int quarter = warp & 3, half = (warp - 2) >> 2;              // of an epilogue warp

    if (warp == 0) {
        // ============================ copies ============================
        if (elect_one()) {
            int s = 0, uses = 0; uint32_t phase = 1;
            for (int kb = kb0; kb < kb1; kb++, uses++) {
                if (!mbar_wait(bar_empty + 8 * s, phase, abort_flag)) { fail = 1; break; }
                mbar_expect_tx(bar_full + 8 * s, S::STAGE);
                const uint32_t dst = smem_u32(ring) + s * S::STAGE;
                tma_load_2d(dst, &P.map_p, kb * kBlk, p0, bar_full + 8 * s);
                tma_load_2d(dst + 128 * kBlk, &P.map_q, kb * kBlk, q0, bar_full + 8 * s);
                if (++s == S::STAGES) { s = 0; phase ^= 1u; }
            }
            // no copy is on its way when the block ends, whoever gave up
            for (int i = 0; i < S::STAGES && i < uses; i++) {
                if (--s < 0) { s = S::STAGES - 1; phase ^= 1u; }
                if (!mbar_wait(bar_full + 8 * s, phase ^ 1u, abort_flag)) fail = 5;
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // ============================ MMA issue ============================
        if (elect_one()) {
            int s = 0, buf = 0; uint32_t phase = 0, acc_phase = 1;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!mbar_wait(bar_acc_empty + 8 * buf, acc_phase, abort_flag)) { fail = 2; break; }
                if (!mbar_wait(bar_full + 8 * s, phase, abort_flag)) { fail = 3; break; }
                tc_fence_after();
                const uint64_t pd = make_desc(smem_u32(ring) + s * S::STAGE), qd = make_desc(smem_u32(ring) + s * S::STAGE + 128 * kBlk);
#pragma unroll
                for (int k = 0; k < 4; k++) umma_fp8(tmem + buf * BN, pd + 2 * k, qd + 2 * k, P.idesc, k ? 1u : 0u);
                umma_commit(bar_empty + 8 * s);
                umma_commit(bar_acc_full + 8 * buf);
                if (++s == S::STAGES) { s = 0; phase ^= 1u; }
                if (++buf == S::BUFS) { buf = 0; acc_phase ^= 1u; }
            }
        }
        __syncwarp();
    } else {
        // ============================ epilogue ============================
        float *mine = scales + (warp - 2) * (2 * S::PER_LANE * 32);
        const int p = p0 + quarter * 32 + lane, q = q0 + half * S::COLS;
        const float *sp = P.scale_p + min(p, P.p_rows - 1) / (1 << P.p_shift);
        float next_p = 0.f, next_q[S::PER_LANE];
        auto fetch = [&](int kb) {
            if (kb >= kb1) return;
            next_p = __ldg(sp + (size_t)kb * P.p_scales);
#pragma unroll
            for (int i = 0; i < S::PER_LANE; i++) {
                const int row = q + i * 32 + lane;
                next_q[i] = row < P.q_rows ? __ldg(P.scale_q + (size_t)kb * P.q_scales + (row >> P.q_shift)) : 0.f;
            }
        };
        fetch(kb0);
        int buf = 0; uint32_t phase = 0;
        for (int kb = kb0; kb < kb1; kb++) {
            float *line = mine + ((buf & 1) * S::PER_LANE) * 32;
#pragma unroll
            for (int i = 0; i < S::PER_LANE; i++) line[i * 32 + lane] = next_q[i];
            const float s_p = next_p;
            __syncwarp();
            fetch(kb + 1);
            if (!mbar_wait_warp(bar_acc_full + 8 * buf, phase, abort_flag)) { fail = 4; break; }
            tc_fence_after();
            const uint32_t base = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN + half * S::COLS);
#pragma unroll
            for (int c = 0; c < S::COLS; c += 16) {
                uint32_t r[16];
                tmem_ld16(base + c, r);
#pragma unroll
                for (int j = 0; j < 16; j += 4) {
                    const float4 s4 = *reinterpret_cast<const float4 *>(line + c + j);
                    acc[c + j] = fmaf(__uint_as_float(r[j]) * s4.x, s_p, acc[c + j]);
                    acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]) * s4.y, s_p, acc[c + j + 1]);
                    acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]) * s4.z, s_p, acc[c + j + 2]);
                    acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]) * s4.w, s_p, acc[c + j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_acc_empty + 8 * buf);
            if (++buf == S::BUFS) { buf = 0; phase ^= 1u; }
        }
        if (P.splits == 1) {
            float *dst = P.c + (size_t)q * P.p_rows + p;
            if (p < P.p_rows) {
#pragma unroll
                for (int i = 0; i < S::COLS; i++)
                    if (q + i < P.q_rows) {
                        float *at = dst + (size_t)i * P.p_rows;
                        *at = P.inc ? *at + acc[i] : acc[i];
                    }
            }
        } else {
            // every operand has been read by an MMA that has completed: the ring takes the partial tile
            float *part = (float *)ring + (half * S::COLS) * 128 + quarter * 32 + lane;
#pragma unroll
            for (int i = 0; i < S::COLS; i++) part[i * 128] = acc[i];
        }
    }
    if (fail) { *abort_flag = 1; *P.status = fail | warp << 8 | 6 << 16; }
    if (P.splits > 1) {
        __syncwarp();
        cluster_arrive(); cluster_wait();
        if (warp >= 2) {
            // a warp a row of C at a time, a lane four neighbouring values: its loads from all blocks are on their way together
            const int p = p0 + lane * 4;
            const bool straight = P.p_rows % 4 == 0 && aligned16(P.c);
#pragma unroll 2
            for (int i = split + P.splits * (warp - 2); i < BN && q0 + i < P.q_rows; i += P.splits * S::EPI) {
                float4 v[8];
#pragma unroll
                for (int r = 0; r < 8; r++) if (r < P.splits) v[r] = lds4_of(smem_u32(ring) + (i * 128 + lane * 4) * 4, r);
                float4 sum = v[0];
#pragma unroll
                for (int r = 1; r < 8; r++) if (r < P.splits) { sum.x += v[r].x; sum.y += v[r].y; sum.z += v[r].z; sum.w += v[r].w; }
                float *at = P.c + (size_t)(q0 + i) * P.p_rows + p;
                if (straight && p < P.p_rows) {
                    if (P.inc) { const float4 o = *reinterpret_cast<const float4 *>(at); sum.x += o.x; sum.y += o.y; sum.z += o.z; sum.w += o.w; }
                    *reinterpret_cast<float4 *>(at) = sum;
                } else {
                    const float each[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
                    for (int k = 0; k < 4; k++) if (p + k < P.p_rows) at[k] = P.inc ? at[k] + each[k] : each[k];
                }
            }
        }
        cluster_arrive(); cluster_wait();                   // a block's shared memory outlives the reads of the others
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM);
}

// ---- product of large matrices -------------------------------------------------------------------------------------------------
// Pairs of CTAs (cta_group::2) that walk over tiles of 256 rows of P x 256 rows of Q: each CTA holds its own 128 rows of P and HALF of the rows of Q, so a
// K-block moves 32 KB into each shared memory and is four instructions of 256 x 256 x 32 into one of two buffers of tensor memory.  Sixteen
// epilogue warps, 32 lanes and 64 columns each, take a buffer out, scale it and add it to fp32 sums in registers while the next K-block
// runs into the other one: four warps a scheduler hide the latencies between them (with eight warps of 128 columns the MMAs waited, 645 us).
// What bounds it is power and operand traffic: 8192 x 8192 x 8192 takes 600 to 625 us on a layer's values, the GPU at its 1000 W and 1.5 GHz (500 on codes
// of one sign); the MMAs alone on operands that are not copied 366 us at the same power, with the copies (64 KB a pair and K-block out of L2, 9 TB/s) 485.
// Which operand is P is chosen so that scaling costs least: a matrix with a scale for 128 rows goes to the N side, where a warp's columns
// share it, and an element takes one multiply-add; with a scale for every row on both sides the N side's are read from shared memory.
// C's rows are P's rows here (ROWS) or Q's; in the first case a warp's values are turned through shared memory on their way out.
// Registers: 640 threads are launched with 96 each; the copy and issue warps keep 56, the epilogue takes 104:
// 128 x 56 + 512 x 104 = 60416 of 640 x 96 = 61440.
constexpr int LG_STAGES = 5, LG_STAGE = 2 * 128 * kBlk, LG_THREADS = 640, LG_LINE = 32 * 17 * 4;
constexpr int LG_SMEM = 1024 + LG_STAGES * LG_STAGE + 16 * LG_LINE;

__device__ __forceinline__ void umma_fp8_pair(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
}
// 16 or 8 columns of the warp's lanes, not waited for
__device__ __forceinline__ void tmem_ask(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ask(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(taddr) : "memory");
}
// the registers of the loads so far may be read: they pass through the wait, so that no use of them is moved ahead of it
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[8]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) :: "memory");
}
__device__ __forceinline__ void sts(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ float lds(uint32_t addr) { float v; asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory"); return v; }
__device__ __forceinline__ float4 lds4(uint32_t addr) {
    float4 v; asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory"); return v;
}

template <bool VEC, bool ROWS, bool HALVES>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(LG_THREADS, 1) fp8_product_large_kernel(const __grid_constant__ ProdParams P) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *ring = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t lines = smem_u32(ring) + LG_STAGES * LG_STAGE;
    __shared__ __align__(8) uint64_t bars[2 * LG_STAGES + 4];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_word;
    volatile int *abort_flag = &abort_word;
    const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * LG_STAGES, bar_acc_full = bar_empty + 8 * LG_STAGES, bar_acc_empty = bar_acc_full + 16;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = (int)(blockIdx.x >> 1), pairs = (int)(gridDim.x >> 1), kblocks = P.kblocks;
    const int tiles_p = P.tiles_p, tail = HALVES ? P.tail : 0, whole = tiles_p * P.splits - tail, jobs = whole + 2 * tail;         // splits: here the tiles along Q
    // Tiles in bands of twelve along P, so that the pairs at work at a time share operands in L2 (8192 cubed: 600 us in the same run that took 635 in bands of eight).
    // The tiles of a last round that fills half of the pairs or less are worked on in halves of 128 rows of Q, job >= whole.
    auto place = [&](int job, int &p0, int &q0) {
        const int tile = !HALVES || job < whole ? job : whole + (job - whole) / 2;
        const int band = tile / (12 * P.splits), in = tile - band * 12 * P.splits, wide = min(12, tiles_p - band * 12);
        p0 = (band * 12 + in % wide) * 256; q0 = in / wide * 256 + (!HALVES || job < whole ? 0 : (job - whole) % 2 * 128);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < LG_STAGES; s++) { mbar_init(bar_full + 8 * s, 1); mbar_init(bar_empty + 8 * s, 1); }
        for (int s = 0; s < 2; s++) { mbar_init(bar_acc_full + 8 * s, 1); mbar_init(bar_acc_empty + 8 * s, 32); }
        abort_word = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        prefetch_map(&P.map_p); prefetch_map(&P.map_q);
    }
    if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot), 512);
    EB_GRID_WAIT();
    tc_fence_before();
    __syncthreads();
    cluster_arrive(); cluster_wait();                        // the other CTA's barriers are initialised before anything arrives on them
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    int fail = 0;

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0 && elect_one()) {
            // ============================ copies ============================
            const uint32_t full_of_first = map_to_rank(bar_full, 0);
            int s = 0, uses = 0; uint32_t phase = 1;
            for (int job = pair; job < jobs && !fail; job += pairs) {
                int p0, q0;
                place(job, p0, q0);
                const bool half = HALVES && job >= whole;
                q0 += (int)rank * (half ? 64 : 128);
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!mbar_wait(bar_empty + 8 * s, phase, abort_flag)) { fail = 1; break; }
                    if (rank == 0) mbar_expect_tx(bar_full + 8 * s, half ? 2 * LG_STAGE - 128 * kBlk : 2 * LG_STAGE);       // the bytes of both CTAs
                    const uint32_t dst = smem_u32(ring) + s * LG_STAGE;
                    tma_load_2d_pair(dst, &P.map_p, kb * kBlk, p0 + (int)rank * 128, full_of_first + 8 * s);
                    tma_load_2d_pair(dst + 128 * kBlk, &P.map_q, kb * kBlk, q0, full_of_first + 8 * s);
                    if (HALVES && !half) tma_load_2d_pair(dst + 192 * kBlk, &P.map_q, kb * kBlk, q0 + 64, full_of_first + 8 * s);
                    uses++;
                    if (++s == LG_STAGES) { s = 0; phase ^= 1u; }
                }
            }
            // the last arrivals on this CTA's barriers come from the other CTA: stay until they are in
            // (after a wait that gave up: until the copies are in, which the first CTA's barriers know for both)
            for (int i = 0; i < LG_STAGES && i < uses; i++) {
                if (--s < 0) { s = LG_STAGES - 1; phase ^= 1u; }
                if (fail) { if (rank == 0) mbar_wait(bar_full + 8 * s, phase ^ 1u, abort_flag); }
                else if (!mbar_wait(bar_empty + 8 * s, phase ^ 1u, abort_flag)) fail = 5;
            }
        } else if (warp == 1 && rank == 0 && elect_one()) {
            // ============================ MMA issue ============================
            int s = 0, buf = 0; uint32_t phase = 0, acc_phase = 1;
            for (int job = pair; job < jobs && !fail; job += pairs) {
                const unsigned idesc = !HALVES || job < whole ? P.idesc : P.idesc - (16u << 17);      // 256 or 128 columns
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!mbar_wait(bar_full + 8 * s, phase, abort_flag)) { fail = 3; break; }
                    if (!mbar_wait(bar_acc_empty + 8 * buf, acc_phase, abort_flag)) { fail = 2; break; }
                    tc_fence_after();
                    const uint64_t pd = make_desc(smem_u32(ring) + s * LG_STAGE), qd = make_desc(smem_u32(ring) + s * LG_STAGE + 128 * kBlk);
#pragma unroll
                    for (int k = 0; k < 4; k++) umma_fp8_pair(tmem + buf * 256, pd + 2 * k, qd + 2 * k, idesc, k ? 1u : 0u);
                    umma_commit_pair(bar_acc_full + 8 * buf);
                    umma_commit_pair(bar_empty + 8 * s);
                    if (++s == LG_STAGES) { s = 0; phase ^= 1u; }
                    if (++buf == 2) { buf = 0; acc_phase ^= 1u; }
                }
            }
        }
        __syncwarp();
    } else {
        // ============================ epilogue ============================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
        const int quarter = warp & 3, group = (warp - 4) >> 2;                 // 32 lanes, COLS columns
        const uint32_t empty_of_first = map_to_rank(bar_acc_empty, 0);
        const uint32_t line = lines + (warp - 4) * LG_LINE;
        uint32_t done = 0;                                       // K-blocks: every other one lies in the first buffer
        auto tile = [&](auto columns, int job) {
            constexpr int COLS = decltype(columns)::value;
            const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(group * COLS);
            int p0, q0;
            place(job, p0, q0);
            const int p = p0 + (int)rank * 128 + quarter * 32 + lane, q = q0 + group * COLS;
            const float *sp = P.scale_p + (min(p, P.p_rows - 1) >> P.p_shift), *sq = P.scale_q + (VEC ? min(q + lane, P.q_rows - 1) : min(q, P.q_rows - 1) >> 7);
            const int second = VEC && COLS == 64 && q + 32 + lane < P.q_rows ? 32 : 0;                // a column past the last one takes another's scale: its products are zero
            float acc[COLS];
#pragma unroll
            for (int i = 0; i < COLS; i++) acc[i] = 0.f;
            // scales of the next two K-blocks, on their way
            float ahead_p[2], ahead_q[2][2];
            int left = kblocks;                              // K-blocks whose scales have not been asked for
            auto fetch = [&](int slot, bool more) {
                if (HALVES ? !more : --left < 0) return;     // the same; each form where it leaves no register spilled (with spills 8192 cubed took 800 us)
                ahead_p[slot] = __ldg(sp);
                ahead_q[slot][0] = __ldg(sq);
                if (VEC && COLS == 64) ahead_q[slot][1] = __ldg(sq + second);
                sp += P.p_scales; sq += P.q_scales;
            };
            auto block = [&](int slot, bool more) {
                const uint32_t scales = line + slot * 256;
                // one factor where a warp's columns share a scale; multiplying by one after the other where their product is no normal number would need
                // registers that are not there (with that path 8192 cubed took 524 us, without 506; with A's scales shared and B's not 660 and 486)
                const float s_p = VEC ? ahead_p[slot] : ahead_p[slot] * ahead_q[slot][0];
                if (VEC) sts(scales + lane * 4, ahead_q[slot][0]);
                if (VEC && COLS == 64) sts(scales + 128 + lane * 4, ahead_q[slot][1]);
                fetch(slot, more);
                const uint32_t buf = done & 1;
                if (!mbar_wait(bar_acc_full + 8 * buf, done >> 1 & 1, abort_flag)) fail = 4;
                if (__any_sync(0xffffffffu, fail)) { fail = 4; return; }
                if (VEC) __syncwarp();                       // the scales of the other lanes
                tc_fence_after();
                const uint32_t base = from + buf * 256;
                constexpr int PIECE = VEC ? 8 : 16,                // the scales from shared memory take registers too (by 16 there: 120 us for 4096 cubed, by 8 110)
                              PIECES = COLS / PIECE;
                uint32_t r[2][PIECE];
                tmem_ask(base, r[0]);
#pragma unroll
                for (int c = 0; c < PIECES; c++) {
                    tmem_wait(r[c & 1]);
                    if (c < PIECES - 1) tmem_ask(base + PIECE * (c + 1), r[(c + 1) & 1]);
                    else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(empty_of_first + 8 * buf);
                    }
#pragma unroll
                    for (int j = 0; j < PIECE; j += 4) {
                        float4 d = make_float4(__uint_as_float(r[c & 1][j]), __uint_as_float(r[c & 1][j + 1]), __uint_as_float(r[c & 1][j + 2]), __uint_as_float(r[c & 1][j + 3]));
                        if (VEC) { const float4 s4 = lds4(scales + (c * PIECE + j) * 4); d.x *= s4.x; d.y *= s4.y; d.z *= s4.z; d.w *= s4.w; }
                        float *to = acc + c * PIECE + j;
                        to[0] = fmaf(d.x, s_p, to[0]); to[1] = fmaf(d.y, s_p, to[1]); to[2] = fmaf(d.z, s_p, to[2]); to[3] = fmaf(d.w, s_p, to[3]);
                    }
                }
                done++;
            };
            fetch(0, true); fetch(1, kblocks > 1);
#pragma unroll 1
            for (int kb = kblocks; kb > 0 && !fail; kb -= 2) {
                block(0, kb > 2);
                if (kb > 1 && !fail) block(1, kb > 3);
            }
            if (fail) return;
            if (ROWS) {
                // C [p_rows][q_rows]: a lane holds a row's values, 32 rows x 16 columns at a time are turned
                const int p_first = p0 + (int)rank * 128 + quarter * 32, rows = min(32, P.p_rows - p_first) - (lane >> 4);
                auto out = [&](auto whole, auto inc) {
#pragma unroll
                    for (int c = 0; c < COLS / 16; c++) {
                        __syncwarp();
#pragma unroll
                        for (int j = 0; j < 16; j++) sts(line + (lane * 17 + j) * 4, acc[c * 16 + j]);
                        __syncwarp();
                        const int col = q + c * 16 + (lane & 15);
                        float *dst = P.c + (size_t)(p_first + (lane >> 4)) * P.q_rows + col;
                        if (col >= P.q_rows) continue;
#pragma unroll 8
                        for (int i = 0; i < 32; i += 2, dst += 2 * (size_t)P.q_rows) {
                            if (!decltype(whole)::value && i >= rows) break;
                            const float v = lds(line + ((i + (lane >> 4)) * 17 + (lane & 15)) * 4);
                            *dst = decltype(inc)::value ? *dst + v : v;
                        }
                    }
                };
                if (P.inc) out(std::false_type(), std::true_type());
                else if (p_first + 32 <= P.p_rows) out(std::true_type(), std::false_type());
                else out(std::false_type(), std::false_type());
                __syncwarp();
            } else if (p < P.p_rows) {
                // C [q_rows][p_rows]: the lanes are neighbours in memory
                float *dst = P.c + (size_t)q * P.p_rows + p;
                const int columns = P.q_rows - q;
                if (!P.inc && columns >= COLS) {
#pragma unroll
                    for (int i = 0; i < COLS; i++, dst += P.p_rows) *dst = acc[i];
                } else {
#pragma unroll
                    for (int i = 0; i < COLS; i++, dst += P.p_rows) if (i < columns) *dst = P.inc ? *dst + acc[i] : acc[i];
                }
            }
            // with an odd number of K-blocks the next tile's first scales take the place of this tile's last ones
            if (VEC) __syncwarp();
        };
        for (int job = pair; job < jobs && !fail; job += pairs) {
            if (!HALVES || job < whole) tile(std::integral_constant<int, 64>(), job);
            else if constexpr (HALVES) tile(std::integral_constant<int, 32>(), job);
        }
    }
    if (fail) { *abort_flag = 1; *P.status = fail | warp << 8 | 7 << 16; }
    tc_fence_before();
    __syncthreads();
    // both CTAs are done with each other's barriers, shared memory and accumulators
    cluster_arrive(); cluster_wait();
    if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

template <bool VEC, bool ROWS, bool HALVES>
int launch_large(DevCtx *cx, int dev, cudaStream_t st, const ProdParams &P) {
    static bool configured[EDDLB200_MAX_DEVICES] = {};
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(fp8_product_large_kernel<VEC, ROWS, HALVES>, cudaFuncAttributeMaxDynamicSharedMemorySize, LG_SMEM);
        if (e != cudaSuccess) return cuda_status(e, "fp8_mult2d(attributes)");
        configured[dev] = true;
    }
    const int jobs = P.tiles_p * P.splits + P.tail, pairs = jobs < EDDLB200_NUM_SMS / 2 ? jobs : EDDLB200_NUM_SMS / 2;
    eb::launch(fp8_product_large_kernel<VEC, ROWS, HALVES>, 2 * pairs, LG_THREADS, LG_SMEM, st, P);
    EB_LAUNCH_CHECK("fp8_mult2d");
    return 0;
}

template <bool HALVES>
int large_product(DevCtx *cx, int dev, cudaStream_t st, const ProdParams &P, int block_a, int block_b) {
    return block_b == kBlk ? launch_large<false, true, HALVES>(cx, dev, st, P) : block_a == kBlk ? launch_large<false, false, HALVES>(cx, dev, st, P) : launch_large<true, false, HALVES>(cx, dev, st, P);
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *, const cuuint32_t *,
                             const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
// the driver entry point is looked up at run time: the library must load (and refuse work) on a machine without a driver
EncodeFn encode_function() {
    static const EncodeFn encode = []() -> EncodeFn {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess) return (EncodeFn)fn;
        cudaGetLastError();
        return nullptr;
    }();
    return encode;
}
// [rows][cols] bytes as boxes of 128 columns and box_rows rows in the K-major 128-byte swizzle; what lies past either edge arrives as zeros
bool encode_bytes_map(CUtensorMap *map, const void *base, size_t ld, int rows, int cols, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)kBlk, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    const EncodeFn encode = encode_function();
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN>
int launch_product(DevCtx *cx, cudaStream_t st, const ProdParams &P, unsigned tiles) {
    using S = ProdShape<BN>;
    if (P.splits > 1) eb::launch_cluster(fp8_product_kernel<BN>, (unsigned)P.splits, tiles * P.splits, S::THREADS, S::SMEM, st, P);
    else eb::launch(fp8_product_kernel<BN>, tiles, S::THREADS, S::SMEM, st, P);
    EB_LAUNCH_CHECK("fp8_mult2d");
    return 0;
}

// What the device holds at once of each tile's kernel: clusters of 1 .. 8 blocks.  A cluster lies within one group of SMs, so their number is not that of
// the blocks divided by the size (1 x 6000 x 6000: 47 clusters of six are two rounds, 15.6 us, 47 of five one, 11.2).  Looked up with the first product on a
// device, along with the kernels' attributes.  The query counts one block an SM of a kernel that uses tensor memory; two of the small tiles' are there
// (10.3 warps of blocks of six active on an SM in a profile of 1 x 8192 x 8192), so its numbers of clusters are doubled.
struct Residents { bool known = false; int of[5][9]; };        // blocks, clusters of 2 .. 8
Residents g_residents[EDDLB200_MAX_DEVICES];
template <int BN>
cudaError_t look_up_residents(int (&of)[9]) {
    using S = ProdShape<BN>;
    cudaError_t e = cudaFuncSetAttribute(fp8_product_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&of[1], fp8_product_kernel<BN>, S::THREADS, S::SMEM);
    const int twice = e == cudaSuccess && of[1] == 1 ? S::PER_SM : 1;
    of[1] *= twice * EDDLB200_NUM_SMS;
    for (int size = 2; size <= 8 && e == cudaSuccess; size++) {
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension; at[0].val.clusterDim.x = size; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t c = {};
        c.gridDim = dim3(EDDLB200_NUM_SMS * S::PER_SM / size * size); c.blockDim = dim3(S::THREADS); c.dynamicSmemBytes = S::SMEM; c.attrs = at; c.numAttrs = 1;
        e = cudaOccupancyMaxActiveClusters(&of[size], fp8_product_kernel<BN>, &c);
        of[size] *= twice;
    }
    return e;
}
int product_residents(int dev, const Residents *&out) {
    Residents &r = g_residents[dev];
    out = &r;
    if (r.known) return 0;
    cudaError_t e = look_up_residents<16>(r.of[0]);
    if (e == cudaSuccess) e = look_up_residents<32>(r.of[1]);
    if (e == cudaSuccess) e = look_up_residents<64>(r.of[2]);
    if (e == cudaSuccess) e = look_up_residents<128>(r.of[3]);
    if (e == cudaSuccess) e = look_up_residents<256>(r.of[4]);
    if (e != cudaSuccess) return cuda_status(e, "fp8_mult2d(occupancy)");
    r.known = true;
    return 0;
}

// Which kernel, tile and split: the least estimated time, in cycles of an SM.  The figures are fitted to a sweep of 19 shapes from 1 x 1024 x 1024 to
// 1024 x 4096 x 4096 over all tiles and splits; the estimates are within 20 % of it.  A K-block costs an SM its operands' way through L2 or, in the
// wide tiles, the epilogue's; alone on its SM a block waits at least for its own chain.  A tile costs its start and its stores and, when split,
// the exchange between the blocks of a cluster.  256 x 4096 x 4096: 128 rows in two splits 15.8 us, pairs 22.0; 2048 cubed: pairs 16.0, 256 rows 24.8.
struct Plan { int bn = 0, splits = 1; size_t tiles = 0, halved = 0; };   // bn 0: the kernel on pairs of CTAs, which halves the last tiles
Plan pick_plan(const Residents &held, int m, int n, int kblocks) {
    Plan best;
    best.tiles = ceil_div(m, 256) * ceil_div(n, 256);
    // a last round for half of the pairs or less is halved (2304 x 2304 x 4096: 52 us, in two whole rounds 63; 4096 cubed 90 and 94; 512 x 4096 x 4096:
    // 17.9, with tiles of 256 x 128 on single CTAs 26)
    const size_t pairs = EDDLB200_NUM_SMS / 2, last = best.tiles % pairs;
    best.halved = last <= pairs / 2 ? last : 0;
    const double last_block = last > pairs / 2 ? 1050.0 : last ? 630.0 : 0.0;
    double least = (best.tiles / pairs * 1050.0 + last_block) * kblocks + (double)ceil_div(best.tiles, pairs) * 8000.0;
    for (int bn = 16; bn <= 256; bn *= 2) {
        if (bn > 16 && bn / 2 >= m) break;                           // half of the tile would be empty
        const int which = bn == 16 ? 0 : bn == 32 ? 1 : bn == 64 ? 2 : bn == 128 ? 3 : 4;
        const size_t tiles = ceil_div(n, 128) * ceil_div(m, bn);
        const double block = bn == 16 ? 410.0 : bn == 32 ? 450.0 : bn == 64 ? 580.0 : bn == 128 ? 950.0 : 1800.0;
        const double alone = bn == 16 ? 600.0 : bn == 32 ? 720.0 : bn == 64 ? 950.0 : block;
        for (int splits = 1; splits <= 8 && splits <= kblocks; splits++) {
            if (held.of[which][splits] < 1) continue;
            const size_t jobs = tiles * splits, rounds = ceil_div(tiles, (size_t)held.of[which][splits]), on_one = ceil_div(jobs, (size_t)EDDLB200_NUM_SMS);
            const double each = (double)ceil_div(kblocks, splits);
            const double work = on_one > 1 ? on_one * each * block : each * alone;
            const double t = work + rounds * (4000.0 + 25.0 * bn + (splits > 1 ? 700.0 * splits + 8.0 * bn : 0.0));
            if (t < least) { least = t; best.bn = bn; best.splits = splits; best.tiles = tiles; }
        }
    }
    return best;
}

size_t matrix_bytes(int rows, int cols, size_t ld) { return rows && cols ? (size_t)(rows - 1) * ld + cols : 0; }
size_t scale_bytes(int rows, int cols, int block_rows) { return ceil_div(cols, kBlk) * ceil_div(rows, block_rows) * sizeof(float); }

}  // namespace

using namespace eb;

extern "C" {

int eddlb200_fp8_quantize(int dev, const float *a, int rows, int cols, int format, int block_rows, int pow2,
                          void *q, size_t ldq, float *scale, void *qt, size_t ldqt, float *scale_t) {
    const char *what = "fp8_quantize";
    EB_REQUIRE(rows >= 0 && cols >= 0, what);
    EB_REQUIRE(format == EDDLB200_E4M3 || format == EDDLB200_E5M2, what);
    EB_REQUIRE(block_rows == 1 || block_rows == kBlk, what);
    EB_REQUIRE(pow2 == 0 || pow2 == 1, what);
    EB_REQUIRE(q || qt, what);
    EB_REQUIRE(!q || (scale && aligned16(q) && ldq % 16 == 0 && ldq >= (size_t)cols), what);
    EB_REQUIRE(!qt || (scale_t && aligned16(qt) && ldqt % 16 == 0 && ldqt >= (size_t)rows), what);
    EB_REQUIRE(!rows || !cols || a, what);
    const size_t tiles = ceil_div(rows, kBlk) * ceil_div(cols, kBlk);
    if (rows > kMaxSide || cols > kMaxSide || tiles > 0x7fffffff) return set_error(EDDLB200_ELIMIT, "%s: %d x %d", what, rows, cols);
    EB_REQUIRE(aligned4(a) && aligned4(scale) && aligned4(scale_t), what);
    const size_t in = (size_t)rows * cols * sizeof(float);
    const void *out[] = {q, scale, qt, scale_t};
    const size_t bytes[] = {matrix_bytes(rows, cols, ldq), scale_bytes(rows, cols, block_rows), matrix_bytes(cols, rows, ldqt), scale_bytes(cols, rows, block_rows)};
    for (int i = 0; i < 4; i++) {
        if (!out[i / 2 * 2]) continue;
        EB_REQUIRE(!overlap(out[i], bytes[i], a, in), what);
        for (int j = 0; j < i; j++) EB_REQUIRE(!out[j / 2 * 2] || !overlap(out[i], bytes[i], out[j], bytes[j]), what);
    }
    EB_CTX(dev);
    if (!rows || !cols) return 0;
    EB_READS(a, in);
    for (int i = 0; i < 4; i++) {
        if (!out[i / 2 * 2]) continue;
        if (i & 1) EB_WRITES(out[i], bytes[i]); else EB_MODIFIES(out[i], bytes[i]);           // bytes between the rows stay
    }
    ProfScope prof(cx, PROF_ELEMENTWISE, (double)rows * cols * (4 + (q ? 1 : 0) + (qt ? 1 : 0)));
    const QuantArgs args{a, (uint8_t *)q, (uint8_t *)qt, scale, scale_t, ldq, ldqt, rows, cols, (int)ceil_div(cols, kBlk), pow2};
    const bool vec = cols % 4 == 0 && aligned16(a);
    auto kernel = format == EDDLB200_E4M3 ? quantize_kernel<EDDLB200_E4M3>(block_rows == kBlk, vec) : quantize_kernel<EDDLB200_E5M2>(block_rows == kBlk, vec);
    eb::launch(kernel, (unsigned)tiles, 512, 0, st, args);
    EB_LAUNCH_CHECK(what);
    return 0;
}

int eddlb200_fp8_mult2d(int dev, const void *qa, size_t lda, const float *scale_a, int format_a, int block_a, const void *qb, size_t ldb,
                        const float *scale_b, int format_b, int block_b, float *c, int inc_c, int m, int n, int k) {
    const char *what = "fp8_mult2d";
    EB_REQUIRE(m >= 0 && n >= 0 && k >= 0, what);
    EB_REQUIRE((format_a == EDDLB200_E4M3 || format_a == EDDLB200_E5M2) && (format_b == EDDLB200_E4M3 || format_b == EDDLB200_E5M2), what);
    EB_REQUIRE((block_a == 1 || block_a == kBlk) && (block_b == 1 || block_b == kBlk), what);
    EB_REQUIRE(lda % 16 == 0 && ldb % 16 == 0 && lda >= (size_t)k && ldb >= (size_t)k, what);
    EB_REQUIRE(lda < ((size_t)1 << 40) && ldb < ((size_t)1 << 40), what);
    EB_REQUIRE(!m || !n || c, what);
    EB_REQUIRE(!m || !n || !k || (qa && qb && scale_a && scale_b && aligned16(qa) && aligned16(qb)), what);
    EB_REQUIRE(aligned4(c) && aligned4(scale_a) && aligned4(scale_b), what);
    if (m > kMaxSide || n > kMaxSide || k > kMaxSide) return set_error(EDDLB200_ELIMIT, "%s: %d x %d x %d", what, m, n, k);
    const size_t out = (size_t)m * n * sizeof(float);
    const void *in[] = {qa, qb, scale_a, scale_b};
    const size_t bytes[] = {matrix_bytes(m, k, lda), matrix_bytes(n, k, ldb), scale_bytes(m, k, block_a), scale_bytes(n, k, block_b)};
    for (int i = 0; i < 4; i++) EB_REQUIRE(!overlap(c, out, in[i], bytes[i]), what);
    EB_CTX(dev);
    if (!m || !n) return 0;
    ProdParams P;
    P.c = c; P.status = fp8_status(cx); P.kblocks = (int)ceil_div(k, kBlk);
    struct Side { const void *q; size_t ld; const float *scale; int rows, block, format; };
    const Side sa{qa, lda, scale_a, m, block_a, format_a}, sb{qb, ldb, scale_b, n, block_b, format_b};
    auto sides = [&](const Side &p, const Side &q, int p_box, int q_box) {
        P.scale_p = p.scale; P.scale_q = q.scale;
        P.p_rows = p.rows; P.q_rows = q.rows;
        P.p_shift = p.block == kBlk ? 7 : 0; P.q_shift = q.block == kBlk ? 7 : 0;
        P.p_scales = (int)ceil_div(p.rows, p.block); P.q_scales = (int)ceil_div(q.rows, q.block);
        return encode_bytes_map(&P.map_p, p.q, p.ld, p.rows, k, p_box) && encode_bytes_map(&P.map_q, q.q, q.ld, q.rows, k, q_box);
    };
    Plan plan;
    if (k) {
        const Residents *held;
        if (int e = product_residents(dev, held)) return e;
        plan = pick_plan(*held, m, n, P.kblocks);
        if (plan.tiles > 0x0fffffff) return set_error(EDDLB200_ELIMIT, "%s: %d x %d", what, m, n);
        // C's rows are P's where only B's scales are shared by 128 rows: the side whose scales cost less is Q (see the kernel on pairs)
        const bool rows = !plan.bn && block_b == kBlk;
        P.tail = plan.bn ? 0 : (int)plan.halved;
        const int p_box = 128, q_box = plan.bn ? plan.bn : P.tail ? 64 : 128;
        if (!(rows ? sides(sa, sb, p_box, q_box) : sides(sb, sa, p_box, q_box))) return set_error(EDDLB200_EINVAL, "%s: the driver refuses a tensor map of the operands", what);
        P.tiles_p = (int)ceil_div(P.p_rows, plan.bn ? 128 : 256);
        P.splits = plan.bn ? plan.splits : (int)ceil_div(P.q_rows, 256);
        const int m_side = plan.bn ? 128 : 256, n_side = plan.bn ? plan.bn : 256;
        P.idesc = rows ? fp8_idesc(format_a, format_b, m_side, n_side) : fp8_idesc(format_b, format_a, m_side, n_side);
    }
    for (int i = 0; i < 4; i++) EB_READS(in[i], bytes[i]);
    if (!inc_c) EB_WRITES(c, out);
    else {
        EB_SETTLE(c, out);
        int status = 0;
        if (lz_take(cx, st, c, out, &status)) inc_c = 0;               // zeros owed to all of C: nothing to add to
        if (status) return status;
    }
    P.inc = inc_c != 0;
    ProfScope prof(cx, PROF_GEMM, 2.0 * m * n * k);
    if (!k) return inc_c ? 0 : launch_zero_fill(cx, st, c, (size_t)m * n);
    if (!plan.bn)
        return P.tail ? large_product<true>(cx, dev, st, P, block_a, block_b) : large_product<false>(cx, dev, st, P, block_a, block_b);
    switch (plan.bn) {
        case 16: return launch_product<16>(cx, st, P, (unsigned)plan.tiles);
        case 32: return launch_product<32>(cx, st, P, (unsigned)plan.tiles);
        case 64: return launch_product<64>(cx, st, P, (unsigned)plan.tiles);
        case 128: return launch_product<128>(cx, st, P, (unsigned)plan.tiles);
        default: return launch_product<256>(cx, st, P, (unsigned)plan.tiles);
    }
}

}  // extern "C"
