// Loss of a student against a teacher's top logits, mixed with the cross-entropy of hard labels, and its gradient with respect to
// the student's logits, in one pass over them.  For a row of logits x, weight w, temperature T and the teacher's k entries
// (id_j, t_j):
//     q = softmax(x / T),   p_j = exp(t_j / T) / sum over the entries     or, given the log of the sum over ALL of the teacher's
//     classes (teacher_lse), p_j = exp(t_j / T - teacher_lse) with the rest p_r = 1 - sum p_j as a class of its own, q_r = the
//     student's mass outside the entries
//     loss  = w [ (1 - alpha) T^2 ( sum_j p_j log(p_j / q_j) + p_r log(p_r / q_r) ) + alpha (log sum exp x - x_label) ]
//     delta = w [ (1 - alpha) T ( q_i - p_i ) + alpha (softmax(x)_i - [i = label]) ],    q_i (1 - p_r / q_r) for i outside the entries
//
// Bound by memory: 8 bytes a logit.  A row lies in shared memory between its one read and its one write -- of one block, or in
// pieces in the blocks of a cluster, which exchange two sets of sums (the maxima, then what depends on them).  Mass outside the
// entries is summed from the values outside, not as 1 minus something: entries are replaced by -infinity first.
#include <type_traits>
#include <cooperative_groups.h>
#include "common.cuh"

namespace {

using namespace eb;
namespace cg = cooperative_groups;

constexpr int kMaxTop = 1024;
constexpr int kMaxPiece = 50176;                 // logits of a row in one block: 196 KB of shared memory, with 12 KB of entries
constexpr int kMaxCluster = 8;
constexpr int kMaxCols = kMaxPiece * kMaxCluster;
constexpr int kSums = 6;

struct Args {
    const float *x, *teacher, *teacher_lse, *weights;
    const int *ids, *labels;
    float *loss, *delta;
    int rows, cols, k, piece;                    // piece: logits of one block, a multiple of 4
    size_t ld;
    float temperature, alpha;
};

__device__ __forceinline__ float minus_inf() { return __int_as_float(0xff800000); }
// a NaN on either side stays
__device__ __forceinline__ float max_nan(float a, float b) { float r; asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ double max_nan(double a, double b) { return b > a || b != b ? b : a; }

// TEAM threads share a row (or a piece of it): a warp, or the whole block.  CLUSTER: the pieces of a row are the blocks of a cluster.
template <int TEAM, bool VEC, bool CLUSTER>
__global__ void __launch_bounds__(TEAM == 32 ? 256 : TEAM) distill_kernel(const Args a) {
    constexpr int TEAMS = TEAM == 32 ? 8 : 1, W = TEAM / 32;
    extern __shared__ __align__(16) float smem[];
    __shared__ double sums[TEAM == 32 ? 1 : 2 * kSums * W];
    __shared__ double peers[CLUSTER ? 2 * kSums * kMaxCluster : 1];
    const int team = threadIdx.x / TEAM, t = threadIdx.x % TEAM, lane = threadIdx.x & 31;
    const int kk = (a.k + 3) & ~3;
    float *x = smem + (size_t)team * (a.piece + 3 * kk);
    float *value = x + a.piece, *prob = value + kk;        // of an entry in this piece: the student's logit, the teacher's weight
    int *cell = reinterpret_cast<int *>(prob + kk);        // where in the piece it lies; -1: not an entry of this piece
    const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0, csize = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
    const int c0 = rank * a.piece, n = max(0, min(a.piece, a.cols - c0));
    const float inv_t = 1.f / a.temperature;
    const bool tail = a.teacher_lse != nullptr, soft = a.alpha != 1.f;
    auto barrier = [&]() { if (TEAM == 32) __syncwarp(); else __syncthreads(); };
    int flip = 0;
    // v[0 .. COUNT) summed (or, LARGEST, the largest) over all threads that share the row, in a fixed order.  Two buffers take turns: one
    // is written again only after the barrier of the exchange in between, which every reader has passed.
    auto combine = [&](auto &v, auto largest) {
        constexpr int COUNT = sizeof(v) / sizeof(double);
        constexpr bool LARGEST = decltype(largest)::value;
#pragma unroll
        for (int i = 0; i < COUNT; i++)
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) { const double u = __shfl_xor_sync(0xffffffffu, v[i], o); v[i] = LARGEST ? max_nan(v[i], u) : v[i] + u; }
        if (TEAM == 32) return;
        double *b = sums + flip * (kSums * W);
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < COUNT; i++) b[i * W + (threadIdx.x >> 5)] = v[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < COUNT; i++) {
            v[i] = b[i * W];
            for (int w = 1; w < W; w++) v[i] = LARGEST ? max_nan(v[i], b[i * W + w]) : v[i] + b[i * W + w];
        }
        if (CLUSTER) {
            cg::cluster_group cl = cg::this_cluster();
            double *mine = peers + flip * (kSums * kMaxCluster);
            if (threadIdx.x < (unsigned)csize) {
                double *there = cl.map_shared_rank(mine, threadIdx.x);
#pragma unroll
                for (int i = 0; i < COUNT; i++) there[i * kMaxCluster + rank] = v[i];
            }
            cl.sync();
#pragma unroll
            for (int i = 0; i < COUNT; i++) {
                v[i] = mine[i * kMaxCluster];
                for (int c = 1; c < csize; c++) v[i] = LARGEST ? max_nan(v[i], mine[i * kMaxCluster + c]) : v[i] + mine[i * kMaxCluster + c];
            }
        }
        flip ^= 1;
    };
    EB_GRID_WAIT();
    const int first = (int)(blockIdx.x / csize) * TEAMS + team, step = (int)(gridDim.x / csize) * TEAMS;
    for (int row = first; row < a.rows; row += step) {
        const float weight = a.weights ? a.weights[row] : 1.f;
        const float *src = a.x + (size_t)row * a.ld + c0;
        float *dst = a.delta ? a.delta + (size_t)row * a.ld + c0 : nullptr;
        // a row without weight, or without a single class that its mask leaves, adds nothing: its values are not looked at
        bool empty = weight == 0.f;
        double most[2] = {minus_inf(), minus_inf()};       // largest logit of the student, of the teacher's entries
        int label = -1;
        float x_label = 0.f;
        if (!empty) {
            float top = minus_inf(), t_top = minus_inf();
            if (VEC) {
#pragma unroll 4
                for (int i = t * 4; i < n; i += TEAM * 4) {
                    const float4 q = *reinterpret_cast<const float4 *>(src + i);
                    *reinterpret_cast<float4 *>(x + i) = q;
                    top = max_nan(max_nan(max_nan(q.x, q.y), max_nan(q.z, q.w)), top);
                }
            } else {
#pragma unroll 4
                for (int i = t; i < n; i += TEAM) { const float q = src[i]; x[i] = q; top = max_nan(top, q); }
            }
            if (a.alpha != 0.f) { label = a.labels[row]; if (label >= a.cols) label = -1; }
            barrier();
            if (t == 0 && label >= c0 && label < c0 + n) x_label = x[label - c0];
            if (soft) {
                // of several entries with the same id the first one counts: a cell holds the least number of an entry with its id
                // until that one puts back what belongs there
                for (int j = t; j < a.k; j += TEAM) {
                    const int id = a.ids[(size_t)row * a.k + j], at = id >= c0 && id < c0 + n ? id - c0 : -1;
                    cell[j] = at;
                    if (at >= 0) value[j] = x[at];
                }
                barrier();
                for (int j = t; j < a.k; j += TEAM) if (cell[j] >= 0) x[cell[j]] = __int_as_float(0x7fffffff);
                barrier();
                for (int j = t; j < a.k; j += TEAM) if (cell[j] >= 0) atomicMin(reinterpret_cast<int *>(x + cell[j]), j);
                barrier();
                for (int j = t; j < a.k; j += TEAM) {
                    if (cell[j] < 0) continue;
                    // only this thread changes cell[j]; the owner's number stays in the cell until the barrier below
                    if (__float_as_int(x[cell[j]]) != j) { cell[j] = -1; continue; }
                    prob[j] = a.teacher[(size_t)row * a.k + j];
                    t_top = max_nan(t_top, prob[j]);
                }
                barrier();
                for (int j = t; j < a.k; j += TEAM) if (cell[j] >= 0) x[cell[j]] = tail ? minus_inf() : value[j];
            }
            most[0] = top; most[1] = t_top;
            combine(most, std::true_type());                          // its barrier lets every thread see the cells
            if (TEAM == 32) __syncwarp();
            empty = most[0] == (double)minus_inf();
        }
        if (empty) {
            if (dst) for (int i = t; i < n; i += TEAM) dst[i] = 0.f;
            if (rank == 0 && t == 0) a.loss[row] = 0.f;
            barrier();
            continue;
        }
        const float m = (float)most[0];
        const bool ce = label >= 0, entries = soft && (tail || most[1] != (double)minus_inf());
        // outside (all of the row unless `tail`), of the entries, with the temperature; the same without it; teacher's sum; KL terms; label
        double v[6] = {0, 0, 0, 0, 0, x_label};
        {
            float zt = 0.f, z1 = 0.f;
            for (int i = t; i < n; i += TEAM) {
                const float d = x[i] - m;
                if (entries) zt += expf(d * inv_t);
                if (ce) z1 += expf(d);
            }
            v[0] = zt; v[2] = z1;
        }
        if (entries) {
            const double temperature = a.temperature, t_off = tail ? (double)a.teacher_lse[row] : most[1] / temperature;
            for (int j = t; j < a.k; j += TEAM) {
                if (cell[j] < 0) continue;
                const double log_p = (double)prob[j] / temperature - t_off, log_q = ((double)value[j] - most[0]) / temperature, p = exp(log_p);
                if (tail) {
                    v[1] += expf((value[j] - m) * inv_t);
                    if (ce) v[2] += expf(value[j] - m);
                }
                v[3] += p;
                if (p != 0.0) v[4] += p * (log_p - log_q);
                prob[j] = (float)p;
            }
        }
        combine(v, std::false_type());
        const double z = v[0] + v[1];
        double kl = 0.0, inside = 0.0, outside = 0.0, p_scale = 0.0;      // factors of q_i at and outside the entries, of p_j
        if (entries) {
            if (tail) {
                const double rest = fmax(0.0, 1.0 - v[3]), q_rest = v[0] / z;
                kl = v[4] + v[3] * log(z) + (rest > 0.0 ? rest * log(rest / q_rest) : 0.0);
                inside = v[3] + rest;
                outside = q_rest > 0.0 ? inside - rest / q_rest : 0.0;
                p_scale = 1.0;
            } else {
                kl = v[4] / v[3] - log(v[3]) + log(z);
                inside = outside = 1.0;
                p_scale = 1.0 / v[3];
            }
        }
        const double ws = entries ? (double)weight * (1.0 - (double)a.alpha) * a.temperature : 0.0, wh = ce ? (double)weight * a.alpha : 0.0;
        if (rank == 0 && t == 0) {
            double l = 0.0;
            if (entries) l += ws * a.temperature * kl;
            if (ce) l += wh * (log(v[2]) - (v[5] - most[0]));
            a.loss[row] = (float)l;
        }
        if (dst) {
            const float f_in = entries ? (float)(ws * inside / z) : 0.f, f_out = entries ? (float)(ws * outside / z) : 0.f, f_p = (float)(ws * p_scale), f_1 = ce ? (float)(wh / v[2]) : 0.f;
            for (int i = t; i < n; i += TEAM) {
                const float d = x[i] - m;
                float g = 0.f;
                if (entries) g = f_out * expf(d * inv_t);
                if (ce) g += f_1 * expf(d);
                x[i] = g;
            }
            barrier();
            if (entries)
                for (int j = t; j < a.k; j += TEAM) {
                    if (cell[j] < 0) continue;
                    const float d = value[j] - m;
                    float g = f_in * expf(d * inv_t) - f_p * prob[j];
                    if (ce) g += f_1 * expf(d);
                    x[cell[j]] = g;
                }
            barrier();
            if (ce && t == 0 && label >= c0 && label < c0 + n) x[label - c0] -= (float)wh;
            barrier();
            if (VEC) for (int i = t * 4; i < n; i += TEAM * 4) *reinterpret_cast<float4 *>(dst + i) = *reinterpret_cast<const float4 *>(x + i);
            else for (int i = t; i < n; i += TEAM) dst[i] = x[i];
        }
        barrier();
    }
    if (CLUSTER) cg::this_cluster().sync();                // a block's slots outlive the writes of the others
}

template <int TEAM, bool CLUSTER>
int launch_distill(DevCtx *cx, int dev, cudaStream_t st, const Args &a, bool vec, unsigned csize, size_t smem) {
    static bool configured[EDDLB200_MAX_DEVICES][2] = {};
    auto kernel = vec ? distill_kernel<TEAM, true, CLUSTER> : distill_kernel<TEAM, false, CLUSTER>;
    if (!configured[dev][vec]) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return cuda_status(e, "distill(attributes)");
        configured[dev][vec] = true;
    }
    constexpr int block = TEAM == 32 ? 256 : TEAM, teams = TEAM == 32 ? 8 : 1;
    size_t per_sm = (size_t)224 * 1024 / (smem + 5 * 1024);
    if (per_sm > 2048 / block) per_sm = 2048 / block;
    const size_t want = ceil_div(a.rows, teams), most = EDDLB200_NUM_SMS * per_sm / csize;
    const unsigned clusters = (unsigned)(want < most ? want : most);
    if (CLUSTER) eb::launch_cluster(kernel, csize, clusters * csize, block, smem, st, a);
    else eb::launch(kernel, clusters, block, smem, st, a);
    EB_LAUNCH_CHECK("distill");
    return 0;
}

}  // namespace

using namespace eb;

extern "C" int eddlb200_distill(int dev, const float *logits, const int *ids, const float *teacher, const float *teacher_lse, const int *labels,
                                const float *weights, int rows, int cols, size_t ld, int k, float temperature, float alpha, float *loss, float *delta) {
    const char *what = "distill";
    EB_REQUIRE(rows >= 0 && cols > 0 && k > 0 && ld >= (size_t)cols, what);
    EB_REQUIRE(temperature > 0.f && temperature < INFINITY, what);
    EB_REQUIRE(alpha >= 0.f && alpha <= 1.f, what);
    if (cols > kMaxCols) return set_error(EDDLB200_ELIMIT, "%s: %d classes, at most %d", what, cols, kMaxCols);
    if (k > kMaxTop) return set_error(EDDLB200_ELIMIT, "%s: %d entries a row, at most %d", what, k, kMaxTop);
    EB_REQUIRE(!rows || (logits && ids && teacher && loss), what);
    EB_REQUIRE(!rows || labels || alpha == 0.f, what);
    const size_t bytes = (rows ? (size_t)(rows - 1) * ld + cols : 0) * sizeof(float), entries = (size_t)rows * k * 4, each = (size_t)rows * 4;
    const void *in[] = {ids, teacher, teacher_lse, labels, weights};
    const size_t in_bytes[] = {entries, entries, each, each, each};
    EB_REQUIRE(delta == logits || !overlap(delta, bytes, logits, bytes), what);
    EB_REQUIRE(!overlap(loss, each, logits, bytes) && !overlap(loss, each, delta, bytes), what);
    for (int i = 0; i < 5; i++) EB_REQUIRE(!overlap(delta, bytes, in[i], in_bytes[i]) && !overlap(loss, each, in[i], in_bytes[i]), what);
    EB_CTX(dev);
    if (!rows) return 0;
    EB_READS(logits, bytes);
    for (int i = 0; i < 5; i++) EB_READS(in[i], in_bytes[i]);
    // columns past `cols` keep what they hold: the range is written in part
    if (ld == (size_t)cols) EB_WRITES(delta, bytes); else EB_MODIFIES(delta, bytes);
    EB_WRITES(loss, each);
    ProfScope prof(cx, PROF_ELEMENTWISE, (delta ? 8.0 : 4.0) * rows * cols);
    const bool vec = cols % 4 == 0 && ld % 4 == 0 && aligned16(logits) && aligned16(delta);
    Args a{logits, teacher, teacher_lse, weights, ids, labels, loss, delta, rows, cols, k, 0, ld, temperature, alpha};
    const size_t own = (size_t)3 * ((k + 3) & ~3);
    auto pieces = [&](unsigned c) { a.piece = (int)((ceil_div(cols, c) + 3) & ~(size_t)3); return ((size_t)a.piece + own) * sizeof(float); };
    if (cols <= 256) { const size_t smem = 8 * pieces(1); return launch_distill<32, false>(cx, dev, st, a, vec, 1, smem); }
    if (cols <= 2048) { const size_t smem = pieces(1); return launch_distill<128, false>(cx, dev, st, a, vec, 1, smem); }
    if (cols <= 16384) { const size_t smem = pieces(1); return launch_distill<512, false>(cx, dev, st, a, vec, 1, smem); }
    const unsigned csize = cols <= 32768 ? 2 : cols <= 65536 ? 4 : 8;
    const size_t smem = pieces(csize);
    return launch_distill<512, true>(cx, dev, st, a, vec, csize, smem);
}
