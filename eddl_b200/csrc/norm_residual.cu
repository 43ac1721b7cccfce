// What stands between two blocks of a residual net, as one pass: normalise the block's output, scale it by a gate, add it to the
// scaled residual stream, normalise the sum for the next block -- and the backward pass of all of it.
//
//     z = norm(f) g1 + b1        r_out = s r + gate z        h = norm(r_out) g2 + b2
//     norm(x) = (x - mean) / sqrt(mean((x - mean)^2) + eps) over a row; the RMS form leaves the mean out
//
// Both passes are bound by memory: 16 bytes a value forward (f, r read, r_out, h written), 24 backward (dh, dr_out, f, r_out read,
// df, dr written).  A row is held in the registers of a team of threads, statistics are two-pass in fp32.
#include <cooperative_groups.h>
#include "common.cuh"

namespace {

using namespace eb;
namespace cg = cooperative_groups;

constexpr int kMaxCols = 16384;            // 1024 threads with four 16-byte pieces each; eight blocks of 256 with two each
constexpr int kMaxCluster = 8;
constexpr int kMaxRows = 0x7ff00000;       // of a group, and groups: counters that go past the last one stay in 32 bits

// Sums of K values over a team of TPR threads (a warp, or the whole block); every thread gets them, added in a fixed order.  K is a power of two:
// the lanes halve the number of values they carry with each of the first exchanges, so K sums of a warp cost K + 1 shuffles or so, not 5 K.
// Two buffers take turns, so one barrier is enough: a buffer is written again only after the barrier of the sums in between,
// which every reader has passed.
template <int TPR, int K>
struct TeamSum {
    static constexpr int W = TPR / 32, LANES = 32 / K;                  // LANES: neighbours that end up with the same sum
    static_assert((K & (K - 1)) == 0 && K <= 8 && W <= 32, "");
    float *buf;
    int flip = 0;
    __device__ __forceinline__ TeamSum(float *b) : buf(b) {}
    __device__ __forceinline__ void operator()(float (&v)[K]) {
        const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
        // after the exchange over `o` lanes a lane holds the values whose number has, in that place, the lane's bit
#pragma unroll
        for (int half = K / 2, o = 16; half > 0; half /= 2, o /= 2) {
            const bool up = lane & o;
#pragma unroll
            for (int k = 0; k < half; k++) {
                const float give = up ? v[k] : v[k + half], keep = up ? v[k + half] : v[k];
                v[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
        float mine = v[0];
#pragma unroll
        for (int o = LANES / 2; o > 0; o /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        const int k = lane / LANES, sub = lane % LANES;                // mine: the warp's sum of value k
        if (W > 1) {
            float *b = buf + flip * (K * W);
            flip ^= 1;
            if (sub == 0) b[k * W + w] = mine;
            __syncthreads();
            mine = 0.f;
#pragma unroll
            for (int i = 0; i < (W + LANES - 1) / LANES; i++) { const int j = i * LANES + sub; mine += j < W ? b[k * W + j] : 0.f; }
#pragma unroll
            for (int o = LANES / 2; o > 0; o /= 2) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        }
#pragma unroll
        for (int i = 0; i < K; i++) v[i] = __shfl_sync(0xffffffffu, mine, i * LANES);
    }
};

// The NV x 4 values that thread t of a team holds of a row: pieces of 16 bytes where VEC, single values a team apart otherwise.
template <int TPR, int NV, bool VEC>
struct Piece {
    int t, cols;
    __device__ __forceinline__ int at(int i) const { return VEC ? ((i / 4) * TPR + t) * 4 + i % 4 : i * TPR + t; }
    __device__ __forceinline__ bool has(int i) const { return at(VEC ? i & ~3 : i) < cols; }
    __device__ __forceinline__ void load(float (&v)[NV * 4], const float *p, float missing) const {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NV * 4; i += 4) {
                float4 q = make_float4(missing, missing, missing, missing);
                if (p && has(i)) q = *reinterpret_cast<const float4 *>(p + at(i));
                v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV * 4; i++) v[i] = p && has(i) ? p[at(i)] : missing;
        }
    }
    // a row of them on its way into shared memory: value c comes to lie at to[misfit(p) + c].  own(): every thread copies what it will read itself (the
    // rows of a warp, few values each, 4 bytes at a time where they are not aligned); else 16 bytes at a time, the team's threads for one another
    static constexpr __device__ __forceinline__ bool own() { return VEC || TPR == 32; }
    static __device__ __forceinline__ int misfit(const float *p) { return own() ? 0 : (int)((uintptr_t)p >> 2) & 3; }
    __device__ __forceinline__ void ask(float *to, const float *p) const {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(to);
        if (!VEC && own()) {
#pragma unroll
            for (int i = 0; i < NV * 4; i++) if (has(i)) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + at(i) * 4), "l"(p + at(i)) : "memory");
            return;
        }
        const int off = misfit(p), end = off + cols;
#pragma unroll
        for (int k = 0; k < NV + (VEC ? 0 : 1); k++) {
            const int u = (k * TPR + t) * 4;
            if (u >= off && u + 4 <= end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + u * 4), "l"(p - off + u) : "memory");
            else if (!VEC && u < end) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (u + i >= off && u + i < end) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + (u + i) * 4), "l"(p - off + u + i) : "memory");
            }
        }
    }
    __device__ __forceinline__ void store(float *p, const float (&v)[NV * 4]) const {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < NV * 4; i += 4)
                if (has(i)) *reinterpret_cast<float4 *>(p + at(i)) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < NV * 4; i++) if (has(i)) p[at(i)] = v[i];
        }
    }
};

struct FwdArgs {
    const float *f, *r, *gate, *g1, *b1, *g2, *b2;
    float *r_out, *h, *stats;
    float res_scale, eps;
    int cols, rows, layer, post;            // rows: of one group
    size_t total;
};

template <int TPR, int NV, bool VEC, bool AHEAD>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, TPR == 512 && AHEAD ? 2 : TPR == 256 ? 3 : 1) norm_residual_fwd_kernel(const FwdArgs a) {
    EB_GRID_WAIT();
    extern __shared__ __align__(16) float staged[];                    // AHEAD: [team][r, f][SPAN]
    __shared__ float sums[2 * (TPR / 32)];
    TeamSum<TPR, 1> sum(sums);
    constexpr int TEAMS = TPR == 32 ? 8 : 1, N = NV * 4, SPAN = TPR * N;
    static_assert(VEC || !AHEAD, "");
    const Piece<TPR, NV, VEC> piece{(int)(threadIdx.x % TPR), a.cols};
    const float inv = 1.f / (float)a.cols;
    // mean and 1 / deviation of the team's row; the values are centred in place
    auto normalise = [&](float (&v)[N], float &mean, float &rstd) {
        float s[1] = {0.f};
        mean = 0.f;
        if (a.layer) {
#pragma unroll
            for (int i = 0; i < N; i++) s[0] += v[i];                   // absent values are zero
            sum(s);
            mean = s[0] * inv;
#pragma unroll
            for (int i = 0; i < N; i++) v[i] = piece.has(i) ? v[i] - mean : 0.f;
        }
        s[0] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) s[0] += v[i] * v[i];
        sum(s);
        rstd = __frcp_rn(sqrtf(s[0] * inv + a.eps));
#pragma unroll
        for (int i = 0; i < N; i++) v[i] *= rstd;
    };
    float *own = staged + (size_t)(threadIdx.x / TPR) * (2 * SPAN);
    const size_t first = (size_t)blockIdx.x * TEAMS + threadIdx.x / TPR, step = (size_t)gridDim.x * TEAMS;
    auto ask = [&](size_t row) {
        if (row < a.total) {
            const size_t base = row * a.cols;
            piece.ask(own, a.r + base);
            if (a.f) piece.ask(own + SPAN, a.f + base);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (AHEAD) ask(first);
    for (size_t row = first; row < a.total; row += step) {
        float v[N], x[N];
        float mean1 = 0.f, rstd1 = 0.f, mean2 = 0.f, rstd2 = 0.f;
        const size_t base = row * a.cols;
        if (AHEAD) {
            // a thread reads what it copied itself, and its places are free again once the values are in registers
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            piece.load(x, own, 0.f);
            if (a.f) piece.load(v, own + SPAN, 0.f);
            ask(row + step);
        } else {
            piece.load(x, a.r + base, 0.f);
            if (a.f) piece.load(v, a.f + base, 0.f);
        }
        if (a.f) {
            if (a.post) normalise(v, mean1, rstd1);
            float p[N];
            if (a.g1) {
                piece.load(p, a.g1, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) v[i] *= p[i];
            }
            if (a.b1) {
                piece.load(p, a.b1, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) v[i] += p[i];
            }
            if (a.gate) {
                piece.load(p, a.gate + row / a.rows * a.cols, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) v[i] *= p[i];
            }
#pragma unroll
            for (int i = 0; i < N; i++) x[i] = a.res_scale * x[i] + v[i];
            piece.store(a.r_out + base, x);
        }
        if (a.h) {
            normalise(x, mean2, rstd2);
            float p[N];
            if (a.g2) {
                piece.load(p, a.g2, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) x[i] *= p[i];
            }
            if (a.b2) {
                piece.load(p, a.b2, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) x[i] += p[i];
            }
            piece.store(a.h + base, x);
        }
        if (a.stats && piece.t == 0) *reinterpret_cast<float4 *>(a.stats + row * 4) = make_float4(mean1, rstd1, mean2, rstd2);
    }
}

constexpr int BWD_THREADS = 512;          // of an SM: 128 registers each
struct BwdArgs {
    const float *dh, *dr_out, *f, *r_out, *gate, *g1, *b1, *g2, *stats;
    float *df, *dr;
    float *param_part, *gate_part;          // [block][4][cols] of dg2, db2, dg1, db1; [unit][cols] of dgate, which is dgate itself where a unit is a group
    float res_scale;
    int cols, chunk, rows, layer, post, inc_df, inc_dr; // chunk: columns of one block of a cluster; inc: 0 store, 1 add, 2 add to a destination known to hold zeros
    int want_gate, want_param, inc_gate;    // want_param: bits dg2, db2, dg1, db1; inc_gate: add to gate_part
    int unit_groups, slices, workers;       // a unit is a slice of a group's rows; workers: blocks (clusters) that share the units
    size_t unit_rows;                       // rows of one unit group
};

// Backward.  With n1, n2 the normalised rows, dn2 = dh g2, G = gate g1 and <> the mean over a row:
//     u  = dr_out + rstd2 (dn2 - <dn2> - n2 <dn2 n2>)                      (the gradient of r_out; RMS: without <dn2>)
//     dr = s u,   dn1 = G u,   df = rstd1 (dn1 - <dn1> - n1 <dn1 n1>)
//     dg2 = sum dh n2, db2 = sum dh, dg1 = sum gate u n1, db1 = sum gate u over all rows, dgate = sum u z over a group's
// u is linear in <dn2> and <dn2 n2>, so the sums of the second norm follow from sums of known values:
//     <dn1>    = <G e> - rstd2 (<dn2> <G>    + <dn2 n2> <G n2>),       e = dr_out + rstd2 dn2
//     <dn1 n1> = <G e n1> - rstd2 (<dn2> <G n1> + <dn2 n2> <G n2 n1>)
// and a row takes one exchange between its threads instead of two.  The column sums stay in registers over all rows of a block
// and are added in a fixed order afterwards: no atomics.
//
// A row's four tensors are copied (cp.async, 16 bytes) while the row before it is worked on.  VEC: 16-byte aligned rows, each value comes to a place
// that only the thread that uses it reads, so the copies need no barrier; else a barrier a row (with 4-byte copies by the thread
// itself 38 x 555 x 1551 took 487 us, forward and backward).  GENERAL: with means or shifts, eight sums a row, else three.
template <int TPR, int NV, bool VEC, bool GENERAL, bool CLUSTER>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR, BWD_THREADS / (TPR == 32 ? 256 : TPR)) norm_residual_bwd_kernel(const BwdArgs a) {
    constexpr int TEAMS = TPR == 32 ? 8 : 1, N = NV * 4, K = GENERAL ? 8 : 4, SPAN = TPR * N + (VEC ? 0 : 4);
    extern __shared__ __align__(16) float staged[];                    // [team][2][dh, dr_out, r_out, f][SPAN]; at a unit's end the column sums of the teams
    __shared__ __align__(16) float sums[2 * K * (TPR / 32)];
    __shared__ __align__(16) float peers[CLUSTER ? 2 * K * kMaxCluster : 4];
    if (CLUSTER) cg::this_cluster().sync();                 // the other blocks have started: their shared memory may be written
    EB_GRID_WAIT();
    TeamSum<TPR, K> sum(sums);
    const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0, csize = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
    const int worker = (int)(blockIdx.x / csize), col0 = rank * a.chunk, cols_here = max(0, min(a.cols - col0, a.chunk));
    const Piece<TPR, NV, VEC> piece{(int)(threadIdx.x % TPR), cols_here};
    const int team = threadIdx.x / TPR;
    float *own = staged + (size_t)team * (8 * SPAN);
    const float inv = 1.f / (float)a.cols;
    int flip = 0, stage = 0;
    // Column sums: dg2, db2, and of u n1 and u over the rows of one gate, from which its dgate and its share of dg1 and db1 follow
    float g2[N], gg[N], dg2[N] = {}, db2[GENERAL ? N : 1] = {}, un[N] = {}, uu[N] = {}, dg1[N] = {}, db1[GENERAL ? N : 1] = {}, gg_sum = 0.f;
    size_t gate_of = 0;
    piece.load(g2, a.g2 ? a.g2 + col0 : nullptr, a.g2 ? 0.f : 1.f);
    auto gate_row = [&](float (&v)[N]) { piece.load(v, a.gate ? a.gate + gate_of * a.cols + col0 : nullptr, a.gate ? 0.f : 1.f); };
    auto take_gate = [&](size_t which) {                       // gg = gate g1
        gate_of = which;
        float v[N];
        gate_row(gg);
        piece.load(v, a.g1 ? a.g1 + col0 : nullptr, a.g1 ? 0.f : 1.f);
        gg_sum = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) { gg[i] = piece.has(i) ? gg[i] * v[i] : 0.f; gg_sum += gg[i]; }
    };
    auto settle = [&](float (&of_gate)[N]) {                   // the sums of this gate's rows go where they belong
        float v[N];
        gate_row(v);
#pragma unroll
        for (int i = 0; i < N; i++) { dg1[i] += v[i] * un[i]; if (GENERAL) db1[GENERAL ? i : 0] += v[i] * uu[i]; }
        if (a.want_gate) {
            piece.load(v, a.g1 ? a.g1 + col0 : nullptr, a.g1 ? 0.f : 1.f);
#pragma unroll
            for (int i = 0; i < N; i++) of_gate[i] = v[i] * un[i];
            if (a.b1) {
                piece.load(v, a.b1 + col0, 0.f);
#pragma unroll
                for (int i = 0; i < N; i++) of_gate[i] += v[i] * uu[i];
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) un[i] = uu[i] = 0.f;
    };
    if (!a.dh) {
#pragma unroll
        for (int i = 0; i < N; i++) g2[i] = 0.f;
    }
    float4 next_stats = make_float4(0.f, 0.f, 0.f, 0.f);
    auto ask = [&](size_t row, int to) {
        const size_t base = row * a.cols + col0;
        float *slot = own + to * (4 * SPAN);
        if (a.dh) { piece.ask(slot, a.dh + base); piece.ask(slot + 2 * SPAN, a.r_out + base); }
        if (a.dr_out) piece.ask(slot + SPAN, a.dr_out + base);
        if (a.f) piece.ask(slot + 3 * SPAN, a.f + base);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next_stats = *reinterpret_cast<const float4 *>(a.stats + row * 4);
    };
    const int units = a.unit_groups * a.slices;
    bool started = false;
    for (int unit = worker; unit < units; unit += a.workers) {
        const size_t group = unit / a.slices, slice = unit % a.slices;
        const size_t first = group * a.unit_rows + a.unit_rows * slice / a.slices, last = group * a.unit_rows + a.unit_rows * (slice + 1) / a.slices;
        if (first + team < last) ask(first + team, stage);
        for (size_t row = first + team; row < last; row += TEAMS, stage ^= 1) {
            const size_t base = row * a.cols + col0;
            const float4 st = next_stats;
            if (row + TEAMS < last) {
                ask(row + TEAMS, stage ^ 1);
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            } else asm volatile("cp.async.wait_group 0;" ::: "memory");
            const float *slot = own + stage * (4 * SPAN);
            if (!started) { take_gate(a.gate ? row / a.rows : 0); started = true; }
            else if (a.gate && row / a.rows != gate_of) {
                float unused[N];
                if (!a.want_gate) settle(unused);
                take_gate(row / a.rows);
            }
            // where the threads copy for one another: a place is copied into again only after the barrier of this row's sums
            if (!piece.own()) __syncthreads();
            float dh[N], e[N], n1[N], n2[N];
            piece.load(dh, a.dh ? slot + piece.misfit(a.dh + base) : nullptr, 0.f);
            piece.load(n2, a.dh ? slot + 2 * SPAN + piece.misfit(a.r_out + base) : nullptr, 0.f);
            piece.load(e, a.dr_out ? slot + SPAN + piece.misfit(a.dr_out + base) : nullptr, 0.f);
            piece.load(n1, a.f ? slot + 3 * SPAN + piece.misfit(a.f + base) : nullptr, 0.f);
            float s[K] = {};
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (!piece.has(i)) { n1[i] = n2[i] = 0.f; continue; }
                n2[i] = (n2[i] - st.z) * st.w;
                if (a.post) n1[i] = (n1[i] - st.x) * st.y;
                const float dn2 = dh[i] * g2[i], gn = gg[i] * n1[i];
                e[i] += st.w * dn2;
                s[0] += dn2 * n2[i];
                s[1] += gn * e[i];
                s[2] += gn * n2[i];
                if (GENERAL) {
                    s[3 % K] += dn2;
                    s[4 % K] += gg[i] * e[i];
                    s[6 % K] += gg[i] * n2[i];
                    s[7 % K] += gn;
                }
            }
            if (GENERAL) s[5 % K] = gg_sum;
            sum(s);
            if (CLUSTER) {
                cg::cluster_group cl = cg::this_cluster();
                float *mine = peers + flip * (K * kMaxCluster);
                flip ^= 1;
                if (threadIdx.x < (unsigned)csize) {
                    float4 *there = reinterpret_cast<float4 *>(cl.map_shared_rank(mine, threadIdx.x) + rank * K);
#pragma unroll
                    for (int k = 0; k < K; k += 4) there[k / 4] = make_float4(s[k], s[k + 1], s[k + 2], s[k + 3]);
                }
                cl.sync();
#pragma unroll
                for (int k = 0; k < K; k++) s[k] = 0.f;
                for (int c = 0; c < csize; c++)
#pragma unroll
                    for (int k = 0; k < K; k++) s[k] += mine[c * K + k];
            }
            const float m_n2 = s[0] * inv, m_1 = GENERAL && a.layer ? s[3 % K] * inv : 0.f;
            const float q_n1 = s[1] * inv - st.w * (m_n2 * (s[2] * inv) + (GENERAL ? m_1 * (s[7 % K] * inv) : 0.f));
            const float q_1 = GENERAL && a.layer ? s[4 % K] * inv - st.w * (m_n2 * (s[6 % K] * inv) + m_1 * (s[5 % K] * inv)) : 0.f;
            float out[N];
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float u = e[i] - st.w * (m_1 + n2[i] * m_n2);
                dg2[i] += dh[i] * n2[i];
                un[i] += u * n1[i];
                if (GENERAL) { db2[GENERAL ? i : 0] += dh[i]; uu[i] += u; }
                e[i] = u;
                const float dn1 = u * gg[i];
                out[i] = a.post ? st.y * (dn1 - q_1 - n1[i] * q_n1) : dn1;
            }
            if (a.df) {
                if (a.inc_df) {
                    float old[N];
                    piece.load(old, a.inc_df == 1 ? a.df + base : nullptr, 0.f);
#pragma unroll
                    for (int i = 0; i < N; i++) out[i] += old[i];
                }
                piece.store(a.df + base, out);
            }
            if (a.dr) {
                if (a.inc_dr) {
                    piece.load(out, a.inc_dr == 1 ? a.dr + base : nullptr, 0.f);
#pragma unroll
                    for (int i = 0; i < N; i++) out[i] += a.res_scale * e[i];
                } else {
#pragma unroll
                    for (int i = 0; i < N; i++) out[i] = a.res_scale * e[i];
                }
                piece.store(a.dr + base, out);
            }
        }
        if (a.want_gate) {
            float of_gate[N] = {};
            if (started) settle(of_gate);
            float *dst = a.gate_part + (size_t)unit * a.cols + col0;
            if (TEAMS == 1) {
                if (a.inc_gate) {
                    float old[N];
                    piece.load(old, dst, 0.f);
#pragma unroll
                    for (int i = 0; i < N; i++) of_gate[i] += old[i];
                }
                piece.store(dst, of_gate);
            } else {
                __syncthreads();                               // no copy is on its way, and no team still reads its places
                piece.store(staged + team * a.cols, of_gate);
                __syncthreads();
                for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
                    float t = 0.f;
                    for (int k = 0; k < TEAMS; k++) t += staged[k * a.cols + c];
                    dst[c] = a.inc_gate ? dst[c] + t : t;
                }
                __syncthreads();
            }
        }
    }
    if (!a.want_gate && started) { float unused[N]; settle(unused); }
    // kinds in the order of param_part: dg2, db2, dg1, db1
    auto leave = [&](int kind, const float (&v)[N]) {
        if (!(a.want_param >> kind & 1)) return;
        float *dst = a.param_part + ((size_t)worker * 4 + kind) * a.cols + col0;
        if (TEAMS == 1) { piece.store(dst, v); return; }
        __syncthreads();
        piece.store(staged + team * a.cols, v);
        __syncthreads();
        for (int c = threadIdx.x; c < a.cols; c += blockDim.x) {
            float t = 0.f;
            for (int k = 0; k < TEAMS; k++) t += staged[k * a.cols + c];
            dst[c] = t;
        }
    };
    leave(0, dg2); leave(2, dg1);
    if constexpr (GENERAL) { leave(1, db2); leave(3, db1); }
    if (CLUSTER) cg::this_cluster().sync();                 // a block's slots outlive the writes of the others
}

// Column sums of the partial rows, in a fixed order: the parameters' gradients over the blocks, dgate over a group's slices.  A block of 32 columns x 32
// rows of threads gives every output as many rows of threads as it has partial rows (a power of two up to 32) and the rest to further
// outputs: 64 groups of six slices are 16 blocks of columns high, not 64.
struct FoldArgs {
    const float *param_part, *gate_part;
    float *out[4], *dgate;
    int cols, workers, slices, groups, inc;
    int param_rows, gate_rows, param_blocks;               // rows of threads for an output (log2), blocks that the parameters take
};
__global__ void __launch_bounds__(1024) norm_residual_fold_kernel(const FoldArgs a) {
    EB_GRID_WAIT();
    __shared__ float part[32][33];
    const int col = blockIdx.x * 32 + threadIdx.x;
    const bool gate = (int)blockIdx.y >= a.param_blocks;
    const int log_rows = gate ? a.gate_rows : a.param_rows, row = threadIdx.y & ((1 << log_rows) - 1);
    const int which = (((int)blockIdx.y - (gate ? a.param_blocks : 0)) << (5 - log_rows)) + (threadIdx.y >> log_rows);
    const bool there = which < (gate ? a.groups : 4) && col < a.cols;
    float *out = !there ? nullptr : gate ? a.dgate + (size_t)which * a.cols : which == 0 ? a.out[0] : which == 1 ? a.out[1] : which == 2 ? a.out[2] : a.out[3];
    const size_t step = gate ? a.cols : (size_t)4 * a.cols;
    const float *src = gate ? a.gate_part + (size_t)which * a.slices * a.cols : a.param_part + (size_t)which * a.cols;
    const int n = gate ? a.slices : a.workers;
    float s = 0.f;
    if (out) {
#pragma unroll 8
        for (int i = row; i < n; i += 1 << log_rows) s += __ldcg(src + i * step + col);
    }
    part[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    if (row || !out) return;
    float t = 0.f;
    for (int i = 0; i < 1 << log_rows; i++) t += part[threadIdx.y + i][threadIdx.x];
    out[col] = a.inc ? out[col] + t : t;
}

template <int TPR, int NV>
struct Fwd {
    // Aligned rows are copied ahead where few blocks share an SM (8192 columns, 4000 rows: 89 us, without 111) or rows are short (128 columns, 100000 rows:
    // 45 us, without 51), not in between (4096 columns, 12288 rows: 142 us, without 132): there the blocks of an SM cover for one another.
    static constexpr bool AHEAD = TPR * NV > 1024 || (TPR == 32 && NV == 1);
    static int run(DevCtx *cx, int dev, cudaStream_t st, const FwdArgs &a, bool vec) {
        constexpr int block = TPR == 32 ? 256 : TPR, teams = TPR == 32 ? 8 : 1;
        const size_t want = ceil_div(a.total, teams), most = (size_t)EDDLB200_NUM_SMS * (2048 / block);
        if constexpr (AHEAD) if (vec) {
            constexpr size_t smem = (size_t)teams * 2 * TPR * NV * 4 * sizeof(float);
            static int known[EDDLB200_MAX_DEVICES] = {};                       // blocks that the device holds at once
            int &n = known[dev];
            auto kernel = norm_residual_fwd_kernel<TPR, NV, true, true>;
            if (!n) {
                cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
                int held = 0;
                if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, kernel, block, smem);
                if (e != cudaSuccess) return cuda_status(e, "norm_residual_fwd(occupancy)");
                n = (held < 1 ? 1 : held) * EDDLB200_NUM_SMS;
            }
            if (want > (size_t)n) {
                eb::launch(kernel, (unsigned)n, block, smem, st, a);
                EB_LAUNCH_CHECK("norm_residual_fwd");
                return 0;
            }
        }
        eb::launch(vec ? norm_residual_fwd_kernel<TPR, NV, true, false> : norm_residual_fwd_kernel<TPR, NV, false, false>, (unsigned)(want < most ? want : most), block, 0, st, a);
        EB_LAUNCH_CHECK("norm_residual_fwd");
        return 0;
    }
};

template <int TPR, int NV, bool CLUSTER>
struct Bwd {
    static constexpr int block = TPR == 32 ? 256 : TPR, teams = TPR == 32 ? 8 : 1;
    static constexpr size_t smem = (size_t)teams * 8 * (TPR * NV * 4 + 4) * sizeof(float);
    static auto kernel(bool vec, bool general) {
        return vec ? (general ? norm_residual_bwd_kernel<TPR, NV, true, true, CLUSTER> : norm_residual_bwd_kernel<TPR, NV, true, false, CLUSTER>)
                   : (general ? norm_residual_bwd_kernel<TPR, NV, false, true, CLUSTER> : norm_residual_bwd_kernel<TPR, NV, false, false, CLUSTER>);
    }
    // blocks (clusters of `csize`) that the device holds at once; 0 with the error set
    static int resident(int dev, bool vec, bool general, unsigned csize) {
        static int known[EDDLB200_MAX_DEVICES][4][kMaxCluster + 1] = {};
        int &n = known[dev][2 * vec + general][csize];
        if (n) return n;
        auto k = kernel(vec, general);
        cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        int held = 0;
        if (e == cudaSuccess && CLUSTER) {
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension; at[0].val.clusterDim.x = csize; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t c = {};
            c.gridDim = dim3(EDDLB200_NUM_SMS / csize * csize); c.blockDim = dim3(block); c.dynamicSmemBytes = smem; c.attrs = at; c.numAttrs = 1;
            e = cudaOccupancyMaxActiveClusters(&held, k, &c);
        } else if (e == cudaSuccess) {
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&held, k, block, smem);
            held *= EDDLB200_NUM_SMS;
        }
        if (e != cudaSuccess) { cuda_status(e, "norm_residual_bwd(occupancy)"); return 0; }
        if (held < 1) { set_error(EDDLB200_ELIMIT, "norm_residual_bwd: the device holds no cluster of %u blocks", csize); return 0; }
        return n = held;
    }
    static int launch(DevCtx *cx, cudaStream_t st, const BwdArgs &a, bool vec, bool general, unsigned csize) {
        if (CLUSTER) eb::launch_cluster(kernel(vec, general), csize, a.workers * csize, block, smem, st, a);
        else eb::launch(kernel(vec, general), a.workers, block, smem, st, a);
        EB_LAUNCH_CHECK("norm_residual_bwd");
        return 0;
    }
};
// The smallest team that holds a row in registers beside its column sums: eight values a thread at most; wider rows are shared by a cluster.  Teams between
// the powers of two where half of the lanes would be idle (10000 x 1300, layer norms: 69 us on 192 threads, 83 on 256; 6000 x 2500: 85 on 320, 112 on 512).
template <typename Go>
auto with_bwd(int cols, Go go) {
    if (cols <= 128) return go(Bwd<32, 1, false>());
    if (cols <= 256) return go(Bwd<32, 2, false>());
    if (cols <= 512) return go(Bwd<128, 1, false>());
    if (cols <= 768) return go(Bwd<96, 2, false>());
    if (cols <= 1024) return go(Bwd<128, 2, false>());
    if (cols <= 1536) return go(Bwd<192, 2, false>());
    if (cols <= 2048) return go(Bwd<256, 2, false>());
    if (cols <= 2560) return go(Bwd<320, 2, false>());
    if (cols <= 4096) return go(Bwd<512, 2, false>());
    return go(Bwd<256, 2, true>());
}

// An output may be an input's own memory (every value is read before it is written, by the thread that writes it), but not part of it.
bool clash(const void *out, size_t out_bytes, const void *in, size_t in_bytes) { return out != in && overlap(out, out_bytes, in, in_bytes); }

const char *const kFwd = "norm_residual_fwd", *const kBwd = "norm_residual_bwd";

}  // namespace

using namespace eb;

extern "C" {

int eddlb200_norm_residual_fwd(int dev, int kind, int post, int groups, int rows, int cols, const float *f, const float *r, const float *gate,
                               const float *g1, const float *b1, float res_scale, const float *g2, const float *b2, float eps,
                               float *r_out, float *h, float *stats) {
    EB_REQUIRE((kind == 0 || kind == 1) && (post == 0 || post == 1), kFwd);
    EB_REQUIRE(groups >= 0 && rows >= 0 && cols > 0, kFwd);
    EB_REQUIRE(eps >= 0.f, kFwd);
    if (cols > kMaxCols) return set_error(EDDLB200_ELIMIT, "%s: rows of %d values, at most %d", kFwd, cols, kMaxCols);
    if (groups > kMaxRows || rows > kMaxRows) return set_error(EDDLB200_ELIMIT, "%s: %d groups of %d rows", kFwd, groups, rows);
    EB_REQUIRE((f != nullptr) == (r_out != nullptr), kFwd);
    EB_REQUIRE(f || (!gate && !g1 && !b1 && !post && res_scale == 1.f), kFwd);
    EB_REQUIRE(post || (!g1 && !b1), kFwd);
    EB_REQUIRE(h || (f && !g2 && !b2), kFwd);
    EB_REQUIRE(aligned16(stats), kFwd);
    const size_t total = (size_t)groups * rows, bytes = total * cols * sizeof(float), vector = (size_t)cols * sizeof(float), gates = groups * vector;
    EB_REQUIRE(!total || r, kFwd);
    const void *in[] = {f, r, gate, g1, b1, g2, b2};
    const size_t in_bytes[] = {bytes, bytes, gates, vector, vector, vector, vector};
    EB_REQUIRE(aligned4(r_out) && aligned4(h), kFwd);
    for (int i = 0; i < 7; i++) {
        EB_REQUIRE(aligned4(in[i]), kFwd);
        EB_REQUIRE(i < 2 ? !clash(r_out, bytes, in[i], in_bytes[i]) : !overlap(r_out, bytes, in[i], in_bytes[i]), kFwd);
        EB_REQUIRE(i < 2 ? !clash(h, bytes, in[i], in_bytes[i]) : !overlap(h, bytes, in[i], in_bytes[i]), kFwd);
        EB_REQUIRE(!overlap(stats, total * 16, in[i], in_bytes[i]), kFwd);
    }
    EB_REQUIRE(!overlap(r_out, bytes, h, bytes) && !overlap(stats, total * 16, r_out, bytes) && !overlap(stats, total * 16, h, bytes), kFwd);
    EB_CTX(dev);
    if (!total) return 0;
    for (int i = 0; i < 7; i++) EB_READS(in[i], in_bytes[i]);
    EB_WRITES(r_out, bytes); EB_WRITES(h, bytes); EB_WRITES(stats, total * 16);
    ProfScope prof(cx, PROF_BN_FWD, (double)bytes * ((f ? 3 : 1) + (h ? 1 : 0)));
    const FwdArgs a{f, r, gate, g1, b1, g2, b2, r_out, h, stats, res_scale, eps, cols, rows, kind, post, total};
    const bool vec = cols % 4 == 0 && aligned16(f) && aligned16(r) && aligned16(gate) && aligned16(g1) && aligned16(b1) && aligned16(g2) && aligned16(b2) && aligned16(r_out) && aligned16(h);
    const bool few = total < (size_t)EDDLB200_NUM_SMS * 8;          // rows for one warp a scheduler or less: several warps a row
    // Twelve to 32 values a thread: a row on fewer threads means fewer to add up and to wait for, and idle lanes cost as much as others (10000 x 1300,
    // layer norms: 44 us on 128 threads, 61 on 256; 12288 x 4096: 132 on 256, 142 on 512; 12544 x 768: 29 on 64, 31 on 32; 6000 x 2400: 41 on 128,
    // 49 on 256; 3000 x 6000: 53 on 512 with 12 values, 55 on 384 with 16).
    auto go = [&](auto k) { return decltype(k)::run(cx, dev, st, a, vec); };
    if (cols <= 128) return go(Fwd<32, 1>());
    if (cols <= 256) return go(Fwd<32, 2>());
    if (cols <= 512) return few ? go(Fwd<128, 1>()) : go(Fwd<32, 4>());
    if (cols <= 768) return few ? go(Fwd<128, 2>()) : go(Fwd<64, 3>());
    if (cols <= 1024) return few ? go(Fwd<128, 2>()) : go(Fwd<32, 8>());
    if (cols <= 1536) return go(Fwd<128, 3>());
    if (cols <= 2048) return go(Fwd<64, 8>());
    if (cols <= 2560) return go(Fwd<128, 5>());
    if (cols <= 4096) return go(Fwd<256, 4>());
    if (cols <= 6144) return go(Fwd<512, 3>());
    if (cols <= 8192) return go(Fwd<512, 4>());
    return go(Fwd<1024, 4>());
}

int eddlb200_norm_residual_bwd(int dev, int kind, int post, int groups, int rows, int cols, const float *dh, const float *dr_out, const float *f,
                               const float *r_out, const float *gate, const float *g1, const float *b1, float res_scale, const float *g2,
                               const float *stats, float *df, float *dr, int inc_d, float *dgate, float *dg1, float *db1, float *dg2, float *db2, int inc_g) {
    EB_REQUIRE((kind == 0 || kind == 1) && (post == 0 || post == 1), kBwd);
    EB_REQUIRE(groups >= 0 && rows >= 0 && cols > 0, kBwd);
    if (cols > kMaxCols) return set_error(EDDLB200_ELIMIT, "%s: rows of %d values, at most %d", kBwd, cols, kMaxCols);
    if (groups > kMaxRows || rows > kMaxRows) return set_error(EDDLB200_ELIMIT, "%s: %d groups of %d rows", kBwd, groups, rows);
    EB_REQUIRE(dh || dr_out, kBwd);
    EB_REQUIRE(dh || (!g2 && !dg2 && !db2), kBwd);
    EB_REQUIRE(f || (!gate && !g1 && !b1 && !post && res_scale == 1.f && !df), kBwd);
    EB_REQUIRE(f || !(dgate || dg1 || db1), kBwd);
    EB_REQUIRE(post || (!g1 && !b1 && !dg1 && !db1), kBwd);
    EB_REQUIRE(gate || !dgate, kBwd);
    const size_t total = (size_t)groups * rows, bytes = total * cols * sizeof(float), vector = (size_t)cols * sizeof(float), gates = groups * vector;
    EB_REQUIRE(!total || (stats && aligned16(stats) && (r_out || !dh)), kBwd);
    const void *in[] = {dh, dr_out, f, r_out, gate, g1, b1, g2, stats};
    const size_t in_bytes[] = {bytes, bytes, bytes, bytes, gates, vector, vector, vector, total * 16};
    float *out[] = {df, dr, dgate, dg1, db1, dg2, db2};
    const size_t out_bytes[] = {bytes, bytes, gates, vector, vector, vector, vector};
    for (int i = 0; i < 9; i++) EB_REQUIRE(aligned4(in[i]), kBwd);
    for (int o = 0; o < 7; o++) {
        EB_REQUIRE(aligned4(out[o]), kBwd);
        for (int i = 0; i < 9; i++) EB_REQUIRE(o < 2 && i < 4 ? !clash(out[o], out_bytes[o], in[i], in_bytes[i]) : !overlap(out[o], out_bytes[o], in[i], in_bytes[i]), kBwd);
        for (int q = 0; q < o; q++) EB_REQUIRE(!overlap(out[o], out_bytes[o], out[q], out_bytes[q]), kBwd);
        EB_REQUIRE(!(o < 2 && inc_d && out[o]) || (out[o] != dh && out[o] != dr_out && out[o] != f && out[o] != r_out), kBwd);
    }
    EB_CTX(dev);
    const bool cluster = cols > 4096, general = kind || db1 || db2 || (dgate && b1);        // dgate with a shift takes the sums of u too
    const unsigned csize = cluster ? (unsigned)ceil_div(cols, 2048) : 1;
    bool vec = cols % 4 == 0;
    for (int i = 0; i < 8; i++) vec = vec && aligned16(in[i]);
    vec = vec && aligned16(df) && aligned16(dr);
    BwdArgs a{dh, dr_out, f, r_out, gate, g1, b1, g2, stats, df, dr, nullptr, nullptr, res_scale, cols, 0, rows, kind, post, 0, 0};
    a.chunk = cluster ? (int)((ceil_div(cols, csize) + 3) & ~(size_t)3) : cols;
    a.want_gate = dgate != nullptr;
    a.want_param = (dg2 ? 1 : 0) | (db2 ? 2 : 0) | (dg1 ? 4 : 0) | (db1 ? 8 : 0);
    a.unit_groups = dgate ? groups : 1;
    a.unit_rows = dgate ? (size_t)rows : total;
    // slices of a group: so many that the rounds of units over the blocks take the fewest rows one after the other
    const size_t passes = total ? ceil_div(a.unit_rows, cols <= 256 ? 8 : 1) : 1;
    size_t most = 1, slices = 1, units = 1;
    auto plan = [&]() {
        most = total ? with_bwd(cols, [&](auto k) { return k.resident(dev, vec, general, csize); }) : 1;
        if (!most) return;
        slices = 1; units = a.unit_groups;
        size_t longest = ceil_div(units, most) * passes;
        for (size_t rounds = 1; rounds <= 4 && a.unit_groups; rounds++) {
            size_t s = rounds * most / a.unit_groups;
            if (s > passes) s = passes;
            if (s > 1 && rounds * ceil_div(passes, s) < longest) { slices = s; units = s * a.unit_groups; longest = rounds * ceil_div(passes, s); }
        }
    };
    plan();
    // a group in one slice: a block of one team writes its dgate itself, as it holds its columns
    if (vec && dgate && slices == 1 && cols > 256 && !aligned16(dgate)) { vec = false; plan(); }
    if (!most) return EDDLB200_ELIMIT;
    a.slices = (int)slices;
    a.workers = (int)(units < most ? units : most);
    const size_t param_floats = a.want_param ? (size_t)a.workers * 4 * cols : 0, gate_floats = dgate && slices > 1 ? units * cols : 0;
    const bool fold = a.want_param || gate_floats;
    a.gate_part = dgate;
    a.inc_gate = dgate && !gate_floats && inc_g;
    if (total && (fold || dgate)) {
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        if (int e = cuda_status(cudaStreamIsCapturing(st, &capturing), kBwd)) return e;
        if (capturing != cudaStreamCaptureStatusNone) return set_error(EDDLB200_EINVAL, "%s: the column sums use the library's scratch memory, which a captured graph must not hold", kBwd);
    }
    if (total && fold) {
        float *scr = (float *)scratch(cx, (param_floats + gate_floats) * sizeof(float));
        if (!scr) return cudaErrorMemoryAllocation;
        a.param_part = scr;
        if (gate_floats) a.gate_part = scr + param_floats;
    }
    if (total) for (int i = 0; i < 9; i++) EB_READS(in[i], in_bytes[i]);
    int inc[2] = {inc_d != 0, inc_d != 0};
    for (int o = 0; o < 7; o++) {
        if (!out[o]) continue;
        if (o < 2 ? !inc_d : !inc_g) EB_WRITES(out[o], out_bytes[o]);
        else if (o >= 2) EB_MODIFIES(out[o], out_bytes[o]);
        else {
            EB_SETTLE(out[o], out_bytes[o]);
            int status = 0;
            if (lz_take(cx, st, out[o], out_bytes[o], &status)) inc[o] = 2;      // zeros owed to all of it: nothing to read
            if (status) return status;
        }
    }
    a.inc_df = inc[0]; a.inc_dr = inc[1];
    if (!total) {                            // the sums over no rows are zero
        for (int o = 2; o < 7 && !inc_g; o++)
            if (out[o] && out_bytes[o]) if (int e = launch_zero_fill(cx, st, out[o], out_bytes[o] / sizeof(float))) return e;
        return 0;
    }
    ProfScope prof(cx, PROF_BN_BWD, (double)bytes * ((dh ? 2 : 0) + (dr_out ? 1 : 0) + (f ? 1 : 0) + (df ? 1 + (inc[0] == 1) : 0) + (dr ? 1 + (inc[1] == 1) : 0)));
    if (int e = with_bwd(cols, [&](auto k) { return k.launch(cx, st, a, vec, general, csize); })) return e;
    if (!fold) return 0;
    auto log_rows = [](int n) { int l = 0; while (l < 5 && (1 << l) < n) l++; return l; };
    FoldArgs fa{a.param_part, a.gate_part, {dg2, db2, dg1, db1}, dgate, cols, a.workers, a.slices, gate_floats ? groups : 0, inc_g, log_rows(a.workers), log_rows(a.slices), 0};
    fa.param_blocks = a.want_param ? (int)ceil_div(4, (size_t)32 >> fa.param_rows) : 0;
    const size_t gate_blocks = ceil_div((size_t)fa.groups, (size_t)32 >> fa.gate_rows);         // fewer groups than blocks that run at a time: far below the grid's limit
    eb::launch(norm_residual_fold_kernel, dim3((unsigned)ceil_div(cols, 32), (unsigned)(fa.param_blocks + gate_blocks)), dim3(32, 32), 0, st, fa);
    EB_LAUNCH_CHECK(kBwd);
    return 0;
}

}  // extern "C"
