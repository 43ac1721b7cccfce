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
// pieces in the blocks of a cluster.  What has to do with the entries (a few dozen a row: look-ups, repeated ids, 64-bit
// exponentials) is a chain of latencies as long as the streaming of the row, so it has a warp of its own that works ahead; the
// other warps keep a running maximum and sum a thread and meet once a row.  Mass outside the entries is summed from the
// values outside, not as 1 minus something: with `teacher_lse` the entries' cells are set to -infinity before the sum.  It stays relative to
// the largest logit outside where that lies far below the entries': a sure student has less there than fp32 holds beside 1.
#include <type_traits>
#include <cooperative_groups.h>
#include "common.cuh"

namespace {

using namespace eb;
namespace cg = cooperative_groups;

constexpr int kMaxTop = 1024;
constexpr int kMaxCluster = 8;
constexpr int kMaxPiece = 43008;                 // logits of a row in one block: 168 KB of shared memory, with up to 36 KB of entries
constexpr int kMaxCols = kMaxPiece * kMaxCluster;

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
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ float exp2_fast(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
constexpr float kLog2e = 1.44269504f;
// exp(d) beside `e`, exp(d / T): an exponential of its own, or e^T by one or two squarings for the temperatures 2 and 4, which doubles or quadruples the
// relative error of `e` (four exponentials of a logit are 110 us of 4096 x 32000 at 16 a cycle and SM: 226 us with them, at temperature 3, 195 with two)
enum : int { kNoExp, kOwnExp, kSquare, kFourth };
template <int HOW> struct Exp { static constexpr int value = HOW; };
template <int HOW>
__device__ __forceinline__ float plain(float d, float e) { return HOW == kSquare ? e * e : HOW == kFourth ? (e * e) * (e * e) : exp2_fast(d * kLog2e); }

// What a row's entries and its label add.  loss = base + per_z ((m - anchor) / T + ln z) - per_rest (ln z_out - ln z) + hard (m - x_label + ln z_1), with
// m the row's largest logit, z and z_1 the sums of exp((x - m) / T) and exp(x - m), z_out the first one outside the entries (and (m_out - m) / T added
// to its logarithm where it is relative to m_out, the largest logit outside); the gradient is
// inside / z - rest / z_out times the exponential outside the entries, inside / z times it minus `less` at an entry.  Where the entries hold less than half
// of the student's mass, z_in / z, the logarithm of z_out / z and that difference come from z_in / z: (entries - inside z_in / z) / z_out; what is
// left of them after subtracting numbers near 1 would be good to a few digits only.
struct Head {
    double base, per_z, per_rest, hard;
    float inside, rest, entries, x_label, anchor;         // anchor: the largest of the entries' logits
    float z, z1;                                 // the entries' sums relative to it, where their cells are closed
    float row_m, row_m_out, row_in, row_out, row_z, row_z1;         // what the other warps found of the row: m, m_out, z_in, z_out, z, z_1; m = -infinity: nothing that counts
    int label, label_is_entry, live;
};
struct Record {
    Head *head;
    float *value, *less;                         // of an entry: the student's logit, what the teacher takes off its gradient
    int *id;                                     // -1: padding, or an id that came before
};

// What the look-up of a row begins with, asked for while the row before is worked on: its numbers and its first entries.
constexpr int kAhead = 4;                        // times 32 entries
struct Ahead {
    float weight = 1.f, lse = 0.f, t[kAhead];
    int label = -1, id[kAhead];
    __device__ __forceinline__ void ask(const Args &a, int row) {
        if (row >= a.rows) return;
        const int lane = threadIdx.x & 31;
        if (a.weights) weight = a.weights[row];
        if (a.teacher_lse) lse = a.teacher_lse[row];
        if (a.alpha != 0.f) label = a.labels[row];
        if (a.alpha != 1.f) entries(a, row, 0, lane);
    }
    __device__ __forceinline__ void entries(const Args &a, int row, int j0, int lane) {
#pragma unroll
        for (int c = 0; c < kAhead; c++) {
            const int j = j0 + c * 32 + lane;
            id[c] = j < a.k ? a.ids[(size_t)row * a.k + j] : -1;
            t[c] = j < a.k ? a.teacher[(size_t)row * a.k + j] : 0.f;
        }
    }
};

// One warp: the record of a row.
__device__ void look_up(const Args &a, int row, int next_row, Ahead &ahead, const Record &r) {
    const int lane = threadIdx.x & 31;
    __syncwarp();                                // the record may be an earlier row's that a lane of this warp still reads
    Ahead now = ahead;
    ahead.ask(a, next_row);
    const float weight = now.weight;
    const float *x = a.x + (size_t)row * a.ld;
    if (weight == 0.f) {
        if (lane == 0) r.head->live = 0;
        __syncwarp();
        return;
    }
    const bool tail = a.teacher_lse != nullptr, soft = a.alpha != 1.f;
    const int label = now.label < a.cols && now.label >= 0 ? now.label : -1;
    const float x_label = label >= 0 ? x[label] : 0.f;
    const double inv_t = 1.0 / (double)a.temperature, lse = now.lse;
    float top = minus_inf(), anchor = minus_inf();
    bool label_seen = false;
    if (soft) {
        // Of several entries with one id the first counts: the lowest lane of 32 at a time, and only if none of the earlier ones, which all lanes look
        // through together, had it (k = 128: some 300 cycles; a table of the ids seen took ten times that).
        for (int j0 = 0; j0 < a.k; j0 += 32 * kAhead) {
            if (j0) now.entries(a, row, j0, lane);
            float value[kAhead];
#pragma unroll
            for (int c = 0; c < kAhead; c++) {
                if (now.id[c] >= a.cols || now.id[c] < 0) now.id[c] = -1;
                value[c] = now.id[c] >= 0 ? x[now.id[c]] : 0.f;
            }
#pragma unroll
            for (int c = 0; c < kAhead; c++) {
                const int j = j0 + c * 32 + lane;
                if (j - lane >= a.k) break;
                int id = now.id[c];
                const unsigned same = __match_any_sync(0xffffffffu, id);
                bool seen = (int)__ffs(same) - 1 != lane;
                const int4 *before = reinterpret_cast<const int4 *>(r.id);
#pragma unroll 4
                for (int q = 0; q < (j - lane) / 4; q++) { const int4 o = before[q]; seen |= o.x == id || o.y == id || o.z == id || o.w == id; }
                if (seen) id = -1;
                if (j < a.k) { r.id[j] = id; r.value[j] = value[c]; r.less[j] = now.t[c]; }
                __syncwarp();
                if (id >= 0) { top = max_nan(top, now.t[c]); anchor = max_nan(anchor, value[c]); label_seen |= id == label; }
            }
        }
        __syncwarp();
        top = warp_max_nan(top); anchor = warp_max_nan(anchor);
        if (!(fabsf(anchor) <= 3.4028235e38f)) anchor = 0.f;
    }
    const bool entries = soft && (tail || top != minus_inf());
    const double ws = entries ? (double)weight * (1.0 - (double)a.alpha) * a.temperature : 0.0;
    double sum = 0.0, terms = 0.0, per_sum = 1.0;
    float z = 0.f, z1 = 0.f;
    if (entries) {
        const float c_t = kLog2e / a.temperature;
        for (int j = lane; j < a.k; j += 32) {
            if (r.id[j] < 0) continue;
            const float below = r.value[j] - anchor;
            float log_p, p;
            if (tail) {                          // 1 - sum p may be small: in 64 bits up to the sum
                const double d = (double)r.less[j] * inv_t - lse, e = exp(d);
                log_p = (float)d; p = (float)e;
                sum += e;
                z += exp2_fast(below * c_t); z1 += exp2_fast(below * kLog2e);
            } else {
                log_p = (r.less[j] - top) * (float)inv_t; p = expf(log_p);
                sum += p;
            }
            if (p != 0.f) terms += p * (log_p - below * (float)inv_t);
            r.less[j] = p;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) { sum += __shfl_xor_sync(0xffffffffu, sum, o); terms += __shfl_xor_sync(0xffffffffu, terms, o); }
        if (tail) { z = warp_sum(z); z1 = warp_sum(z1); }
        else per_sum = 1.0 / sum;
        const float scale = (float)(ws * per_sum);
        for (int j = lane; j < a.k; j += 32) r.less[j] *= scale;
    } else if (soft) {
        for (int j = lane; j < a.k; j += 32) r.id[j] = -1;
    }
    label_seen = __any_sync(0xffffffffu, entries && label_seen);
    if (lane == 0) {
        const double rest = tail && entries ? fmax(0.0, 1.0 - sum) : 0.0, wt = ws * a.temperature;
        Head h;
        h.hard = label >= 0 ? (double)weight * a.alpha : 0.0;
        h.base = entries ? wt * (tail ? terms + (rest > 0.0 ? rest * (sum < 0.5 ? log1pf((float)-sum) : logf((float)rest)) : 0.0) : terms * per_sum - logf((float)sum)) : 0.0;
        h.per_z = entries ? wt * (tail ? sum : 1.0) : 0.0;
        h.per_rest = wt * rest;
        h.inside = (float)(ws * (tail ? sum + rest : 1.0));
        h.rest = (float)(ws * rest);
        h.entries = (float)(ws * sum);
        h.x_label = x_label; h.anchor = anchor; h.z = z; h.z1 = z1;
        h.label = label; h.label_is_entry = label_seen; h.live = 1;
        *r.head = h;
    }
    __syncwarp();
}

// Largest logit and sums of exponentials below it, of a thread, a warp, a row: z with the temperature (outside the entries where their cells are
// -infinity), z1 without.
struct Run {
    float m, z, z1;
    // relative to a common maximum; with nothing but -infinity so far the sums are zero and stay it
    __device__ __forceinline__ void meet(float top, float c_t) {
        const float d = m == top ? 0.f : m - top;
        z *= exp2_fast(d * c_t); z1 *= exp2_fast(d * kLog2e);
        m = top;
    }
};

// TEAM threads share a row (or a piece of it): a warp of eight, or all warps of the block but the last.  CLUSTER: the pieces of a row are the blocks
// of a cluster.  16-byte accesses whatever the row's alignment: the piece is laid out in shared memory with the alignment it has in
// global memory, -infinity around it, so the sums need no bounds.  A thread copies (cp.async), sums and writes the same pieces of the row, so
// between those steps nobody waits.  ex2 of one product: 2^-22 relative, the argument's roundings as in any fp32 softmax.
constexpr int blocks_per_sm(int team) { return team == 32 ? 4 : team == 128 ? 4 : 3; }
constexpr int entry_warps(bool cluster) { return cluster ? 1 : 2; }
constexpr int block_of(int team, bool cluster) { return team == 32 ? 256 : team + 32 * entry_warps(cluster); }
template <int TEAM, bool CLUSTER>
__global__ void __launch_bounds__(block_of(TEAM, CLUSTER), blocks_per_sm(TEAM)) distill_kernel(const Args a) {
    constexpr bool OWN = TEAM == 32;                       // every warp its own rows, entries and all
    constexpr int TEAMS = OWN ? 8 : 1, W = TEAM / 32, RECORDS = OWN ? 1 : CLUSTER ? 3 : 4;
    extern __shared__ __align__(16) float smem[];
    __shared__ Head heads[OWN ? 8 : RECORDS];
    __shared__ float4 runs[OWN ? 1 : 2][CLUSTER ? kMaxCluster : 1][W];
    const int team = OWN ? threadIdx.x / 32 : 0, t = OWN ? threadIdx.x % 32 : threadIdx.x, lane = threadIdx.x & 31, warp = t >> 5;
    const int kk = (a.k + 3) & ~3;
    float *x = smem + (size_t)team * (a.piece + 4 + 3 * RECORDS * kk), *lists = x + a.piece + 4;
    auto record = [&](int i) {
        float *p = lists + 3 * kk * i;
        return Record{heads + team + i, p, p + kk, reinterpret_cast<int *>(p + 2 * kk)};
    };
    const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0, csize = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
    const int c0 = rank * a.piece, n = max(0, min(a.piece, a.cols - c0));
    const bool tail = a.teacher_lse != nullptr && a.alpha != 1.f, one_exp = a.temperature == 1.f, any_entries = a.alpha != 1.f;
    const float c_t = kLog2e / a.temperature;
    // Clusters: all threads of all blocks meet once a row, the one entry warp with the next row's record.  Single blocks: the records are passed on by
    // barriers of their own (2 + i: record i is there, 6 + i: it has been used), between the team and one of two entry warps that
    // take the rows in turn; beside busy warps a look-up takes 8 to 13 k cycles, several times its row where rows are short.
    auto meeting = [&]() { if (CLUSTER) cg::this_cluster().sync(); };
    auto wait_for = [&](int id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(TEAM + 32) : "memory"); };
    auto tell = [&](int id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(TEAM + 32) : "memory"); };
    auto team_barrier = [&]() { if (OWN) __syncwarp(); else asm volatile("bar.sync 1, %0;" ::"n"(TEAM) : "memory"); };
    const int first = (int)(blockIdx.x / csize) * TEAMS + team, step = (int)(gridDim.x / csize) * TEAMS;
    EB_GRID_WAIT();

    // the row's maximum and sums from its warps' lines; with the entries' cells closed the maximum is theirs too
    auto combine = [&](int flip) {
        Run run{minus_inf(), 0.f, 0.f};
        for (int l = lane; l < csize * W; l += 32) {
            const float4 q = runs[flip][l / W][l % W];
            Run one{q.x, q.y, q.z};
            const float top = max_nan(run.m, one.m);
            run.meet(top, c_t); one.meet(top, c_t);
            run.z += one.z; run.z1 += one.z1;
        }
        run.meet(warp_max_nan(run.m), c_t);
        run.z = warp_sum(run.z); run.z1 = warp_sum(run.z1);
        return run;
    };
    // The row's sums with the entries' own.  Where the largest logit outside is 2^-32 of the row's largest or less, after the temperature, the sum outside
    // stays relative to it: beside the row's largest those classes would be zero from 2^-126 on.
    struct Sums { float m, m_out, in, out, z, z1; };
    auto with_entries = [&](Run run, const Head &h) {
        Run own{h.anchor, h.z, h.z1};
        if (!tail || h.z == 0.f) own.m = minus_inf();
        const float top = max_nan(run.m, own.m);
        const bool far = tail && run.m > minus_inf() && (top - run.m) * c_t > 32.f;
        Sums s{top, far ? run.m : top, 0.f, run.z, 0.f, 0.f};
        run.meet(top, c_t); own.meet(top, c_t);
        s.in = own.z; s.z = run.z + own.z; s.z1 = one_exp && any_entries ? s.z : run.z1 + own.z1;
        if (!far) s.out = run.z;
        return s;
    };
    auto loss_of = [&](const Head &h, const Sums &s) {
        double l = h.base;
        if (any_entries) l += h.per_z * (((double)s.m - (double)h.anchor) / (double)a.temperature + (double)logf(s.z));
        if (h.per_rest > 0.0) l -= h.per_rest * (s.in < 0.5f * s.z ? (double)log1pf(-s.in / s.z) : (double)logf(s.out / s.z) + (s.m_out < s.m ? ((double)s.m_out - (double)s.m) / (double)a.temperature : 0.0));
        if (h.label >= 0) l += h.hard * ((double)s.m - (double)h.x_label + (double)logf(s.z1));
        return (float)l;
    };

    if (!OWN && warp >= W) {
        // ============================ the entries, ahead of their rows; the loss ============================
        if (CLUSTER) {
            Ahead ahead;
            ahead.ask(a, first);
            if (first < a.rows) look_up(a, first, first + step, ahead, record(0));
            meeting();
            int i = 0, flip = 0;
            for (int row = first; row < a.rows; row += step, flip ^= 1) {
                const Head &h = *record(i).head;
                // the record written here was last read two meetings ago
                i = i == 2 ? 0 : i + 1;
                if (row + step < a.rows) look_up(a, row + step, row + 2 * step, ahead, record(i));
                meeting();
                if (rank) continue;
                float loss = 0.f;
                if (h.live) {
                    const Sums s = with_entries(combine(flip), h);
                    if (s.m != minus_inf()) loss = loss_of(h, s);
                }
                if (lane == 0) a.loss[row] = loss;
            }
        } else {
            auto finish = [&](int n) {                       // row n of the block is done: its loss, and its record may be written again
                wait_for(6 + (n & 3));
                const Head &h = *record(n & 3).head;
                const float loss = h.row_m == minus_inf() ? 0.f : loss_of(h, Sums{h.row_m, h.row_m_out, h.row_in, h.row_out, h.row_z, h.row_z1});
                if (lane == 0) a.loss[first + n * step] = loss;
            };
            Ahead ahead;
            int n = warp - W;
            ahead.ask(a, first + n * step);
            for (; first + n * step < a.rows; n += 2) {
                if (n >= 4) finish(n - 4);
                look_up(a, first + n * step, first + (n + 2) * step, ahead, record(n & 3));
                tell(2 + (n & 3));
            }
            for (int m = n >= 4 ? n - 4 : n - 2; m < n; m += 2) if (m >= 0) finish(m);
        }
    } else {
        // piece v of the row, 16 bytes, on its way into its place; -infinity where there is no logit
        auto fetch = [&](const float *src, int off, int end, int v) {
            const int u = v * 4;
            if (u >= off && u + 4 <= end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(x + u)), "l"(src - off + u) : "memory");
            else {
#pragma unroll
                for (int q = 0; q < 4; q++) x[u + q] = u + q >= off && u + q < end ? src[u + q - off] : minus_inf();
            }
        };
        auto source = [&](int row) { return a.x + (size_t)row * a.ld + c0; };
        auto misfit = [&](const float *p) { return (int)((uintptr_t)p >> 2) & 3; };
        auto fetch_row = [&](int row) {
            if (row >= a.rows) return;
            const float *src = source(row);
            const int off = misfit(src), end = off + n;
            for (int v = t; v * 4 < end; v += TEAM) fetch(src, off, end, v);
        };
        int i = 0, flip = 0;
        Ahead ahead;
        if (OWN) ahead.ask(a, first);
        fetch_row(first);
        meeting();
        for (int row = first; row < a.rows; row += step, flip ^= 1) {
            const Record r = record(i);
            const int turn = i;
            if (OWN) look_up(a, row, row + step, ahead, r);
            else i = i == RECORDS - 1 ? 0 : i + 1;
            if (!OWN && !CLUSTER) wait_for(2 + turn);
            auto done = [&](const Sums &s) {
                if (OWN) {
                    if (t == 0) a.loss[row] = s.m == minus_inf() ? 0.f : loss_of(*r.head, s);
                    __syncwarp();
                } else if (!CLUSTER) {
                    if (t == 0) { r.head->row_m = s.m; r.head->row_m_out = s.m_out; r.head->row_in = s.in; r.head->row_out = s.out; r.head->row_z = s.z; r.head->row_z1 = s.z1; }
                    tell(6 + turn);
                }
            };
            float *dst = a.delta ? a.delta + (size_t)row * a.ld + c0 : nullptr;
            const bool live = r.head->live != 0;
            const int off = misfit(source(row)), end = off + n, nv = (end + 3) >> 2, label = live ? r.head->label : -1;
            const bool ce = label >= 0;
            Run run{minus_inf(), 0.f, 0.f};
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (live) {
                if (tail) {
                    team_barrier();
                    for (int j = t; j < a.k; j += TEAM) {
                        const int at = r.id[j] - c0;
                        if (r.id[j] >= 0 && at >= 0 && at < n) x[at + off] = minus_inf();
                    }
                    team_barrier();
                }
                auto add = [&](auto want_t, auto want_1) {
#pragma unroll 2
                    for (int v = t; v < nv; v += TEAM) {
                        const float4 q = *reinterpret_cast<const float4 *>(x + v * 4);
                        const float top = max_nan(max_nan(q.x, q.y), max_nan(q.z, q.w));
                        if (!(top <= run.m)) run.meet(max_nan(top, run.m), c_t);
                        const float m = run.m == minus_inf() ? 0.f : run.m;
                        const float d0 = q.x - m, d1 = q.y - m, d2 = q.z - m, d3 = q.w - m;
                        float e0 = 0.f, e1 = 0.f, e2 = 0.f, e3 = 0.f;
                        if (decltype(want_t)::value) {
                            e0 = exp2_fast(d0 * c_t); e1 = exp2_fast(d1 * c_t); e2 = exp2_fast(d2 * c_t); e3 = exp2_fast(d3 * c_t);
                            run.z += (e0 + e1) + (e2 + e3);
                        }
                        if (decltype(want_1)::value != kNoExp) run.z1 += (plain<decltype(want_1)::value>(d0, e0) + plain<decltype(want_1)::value>(d1, e1)) + (plain<decltype(want_1)::value>(d2, e2) + plain<decltype(want_1)::value>(d3, e3));
                    }
                };
                if (any_entries && ce && !one_exp) {
                    if (a.temperature == 2.f) add(std::true_type(), Exp<kSquare>());
                    else if (a.temperature == 4.f) add(std::true_type(), Exp<kFourth>());
                    else add(std::true_type(), Exp<kOwnExp>());
                } else if (any_entries) { add(std::true_type(), Exp<kNoExp>()); run.z1 = run.z; }
                else add(std::false_type(), Exp<kOwnExp>());
                run.meet(warp_max_nan(run.m), c_t);
                run.z = warp_sum(run.z); run.z1 = warp_sum(run.z1);
                if (!OWN) {
                    // a warp's line in every block of the cluster; the lines of two rows take turns
                    float4 *mine = &runs[flip][rank][warp];
                    if (CLUSTER) { if (lane < csize) *cg::this_cluster().map_shared_rank(mine, lane) = make_float4(run.m, run.z, run.z1, 0.f); }
                    else if (lane == 0) *mine = make_float4(run.m, run.z, run.z1, 0.f);
                }
            }
            if (!OWN) {
                if (CLUSTER) meeting(); else team_barrier();
                if (live) run = combine(flip);
            }
            Sums sums{minus_inf(), 0.f, 0.f, 0.f, 0.f, 0.f};
            if (live) sums = with_entries(run, *r.head);
            if (sums.m == minus_inf()) {                   // no weight, or a mask leaves nothing of the row
                fetch_row(row + step);
                if (dst) for (int q = t; q < n; q += TEAM) dst[q] = 0.f;
                done(sums);
                continue;
            }
            if (!dst) { fetch_row(row + step); done(sums); continue; }
            const float m = sums.m, m_out = sums.m_out;
            const bool far = tail && m_out < m;
            const float f_in = any_entries ? r.head->inside / sums.z : 0.f, f_1 = ce ? (float)r.head->hard / sums.z1 : 0.f;
            const float f_out = !tail ? f_in : !(sums.out > 0.f) ? 0.f : sums.in < 0.5f * sums.z ? (r.head->entries - r.head->inside * (sums.in / sums.z)) / sums.out
                              : (far ? f_in * exp2_fast((m_out - m) * c_t) : f_in) - r.head->rest / sums.out;
            const bool straight = misfit(dst) == off;
            // the next row's pieces follow this row's out of their places
            const bool more = row + step < a.rows;
            const float *next = source(more ? row + step : row);
            const int next_off = misfit(next), next_end = more ? next_off + n : 0;
            auto put = [&](auto want_t, auto want_1, float f) {
#pragma unroll 2
                for (int v = t; v < nv; v += TEAM) {
                    const int u = v * 4;
                    const float4 q = *reinterpret_cast<const float4 *>(x + u);
                    const float v4[4] = {q.x, q.y, q.z, q.w};
                    float g[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float x = exp2_fast((v4[e] - m_out) * (decltype(want_t)::value ? c_t : kLog2e));
                        g[e] = f * x;
                        if (decltype(want_1)::value != kNoExp) g[e] = fmaf(f_1, plain<decltype(want_1)::value>(v4[e] - m, x), g[e]);
                    }
                    if (straight && u >= off && u + 4 <= end) *reinterpret_cast<float4 *>(dst - off + u) = make_float4(g[0], g[1], g[2], g[3]);
                    else {
#pragma unroll
                        for (int e = 0; e < 4; e++) if (u + e >= off && u + e < end) dst[u + e - off] = g[e];
                    }
                    if (u < next_end) fetch(next, next_off, next_end, v);
                }
            };
            if (any_entries && (far || (ce && !one_exp))) {
                if (far) put(std::true_type(), Exp<kOwnExp>(), f_out);
                else if (a.temperature == 2.f) put(std::true_type(), Exp<kSquare>(), f_out);
                else if (a.temperature == 4.f) put(std::true_type(), Exp<kFourth>(), f_out);
                else put(std::true_type(), Exp<kOwnExp>(), f_out);
            } else if (any_entries) put(std::true_type(), Exp<kNoExp>(), f_out + f_1);
            else put(std::false_type(), Exp<kNoExp>(), f_1);
            if (nv * 4 < next_end && t == nv % TEAM) fetch(next, next_off, next_end, nv);      // a row that reaches one piece further
            team_barrier();                                // the entries' and the label's places are written again, after the above
            const float hard = (float)r.head->hard;
            if (any_entries)
                for (int j = t; j < a.k; j += TEAM) {
                    const int at = r.id[j] - c0;
                    if (r.id[j] < 0 || at < 0 || at >= n) continue;
                    const float d = r.value[j] - m;
                    float g = f_in * exp2_fast(d * c_t) - r.less[j];
                    if (ce) g += f_1 * exp2_fast(d * kLog2e);
                    if (r.id[j] == label) g -= hard;
                    dst[at] = g;
                }
            if (ce && t == 0 && label >= c0 && label < c0 + n && !r.head->label_is_entry) {
                const float d = r.head->x_label - m;
                dst[label - c0] = f_1 * exp2_fast(d * kLog2e) + f_out * exp2_fast((r.head->x_label - m_out) * c_t) - hard;
            }
            done(sums);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (CLUSTER) cg::this_cluster().sync();                // a block's lines outlive the writes of the others
}

constexpr size_t kSmemSM = 227 * 1024, kStatic = 4 * 1024;             // of an SM; what a block takes beside its own
int blocks_held(size_t smem, int team) {
    const size_t n = kSmemSM / (smem + kStatic);
    return (int)(n < 1 ? 1 : n > (size_t)blocks_per_sm(team) ? (size_t)blocks_per_sm(team) : n);
}
template <int TEAM, bool CLUSTER>
int set_attributes(int dev) {
    static bool configured[EDDLB200_MAX_DEVICES] = {};
    if (configured[dev]) return 0;
    const cudaError_t e = cudaFuncSetAttribute(distill_kernel<TEAM, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, 222 * 1024);
    if (e != cudaSuccess) return cuda_status(e, "distill(attributes)");
    configured[dev] = true;
    return 0;
}
template <int TEAM>
int launch_distill(DevCtx *cx, int dev, cudaStream_t st, const Args &a, size_t smem) {
    if (int e = set_attributes<TEAM, false>(dev)) return e;
    const size_t want = ceil_div(a.rows, TEAM == 32 ? 8 : 1), most = (size_t)EDDLB200_NUM_SMS * blocks_held(smem, TEAM);
    eb::launch(distill_kernel<TEAM, false>, (unsigned)(want < most ? want : most), block_of(TEAM, false), smem, st, a);
    EB_LAUNCH_CHECK("distill");
    return 0;
}
// Clusters of `csize` blocks, `per_sm` of which fit an SM, that the device holds at once.  The blocks of a cluster share a group of SMs, whose number need
// not divide by what they take: with more clusters than the GPU holds the rows of the last ones would wait for a whole round (1023 x 131071,
// 55 clusters of eight of which 48 fit: 434 us, with 48 252).
int clusters_held(int dev, int csize, int per_sm, int &out) {
    static int known[EDDLB200_MAX_DEVICES][kMaxCluster + 1][4] = {};
    int &n = known[dev][csize][per_sm];
    if (!n) {
        if (int e = set_attributes<256, true>(dev)) return e;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension; at[0].val.clusterDim.x = csize; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
        cudaLaunchConfig_t c = {};
        c.gridDim = dim3((unsigned)(EDDLB200_NUM_SMS * per_sm / csize * csize)); c.blockDim = dim3(block_of(256, true));
        c.dynamicSmemBytes = kSmemSM / per_sm - kStatic; c.attrs = at; c.numAttrs = 1;
        if (c.dynamicSmemBytes > 222 * 1024) c.dynamicSmemBytes = 222 * 1024;
        int held = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&held, distill_kernel<256, true>, &c);
        if (e != cudaSuccess) return cuda_status(e, "distill(clusters)");
        n = held < 1 ? -1 : held;
    }
    out = n < 0 ? 0 : n;
    return 0;
}

}  // namespace

using namespace eb;

extern "C" int eddlb200_distill(int dev, const float *logits, const int *ids, const float *teacher, const float *teacher_lse, const int *labels,
                                const float *weights, int rows, int cols, size_t ld, int k, float temperature, float alpha, float *loss, float *delta) {
    const char *what = "distill";
    EB_REQUIRE(rows >= 0 && cols > 0 && k > 0 && ld >= (size_t)cols, what);
    EB_REQUIRE(temperature >= 1.17549435e-38f && temperature < INFINITY, what);
    EB_REQUIRE(alpha >= 0.f && alpha <= 1.f, what);
    if (cols > kMaxCols) return set_error(EDDLB200_ELIMIT, "%s: %d classes, at most %d", what, cols, kMaxCols);
    if (rows > 0x7ff00000) return set_error(EDDLB200_ELIMIT, "%s: %d rows", what, rows);
    if (k > kMaxTop) return set_error(EDDLB200_ELIMIT, "%s: %d entries a row, at most %d", what, k, kMaxTop);
    EB_REQUIRE(!rows || (logits && ids && teacher && loss), what);
    EB_REQUIRE(!rows || labels || alpha == 0.f, what);
    const size_t bytes = (rows ? (size_t)(rows - 1) * ld + cols : 0) * sizeof(float), entries = (size_t)rows * k * 4, each = (size_t)rows * 4;
    const void *in[] = {ids, teacher, teacher_lse, labels, weights};
    const size_t in_bytes[] = {entries, entries, each, each, each};
    EB_REQUIRE(delta == logits || !overlap(delta, bytes, logits, bytes), what);
    EB_REQUIRE(!overlap(loss, each, logits, bytes) && !overlap(loss, each, delta, bytes), what);
    EB_REQUIRE(aligned4(logits) && aligned4(delta) && aligned4(loss), what);
    for (int i = 0; i < 5; i++) EB_REQUIRE(aligned4(in[i]), what);
    for (int i = 0; i < 5; i++) EB_REQUIRE(!overlap(delta, bytes, in[i], in_bytes[i]) && !overlap(loss, each, in[i], in_bytes[i]), what);
    EB_CTX(dev);
    if (!rows) return 0;
    EB_READS(logits, bytes);
    for (int i = 0; i < 5; i++) EB_READS(in[i], in_bytes[i]);
    // columns past `cols` keep what they hold: the range is written in part
    if (ld == (size_t)cols) EB_WRITES(delta, bytes); else EB_MODIFIES(delta, bytes);
    EB_WRITES(loss, each);
    ProfScope prof(cx, PROF_ELEMENTWISE, (delta ? 8.0 : 4.0) * rows * cols);
    Args a{logits, teacher, teacher_lse, weights, ids, labels, loss, delta, rows, cols, k, 0, ld, temperature, alpha};
    const size_t kk = (k + 3) & ~3;
    auto smem = [&](unsigned c, int records) { a.piece = (int)((ceil_div(cols, c) + 3) & ~(size_t)3); return ((size_t)a.piece + 4 + 3 * records * kk) * sizeof(float); };
    // A warp a row, entries and all, as long as two blocks of eight rows fit an SM and there are rows for every SM: nothing waits for anything but its own
    // latencies (40000 x 1300, 32 entries: 119 us, with a block a row 233; 16384 x 4000, where one block fits: 180 and 147).
    if (cols <= 256 || (8 * smem(1, 1) <= 112 * 1024 && rows >= EDDLB200_NUM_SMS * 8)) { const size_t b = 8 * smem(1, 1); return launch_distill<32>(cx, dev, st, a, b); }
    if (cols <= 8192) { const size_t b = smem(1, 4); return launch_distill<128>(cx, dev, st, a, b); }
    if (cols <= 16384) { const size_t b = smem(1, 4); return launch_distill<256>(cx, dev, st, a, b); }
    // A cluster's size: the least of rounds x time of a round, 3.6 us and 0.21, 0.35 or 0.48 ns a logit of a block with one, two or three of them on its SM,
    // or the look-up of many entries if that is longer (within 8 % of 50 measured pairs of shape and size).  1023 x 131071: five blocks 241 us,
    // eight 252, four 286; 1000 x 80000: five 137, eight 165; 2000 x 50257: three 163, four 176; 4096 x 32000: two 208, three 242.
    unsigned csize = 0, clusters = 0;
    double least = 0.0;
    for (int c = kMaxCluster; c >= 2; c--) {
        const size_t b = smem(c, 3);
        if (a.piece > kMaxPiece) break;
        const int per_sm = blocks_held(b, 256);
        int held = 0;
        if (int e = clusters_held(dev, c, per_sm, held)) return e;
        if (!held) continue;
        const int at_once = rows < held ? rows : held, full = (int)ceil_div((size_t)at_once * c, (size_t)EDDLB200_NUM_SMS), on_sm = full < per_sm ? full : per_sm;
        const double round = 3570.0 + a.piece * (on_sm == 1 ? 0.21 : on_sm == 2 ? 0.35 : 0.48), look = 0.09 * k * k;
        const double t = (double)ceil_div(rows, held) * (round > look ? round : look);
        if (!csize || t < least) { csize = c; clusters = at_once; least = t; }
    }
    if (!csize) return set_error(EDDLB200_ELIMIT, "%s: the device holds no cluster for rows of %d classes", what, cols);
    const size_t b = smem(csize, 3);
    eb::launch_cluster(distill_kernel<256, true>, csize, clusters * csize, block_of(256, true), b, st, a);
    EB_LAUNCH_CHECK(what);
    return 0;
}
