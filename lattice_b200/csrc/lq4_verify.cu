// Verification of drafted tokens (a chain or a tree) against the target's distribution, from given uniforms.
//
// At a node with target distribution p and draft distribution q the children are tried in index order, and a
// refused child leaves the residual norm(max(p' - q, 0)) of what was there before it.  Unrolled, the residual
// after r refusals is max(p - a_r q, 0) / Z_r with a_0 = 0, Z_0 = 1 and
//
//     a_{r+1} = a_r + Z_r,     Z_{r+1} = sum_j max(p_j - a_{r+1} q_j, 0):
//
// two numbers carry the whole state, and a refusal costs one sum over the vocabulary.  A child with token t is
// accepted iff u q(t) Z < max(p(t) - a q(t), 0).  Certain drafts (no draft distribution) take the refused tokens
// out of p instead: accepted iff u Z < p(t), Z -= p(t) on refusal.  The last token is the smallest j whose
// cumulated residual exceeds u_0 times its sum; temperature 0 compares with the argmax throughout.
//
// One thread-block cluster per sequence walks down from the root and reads only the rows of the nodes it
// visits (a tree of 64 nodes has few on its path); the vocabulary is cut over the cluster, 512 bytes of logits per
// warp step.  The rows of a node are read once: a warp's share (32 logits a lane at most, as a rule) stays in registers as
// masses relative to the warp's own maximum, (max, sum) of p and q go through distributed shared memory with one
// cluster barrier, a refusal is a pass over the registers with another barrier, and the last token comes from the one
// warp that the border falls into.  Longer shares are read again instead.  Every CTA takes every decision itself from the
// same numbers, in the same order.
//
// A cluster lives in one GPC and gets some 0.8 TB/s: two rows of 248320 f32 logits are 2.5 us and more per node, one node after
// the other.  Where there are few enough rows (stat_splits), verify_stats_kernel takes (max, sum) of every row over the
// whole GPU first; the walk then only reads the rows of a node where a draft is refused or the last token is drawn.  What
// bounds it is the chain of latencies per node (rows, two reductions, a barrier); without statistics the first child's rows
// are fetched into L2 meanwhile.  B200, device time: a chain of 5 over 248320 f32 logits 26 to 31 us with the data (10 MB of rows:
// 1.5 us at HBM rate); 16 trees of 24 over 100003 bf16 logits 49 to 101 us.  Under ncu the chain waits at barriers most of
// all, then for instructions and loads.  The held form does not fit 128 registers: 1012 bytes of spill loads with f32
// logits, 236 with bf16, none in the form that reads long shares again.
//
// Decisions lie next to borders.  Masses are f32 (ex2.approx of the rounded distance from the maximum: a few 2^-23, and
// exactly 1 at the maximum; four or eight at a time are added in f32); all further sums are pairs of f32 (some 48 bits, any size of
// residual; sums of equal masses are exact, so that they meet a border where they should).  f64 is left to one lane: this
// part does about two f64 operations a cycle and SM.  Code is kept short for the same reason as the loads are early: a
// node's pass runs through it once, and instruction fetches count.
#include "lq4_attend.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace lq4 {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kVThreads = 512, kVWarps = kVThreads / 32, kMaxCluster = 16;
constexpr uint32_t kNoToken = 0xffffffffu;

struct VerifyParams {
    const void* target;
    const void* draft;                  // NULL: certain drafts
    uint64_t target_batch, target_node, draft_batch, draft_node;
    uint32_t nodes, vocab;
    const int32_t* tokens;
    const int32_t* parents;
    const int32_t* node_counts;
    const float* uniforms;
    const float* temperature;
    int32_t* path;
    int32_t* path_len;
    int32_t* next_token;
    int32_t* status;
    struct Stat* stats;                 // [2: target, draft][batch * nodes][splits], or NULL
    uint32_t batch, splits;
};

// An unevaluated sum h + l of two f32, |l| at most half a step of h.
struct Pair {
    float h, l;
};
__device__ __forceinline__ Pair plus(const Pair& a, const Pair& b) {
    const float s = __fadd_rn(a.h, b.h), t = __fsub_rn(s, a.h);
    const float e = __fadd_rn(__fadd_rn(__fsub_rn(a.h, __fsub_rn(s, t)), __fsub_rn(b.h, t)), __fadd_rn(a.l, b.l));
    const float h = __fadd_rn(s, e);
    return {h, __fsub_rn(e, __fsub_rn(h, s))};
}
__device__ __forceinline__ bool above(const Pair& a, const Pair& b) { return a.h > b.h || (a.h == b.h && a.l > b.l); }
__device__ __forceinline__ double value(const Pair& a) { return (double)a.h + (double)a.l; }
__device__ __forceinline__ Pair pair_of(double x) {
    const float h = (float)x;
    return {h, (float)(x - (double)h)};
}
__device__ __forceinline__ Pair lanes_sum(Pair x, int first = 16) {
    for (int o = first; o; o >>= 1) x = plus(x, {__shfl_xor_sync(0xffffffffu, x.h, o), __shfl_xor_sync(0xffffffffu, x.l, o)});
    return x;
}
__device__ __forceinline__ Pair lanes_prefix(Pair x, uint32_t lane) {      // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Pair up = {__shfl_up_sync(0xffffffffu, x.h, o), __shfl_up_sync(0xffffffffu, x.l, o)};
        if (lane >= (uint32_t)o) x = plus(up, x);
    }
    return x;
}

// (max, sum of exp((x - max) / tau)) of a share of a row
struct WarpSum {
    float m;
    Pair s;
};

// log2(e) / tau.  Above zero for an infinite temperature too: that is the limit in which everything above -inf weighs the same,
// and 0 * -inf would be NaN.
__device__ __forceinline__ float per_tau(float tau) { return fmaxf(1.44269504088896340736f / tau, 1.4e-45f); }
// exp((x - m) / tau), c = per_tau(tau); a row whose maximum is +inf has all its mass on the entries that are.
__device__ __forceinline__ float mass(float x, float m, float c) {
    if (m == INFINITY) return x == m ? 1.0f : 0.0f;
    return exp2_fast((x - (m == -INFINITY ? 0.0f : m)) * c);
}
// The same beyond f32's range and free of the distance's rounding, for the drafted tokens: their p and q are compared however
// small they are.
__device__ __forceinline__ double mass_wide(float x, float m, float c) {
    if (x == -INFINITY || m == INFINITY) return x == m ? 1.0 : 0.0;
    const float d = __fsub_rn(x, m), t = __fsub_rn(d, x);
    const float e = __fsub_rn(__fsub_rn(x, __fsub_rn(d, t)), __fadd_rn(m, t));      // d + e = x - m
    const float y = d * c, n = rintf(y);
    if (!(y > -1000.0f)) return 0.0;
    const double f = exp2_fast((y - n) + fmaf(d, c, -y) + e * c);
    return __hiloint2double(__double2hiint(f) + ((int)n << 20), __double2loint(f));
}
// The sums of several shares, over lanes that differ in bits first, first / 2, .. 1: one maximum, scaled sums.
__device__ __forceinline__ WarpSum join_lanes(WarpSum a, int first, float c) {
    float m = a.m;
    for (int o = first; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float f = mass(a.m, m, c);                                     // (nothing has mass: 0)
    return {m, lanes_sum({a.s.h * f, a.s.l * f}, first)};
}
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }      // NaN carries no mass

// A cluster's start: another CTA's shared memory may be touched once all of them are known to run.  In two halves, so that the
// way between them hides behind a load.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Order of candidates: higher logit first, ties to the lower id (0: nothing that ranks).
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t id) {
    if (v == -INFINITY) return 0;
    if (v == 0.0f) v = 0.0f;
    uint32_t u = __float_as_uint(v);
    u = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return ((uint64_t)u << 32) | (uint32_t)~id;
}

// A lane's V logits (16 bytes), from element j of a row on: fetched as they lie where the load fits, and then read as f32,
// -inf outside the row and for NaN.  In two steps, so that many fetches can be under way before the first value is used.  The
// few at a row's ends, and rows of the draft that lie otherwise than the target's, come one by one.
template <typename T>
constexpr int kLane = 16 / sizeof(T);
template <int V>
struct Few {
    float x[V];
};
template <typename T>
__device__ __noinline__ Few<kLane<T>> edge(const T* row, int32_t j, int32_t end) {
    Few<kLane<T>> r;
#pragma unroll
    for (int i = 0; i < kLane<T>; ++i) {
        r.x[i] = -INFINITY;
        if (j + i >= 0 && j + i < end) {
            if constexpr (std::is_same<T, float>::value)
                r.x[i] = __ldg(row + j + i);
            else
                r.x[i] = bf16_to_f32(__ldg(row + j + i));
        }
    }
    return r;
}
template <typename T>
__device__ __forceinline__ void fetch(const T* row, int32_t j, bool fits, uint4& r) {
    if (fits) r = __ldg(reinterpret_cast<const uint4*>(row + j));
}
template <typename T>
__device__ __forceinline__ void read(const T* row, int32_t j, int32_t end, bool fits, const uint4& r, float (&x)[kLane<T>]) {
    if (fits) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, float>::value) {
                x[i] = __uint_as_float(w[i]);
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    } else {
        const Few<kLane<T>> e = edge(row, j, end);
#pragma unroll
        for (int i = 0; i < kLane<T>; ++i) x[i] = e.x[i];
    }
#pragma unroll
    for (int i = 0; i < kLane<T>; ++i) x[i] = clean(x[i]);
}
template <typename T>
__device__ __forceinline__ void load(const T* row, int32_t j, int32_t end, bool fits, float (&x)[kLane<T>]) {
    uint4 r;
    fetch(row, j, fits, r);
    read(row, j, end, fits, r, x);
}

template <typename T>
__device__ __forceinline__ float one_logit(const T* row, uint32_t j) {
    if constexpr (std::is_same<T, float>::value)
        return clean(row[j]);
    else
        return clean(bf16_to_f32(row[j]));
}

struct Stat {                           // of a split of a row, for the walk
    WarpSum s;
    uint64_t best;
};
struct Exchange {                       // what a CTA tells the others
    WarpSum p, q;
    uint64_t best;
    Pair total;
};
struct Row {                            // the current node's distributions, for all warps of a CTA
    float pm, qm, q_over_p;             // maxima; q(t) in units of p's masses is (mass of q) * q_over_p
    uint64_t best;
};

// Logits of a warp step; steps of a warp's share that stay in registers (32 logits a lane).
template <typename T>
constexpr uint32_t kStep = 32 * kLane<T>;
template <typename T>
constexpr uint32_t kHeldSteps = 32 / kLane<T>;

// HELD: every warp's share is at most that many steps.
template <typename T, bool HELD>
__global__ void __launch_bounds__(kVThreads, 1) verify_kernel(const __grid_constant__ VerifyParams p) {
    const cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ranks = cluster.num_blocks(), rank = cluster.block_rank();
    constexpr uint32_t V = kLane<T>, STEP = kStep<T>, kHeld = kHeldSteps<T>;
    const uint32_t b = blockIdx.x / ranks, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    __shared__ Exchange slots[2][kMaxCluster];
    __shared__ WarpSum wp[kVWarps], wq[kVWarps];
    __shared__ uint64_t wbest[kVWarps];
    __shared__ Pair wtot[kVWarps], s_base, s_border;
    __shared__ uint32_t s_who;
    __shared__ Row row;
    __shared__ double s_ip;                                              // 1 / (sum of p's masses)
    __shared__ int32_t parent[LQ4_MAX_TREE_NODES], token[LQ4_MAX_TREE_NODES];
    __shared__ float uni[LQ4_MAX_TREE_NODES];
    __shared__ double child_p[LQ4_MAX_TREE_NODES], child_q[LQ4_MAX_TREE_NODES];
    __shared__ uint32_t gone[LQ4_MAX_TREE_NODES];
    __shared__ uint32_t s_action, s_child, s_gone;
    __shared__ double s_a, s_z;
    __shared__ Row row_of[LQ4_MAX_TREE_NODES];                           // with statistics: every node's, known from the start
    __shared__ double ip_of[LQ4_MAX_TREE_NODES];

    cluster_arrive();
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    int32_t n = p.node_counts ? p.node_counts[b] : (int32_t)p.nodes;
    cluster_wait();                                                      // the other CTAs' slots exist from here on
    if (n > (int32_t)p.nodes) {
        n = (int32_t)p.nodes;
        if (tid == 0 && rank == 0) atomicOr(p.status, kDevErrBadIndex);
    }
    const uint64_t first = (uint64_t)b * p.nodes;
    if (n <= 0) {                                                        // uniform over the cluster
        if (rank == 0) {
            if (tid < p.nodes) p.path[first + tid] = -1;
            if (tid == 0) p.path_len[b] = 0, p.next_token[b] = -1;
        }
        return;
    }
    if (tid < (uint32_t)n) {
        parent[tid] = p.parents ? p.parents[first + tid] : (int32_t)tid - 1;
        token[tid] = tid ? p.tokens[first + tid] : -1;
        uni[tid] = p.uniforms[first + tid];
    }
    const float tau = p.temperature ? p.temperature[b] : 1.0f;
    const bool greedy = !(tau >= 1e-20f);
    const float it = greedy ? 1.0f : per_tau(tau);
    const bool sampled = p.draft != nullptr && !greedy;
    const T* target_rows = static_cast<const T*>(p.target) + b * p.target_batch;
    const T* draft_rows = static_cast<const T*>(p.draft) + b * p.draft_batch;
    uint32_t turn = 0;                                                   // which half of `slots` comes next
    if (rank == 0 && tid < p.nodes) p.path[first + tid] = tid == 0 ? 0 : -1;
    uint32_t cur = 0, count = 1;
    __syncthreads();

    // One warp: a row's shares, one per lane, to what the walk needs of it.
    auto join_row = [&](WarpSum P, WarpSum Q, uint64_t best, bool with_q, Row& to, double& ip) {
        P = join_lanes(P, 16, it);
        Q = join_lanes(Q, 16, it);
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
            best = k > best ? k : best;
        }
        const bool has_p = P.m != -INFINITY, has_q = with_q && Q.m != -INFINITY;      // (a row without mass has neither)
        if (lane == 0) {
            ip = has_p ? 1.0 / value(P.s) : 0.0;
            to = {P.m, with_q ? Q.m : -INFINITY, has_q ? (float)(value(P.s) / value(Q.s)) : 0.0f, best};
        }
        __syncwarp();
    };
    auto child_masses = [&](uint32_t c, const T* prow, const T* qrow, const Row& r) {      // of a child's token behind its parent
        if ((uint32_t)token[c] >= p.vocab) return;
        child_p[c] = r.pm != -INFINITY ? mass_wide(one_logit(prow, token[c]), r.pm, it) : 0.0;
        child_q[c] = r.qm != -INFINITY ? mass_wide(one_logit(qrow, token[c]), r.qm, it) : 0.0;
    };
    if (p.stats != nullptr) {
        for (uint32_t node = warp; node < (uint32_t)n; node += kVWarps) {
            bool with_q = false;
            for (uint32_t c = node + 1; c < (uint32_t)n && sampled; ++c) with_q |= parent[c] == (int32_t)node;
            const Stat* of = p.stats + (first + node) * p.splits;
            Stat x{{-INFINITY, {0.0f, 0.0f}}, 0}, y = x;
            if (lane < p.splits) {
                x = of[lane];
                if (with_q) y = of[(uint64_t)p.batch * p.nodes * p.splits + lane];
            }
            join_row(x.s, y.s, x.best, with_q, row_of[node], ip_of[node]);
        }
        __syncthreads();
        if (tid < (uint32_t)n && tid > 0 && !greedy && parent[tid] >= 0 && parent[tid] < (int32_t)tid)
            child_masses(tid, target_rows + parent[tid] * p.target_node, draft_rows + parent[tid] * p.draft_node, row_of[parent[tid]]);
        __syncthreads();
    }

    const uint32_t all_warps = ranks * kVWarps, me = rank * kVWarps + warp;
    for (;;) {
        // this warp's part of the row, in steps from the row's own 16-byte border on
        const T* prow = target_rows + cur * p.target_node;
        const T* qrow = sampled ? draft_rows + cur * p.draft_node : nullptr;
        const int32_t shift = (int32_t)((reinterpret_cast<uintptr_t>(prow) & 15) / sizeof(T));
        const uint32_t steps = (p.vocab + shift + STEP - 1) / STEP, per = (steps + all_warps - 1) / all_warps;
        const uint32_t c0 = min(me * per, steps), c1 = min(c0 + per, steps);
        const bool q_alike = ((reinterpret_cast<uintptr_t>(prow) ^ reinterpret_cast<uintptr_t>(qrow)) & 15) == 0;
        auto at = [&](uint32_t c) { return (int32_t)(c * STEP + lane * V) - shift; };      // this lane's first logit of step c
        auto fits = [&](int32_t j, int32_t end) { return j >= 0 && j + (int32_t)V <= end; };
        uint32_t child = (uint32_t)n;                                    // the first one
        for (uint32_t c = (uint32_t)n - 1; c > cur; --c)
            if (parent[c] == (int32_t)cur) child = c;
        const bool with_q = sampled && child < (uint32_t)n;

        // ---- (max, sum) of p, of q where children need it; the argmax for greedy sequences
        WarpSum sp{-INFINITY, {0.0f, 0.0f}}, sq = sp;                    // of this warp
        const int32_t vocab = (int32_t)p.vocab;
        uint64_t best = 0;
        float ep[HELD ? kHeld : 1][V], eq[HELD ? kHeld : 1][V];          // masses relative to sp.m and sq.m
        // The warp's logits of p, and of q where children need it, into ep and eq.
        auto hold = [&]() {
            if constexpr (HELD) {
                uint4 rp[kHeld], rq[kHeld];                                  // all loads are under way before the first use
#pragma unroll
                for (uint32_t h = 0; h < kHeld; ++h) {
                    const int32_t j = at(c0 + h);
                    const bool f = fits(j, c0 + h < c1 ? vocab : 0);
                    fetch(prow, j, f, rp[h]);
                    fetch(qrow, j, f && q_alike && with_q, rq[h]);
                }
#pragma unroll
                for (uint32_t h = 0; h < kHeld; ++h) {
                    const int32_t j = at(c0 + h), end = c0 + h < c1 ? vocab : 0;
                    read(prow, j, end, fits(j, end), rp[h], ep[h]);
                    if (with_q) read(qrow, j, end, fits(j, end) && q_alike, rq[h], eq[h]);
                }
            }
        };
        if constexpr (HELD) {
            if (p.stats == nullptr) {
                hold();
                if (child < (uint32_t)n) {                                   // most likely the next node: its rows into L2
                    const T* next_p = target_rows + child * p.target_node;
                    const T* next_q = sampled ? draft_rows + child * p.draft_node : next_p;
                    for (uint32_t h = 0; h < kHeld; ++h) {
                        const uint32_t j = (c0 + h) * STEP + lane * V;
                        if (c0 + h < c1 && j < p.vocab && (lane & 7) == 0) {
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(next_p + j));
                            asm volatile("prefetch.global.L2 [%0];" ::"l"(next_q + j));
                        }
                    }
                }
                if (greedy) {
                    float top = -INFINITY;
                    int32_t id = -1;
#pragma unroll
                    for (uint32_t h = 0; h < kHeld; ++h)
#pragma unroll
                        for (int i = 0; i < (int)V; ++i)
                            if (ep[h][i] > top) top = ep[h][i], id = at(c0 + h) + i;      // (rising ids: ties stay with the lower)
                    best = rank_key(top, (uint32_t)id);
                } else {
                    auto masses = [&](float (&v)[HELD ? kHeld : 1][V], WarpSum& s) {
                        float m = -INFINITY;
#pragma unroll
                        for (uint32_t h = 0; h < kHeld; ++h)
#pragma unroll
                            for (int i = 0; i < (int)V; ++i) m = fmaxf(m, v[h][i]);
#pragma unroll
                        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                        const float base = m == -INFINITY ? 0.0f : m;
                        Pair sum{0.0f, 0.0f};
#pragma unroll
                        for (uint32_t h = 0; h < kHeld; ++h) {
                            float t = 0.0f;
                            if (m == INFINITY) {
#pragma unroll
                                for (int i = 0; i < (int)V; ++i) v[h][i] = v[h][i] == m ? 1.0f : 0.0f;
                            } else {
#pragma unroll
                                for (int i = 0; i < (int)V; ++i) v[h][i] = exp2_fast((v[h][i] - base) * it);
                            }
#pragma unroll
                            for (int i = 0; i < (int)V; ++i) t += v[h][i];
                            sum = plus(sum, {t, 0.0f});
                        }
                        s = {m, lanes_sum(sum)};
                    };
                    masses(ep, sp);
                    if (with_q) masses(eq, sq);
                }
            }
        } else {
            for (uint32_t c = c0; c < c1; ++c) {
                const int32_t j = at(c);
                const bool f = fits(j, vocab);
                float x[V], y[V];
                load(prow, j, vocab, f, x);
                if (with_q) load(qrow, j, vocab, f && q_alike, y);
                if (greedy) {
#pragma unroll
                    for (int i = 0; i < (int)V; ++i) {
                        const uint64_t k = rank_key(x[i], (uint32_t)(j + i));
                        best = k > best ? k : best;
                    }
                    continue;
                }
                auto add = [&](WarpSum& s, const float (&v)[V]) {
                    float m = v[0];
#pragma unroll
                    for (int i = 1; i < (int)V; ++i) m = fmaxf(m, v[i]);
#pragma unroll
                    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                    if (m == -INFINITY) return;                          // (one maximum for the warp)
                    if (m > s.m) {
                        const float f = s.m == -INFINITY ? 0.0f : mass(s.m, m, it);
                        s.s = {s.s.h * f, s.s.l * f};
                        s.m = m;
                    }
                    float t = 0.0f;
#pragma unroll
                    for (int i = 0; i < (int)V; ++i) t += mass(v[i], s.m, it);
                    s.s = plus(s.s, {t, 0.0f});
                };
                add(sp, x);
                if (with_q) add(sq, y);
            }
            if (!greedy) sp.s = lanes_sum(sp.s), sq.s = lanes_sum(sq.s);
        }
        if (greedy) {
#pragma unroll
            for (int o = 16; o; o >>= 1) {
                const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
                best = k > best ? k : best;
            }
        }
        if (p.stats == nullptr) {
            if (lane == 0) wp[warp] = sp, wq[warp] = sq, wbest[warp] = best;
            __syncthreads();
            if (warp == 0) {                                                 // the CTA's, told to all CTAs
                Exchange e;
                e.p = join_lanes(wp[lane & (kVWarps - 1)], kVWarps / 2, it);
                e.q = join_lanes(wq[lane & (kVWarps - 1)], kVWarps / 2, it);
                e.best = wbest[lane & (kVWarps - 1)];
#pragma unroll
                for (int o = kVWarps / 2; o; o >>= 1) {
                    const uint64_t k = __shfl_xor_sync(0xffffffffu, e.best, o);
                    e.best = k > e.best ? k : e.best;
                }
                e.total = {0.0f, 0.0f};
                if (lane < ranks) *cluster.map_shared_rank(&slots[turn][rank], lane) = e;
            }
            cluster.sync();
        }
        if (warp == 0) {
            if (p.stats != nullptr) {
                if (lane == 0) row = row_of[cur], s_ip = ip_of[cur];
            } else {
                WarpSum P{-INFINITY, {0.0f, 0.0f}}, Q = P;
                best = 0;
                if (lane < ranks) P = slots[turn][lane].p, Q = slots[turn][lane].q, best = slots[turn][lane].best;
                join_row(P, Q, best, with_q, row, s_ip);
                // the children's masses
                for (uint32_t c = lane; c < (uint32_t)n && !greedy; c += 32)
                    if (c > cur && parent[c] == (int32_t)cur) child_masses(c, prow, qrow, row);
            }
            if (lane == 0) s_child = cur + 1, s_gone = 0, s_a = 0.0, s_z = 1.0;
        }
        if (p.stats == nullptr) turn ^= 1;
        __syncthreads();
        const float pm = row.pm, qm = row.qm;
        best = row.best;
        bool held = p.stats == nullptr;                                  // (with statistics the rows are read where they are needed)
        float fp = mass(sp.m, pm, it), fq = mass(sq.m, qm, it);          // the warp's masses -> the row's

        // The residual, in units of p's masses: without a refusal its terms are those masses.  Step h of the share, at logit j.
        auto residual = [&](uint32_t h, int32_t j, float a, uint32_t ngone, float (&w)[V]) {
            const float k = a * row.q_over_p;
            if constexpr (HELD) {
                const float kq = k * fq;
                if (a != 0.0f) {
#pragma unroll
                    for (int i = 0; i < (int)V; ++i) w[i] = fmaxf(fmaf(-eq[h][i], kq, ep[h][i] * fp), 0.0f);
                } else {
#pragma unroll
                    for (int i = 0; i < (int)V; ++i) w[i] = ep[h][i] * fp;
                }
            } else {
                float x[V], y[V];
                const bool f = fits(j, vocab);
                load(prow, j, vocab, f, x);
                if (a != 0.0f) load(qrow, j, vocab, f && q_alike, y);
#pragma unroll
                for (int i = 0; i < (int)V; ++i) {
                    w[i] = mass(x[i], pm, it);
                    if (a != 0.0f && qm != -INFINITY) w[i] = fmaxf(fmaf(-mass(y[i], qm, it), k, w[i]), 0.0f);
                }
            }
            for (uint32_t g = 0; g < ngone; ++g) {
                const int32_t d = (int32_t)gone[g] - j;
#pragma unroll
                for (int i = 0; i < (int)V; ++i)
                    if (d == i) w[i] = 0.0f;
            }
        };
        // Its sum over the vocabulary; every warp's share stays in wtot, every CTA's in the slots.
        uint32_t last_turn = 0;
        auto residual_pass = [&](float a, uint32_t ngone) -> Pair {
            if (HELD && !held) {
                held = true;
                hold();
#pragma unroll
                for (uint32_t h = 0; h < (HELD ? kHeld : 1); ++h)
#pragma unroll
                    for (int i = 0; i < (int)V; ++i) {
                        ep[h][i] = mass(ep[h][i], pm, it);
                        if (with_q) eq[h][i] = mass(eq[h][i], qm, it);
                    }
                fp = fq = 1.0f;
            }
            Pair sum{0.0f, 0.0f};
            auto step = [&](uint32_t h) {
                float w[V], t = 0.0f;
                residual(h, at(c0 + h), a, ngone, w);
#pragma unroll
                for (int i = 0; i < (int)V; ++i) t += w[i];
                sum = plus(sum, {t, 0.0f});
            };
            if constexpr (HELD) {
#pragma unroll
                for (uint32_t h = 0; h < kHeld; ++h) step(h);
            } else {
                for (uint32_t h = 0; h < c1 - c0; ++h) step(h);
            }
            sum = lanes_sum(sum);
            __syncthreads();                                             // wtot of the pass before is read
            if (lane == 0) wtot[warp] = sum;
            __syncthreads();
            if (warp == 0) {
                const Pair t = lanes_sum(wtot[lane & (kVWarps - 1)], kVWarps / 2);
                if (lane < ranks) cluster.map_shared_rank(&slots[turn][rank], lane)->total = t;
            }
            cluster.sync();
            const Pair t = lanes_sum(lane < ranks ? slots[turn][lane].total : Pair{0.0f, 0.0f}, kMaxCluster / 2);      // (lanes 0..15)
            last_turn = turn;
            turn ^= 1;
            return {__shfl_sync(0xffffffffu, t.h, 0), __shfl_sync(0xffffffffu, t.l, 0)};
        };

        // ---- the children, one after the other
        constexpr uint32_t kFinish = 0, kAccept = 1, kRefused = 2;
        bool passed = false;                                             // wtot holds the residual of (s_a, 0 gone)
        Pair last_sum{0.0f, 0.0f};
        uint32_t action;
        for (;;) {
            if (tid == 0) {
                uint32_t c = s_child, act = kFinish;
                for (; c < (uint32_t)n; ++c) {
                    if (parent[c] != (int32_t)cur || (uint32_t)token[c] >= p.vocab) continue;
                    const double u = uni[c];
                    if (greedy) {
                        if (best && (uint32_t)token[c] == ~(uint32_t)best) { act = kAccept; break; }
                    } else if (sampled) {
                        // u q Z < max(p - a q, 0), times the sum of p's masses
                        const double q = child_q[c] * row.q_over_p;
                        if (u * q * s_z < fmax(child_p[c] - s_a * q, 0.0)) { act = kAccept; break; }
                        s_a += s_z;
                        act = kRefused;
                        break;
                    } else {
                        bool before = false;
                        for (uint32_t g = 0; g < s_gone; ++g) before |= gone[g] == (uint32_t)token[c];
                        if (before) continue;
                        if (u * s_z < child_p[c] * s_ip) { act = kAccept; break; }
                        s_z -= child_p[c] * s_ip;
                        gone[s_gone++] = token[c];
                    }
                }
                s_action = act;
                s_child = c;
            }
            __syncthreads();
            action = s_action;
            if (action != kRefused) break;
            last_sum = residual_pass((float)s_a, 0);
            passed = true;
            __syncthreads();
            if (tid == 0) s_z = value(last_sum) * s_ip, s_child += 1;
            __syncthreads();
        }
        if (action == kAccept) {
            cur = s_child;
            if (rank == 0 && tid == 0) p.path[first + count] = (int32_t)cur;
            ++count;
            __syncthreads();
            continue;
        }

        // ---- the last token
        if (rank == 0 && tid == 0) p.path_len[b] = (int32_t)count;
        if (greedy) {
            if (rank == 0 && tid == 0) p.next_token[b] = best ? (int32_t)~(uint32_t)best : -1;
            break;
        }
        float a = (float)s_a;
        uint32_t ngone = s_gone;
        if (!passed) last_sum = residual_pass(a, ngone);
        Pair z = last_sum;
        if (!(z.h > 0.0f) && (a != 0.0f || ngone)) a = 0.0f, ngone = 0, z = residual_pass(0.0f, 0);   // nothing is left of p: p itself
        if (!(z.h > 0.0f)) {
            if (rank == 0 && tid == 0) p.next_token[b] = -1;             // the row is empty
            break;
        }
        // The smallest j whose prefix exceeds u z: the CTA, the warp, the lane, the entry.  (By rounding, or for a uniform of 1
        // or more, there may be none: then the last entry with mass.)
        if (warp == 0) {
            auto find = [&](const Pair share, const Pair before, const Pair border, Pair& base) -> uint32_t {
                const Pair incl = plus(before, lanes_prefix(share, lane));
                const uint32_t hits = __ballot_sync(0xffffffffu, above(incl, border)), some = __ballot_sync(0xffffffffu, share.h > 0.0f);
                const uint32_t who = hits & some ? __ffs(hits & some) - 1 : some ? 31 - __clz(some) : 0;
                base = {__shfl_sync(0xffffffffu, incl.h, who ? who - 1 : 0), __shfl_sync(0xffffffffu, incl.l, who ? who - 1 : 0)};
                if (who == 0) base = before;
                return who;
            };
            const Pair none{0.0f, 0.0f}, border = pair_of((double)uni[0] * value(z));
            Pair base;
            const uint32_t owner = find(lane < ranks ? slots[last_turn][lane].total : none, none, border, base);
            uint32_t who = kNoToken;
            if (owner == rank) who = find(lane < kVWarps ? wtot[lane] : none, base, border, base);
            if (lane == 0) s_who = who, s_base = base, s_border = border;
        }
        __syncthreads();
        if (s_who == warp) {
            Pair base = s_base;
            const Pair border = s_border;
            uint32_t found = kNoToken, last = kNoToken;
            auto scan = [&](uint32_t h) {
                const int32_t j = at(c0 + h);
                float w[V], part[V], t = 0.0f;
                residual(h, j, a, ngone, w);
                uint32_t mine = kNoToken, end = kNoToken;
#pragma unroll
                for (int i = 0; i < (int)V; ++i) {
                    t += w[i];
                    part[i] = t;
                    if (w[i] > 0.0f) end = (uint32_t)(j + i);
                }
                const Pair incl = plus(base, lanes_prefix({t, 0.0f}, lane));
                Pair before = {__shfl_up_sync(0xffffffffu, incl.h, 1), __shfl_up_sync(0xffffffffu, incl.l, 1)};
                if (lane == 0) before = base;
#pragma unroll
                for (int i = 0; i < (int)V; ++i)
                    if (mine == kNoToken && w[i] > 0.0f && above(plus(before, {part[i], 0.0f}), border)) mine = (uint32_t)(j + i);
                const uint32_t hits = __ballot_sync(0xffffffffu, mine != kNoToken), some = __ballot_sync(0xffffffffu, end != kNoToken);
                if (hits && found == kNoToken) found = __shfl_sync(0xffffffffu, mine, __ffs(hits) - 1);
                if (some) last = __shfl_sync(0xffffffffu, end, 31 - __clz(some));
                base = {__shfl_sync(0xffffffffu, incl.h, 31), __shfl_sync(0xffffffffu, incl.l, 31)};
            };
            if constexpr (HELD) {
#pragma unroll
                for (uint32_t h = 0; h < kHeld; ++h) scan(h);
            } else {
                for (uint32_t h = 0; h < c1 - c0 && found == kNoToken; ++h) scan(h);
            }
            if (lane == 0) p.next_token[b] = (int32_t)(found != kNoToken ? found : last);
        }
        break;
    }
    cluster.sync();                                                      // nobody leaves while others may still write its slots
}

// (max, sum) and the best candidate of every row that the walk may visit: one CTA per split of a row.
constexpr uint32_t kStatThreads = 256, kMaxSplits = 32;
// When the statistics come first.  They cost the rows of nodes that the walk never visits, and save it a pass over a row per
// visited one.  Without and with them, us on a B200, means of six inputs that get differently far:
//   rows       chains of 5, f32: 1 over 2048 (10 rows) 54 and 29, 64 over 2048 (640) 66 and 34, 64 over 8192 68 and 33, 1 over
//              32000 56 and 31; trees of 24 over 32000, bf16: 16 (768 rows) 73 and 63; trees of 64 over 2048, bf16: 64 (8192
//              rows, of which few are visited) 77 and 110
//   bytes      trees of 24 over 100003, bf16: 8 (77 MB) 89 and 77, 10 (96 MB) 58 and 67, 16 (154 MB) 80 and 109; a chain's rows are
//              more likely to be visited: 9 of 5 over 248320, f32 (89 MB) 94 and 77, 9 of 8 (143 MB) 147 and 107
// With one node there is nothing to walk.
constexpr uint64_t kMaxStatRows = 2048, kTreeBytes = 80ull << 20, kChainBytes = 144ull << 20;

template <typename T>
__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const __grid_constant__ VerifyParams p) {
    constexpr uint32_t V = kLane<T>, STEP = kStep<T>, WARPS = kStatThreads / 32;
    __shared__ WarpSum ws[WARPS];
    __shared__ uint64_t wbest[WARPS];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t split = blockIdx.x % p.splits, id = blockIdx.x / p.splits, rows = p.batch * p.nodes;
    const bool draft = id >= rows;
    const uint32_t at_row = draft ? id - rows : id, b = at_row / p.nodes, node = at_row - b * p.nodes;
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const int32_t n = p.node_counts ? min(p.node_counts[b], (int32_t)p.nodes) : (int32_t)p.nodes;
    if ((int32_t)node >= n) return;
    const float tau = p.temperature ? p.temperature[b] : 1.0f;
    const bool greedy = !(tau >= 1e-20f);
    const float it = greedy ? 1.0f : per_tau(tau);
    if (draft) {                                                         // read for the children of a node, if it has any
        bool inner = false;
        for (uint32_t c = node + 1; c < (uint32_t)n && !inner; ++c) inner = (p.parents ? p.parents[(uint64_t)b * p.nodes + c] : (int32_t)c - 1) == (int32_t)node;
        if (greedy || !inner) return;
    }
    const T* row = draft ? static_cast<const T*>(p.draft) + b * p.draft_batch + node * p.draft_node
                         : static_cast<const T*>(p.target) + b * p.target_batch + node * p.target_node;
    const int32_t vocab = (int32_t)p.vocab, shift = (int32_t)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const uint32_t steps = (p.vocab + shift + STEP - 1) / STEP, all = p.splits * WARPS, per = (steps + all - 1) / all;
    const uint32_t me = split * WARPS + warp, c0 = min(me * per, steps), c1 = min(c0 + per, steps);
    WarpSum s{-INFINITY, {0.0f, 0.0f}};
    float top = -INFINITY;
    int32_t top_id = -1;
    constexpr uint32_t kAtATime = 32 / V;
    for (uint32_t c = c0; c < c1; c += kAtATime) {
        uint4 raw[kAtATime];
        float x[kAtATime][V];
#pragma unroll
        for (uint32_t h = 0; h < kAtATime; ++h) {
            const int32_t j = (int32_t)((c + h) * STEP + lane * V) - shift, end = c + h < c1 ? vocab : 0;
            fetch(row, j, j >= 0 && j + (int32_t)V <= end, raw[h]);
        }
        float m = -INFINITY;
#pragma unroll
        for (uint32_t h = 0; h < kAtATime; ++h) {
            const int32_t j = (int32_t)((c + h) * STEP + lane * V) - shift, end = c + h < c1 ? vocab : 0;
            read(row, j, end, j >= 0 && j + (int32_t)V <= end, raw[h], x[h]);
#pragma unroll
            for (int i = 0; i < (int)V; ++i) {
                m = fmaxf(m, x[h][i]);
                if (x[h][i] > top) top = x[h][i], top_id = j + i;
            }
        }
        if (greedy) continue;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (m > s.m) {
            const float f = s.m == -INFINITY ? 0.0f : mass(s.m, m, it);
            s = {m, {s.s.h * f, s.s.l * f}};
        }
#pragma unroll
        for (uint32_t h = 0; h < kAtATime; ++h) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < (int)V; ++i) t += mass(x[h][i], s.m, it);
            s.s = plus(s.s, {t, 0.0f});
        }
    }
    s.s = lanes_sum(s.s);
    uint64_t best = rank_key(top, (uint32_t)top_id);
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
        best = k > best ? k : best;
    }
    if (lane == 0) ws[warp] = s, wbest[warp] = best;
    __syncthreads();
    if (warp == 0) {
        const WarpSum all_s = join_lanes(ws[lane & (WARPS - 1)], WARPS / 2, it);
        best = wbest[lane & (WARPS - 1)];
#pragma unroll
        for (int o = WARPS / 2; o; o >>= 1) {
            const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
            best = k > best ? k : best;
        }
        if (lane == 0) p.stats[(uint64_t)id * p.splits + split] = {all_s, best};
    }
}

// CTAs per sequence, and whether a warp's share of a row stays in its registers.
struct WalkShape {
    uint32_t ranks;
    bool held;
};
template <typename T>
WalkShape walk_shape(uint32_t batch, uint32_t vocab, int sm_count) {
    // as many CTAs per sequence as keep every SM at one CTA, and at least 2048 logits for each of them
    uint32_t ranks = kMaxCluster;
    while (ranks > 1 && ((uint64_t)batch * ranks > (uint64_t)sm_count || vocab / ranks < 2048)) ranks >>= 1;
    const uint64_t steps = ((uint64_t)vocab + kLane<T> - 1 + kStep<T> - 1) / kStep<T>;      // (a row may start behind a 16-byte border)
    return {ranks, (steps + ranks * kVWarps - 1) / (ranks * kVWarps) <= kHeldSteps<T>};
}

// Splits of a row that the statistics are taken in; 0: the walk takes them itself.  Only the form that holds its share works with
// them; beyond it the time goes up in a step: chains of 5 over 248320 logits, f32, 9 sequences 78 us and 10 (8 CTAs each) 92; bf16,
// 18 sequences 92 us and 19 (4 CTAs each) 119.
uint32_t stat_splits(const lq4_verify_args& a, int sm_count) {
    const bool f32 = a.dtype == LQ4_DTYPE_F32;
    const uint64_t rows = (uint64_t)a.batch * a.nodes * (a.draft_logits ? 2 : 1), row = (uint64_t)a.vocab * (f32 ? 4 : 2);
    // (a division: rows * row may pass 64 bits where rows are broadcast)
    if (a.nodes < 2 || rows > kMaxStatRows || rows > (a.parents ? kTreeBytes : kChainBytes) / row) return 0;
    if (!(f32 ? walk_shape<float>(a.batch, a.vocab, sm_count) : walk_shape<uint16_t>(a.batch, a.vocab, sm_count)).held) return 0;
    uint64_t splits = (4ull * sm_count + rows - 1) / rows;
    return splits > kMaxSplits ? kMaxSplits : splits < 1 ? 1 : (uint32_t)splits;
}

template <typename T>
cudaError_t run(VerifyParams p, int sm_count, int use_pdl, cudaStream_t s, int* launches) {
    const uint32_t batch = p.batch;
    const WalkShape shape = walk_shape<T>(batch, p.vocab, sm_count);
    const uint32_t ranks = shape.ranks;
    const bool held = shape.held;
    auto fn = held ? verify_kernel<T, true> : verify_kernel<T, false>;
    static DeviceOnce once_of[2];
    DeviceOnce& once = once_of[held];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    if (once.needs(dev)) {
        if ((e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
        once.mark(dev);
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(batch * ranks);
    cfg.blockDim = dim3(kVThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl ? 2 : 1;
    *launches = 1;
    if (p.stats) {
        cudaLaunchConfig_t first = cfg;
        first.gridDim = dim3(p.batch * p.nodes * (p.draft ? 2 : 1) * p.splits);
        first.blockDim = dim3(kStatThreads);
        first.attrs = attr + 1;
        first.numAttrs = use_pdl ? 1 : 0;
        if ((e = cudaLaunchKernelEx(&first, verify_stats_kernel<T>, p)) != cudaSuccess) return e;
        *launches = 2;
    }
    return cudaLaunchKernelEx(&cfg, fn, p);
}

}  // namespace

size_t verify_workspace_bytes(const lq4_verify_args& a, int sm_count) {
    return (size_t)a.batch * a.nodes * (a.draft_logits ? 2 : 1) * stat_splits(a, sm_count) * sizeof(Stat);      // (64 KB at most)
}

cudaError_t launch_verify_draft(const lq4_verify_args& a, void* workspace, int32_t* status, int sm_count, int use_pdl, cudaStream_t s, int* launches) {
    VerifyParams p{};
    p.target = a.target_logits;
    p.draft = a.draft_logits;
    p.target_batch = a.target_batch, p.target_node = a.target_node;
    p.draft_batch = a.draft_batch, p.draft_node = a.draft_node;
    p.nodes = a.nodes;
    p.vocab = a.vocab;
    p.tokens = a.tokens;
    p.parents = a.parents;
    p.node_counts = a.node_counts;
    p.uniforms = a.uniforms;
    p.temperature = a.temperature;
    p.path = a.path;
    p.path_len = a.path_len;
    p.next_token = a.next_token;
    p.status = status;
    p.batch = a.batch;
    p.splits = stat_splits(a, sm_count);
    p.stats = static_cast<Stat*>(workspace);
    return a.dtype == LQ4_DTYPE_F32 ? run<float>(p, sm_count, use_pdl, s, launches) : run<uint16_t>(p, sm_count, use_pdl, s, launches);
}

}  // namespace lq4
