// lq4_tree_attention for bf16 activations and many rows per kv head (a large tree), on the 5th-generation tensor cores.
//
// With R query rows on a key/value head there are R flops per byte of cache, so beyond some 50 rows the HBM
// stream is no longer the bound and mma.sync (552 TFLOP/s measured here) is; tcgen05.mma has three times that.  The work
// is cut exactly as in lq4_attend.cu (tiles of 64 keys, an even share of all tiles per persistent CTA, partials
// joined by attend_join_kernel); only what happens inside a piece differs.  An item has 128 rows (the lanes of
// tensor memory).  Per tile:
//
//   S[128, 64] = Q K^T     A = Q, B = K, both K-major in shared memory with the 128-byte swizzle
//   P = exp2(S - max)      one thread per row: no shuffles; bf16 pairs back to tensor memory
//   O[128, D] += P V       A = P from tensor memory, B = V as it lies in the cache (keys outer: MN-major)
//
// The exponentials cost as much as the MMAs, so up to D = 128 a CTA runs two streams, each with its own S, P and O: while
// one is exponentiated the tensor cores work on the other.  With up to 128 rows per item the streams take the
// key tiles in turn and their O meet at the end of a piece; with more the item has 256 rows and each stream has 128 of
// them, so that a tile of keys in shared memory serves both.  (At D = 256 tensor memory holds one O.)
//
//   warps 0..4N-1   softmax, four warps per stream: a thread reads its row of S, hands the buffer back at once (the
//                   stream's next S is computed while this one is exponentiated), writes P, and drains O at the end
//   next warp       tensor memory allocation; one lane issues all MMAs
//   last 4 warps    loaders: cp.async of K and V rows, each looked up through the page table, into one ring of slots
//                   (K, V, K, V, ...); they run ahead over the borders of pieces
//
// The running maximum only moves when it has grown by more than 2^8 (the final division takes the same base out
// again), so O is rescaled in tensor memory a few times per sequence instead of per tile.
#include "lq4_attend_dev.cuh"

#include <atomic>
#include <type_traits>

namespace lq4 {

namespace {

constexpr int kTcRows = 128, kLoaders = 128;
constexpr float kLazy = 8.0f;                  // how far (log2) a row's maximum may outgrow its base

__device__ __forceinline__ void tmem_alloc(uint32_t* smem_dst, uint32_t ncols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(smem_dst)), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish() { asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// D[tmem] (+)= A[smem] B[smem]; bf16, f32 accumulation; one thread issues.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// The same with A in tensor memory (a lane per row, two consecutive k per column).
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_lane() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
template <int AT, int N>
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[N]) {      // 32 columns -> r[AT .. AT + 32)
    uint32_t u[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]),
          "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]),
          "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
        : "r"(taddr)
        : "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) r[AT + i] = __uint_as_float(u[i]);
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&u)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(u[0]),
        "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]), "r"(u[11]), "r"(u[12]),
        "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]), "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]),
        "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]), "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory matrix descriptors, 128-byte swizzle (version 1 at bits 46-47, swizzle mode 2 at 61-63); a tile is
// [rows][128 bytes], 8 rows = 1024 bytes.
//   K-major (Q, K): the 128 bytes are 64 channels of k; stride offset = 8 rows, leading offset unused.
//   MN-major (V): the 128 bytes are 64 columns of O and the rows are k; leading offset = from 64 columns to the
//   next 64, stride offset = 8 rows of k.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16 with f32 accumulators (bit 4), bf16 A and B (1 at bits 7 and 10), B MN-major (bit 16), N >> 3 at 17, M >> 4 at 24.
__host__ __device__ constexpr uint32_t instr_desc(uint32_t n, uint32_t b_mn) {
    return 1u << 4 | 1u << 7 | 1u << 10 | b_mn << 16 | (n >> 3) << 17 | (uint32_t)(kTcRows >> 4) << 24;
}

// Byte offset of 16-byte chunk c (of D / 8) of row r in a tile stored as [D / 64][rows][128 bytes], swizzled.
__device__ __forceinline__ uint32_t swz(uint32_t rows, uint32_t r, uint32_t c) {
    return (c >> 3) * (rows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// NS streams; WIDE: items of 256 rows.
template <int D, int NS, bool WIDE>
struct TcShape {
    static constexpr int kSoftmax = 128 * NS, kThreads = kSoftmax + 32 + kLoaders, kItemRows = WIDE ? 256 : 128;
    static constexpr uint32_t kSlot = kKeys * D * 2, kQ = kTcRows * D * 2 * (WIDE ? 2 : 1);
    static constexpr uint32_t kFit = ((uint32_t)kMaxSmem - kQ - 5120) / kSlot, kSlots = kFit > 12 ? 12 : kFit;
    static constexpr uint32_t kOffs = kSlots * kSlot + kQ, kValid = kOffs + 2 * kKeys * 8, kAnc = kValid + 16 * 8, kMeet = kAnc + kMaxNodes * 8;
    static constexpr uint32_t kBars = kMeet + kTcRows * 8, kCtl = kBars + 48 * 8, kSmem = kCtl + 256 + 1024;      // + alignment slack
    static constexpr uint32_t kColO = 0, kColS = NS * D, kColP = kColS + NS * 64, kCols = kColP + NS * 32 <= 256 ? 256 : 512;
    static_assert(kSlots >= 4 && kSmem <= (uint32_t)kMaxSmem && kColP + NS * 32 <= 512, "shared or tensor memory");
    static_assert(NS == 2 || !WIDE, "256 rows take two streams");
    static_assert(kTcRows * 32 * 4 <= kQ, "the streams meet in Q's place");
};

template <int D, int NS, bool WIDE>
__global__ void __launch_bounds__((TcShape<D, NS, WIDE>::kThreads), 1) attend_tc_kernel(const __grid_constant__ AttendParams p) {
    using S = TcShape<D, NS, WIDE>;
    constexpr int CPR = D / 8, kSoftmax = S::kSoftmax, kMmaWarp = kSoftmax / 32;
    constexpr uint32_t SL = S::kSlots;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);      // swizzle atoms are 1024 bytes
    uint64_t* offs = reinterpret_cast<uint64_t*>(smem + S::kOffs);      // [2][64] element offset of a key's row
    volatile uint64_t* valid = reinterpret_cast<uint64_t*>(smem + S::kValid);    // [16] which of a tile's keys there are
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + S::kAnc);        // [nodes] of the piece's sequence
    float2* meet = reinterpret_cast<float2*>(smem + S::kMeet);          // [128] (max, sum) of stream 1's rows
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* ctl = reinterpret_cast<uint64_t*>(smem + S::kCtl);        // 0, 1: cursor; 2..14: warp sums; 16: tensor memory; 18..25: fixes
    uint64_t *full = bars, *empty = bars + SL, *s_full = bars + 2 * SL, *s_free = s_full + 2, *p_full = s_full + 4, *o_done = s_full + 6;
    uint64_t *q_full = s_full + 8, *drained = s_full + 9;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 16);
    volatile uint32_t* fixes = reinterpret_cast<uint32_t*>(ctl + 18);    // [16] a tile's V held inf or NaN
    const uint32_t sbase = smem_u32(smem), qbase = sbase + SL * S::kSlot;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    pdl_wait_prior_grids();
    const Range range = cta_range<S::kThreads>(p, ctl, ctl + 2);
    if (range.begin >= range.end) return;
    if (warp == kMmaWarp) {
        tmem_alloc(tmem_slot, S::kCols);
        tmem_relinquish();
        if (lane == 0) {
            for (uint32_t i = 0; i < SL; ++i) {
                mbar_init(full + i, kLoaders / 32);                      // one arrival per warp
                mbar_init(empty + i, 1);
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(s_full + i, 1);
                mbar_init(s_free + i, 4);
                mbar_init(p_full + i, 4);
                mbar_init(o_done + i, 1);
            }
            mbar_init(q_full, kSoftmax / 32);
            mbar_init(drained, 1);
            mbar_fence_init();
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    // Only now may the next kernel's CTAs come: they allocate tensor memory too, and wait for this grid.
    pdl_launch_dependents();

    uint64_t u = range.begin, seq_first = range.seq_first;
    const uint64_t u_end = range.end;
    uint32_t b = range.seq;
    uint32_t tile = 0;                                                   // tiles of this CTA before the current piece
    // Once a wait has run out the CTA goes on without waiting, so that its barriers still match; the results are
    // rubbish then, and reported.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity);
    };
    auto wait_group = [&](uint32_t g) { wait(full + g % SL, (g / SL) & 1); };      // group 2n: K of tile n, 2n + 1: V

    if (tid < (uint32_t)kSoftmax) {
        // ---- softmax: thread = row ---------------------------------------------------------------------
        const uint32_t str = tid >> 7, r = tid & 127;
        const uint32_t lanes = tmem + ((warp & 3) << 21);                // this warp's 32 lanes, at bit 16
        const uint32_t col_o = lanes + S::kColO + str * D, col_s = lanes + S::kColS + str * 64, col_p = lanes + S::kColP + str * 32;
        const uint32_t rows = p.nodes * p.group;
        uint32_t used = 0;                                               // steps of this stream so far
        while (u < u_end) {
            const Piece x = next_piece(p, u, u_end, b, seq_first);
            if (x.sq.bad && tid == 0) atomicOr(p.status, kDevErrBadIndex);
            const uint32_t row = x.rt * S::kItemRows + (WIDE ? tid : r), t = row / p.group, g = row - t * p.group;
            const bool live = row < rows && (int32_t)t < x.sq.nodes;
            // Q: all MMAs that read the last one are done (o_done of its last step)
#pragma unroll 4
            for (uint32_t i = tid; i < S::kItemRows * CPR; i += kSoftmax) {
                const uint32_t qr = i / CPR, c = i % CPR, qrow = x.rt * S::kItemRows + qr, qt = qrow / p.group, qg = qrow - qt * p.group;
                uint32_t w[4] = {0, 0, 0, 0};
                if (qrow < rows && (int32_t)qt < x.sq.nodes && c * 8 < p.head_dim) {
                    const uint16_t* src = static_cast<const uint16_t*>(p.q) + b * p.q_batch + qt * p.q_node + (uint64_t)(x.h * p.group + qg) * p.q_head + c * 8;
                    if (p.q_vec) {
                        const uint4 v = *reinterpret_cast<const uint4*>(src);
                        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = src[2 * e] | (uint32_t)src[2 * e + 1] << 16;
                    }
                    if (p.q_sign != 1.0f) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(w[e] << 16) * p.q_sign, __uint_as_float(w[e] & 0xffff0000u) * p.q_sign);
                            w[e] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                    }
                }
                *reinterpret_cast<uint4*>(smem + SL * S::kSlot + (qr >> 7) * (kTcRows * D * 2) + swz(kTcRows, qr & 127, c)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (x.has_nodes && tid < p.nodes) {
                bool bad = false;
                anc[tid] = node_path(p, b, tid, bad);
                if (bad && (int32_t)tid < x.sq.nodes) atomicOr(p.status, kDevErrBadIndex);
            }
            fence_async_smem();
            named_bar_sync(2, kSoftmax);                                 // (anc is read by other threads)
            if (lane == 0) mbar_arrive(q_full);

            float m = -INFINITY, l = 0.0f;                               // base (log2) and sum of this row
            bool first = true;
            for (uint32_t i = WIDE || NS == 1 ? 0 : str; i < x.n_tiles; i += WIDE || NS == 1 ? 1 : 2) {
                const uint32_t n = tile + i;
                // (V's slot cannot be filled again before this thread has handed over P; V's barrier covers `valid` and `fixes`)
                wait_group(2 * n + 1);
                wait(s_full + str, used & 1);
                __syncwarp();
                tc_fence_after();
                float s[64];
                tmem_ld32<0>(col_s, s);
                tmem_ld32<32>(col_s + 32, s);
                uint64_t see = valid[n & 15];
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_free + str);
                if (x.t0 + i + 1 == x.sq.tiles && t < p.nodes) see &= anc[t];
                if (see != ~0ull) {
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (!((see >> j) & 1)) s[j] = -INFINITY;
                }
                float top;
                {
                    float t4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
                    for (int j = 4; j < 64; ++j) t4[j & 3] = fmaxf(t4[j & 3], s[j]);
                    top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale_log2;
                }
                // P's buffer and O are free once the stream's MMA before has read and written them
                if (!first) wait(o_done + str, (used - 1) & 1);
                __syncwarp();
                tc_fence_after();
                if (first) {
                    m = top;
                } else {
                    const bool grow = top > m + kLazy;                   // (m -inf: at the first finite score)
                    if (__any_sync(0xffffffffu, grow)) {
                        const float f = grow ? exp2_fast(m - top) : 1.0f;
                        l *= f;
                        m = grow ? top : m;
#pragma unroll 1
                        for (int d = 0; d < D; d += 32) {
                            float o[32];
                            tmem_ld32<0>(col_o + d, o);
                            tmem_ld_wait();
                            uint32_t w[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * f);
                            tmem_st32(col_o + d, w);
                        }
                        tmem_st_wait();
                    }
                }
                const float base = m == -INFINITY ? 0.0f : m;
                float sum0 = 0.0f, sum1 = 0.0f;
                uint32_t w[32];
#pragma unroll
                for (int j = 0; j < 32; ++j) {
                    const float a = exp2_fast(fmaf(s[2 * j], p.scale_log2, -base)), c = exp2_fast(fmaf(s[2 * j + 1], p.scale_log2, -base));
                    sum0 += a;
                    sum1 += c;
                    const __nv_bfloat162 y = __floats2bfloat162_rn(a, c);
                    w[j] = *reinterpret_cast<const uint32_t*>(&y);
                }
                l += sum0 + sum1;
                tmem_st32(col_p, w);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + str);
                first = false;
                ++used;
            }
            if (!first) wait(o_done + str, (used - 1) & 1);
            __syncwarp();
            tc_fence_after();
            // ---- O of this piece: the result, or a partial.  Two streams over the keys: stream 1 hands its O to stream 0
            // through Q's place, 32 columns at a time (both have waited for all MMAs of their own that read Q; the
            // barrier below covers the other's).
            constexpr bool kMeets = NS == 2 && !WIDE;
            float f = 1.0f, f_other = 0.0f;
            if constexpr (kMeets) {
                if (str == 1) meet[r] = make_float2(m, l);
                named_bar_sync(2, kSoftmax);
                if (str == 0) {
                    const float2 e = meet[r];
                    const float top = fmaxf(m, e.x), safe = top == -INFINITY ? 0.0f : top;
                    f = exp2_fast(m - safe);
                    f_other = exp2_fast(e.x - safe);
                    l = l * f + e.y * f_other;
                    m = top;
                }
            }
            const bool whole = x.t0 == 0 && x.has_nodes;
            const uint64_t slot = ((uint64_t)2 * blockIdx.x + (x.t0 == 0 ? 1 : 0)) * S::kItemRows + (WIDE ? tid : r);
            const bool fix = x.has_nodes && fixes[(tile + x.n_tiles - 1) & 15];      // (the nodes' tile is a piece's last one)
            const float inv = 1.0f / l;
            if (!whole && live && (!kMeets || str == 0)) p.part_ml[slot] = make_float2(m, l);
            const uint64_t to = b * p.out_batch + t * p.out_node + (uint64_t)(x.h * p.group + g) * p.out_head;
            float* pass = reinterpret_cast<float*>(smem + SL * S::kSlot) + r;      // [columns][128]: lanes side by side
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
                float o[32];
                __syncwarp();
                if (kMeets && str == 1) {
                    if (first) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                    } else {
                        tmem_ld32<0>(col_o + d, o);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int e = 0; e < 32; ++e) pass[e * 128] = o[e];
                    named_bar_sync(3, 256);
                    named_bar_sync(4, 256);                              // stream 0 has it
                    continue;
                }
                tmem_ld32<0>(col_o + d, o);
                tmem_ld_wait();
                if constexpr (kMeets) {
                    named_bar_sync(3, 256);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = o[e] * f + (f_other == 0.0f ? 0.0f : pass[e * 128] * f_other);
                    named_bar_sync(4, 256);
                }
                if (!live) continue;
                if (fix) {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        if (d + e < (int)p.head_dim) o[e] += nonfinite_sum(p, x, anc[t], d + e);
                }
                if (!whole) {
                    float4* dst = reinterpret_cast<float4*>(p.part_o + slot * D + d);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                } else {
                    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + to + d;
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        if (d + e >= (int)p.head_dim) break;             // (a multiple of 8)
                        uint32_t w[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const __nv_bfloat162 y = __floats2bfloat162_rn(o[e + 2 * k] * inv, o[e + 2 * k + 1] * inv);
                            w[k] = *reinterpret_cast<const uint32_t*>(&y);
                        }
                        if (p.out_vec) {
                            *reinterpret_cast<uint4*>(out + e) = make_uint4(w[0], w[1], w[2], w[3]);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; ++k) out[e + k] = __ushort_as_bfloat16((unsigned short)(w[k >> 1] >> (16 * (k & 1))));
                        }
                    }
                }
            }
            __syncwarp();
            tc_fence_before();
            named_bar_sync(2, kSoftmax);                                 // everybody has read anc, meet and O
            tile += x.n_tiles;
            u += x.n_tiles;
        }
    } else if (warp == kMmaWarp) {
        // ---- MMA issue --------------------------------------------------------------------------------------
        // Steps v of a piece: NS streams in turn over the tiles; with 256 rows both streams take every tile.  The whole warp
        // walks through the steps with warp-uniform values (descriptors then live in uniform registers); one lane issues.
        const bool leader = elect_lane();
        auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
        const uint32_t tm = uniform(tmem), ring = uniform(sbase) >> 4, q0 = uniform(qbase) >> 4;
        const uint64_t kmajor = smem_desc(0, 16), mnmajor = smem_desc(0, kKeys * 128);
        // Everything an iteration looks up is kept running: the ring position of the next K and V group with its phase, and
        // the phases of the streams' barriers.
        struct Ring {
            uint32_t slot, phase;
            __device__ __forceinline__ void step() {                     // K to K or V to V: two groups on
                slot += 2;
                if (slot >= SL) slot -= SL, phase ^= 1;
            }
        } kr{0, 0}, vr{1, 0};
        uint32_t piece = 0, ph_s[NS], ph_p[NS], s_any = 0;
#pragma unroll
        for (int i = 0; i < NS; ++i) ph_s[i] = 1, ph_p[i] = 0;           // s_free: phase 1 of the step before the first
        auto scores = [&](auto stream) {                                 // next S of a stream, from K's ring position
            constexpr uint32_t str = decltype(stream)::value;
            constexpr bool new_k = !WIDE || str == 0, last_use = !WIDE || str == NS - 1;
            if (new_k) wait(full + kr.slot, kr.phase);
            if (s_any >> str & 1) wait(s_free + str, ph_s[str]);
            s_any |= 1u << str;
            ph_s[str] ^= 1;
            __syncwarp();
            tc_fence_after();
            const uint64_t k = kmajor + (ring + kr.slot * (S::kSlot >> 4)), q = kmajor + (q0 + (WIDE ? str * (kTcRows * D * 2 >> 4) : 0));
            const uint32_t d = tm + S::kColS + str * 64;
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                    mma_ss(d, q + ((ks >> 2) * (kTcRows * 128) + (ks & 3) * 32 >> 4), k + ((ks >> 2) * (kKeys * 128) + (ks & 3) * 32 >> 4), instr_desc(kKeys, 0), ks > 0);
                if (last_use) mma_commit(empty + kr.slot);
                mma_commit(s_full + str);
            }
            if (last_use) kr.step();
        };
        auto values = [&](auto stream, uint32_t accumulate) {            // O of a stream += its P times V at the ring position
            constexpr uint32_t str = decltype(stream)::value;
            constexpr bool new_v = !WIDE || str == 0, last_use = !WIDE || str == NS - 1;
            if (new_v) wait(full + vr.slot, vr.phase);
            wait(p_full + str, ph_p[str]);
            ph_p[str] ^= 1;
            __syncwarp();
            tc_fence_after();
            const uint64_t vt = mnmajor + (ring + vr.slot * (S::kSlot >> 4));
            const uint32_t o = tm + S::kColO + str * D, pr = tm + S::kColP + str * 32;
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < (int)kKeys / 16; ++ks) mma_ts(o, pr + ks * 8, vt + (ks * 2048 >> 4), instr_desc(D, 1), ks > 0 ? 1u : accumulate);
                if (last_use) mma_commit(empty + vr.slot);
                mma_commit(o_done + str);
            }
            if (last_use) vr.step();
        };
        constexpr std::integral_constant<uint32_t, 0> stream0{};
        constexpr std::integral_constant<uint32_t, NS - 1> stream1{};    // (stream 0 again where there is one)
        while (u < u_end) {
            const Piece x = next_piece(p, u, u_end, b, seq_first);
            const uint32_t tiles = uniform(x.n_tiles);
            wait(q_full, piece & 1);
            // rounds of NS steps; with 128 rows and two streams the last round may have one
            const uint32_t steps = WIDE ? 2 * tiles : tiles;
            scores(stream0);
            if (NS == 2 && steps > 1) scores(stream1);
            for (uint32_t v = 0; v < steps; v += NS) {
                if (v + NS < steps) scores(stream0);
                values(stream0, v > 0);
                if (NS == 2) {
                    if (v + NS + 1 < steps) scores(stream1);
                    if (v + 1 < steps) values(stream1, v > 0);
                }
            }
            ++piece;
            u += tiles;
        }
        if (leader) mma_commit(drained);                                 // tensor memory is freed behind the last MMA
        if (!mbar_wait(drained, 0)) ok = false;
        __syncwarp();
    } else {
        // ---- loaders ---------------------------------------------------------------------------------------
        // A group is handed on when it has landed, kLag groups behind the newest one; before a thread blocks on a slot
        // that is still in use it hands on all it has, oldest first, since the slot may only become free after them.
        constexpr uint32_t kLag = SL > 6 ? 4 : 2;
        const uint32_t lt = tid - (S::kThreads - kLoaders);
        uint32_t issued = 0, handed = 0;
        auto hand = [&](uint32_t upto) {
            if (handed >= upto) return;
            fence_async_smem();
            __syncwarp();
            for (; handed < upto; ++handed)
                if (lane == 0) mbar_arrive(full + handed % SL);
        };
        auto acquire = [&]() {
            if (issued < SL) return;
            uint64_t* bar = empty + issued % SL;
            const uint32_t parity = (issued / SL - 1) & 1;
            if (__any_sync(0xffffffffu, !ok || mbar_try_wait(bar, parity))) return;      // (what one lane has seen, all have)
            if (issued - handed > 3) cp_wait<3>(), hand(issued - 3);
            if (issued - handed > 2) cp_wait<2>(), hand(issued - 2);
            if (issued - handed > 1) cp_wait<1>(), hand(issued - 1);
            cp_wait<0>();
            hand(issued);
            wait(bar, parity);
            __syncwarp();
        };
        while (u < u_end) {
            const Piece x = next_piece(p, u, u_end, b, seq_first);
            int32_t page = lt < kKeys ? key_page(p, x, 0, lt) : -1;
            for (uint32_t i = 0; i < x.n_tiles; ++i, ++tile) {
                __syncwarp();
                if (lt < kKeys) {
                    const uint64_t at = key_offset(p, x, i, lt, page);
                    offs[(tile & 1) * kKeys + lt] = at;
                    __syncwarp();
                    const uint32_t bits = __ballot_sync(0xffffffffu, at != ~0ull);
                    if (lane == 0) reinterpret_cast<volatile uint32_t*>(valid + (tile & 15))[lt >> 5] = bits;
                    if (lt == 0) fixes[tile & 15] = 0;
                    page = key_page(p, x, i + 1, lt);
                }
                __syncwarp();
                named_bar_sync(1, kLoaders);
                const bool own = x.t0 + i + 1 == x.sq.tiles;
                auto load = [&](const uint16_t* base) {
                    acquire();
                    const uint32_t slot = sbase + (issued % SL) * S::kSlot;
#pragma unroll 8
                    for (uint32_t n = 0; n < kKeys * CPR / kLoaders; ++n) {
                        const uint32_t idx = n * kLoaders + lt, r = idx / CPR, c = idx % CPR;
                        const uint64_t at = offs[(tile & 1) * kKeys + r];
                        const bool here = at != ~0ull && c * 8 < p.head_dim;
                        cp_async16(slot + swz(kKeys, r, c), here ? base + at + c * 8 : p.k, here);
                    }
                    cp_commit();
                    ++issued;
                };
                load(own ? p.k : p.c.k);
                load(own ? p.v : p.c.v);
                if (own) {                                               // clear non-finite V of the nodes before it is used
                    cp_wait<0>();
                    bool odd = false;
                    for (uint32_t n = 0; n < kKeys * CPR / kLoaders; ++n) {
                        const uint32_t idx = n * kLoaders + lt;
                        odd |= clear_nonfinite(reinterpret_cast<uint4*>(smem + ((issued - 1) % SL) * S::kSlot + swz(kKeys, idx / CPR, idx % CPR)));
                    }
                    if (odd) fixes[tile & 15] = 1;
                    hand(issued);
                } else if (issued - handed > kLag) {
                    cp_wait<kLag>();
                    hand(issued - kLag);
                }
            }
            u += x.n_tiles;
        }
        cp_wait<0>();
        hand(issued);
    }
    if (!ok) atomicOr(p.status, kDevErrBarrierTimeout);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, S::kCols);
}

template <int D, int NS, bool WIDE>
cudaError_t run(AttendParams p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    using S = TcShape<D, NS, WIDE>;
    static DeviceOnce once;
    auto fn = attend_tc_kernel<D, NS, WIDE>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void*>(fn), S::kSmem, once);
    if (e != cudaSuccess) return e;
    p.grid = (uint32_t)sm_count;
    p.row_tiles = (p.nodes * p.group + S::kItemRows - 1) / S::kItemRows;
    if (!attend_workspace(p, ws, S::kItemRows, D)) return cudaSuccess;
    if ((e = attend_launch(fn, dim3(p.grid), S::kThreads, S::kSmem, use_pdl, s, p)) != cudaSuccess) return e;
    return launch_attend_join(p, S::kItemRows, D, true, ws, use_pdl, s);
}

}  // namespace

cudaError_t launch_attend_tc(const AttendParams& p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    const bool wide = p.nodes * p.group > (uint32_t)kTcRows;
    if (p.head_dim <= 64) return wide ? run<64, 2, true>(p, ws, sm_count, use_pdl, s) : run<64, 2, false>(p, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 128) return wide ? run<128, 2, true>(p, ws, sm_count, use_pdl, s) : run<128, 2, false>(p, ws, sm_count, use_pdl, s);
    return run<256, 1, false>(p, ws, sm_count, use_pdl, s);
}

}  // namespace lq4
