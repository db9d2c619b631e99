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
//   warps 0..3   softmax: a thread reads its row of S, hands the buffer back at once (the next S is computed
//                while this one is exponentiated), writes P, and at the end of a piece drains O
//   warp 4       tensor memory allocation; one lane issues all MMAs
//   warps 5..7   loaders: cp.async of K and V rows, each looked up through the page table, two stages; they run
//                ahead over the borders of pieces
//
// The running maximum only moves when it has grown by more than 2^8 (the final division takes the same base out
// again), so O is rescaled in tensor memory a few times per sequence instead of per tile.  Up to D = 128 a CTA
// takes half an SM (256 columns, 100 KB): one CTA's softmax runs beside the other's MMAs.
#include "lq4_attend_dev.cuh"

#include <atomic>

namespace lq4 {

namespace {

constexpr int kTcThreads = 256, kTcRows = 128, kSoftmax = 128, kLoaders = 96, kTcStages = 2;
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

template <int D>
struct TcShape {
    static constexpr uint32_t kTile = kKeys * D * 2, kStage = 2 * kTile, kQ = kTcRows * D * 2;
    static constexpr uint32_t kOffs = kTcStages * kStage + kQ, kValid = kOffs + 2 * kKeys * 8, kAnc = kValid + 8 * 8;
    static constexpr uint32_t kBars = kAnc + 2 * kMaxNodes * 8, kCtl = kBars + 16 * 8, kSmem = kCtl + 192 + 1024;      // + alignment slack
    static constexpr uint32_t kColS = D, kColP = D + 64, kCols = D + 96 <= 256 ? 256 : 512;
    static constexpr int kPerSm = D <= 128 ? 2 : 1;
    static_assert(kSmem <= (uint32_t)kMaxSmem, "shared memory");
};

template <int D>
__global__ void __launch_bounds__(kTcThreads, TcShape<D>::kPerSm) attend_tc_kernel(const __grid_constant__ AttendParams p) {
    using S = TcShape<D>;
    constexpr int CPR = D / 8;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);      // swizzle atoms are 1024 bytes
    uint64_t* offs = reinterpret_cast<uint64_t*>(smem + S::kOffs);      // [2][64] element offset of a key's row
    volatile uint64_t* valid = reinterpret_cast<uint64_t*>(smem + S::kValid);    // [8] which of a tile's keys there are
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + S::kAnc);        // [nodes] (the piece's)
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* ctl = reinterpret_cast<uint64_t*>(smem + S::kCtl);        // 0, 1: cursor; 2..10: warp sums; 12: tensor memory; 16..19: fixes
    uint64_t *k_full = bars, *k_empty = bars + 2, *v_full = bars + 4, *v_empty = bars + 6;      // two stages each
    uint64_t *s_full = bars + 8, *s_free = bars + 9, *p_full = bars + 10, *o_done = bars + 11, *q_full = bars + 12, *drained = bars + 13;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 12);
    volatile uint32_t* fixes = reinterpret_cast<uint32_t*>(ctl + 16);    // [8] a tile's V held inf or NaN
    const uint32_t sbase = smem_u32(smem), qbase = sbase + kTcStages * S::kStage;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    pdl_wait_prior_grids();
    const Range range = cta_range<kTcThreads>(p, ctl, ctl + 2);
    if (range.begin >= range.end) return;
    if (warp == 4) {
        tmem_alloc(tmem_slot, S::kCols);
        tmem_relinquish();
        if (lane == 0) {
            for (int i = 0; i < kTcStages; ++i) {
                mbar_init(k_full + i, kLoaders);
                mbar_init(k_empty + i, 1);
                mbar_init(v_full + i, kLoaders);
                mbar_init(v_empty + i, 1);
            }
            mbar_init(s_full, 1);
            mbar_init(s_free, kSoftmax);
            mbar_init(p_full, kSoftmax);
            mbar_init(o_done, 1);
            mbar_init(q_full, kSoftmax);
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
    uint32_t tile = 0;                                                   // tiles of this CTA so far
    // Once a wait has run out the CTA goes on without waiting, so that its barriers still match; the results are
    // rubbish then, and reported.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity);
    };

    if (warp < 4) {
        // ---- softmax: thread = row ---------------------------------------------------------------------
        const uint32_t lanes = tmem + (warp << 21);                      // this warp's lanes: 32 * warp << 16
        const uint32_t rows = p.nodes * p.group;
        while (u < u_end) {
            const Piece x = next_piece(p, u, u_end, b, seq_first);
            if (x.sq.bad && tid == 0) atomicOr(p.status, kDevErrBadIndex);
            const uint32_t row = x.rt * kTcRows + tid, t = row / p.group, g = row - t * p.group;
            const bool live = row < rows && (int32_t)t < x.sq.nodes;
            // Q: all MMAs that read the last one are done (o_done of its last tile)
            for (uint32_t i = tid; i < kTcRows * CPR; i += kSoftmax) {
                const uint32_t r = i / CPR, c = i % CPR, qrow = x.rt * kTcRows + r, qt = qrow / p.group, qg = qrow - qt * p.group;
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
                *reinterpret_cast<uint4*>(smem + kTcStages * S::kStage + swz(kTcRows, r, c)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (x.has_nodes && tid < p.nodes) {
                bool bad = false;
                anc[tid] = node_path(p, b, tid, bad);
                if (bad && (int32_t)tid < x.sq.nodes) atomicOr(p.status, kDevErrBadIndex);
            }
            fence_async_smem();
            named_bar_sync(2, kSoftmax);                                 // (anc is read by other threads)
            mbar_arrive(q_full);

            float m = -INFINITY, l = 0.0f;                               // base (log2) and sum of this row
            for (uint32_t i = 0; i < x.n_tiles; ++i, ++tile) {
                // (V's barrier cannot move on before this thread has handed over P; it also covers `valid` and `fixes`)
                wait(v_full + tile % kTcStages, (tile / kTcStages) & 1);
                wait(s_full, tile & 1);
                __syncwarp();
                tc_fence_after();
                float s[64];
                tmem_ld32<0>(lanes + S::kColS, s);
                tmem_ld32<32>(lanes + S::kColS + 32, s);
                uint64_t see = valid[tile & 7];
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(s_free);
                if (x.t0 + i + 1 == x.sq.tiles && t < p.nodes) see &= anc[t];
                if (see != ~0ull) {
#pragma unroll
                    for (int j = 0; j < 64; ++j)
                        if (!((see >> j) & 1)) s[j] = -INFINITY;
                }
                float top = s[0];
#pragma unroll
                for (int j = 1; j < 64; ++j) top = fmaxf(top, s[j]);
                top *= p.scale_log2;
                // P's buffer and O are free once the MMA before has read and written them
                if (i > 0) wait(o_done, (tile - 1) & 1);
                __syncwarp();
                tc_fence_after();
                if (i == 0) {
                    m = top;
                } else {
                    const bool grow = top > m + kLazy;                   // (m -inf: at the first finite score)
                    if (__any_sync(0xffffffffu, grow)) {
                        const float base = grow ? top : m;
                        const float f = grow ? exp2_fast(m - top) : 1.0f;
                        l *= f;
                        m = base;
#pragma unroll 1
                        for (int d = 0; d < D; d += 32) {
                            float o[32];
                            tmem_ld32<0>(lanes + d, o);
                            tmem_ld_wait();
                            uint32_t w[32];
#pragma unroll
                            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * f);
                            tmem_st32(lanes + d, w);
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
                tmem_st32(lanes + S::kColP, w);
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(p_full);
            }
            wait(o_done, (tile - 1) & 1);
            __syncwarp();
            tc_fence_after();
            // ---- O of this piece: the result, or a partial
            const bool whole = x.t0 == 0 && x.has_nodes;
            const uint64_t slot = ((uint64_t)2 * blockIdx.x + (x.t0 == 0 ? 1 : 0)) * kTcRows + tid;
            const bool fix = x.has_nodes && fixes[(tile - 1) & 7];       // (the nodes' tile is a piece's last one)
            const float inv = 1.0f / l;
            if (!whole && live) p.part_ml[slot] = make_float2(m, l);
            const uint64_t to = b * p.out_batch + t * p.out_node + (uint64_t)(x.h * p.group + g) * p.out_head;
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
                float o[32];
                __syncwarp();
                tmem_ld32<0>(lanes + d, o);
                tmem_ld_wait();
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
            named_bar_sync(2, kSoftmax);                                 // everybody has read anc and O
            u += x.n_tiles;
        }
    } else if (warp == 4) {
        // ---- MMA issue: one lane ----------------------------------------------------------------------------
        if (lane == 0) {
            uint32_t piece = 0;
            auto scores = [&](uint32_t n) {                              // S of tile n
                wait(k_full + n % kTcStages, (n / kTcStages) & 1);
                if (n > 0) wait(s_free, (n - 1) & 1);
                tc_fence_after();
                const uint32_t k = sbase + (n % kTcStages) * S::kStage;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t chunk = ks >> 2, in = (ks & 3) * 32;
                    mma_ss(tmem + S::kColS, smem_desc(qbase + chunk * (kTcRows * 128) + in, 16), smem_desc(k + chunk * (kKeys * 128) + in, 16),
                           instr_desc(kKeys, 0), ks > 0);
                }
                mma_commit(k_empty + n % kTcStages);
                mma_commit(s_full);
            };
            while (u < u_end) {
                const Piece x = next_piece(p, u, u_end, b, seq_first);
                wait(q_full, piece & 1);
                scores(tile);
                for (uint32_t i = 0; i < x.n_tiles; ++i, ++tile) {
                    if (i + 1 < x.n_tiles) scores(tile + 1);
                    wait(v_full + tile % kTcStages, (tile / kTcStages) & 1);
                    wait(p_full, tile & 1);
                    tc_fence_after();
                    const uint32_t v = sbase + (tile % kTcStages) * S::kStage + S::kTile;
#pragma unroll
                    for (int ks = 0; ks < (int)kKeys / 16; ++ks)
                        mma_ts(tmem, tmem + S::kColP + ks * 8, smem_desc(v + ks * 2048, kKeys * 128), instr_desc(D, 1), i > 0 || ks > 0);
                    mma_commit(v_empty + tile % kTcStages);
                    mma_commit(o_done);
                }
                ++piece;
                u += x.n_tiles;
            }
            mma_commit(drained);                                         // tensor memory is freed behind the last MMA
            if (!mbar_wait(drained, 0)) ok = false;
        }
        __syncwarp();
    } else {
        // ---- loaders ---------------------------------------------------------------------------------------
        // Groups of copies in order: K and V of a tile, then the next tile's.  A group is handed on when it has landed,
        // kLag groups behind the newest one; before a thread blocks on a stage that is still in use it hands on all
        // it has, since that stage may only become free after them.
        constexpr uint32_t kLag = 2;
        const uint32_t lt = tid - (kTcThreads - kLoaders);
        uint32_t issued = 0, handed = 0;
        auto hand = [&](uint32_t upto) {
            fence_async_smem();
            for (; handed < upto; ++handed) mbar_arrive((handed & 1 ? v_full : k_full) + (handed >> 1) % kTcStages);
        };
        auto acquire = [&](uint64_t* empty) {
            if (tile < (uint32_t)kTcStages) return;
            uint64_t* bar = empty + tile % kTcStages;
            const uint32_t parity = (tile / kTcStages - 1) & 1;
            if (!ok || mbar_try_wait(bar, parity)) return;
            cp_wait<0>();
            hand(issued);
            wait(bar, parity);
        };
        // (threads of a warp may part company here; they meet again at the barrier of the next tile)
        while (u < u_end) {
            const Piece x = next_piece(p, u, u_end, b, seq_first);
            int32_t page = lt < kKeys ? key_page(p, x, 0, lt) : -1;
            for (uint32_t i = 0; i < x.n_tiles; ++i, ++tile) {
                const uint32_t st = tile % kTcStages;
                __syncwarp();
                if (lt < kKeys) {
                    const uint64_t at = key_offset(p, x, i, lt, page);
                    offs[(tile & 1) * kKeys + lt] = at;
                    __syncwarp();
                    const uint32_t bits = __ballot_sync(0xffffffffu, at != ~0ull);
                    if (lane == 0) reinterpret_cast<volatile uint32_t*>(valid + (tile & 7))[lt >> 5] = bits;
                    if (lt == 0) fixes[tile & 7] = 0;
                    page = key_page(p, x, i + 1, lt);
                }
                __syncwarp();
                named_bar_sync(1, kLoaders);
                const bool own = x.t0 + i + 1 == x.sq.tiles;
                auto load = [&](const uint16_t* base, uint32_t stage) {
#pragma unroll 4
                    for (uint32_t idx = lt; idx < kKeys * CPR; idx += kLoaders) {
                        const uint32_t r = idx / CPR, c = idx % CPR;
                        const uint64_t at = offs[(tile & 1) * kKeys + r];
                        const bool here = at != ~0ull && c * 8 < p.head_dim;
                        cp_async16(stage + swz(kKeys, r, c), here ? base + at + c * 8 : p.k, here);
                    }
                    cp_commit();
                    ++issued;
                };
                const uint32_t kst = sbase + st * S::kStage;
                acquire(k_empty);
                load(own ? p.k : p.c.k, kst);
                acquire(v_empty);
                load(own ? p.v : p.c.v, kst + S::kTile);
                if (own) {                                               // clear non-finite V of the nodes before it is used
                    cp_wait<0>();
                    bool odd = false;
                    for (uint32_t idx = lt; idx < kKeys * CPR; idx += kLoaders)
                        odd |= clear_nonfinite(reinterpret_cast<uint4*>(smem + st * S::kStage + S::kTile + swz(kKeys, idx / CPR, idx % CPR)));
                    if (odd) fixes[tile & 7] = 1;
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
    if (warp == 4) tmem_dealloc(tmem, S::kCols);
}

template <int D>
cudaError_t run(AttendParams p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    using S = TcShape<D>;
    static DeviceOnce once;
    auto fn = attend_tc_kernel<D>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void*>(fn), S::kSmem, once);
    if (e != cudaSuccess) return e;
    p.grid = (uint32_t)(sm_count * S::kPerSm);
    p.row_tiles = (p.nodes * p.group + kTcRows - 1) / kTcRows;
    if (!attend_workspace(p, ws, kTcRows, D)) return cudaSuccess;
    if ((e = attend_launch(fn, dim3(p.grid), kTcThreads, S::kSmem, use_pdl, s, p)) != cudaSuccess) return e;
    return launch_attend_join(p, kTcRows, D, true, ws, use_pdl, s);
}

}  // namespace

cudaError_t launch_attend_tc(const AttendParams& p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    if (p.head_dim <= 64) return run<64>(p, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 128) return run<128>(p, ws, sm_count, use_pdl, s);
    return run<256>(p, ws, sm_count, use_pdl, s);
}

}  // namespace lq4
