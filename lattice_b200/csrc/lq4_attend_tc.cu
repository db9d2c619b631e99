// lq4_tree_attention for many rows per kv head (a large tree), on the 5th-generation tensor cores.
//
// With R query rows on a key/value head there are R flops per byte of cache, so with some dozens of rows the HBM
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
//   next N warps    MMA issue, a warp per stream (the first one allocates tensor memory)
//   last warps      loaders: cp.async of K and V rows, each looked up through the page table, into one ring of slots
//                   (K, V, K, V, ...), a warp per tile; they run ahead over the borders of pieces
//
// The running maximum only moves when it has grown by more than 2^8 (the final division takes the same base out
// again), so O is rescaled in tensor memory a few times per sequence instead of per tile.
//
// f32 activations (up to D = 128): q and P are three bf16 terms each, 24 bits, smallest products first.  The accumulators
// in tensor memory cut off below their last bit at every MMA, some 10^-5 over a few hundred of them, so P V of a tile
// starts from zero and the softmax threads add it to O in their registers, a tile later; one stream, two buffers of P and
// of P V.
//
// B200, device time: 4 trees of 64 nodes over 16384 tokens, 32 heads on 8 of 128, bf16: 119 us (0.6 PFLOP/s); 8 trees of 13
// nodes over 2000 to 4000, 40 heads on 8 of 128, f32: 86 us.  Neither HBM nor the tensor cores are busy (22 % and 26 % at
// half the first one's length, 16 % and 27 % in the second): a stream waits for its own scores, exponentials and products in
// turn, and with f32 activations, where a scheduler has one softmax warp, most of all for its instructions.
#include "lq4_attend_dev.cuh"

namespace lq4 {

namespace {

constexpr int kTcRows = 128;
constexpr float kLazy = 8.0f;                  // how far (log2) a row's maximum may outgrow its base

// D[tmem] (+)= A[tmem] B[smem]: A has a lane per row and two consecutive k per column; one thread issues.
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
template <int AT, int N>
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[N]) {      // 32 columns -> r[AT .. AT + 32)
    uint32_t u[32];
    tmem_ld_32x32(taddr, u);
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
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&u)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0,%1,%2,%3,%4,%5,%6,%7};" ::"r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                 "r"(u[6]), "r"(u[7]), "r"(taddr)
                 : "memory");
}
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

// Adds what the item's pieces before have left of a row (ml, and D floats at `from`) to the row's O in tensor memory, maximum and sum;
// none: there is no O yet.  A call of its own: the end of a piece runs once or twice per CTA, and what it has to fetch of the
// program counts (inline this cost 6 us of 126 where no item had several pieces).
template <int D>
__device__ __noinline__ float2 resume(uint32_t col_o, bool none, float m, float l, float2 ml, const float* from) {
    const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.0f : top, f = exp2_fast(m - base), g = exp2_fast(ml.x - base);
    __syncwarp();
#pragma unroll 1
    for (int d = 0; d < D; d += 32) {
        float o[32];
        tmem_ld32<0>(col_o + d, o);
        tmem_ld_wait();
        uint32_t w[32];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float4 v = reinterpret_cast<const float4*>(from + d)[e];
            w[4 * e] = __float_as_uint((none ? 0.0f : o[4 * e] * f) + v.x * g), w[4 * e + 1] = __float_as_uint((none ? 0.0f : o[4 * e + 1] * f) + v.y * g);
            w[4 * e + 2] = __float_as_uint((none ? 0.0f : o[4 * e + 2] * f) + v.z * g), w[4 * e + 3] = __float_as_uint((none ? 0.0f : o[4 * e + 3] * f) + v.w * g);
        }
        tmem_st32(col_o + d, w);
    }
    tmem_st_wait();
    return make_float2(top, l * f + ml.y * g);
}

// NS streams; WIDE: items of 256 rows; NQ bf16 terms of q and P: 1 for bf16 activations, 3 for f32.
template <int D, int NS, bool WIDE, int NQ>
struct TcShape {
    static constexpr int kSoftmax = 128 * NS, kItemRows = WIDE ? 256 : 128;
    static constexpr uint32_t kSlot = kKeys * D * 2, kQTerm = kTcRows * D * 2, kQ = kQTerm * (WIDE ? 2 : 1) * NQ;
    // Rings of slots: one that all streams read in order, or one per stream where they take the tiles in turn (a wait on a slot's
    // barrier is only good as long as the reader goes through the slot's uses one by one).
    static constexpr uint32_t kRings = NS == 2 && !WIDE ? 2 : 1;
    static constexpr uint32_t kFit = ((uint32_t)kMaxSmem - kQ - 5120) / kSlot / kRings, kRing = kFit > 12 / kRings ? 12 / kRings : kFit, kSlots = kRing * kRings;
    static constexpr uint32_t kValid = kSlots * kSlot + kQ, kFixes = kValid + 16 * 8, kAnc = kFixes + 16 * 8, kMeet = kAnc + kMaxNodes * 8;
    static constexpr uint32_t kBars = kMeet + kTcRows * 8, kCtl = kBars + 56 * 8, kSmem = kCtl + 160 + 1024;      // + alignment slack
    // Three terms: two buffers of O and P, so that a tile's P V runs beside the next tile's softmax.
    static constexpr uint32_t kBufs = NQ == 1 ? NS : 2, kColO = 0, kColS = kBufs * D, kColP = kColS + NS * 64, kEnd = kColP + kBufs * 32 * NQ, kCols = kEnd <= 256 ? 256 : 512;
    // Loaders: teams, warps of a team.  (Seven warps for three terms: with nine a thread has 168 registers, and O spills.)
    static constexpr uint32_t kTeams = NQ == 1 && kSlots >= 8 ? 4 : 2, kTeam = NQ == 1 ? 4 / kTeams : 1;
    static constexpr int kLoaders = 32 * kTeams * kTeam, kThreads = kSoftmax + 32 * NS + kLoaders;
    static_assert(2 * kTeams / kRings <= kRing, "a team's next tile is at most a ring ahead of its last one");
    static_assert(kSlots >= 4 && kSmem <= (uint32_t)kMaxSmem && kEnd <= 512, "shared or tensor memory");
    static_assert(NQ == 1 || NS == 1, "three terms take one stream");
    static_assert(NS == 2 || !WIDE, "256 rows take two streams");
    static_assert(kTcRows * 32 * 4 <= kQ, "the streams meet in Q's place");
};

template <int D, int NS, bool WIDE, int NQ>
__global__ void __launch_bounds__((TcShape<D, NS, WIDE, NQ>::kThreads), 1) attend_tc_kernel(const __grid_constant__ AttendParams p) {
    using S = TcShape<D, NS, WIDE, NQ>;
    constexpr int CPR = D / 8, kSoftmax = S::kSoftmax, kMmaWarp = kSoftmax / 32;
    constexpr uint32_t SL = S::kSlots, RING = S::kRing, RINGS = S::kRings;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);      // swizzle atoms are 1024 bytes
    volatile uint32_t* valid = reinterpret_cast<uint32_t*>(smem + S::kValid);    // [16][2] which of a tile's 64 keys there are
    volatile uint32_t* fixes = reinterpret_cast<uint32_t*>(smem + S::kFixes);    // [16][2] V of the tile held inf or NaN (by warp of a team)
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + S::kAnc);        // [nodes] of the piece's sequence
    float2* meet = reinterpret_cast<float2*>(smem + S::kMeet);          // [128] (max, sum) of stream 1's rows
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t* ctl = reinterpret_cast<uint64_t*>(smem + S::kCtl);        // 0, 1: cursor; 2..15: warp sums, then 2: the range's first unit; 16: tensor memory
    uint64_t *full = bars, *empty = bars + SL, *s_full = bars + 2 * SL, *s_free = s_full + 2, *p_full = s_full + 4, *o_done = s_full + 6;
    uint64_t *q_full = s_full + 8, *drained = s_full + 9, *info = s_full + 10;      // info: [16], the loaders are at most 7 tiles ahead
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctl + 16);
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
                mbar_init(full + i, S::kTeam);
                mbar_init(empty + i, WIDE ? 2 : 1);                      // by the streams that read the tile
            }
            for (int i = 0; i < 2; ++i) {
                mbar_init(s_full + i, 1);
                mbar_init(s_free + i, 4);
                mbar_init(p_full + i, 4);
                mbar_init(o_done + i, 1);
            }
            mbar_init(q_full, kSoftmax / 32);
            mbar_init(drained, NS);
            for (int i = 0; i < 16; ++i) mbar_init(info + i, S::kTeam);
            mbar_fence_init();
            ctl[2] = range.begin;
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

    if (tid < (uint32_t)kSoftmax) {
        // ---- softmax: thread = row ---------------------------------------------------------------------
        const uint32_t str = tid >> 7, r = tid & 127;
        const uint32_t lanes = tmem + ((warp & 3) << 21);                // this warp's 32 lanes, at bit 16
        const uint32_t col_o = lanes + S::kColO + str * D, col_s = lanes + S::kColS + str * 64, col_p = lanes + S::kColP + str * 32;
        const uint32_t rows = p.nodes * p.group;
        uint32_t used = 0;                                               // steps of this stream so far
        while (u < u_end) {
            const Piece x = next_piece<kPieceTiles<NQ>>(p, u, u_end, b, seq_first);
            if (x.sq.bad && tid == 0) atomicOr(p.status, kDevErrBadIndex);
            const uint32_t row = x.rt * S::kItemRows + (WIDE ? tid : r), t = row / p.group, g = row - t * p.group;
            const bool live = row < rows && (int32_t)t < x.sq.nodes;
            // Q: all MMAs that read the last one are done (o_done of its last step)
#pragma unroll 4
            for (uint32_t i = tid; i < S::kItemRows * CPR; i += kSoftmax) {
                const uint32_t qr = i / CPR, c = i % CPR, qrow = x.rt * S::kItemRows + qr, qt = qrow / p.group, qg = qrow - qt * p.group;
                const bool here = qrow < rows && (int32_t)qt < x.sq.nodes && c * 8 < p.head_dim;
                const uint64_t from = b * p.q_batch + qt * p.q_node + (uint64_t)(x.h * p.group + qg) * p.q_head + c * 8;
                const uint32_t to = SL * S::kSlot + (qr >> 7) * S::kQTerm + swz(kTcRows, qr & 127, c);
                if constexpr (NQ == 1) {
                    uint32_t w[4] = {0, 0, 0, 0};
                    if (here) {
                        const uint16_t* src = static_cast<const uint16_t*>(p.q) + from;
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
                    *reinterpret_cast<uint4*>(smem + to) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
                    if (here) {
                        const float* src = static_cast<const float*>(p.q) + from;
                        if (p.q_vec) {
                            const float4 lo = reinterpret_cast<const float4*>(src)[0], hi = reinterpret_cast<const float4*>(src)[1];
                            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e) v[e] = src[e];
                        }
#pragma unroll
                        for (int e = 0; e < 8; ++e) v[e] *= p.q_sign;
                    }
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) w[e] = split_pair(v[2 * e], v[2 * e + 1]);
                        *reinterpret_cast<uint4*>(smem + to + n * S::kQTerm) = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
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
            float acc[NQ == 1 ? 1 : D];                                  // f32 activations: O
            auto fold = [&](float f) {                                   // O = f (O + P V of the tile before)
                if constexpr (NQ > 1) {
                    const uint32_t last = used - 1;
                    wait(o_done + (last & 1), last >> 1 & 1);
                    __syncwarp();
                    tc_fence_after();
#pragma unroll
                    for (int d = 0; d < D; d += 32) {
                        float o[32];
                        tmem_ld32<0>(col_o + (last & 1) * D + d, o);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e) acc[d + e] = (acc[d + e] + o[e]) * f;
                    }
                }
            };
#pragma unroll
            for (int d = 0; d < (NQ == 1 ? 1 : D); ++d) acc[d] = 0.0f;
            for (uint32_t i = RINGS == 2 ? (str - tile) & 1 : 0; i < x.n_tiles; i += RINGS) {      // (tile n belongs to stream n & 1)
                const uint32_t n = tile + i;
                wait(info + (n & 15), (n >> 4) & 1);                     // `valid` of this tile is there
                wait(s_full + str, used & 1);
                __syncwarp();
                tc_fence_after();
                float s[64];
                tmem_ld32<0>(col_s, s);
                tmem_ld32<32>(col_s + 32, s);
                uint64_t see = (uint64_t)valid[(n & 15) * 2 + 1] << 32 | valid[(n & 15) * 2];
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
                    for (int j = 4; j < 60; j += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) t4[e] = fmaxf(fmaxf(t4[e], s[j + e]), s[j + 4 + e]);      // (one instruction)
#pragma unroll
                    for (int e = 0; e < 4; ++e) t4[e] = fmaxf(t4[e], s[60 + e]);
                    top = fmaxf(fmaxf(t4[0], t4[1]), fmaxf(t4[2], t4[3])) * p.scale_log2;
                }
                // P's buffer and O are free once the stream's MMA before has read and written them (three terms: two tiles
                // before, which the last fold has waited for)
                if (NQ == 1 && !first) wait(o_done + str, (used - 1) & 1);
                __syncwarp();
                tc_fence_after();
                float f = 1.0f;
                if constexpr (NQ > 1) {
                    const float up = fmaxf(m, top);
                    if (m != up) f = exp2_fast(m - up);                  // (m -inf: 0)
                    l *= f;
                    m = up;
                } else if (first) {
                    m = top;
                } else {
                    const bool grow = top > m + kLazy;                   // (m -inf: at the first finite score)
                    if (__any_sync(0xffffffffu, grow)) {
                        f = grow ? exp2_fast(m - top) : 1.0f;
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
                if constexpr (NQ == 1) {
                    uint32_t w[32];
#pragma unroll
                    for (int j = 0; j < 32; ++j) {
                        const float a = exp2_fast(fmaf(s[2 * j], p.scale_log2, -base)), c = exp2_fast(fmaf(s[2 * j + 1], p.scale_log2, -base));
                        sum0 += a;
                        sum1 += c;
                        const __nv_bfloat162 y = __floats2bfloat162_rn(a, c);
                        w[j] = *reinterpret_cast<const uint32_t*>(&y);
                    }
                    tmem_st32(col_p, w);
                } else {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {                        // 16 keys at a time
                        float e[16];
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            e[j] = exp2_fast(fmaf(s[16 * k + j], p.scale_log2, -base));
                            (j & 1 ? sum1 : sum0) += e[j];
                        }
#pragma unroll
                        for (int n = 0; n < NQ; ++n) {
                            uint32_t w[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) w[j] = split_pair(e[2 * j], e[2 * j + 1]);
                            tmem_st8(col_p + (used & 1) * (32 * NQ) + 32 * n + 8 * k, w);
                        }
                    }
                }
                l += sum0 + sum1;
                tmem_st_wait();
                // the nodes' tile: `fixes` comes with V, whose slot is not filled again before this P is handed over
                if (x.t0 + i + 1 == x.sq.tiles) wait(full + (n & (RINGS - 1)) * RING + (2 * (n / RINGS) + 1) % RING, (2 * (n / RINGS) + 1) / RING & 1);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + str);
                if (NQ > 1 && !first) fold(f);                           // (its P V has had this tile's softmax to finish in)
                first = false;
                ++used;
            }
            if (NQ == 1 && !first) wait(o_done + str, (used - 1) & 1);
            __syncwarp();
            tc_fence_after();
            if (NQ > 1 && !first) fold(1.0f);
            // ---- O of this piece: the result, or a partial.  Two streams over the keys: stream 1 hands its O to stream 0
            // through Q's place, 32 columns at a time (both have waited for all MMAs of their own that read Q; the
            // barrier below covers the other's).
            constexpr bool kMeets = NS == 2 && !WIDE;
            const Fate fates = fate<NQ>(x, u, ctl[2]);
            const bool whole = fates.whole;
            const uint64_t slot = (uint64_t)fates.slot * S::kItemRows + (WIDE ? tid : r);
            if (NQ == 1 && fates.goes_on && (!kMeets || str == 0)) {
                const float2 ml = resume<D>(col_o, first, m, l, p.part_ml[slot], p.part_o + slot * D);
                m = ml.x, l = ml.y;
                first = false;
            }
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
            const bool fix = x.has_nodes && (fixes[((tile + x.n_tiles - 1) & 15) * 2] | (S::kTeam == 2 ? fixes[((tile + x.n_tiles - 1) & 15) * 2 + 1] : 0));      // (the nodes' tile is a piece's last one)
            const float inv = 1.0f / l;
            if (!whole && live && (!kMeets || str == 0)) p.part_ml[slot] = make_float2(m, l);
            const uint64_t to = b * p.out_batch + t * p.out_node + (uint64_t)(x.h * p.group + g) * p.out_head;
            float* pass = reinterpret_cast<float*>(smem + SL * S::kSlot) + r;      // [columns][128]: lanes side by side
            auto put = [&](int d, float (&o)[32]) {                      // 32 columns of this row
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
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        if (d + e >= (int)p.head_dim) break;             // (a multiple of 8)
                        if constexpr (NQ > 1) {
                            float* out = static_cast<float*>(p.out) + to + d + e;
                            if (p.out_vec) {
                                reinterpret_cast<float4*>(out)[0] = make_float4(o[e] * inv, o[e + 1] * inv, o[e + 2] * inv, o[e + 3] * inv);
                                reinterpret_cast<float4*>(out)[1] = make_float4(o[e + 4] * inv, o[e + 5] * inv, o[e + 6] * inv, o[e + 7] * inv);
                            } else {
#pragma unroll
                                for (int k = 0; k < 8; ++k) out[k] = o[e + k] * inv;
                            }
                            continue;
                        }
                        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + to + d;
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
            };
            if constexpr (NQ > 1) {
#pragma unroll
                for (int d = 0; d < D; d += 32) {
                    float o[32];
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = acc[d + e];
                    if (live) put(d, o);
                }
            } else {
#pragma unroll 1
            for (int d = 0; d < D; d += 32) {
                float o[32];
                __syncwarp();
                if (kMeets && first) {                                   // this stream had no tile of the piece
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = 0.0f;
                } else {
                    tmem_ld32<0>(col_o + d, o);
                    tmem_ld_wait();
                }
                if (kMeets && str == 1) {
#pragma unroll
                    for (int e = 0; e < 32; ++e) pass[e * 128] = o[e];
                    named_bar_sync(3, 256);
                    named_bar_sync(4, 256);                              // stream 0 has it
                    continue;
                }
                if constexpr (kMeets) {
                    named_bar_sync(3, 256);
#pragma unroll
                    for (int e = 0; e < 32; ++e) o[e] = o[e] * f + pass[e * 128] * f_other;      // (0 of a stream without tiles)
                    named_bar_sync(4, 256);
                }
                if (live) put(d, o);
            }
            }
            if (live && whole && (!kMeets || str == 0) && !(l > 0.0f)) mark(p, NQ == 1, to);
            __syncwarp();
            tc_fence_before();
            named_bar_sync(2, kSoftmax);                                 // everybody has read anc, meet and O
            tile += x.n_tiles;
            u += x.n_tiles;
        }
    } else if (warp < kMmaWarp + NS) {
        // ---- MMA issue: a warp per stream ------------------------------------------------------------------
        // The whole warp walks through the stream's tiles with warp-uniform values (descriptors then live in uniform
        // registers); one lane issues.  Everything a step looks up is kept running: ring position and phase of the next K
        // and V group, phases of the stream's barriers.
        const bool leader = elect_lane();
        auto uniform = [](uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); };
        const uint32_t str = uniform(warp - kMmaWarp);
        const uint32_t tm = uniform(tmem), ring = uniform(sbase) >> 4;
        const uint32_t col_s = tm + S::kColS + str * 64, col_p = tm + S::kColP + str * 32, col_o = tm + S::kColO + str * D;
        const uint64_t kmajor = smem_desc(0, 16), mnmajor = smem_desc(0, kKeys * 128);
        const uint64_t q = kmajor + (uniform(qbase) >> 4) + (WIDE ? str * (S::kQTerm >> 4) : 0);
        struct Ring {
            uint32_t slot, phase;
            __device__ __forceinline__ void move(uint32_t groups) {
                slot += groups;
                if (slot >= RING) slot -= RING, phase ^= 1;
            }
        } kr{0, 0}, vr{1, 0};
        const uint32_t ring0 = RINGS == 2 ? str * RING : 0;              // first slot of the stream's ring
        uint32_t piece = 0, ph_s = 1, ph_p = 0, at = 0, buf = 0;         // s_free: phase 1 of the step before the first; tiles so far; O and P in turn
        bool s_any = false;
        auto scores = [&]() {
            wait(full + ring0 + kr.slot, kr.phase);
            if (s_any) wait(s_free + str, ph_s);
            s_any = true;
            ph_s ^= 1;
            __syncwarp();
            tc_fence_after();
            const uint64_t k = kmajor + (ring + (ring0 + kr.slot) * (S::kSlot >> 4));
            if (leader) {
#pragma unroll
                for (int ks = 0; ks < NQ * (D / 16); ++ks) {             // the smallest term first
                    const int n = NQ - 1 - ks / (D / 16), c = ks % (D / 16) >> 2, in = (ks & 3) * 32;
                    umma_f16(col_s, q + (n * S::kQTerm + c * (kTcRows * 128) + in >> 4), k + (c * (kKeys * 128) + in >> 4), instr_desc(kKeys, 0), ks > 0);
                }
                umma_commit(empty + ring0 + kr.slot);
                umma_commit(s_full + str);
            }
            kr.move(2);
        };
        while (u < u_end) {
            const Piece x = next_piece<kPieceTiles<NQ>>(p, u, u_end, b, seq_first);
            const uint32_t tiles = uniform(x.n_tiles);
            const uint32_t steps = RINGS == 2 ? (tiles + 1 - ((str - at) & 1)) / 2 : tiles;      // of this stream
            wait(q_full, piece & 1);
            if (steps > 0) scores();
            for (uint32_t v = 0; v < steps; ++v) {
                if (v + 1 < steps) scores();
                wait(full + ring0 + vr.slot, vr.phase);
                wait(p_full + str, ph_p);
                ph_p ^= 1;
                __syncwarp();
                tc_fence_after();
                const uint64_t vt = mnmajor + (ring + (ring0 + vr.slot) * (S::kSlot >> 4));
                if (leader) {
#pragma unroll
                    for (int ks = 0; ks < NQ * ((int)kKeys / 16); ++ks) {
                        const int n = NQ - 1 - ks / 4, c = ks & 3;
                        mma_ts(col_o + buf * D, col_p + buf * (32 * NQ) + n * 32 + c * 8, vt + (c * 2048 >> 4), instr_desc(D, 1), (NQ == 1 && v > 0) || ks > 0);
                    }
                    umma_commit(empty + ring0 + vr.slot);
                    umma_commit(o_done + (NQ == 1 ? str : buf));
                }
                if (NQ > 1) buf ^= 1;
                vr.move(2);
            }
            at += tiles;
            ++piece;
            u += tiles;
        }
        if (leader) umma_commit(drained);                                 // tensor memory is freed behind the last MMA
        if (!mbar_wait(drained, 0)) ok = false;
        __syncwarp();
    } else {
        // ---- loaders -----------------------------------------------------------------------------------------
        load_stream<D, RING, RINGS, S::kTeams, S::kTeam, kPieceTiles<NQ>>(p, u, u_end, b, seq_first, warp - (S::kThreads - S::kLoaders) / 32, smem, full, empty, info, valid, fixes, ok,
                                                         [](uint32_t r, uint32_t c) { return swz(kKeys, r, c); });
    }
    if (!ok) atomicOr(p.status, kDevErrBarrierTimeout);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, S::kCols);
}

template <int D, int NS, bool WIDE, int NQ>
cudaError_t run(AttendParams p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    using S = TcShape<D, NS, WIDE, NQ>;
    static DeviceOnce once;
    auto fn = attend_tc_kernel<D, NS, WIDE, NQ>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void*>(fn), S::kSmem, once);
    if (e != cudaSuccess) return e;
    p.grid = (uint32_t)sm_count;
    p.row_tiles = (p.nodes * p.group + S::kItemRows - 1) / S::kItemRows;
    if (!attend_workspace(p, ws, S::kItemRows, D)) return cudaSuccess;
    if ((e = attend_launch(fn, dim3(p.grid), S::kThreads, S::kSmem, use_pdl, s, p)) != cudaSuccess) return e;
    return launch_attend_join(p, S::kItemRows, D, NQ == 1, ws, use_pdl, s);
}

}  // namespace

cudaError_t launch_attend_tc(const AttendParams& p, bool f32, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    const bool wide = p.nodes * p.group > (uint32_t)kTcRows;
    if (f32) return p.head_dim <= 64 ? run<64, 1, false, 3>(p, ws, sm_count, use_pdl, s) : run<128, 1, false, 3>(p, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 64) return wide ? run<64, 2, true, 1>(p, ws, sm_count, use_pdl, s) : run<64, 2, false, 1>(p, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 128) return wide ? run<128, 2, true, 1>(p, ws, sm_count, use_pdl, s) : run<128, 2, false, 1>(p, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 192) return run<192, 1, false, 1>(p, ws, sm_count, use_pdl, s);
    return run<256, 1, false, 1>(p, ws, sm_count, use_pdl, s);
}

}  // namespace lq4
