// Attention of a tree of drafted tokens (one token: ordinary decode) over a paged bf16 cache and the nodes' own
// rows, in one pass over the keys:
//
//   o[t, h] = sum_j softmax_j(scale q[t, h] . k[j]) v[j],   j over the committed slots of the sequence and over
//             the nodes on the path from the root to t.
//
// The query rows that share a key/value head (nodes x q_heads / kv_heads of them) are the rows of one matrix, so
// every key is read once for all of them.  With few rows the bound is HBM (4 bytes of cache per row and channel
// against 4 flops), so the design is about keeping the key stream going:
//
//   work       the (sequence, kv head, row tile) items, cut into tiles of 64 keys, form one range that is split
//              evenly over a persistent grid.  The lengths are only known on the device: every CTA sums them
//              itself.  A ragged batch is balanced to one tile, and the launch does not depend on the lengths
//              (a captured graph replays with others).  An item cut by a CTA border leaves (max, sum, O) partials,
//              at most two per CTA, which attend_join_kernel merges in the order of the CTAs: the same lengths
//              give the same bits.
//   loads      four warps of their own (load_stream): cp.async, 16 bytes a lane, into a ring of K and V tiles.  Every
//              key's address is looked up on its own (slot -> page), so pages of any size may end anywhere inside a tile.
//   math       mma.sync m16n8k16 on bf16.  K and V are bf16 in memory and exact.  q and the probabilities are one
//              bf16 term each for bf16 activations (q is one; the weights' rounding is of the size of the output's own), and
//              three terms each (24 bits) for f32 ones, so that an f32 result keeps 32-bit accuracy.  A second term of the
//              weights would take the error of the batch below from 1.83e-3 to 1.67e-3 (2-norm; what the result's own rounding
//              leaves) for 154 -> 164 us a call, and with tcgen05 that of large trees from 2.27e-3 to 1.67e-3 for 126 -> 162 us.
//   warps      four for the math, WM x WN: WM bands of 16 rows, WN shares of the 64 keys.  Each warp keeps its own running
//              maximum, sum and O over its keys; they meet in shared memory once per piece.
//
// B200, device time: 32 sequences of 4096 to 8191 tokens, 40 heads on 8 of 128, bf16: 144 us (5.7 TB/s; every key is read
// once).  One of 120001, 24 heads on 4 of 256, f32: 148 us (3.3 TB/s; 6 rows fill 16, and each product is three: tensor pipe 34 %,
// issue active 30 %, and one math warp a scheduler has nobody to hide its waits).  f32 above a head_dim of 128 is at the limit of
// 255 registers and spills: 120 bytes of loads at 256 with up to 16 rows and 272 with 32, 68 and 160 at 192.
//
// A key that a row may not see contributes nothing whatever it holds: its score is replaced by -inf, and a
// non-finite V entry of a node (0 * inf would reach the rows that do not see it) is cleared in shared memory
// and added back at the end for the rows that do see it.  A cached one is seen by all rows of its sequence; what a weight of
// zero makes NaN of it is put right by the join (kMark).
#include "lq4_attend_dev.cuh"

namespace lq4 {

namespace {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Byte offset of 16-byte chunk `c` of row `r` in a tile of D-element bf16 rows: the chunk's low bits are mixed
// with the row's, so that eight rows of one chunk (an ldmatrix) lie in eight different bank groups.
template <int D>
__device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t c) { return r * (D * 2) + ((c ^ (r & 7)) << 4); }

// More rows than this per kv head take the tcgen05 kernel.  16 sequences of 8192 tokens, 8 kv heads of 128 (B200), bf16: 16
// rows 108 us here and 126 us there, 25 rows 164 and 128 us, 64 rows 217 and 132 us; f32: 25 rows 238 and 304 us, 64
// rows 357 and 304 us, 128 rows 691 and 325 us.  (f32 and head_dim above 128: three terms of Q leave no room there.)
constexpr uint32_t kTcMinRows = 16, kTcMinRowsF32 = 32;

// WM bands of 16 rows, four warps on them (WN shares of the keys); NQ bf16 terms of q and P.
template <int D, int WM, int NQ>
struct Shape {
    static constexpr int WN = 4 / WM, BM = 16 * WM, NK = kKeys / WN;                  // NK keys of a warp
    static constexpr int kMath = 128, kLoaders = 128, NT = kMath + kLoaders;
    // two CTAs an SM where 128 registers a thread are enough
    static constexpr int kPerSm = D <= 128 && NQ == 1 ? 2 : 1;
    static constexpr uint32_t kSlot = kKeys * D * 2, kQ = NQ * BM * D * 2, kMeet = WN * BM * 36 * 4;
    static constexpr uint32_t kRest = 16 * 8 + 16 * 8 + kMaxNodes * 8 + WN * BM * 8 + 256 + 64 * 8;
    static constexpr uint32_t kFit = ((uint32_t)kMaxSmem / kPerSm - 1024 * (kPerSm - 1) - kQ - kMeet - kRest) / kSlot, kRing = kFit > 12 ? 12 : kFit;
    static constexpr uint32_t kTeams = kRing >= 8 ? 4 : 2, kTeam = 4 / kTeams;
    static constexpr uint32_t kOffQ = kRing * kSlot, kOffMeet = kOffQ + kQ, kValid = kOffMeet + kMeet, kFixes = kValid + 16 * 8, kAnc = kFixes + 16 * 8;
    static constexpr uint32_t kMl = kAnc + kMaxNodes * 8, kCtl = kMl + WN * BM * 8, kBars = kCtl + 256, kSmem = kBars + 64 * 8;
    static_assert(kRing >= 4 && kSmem <= (uint32_t)kMaxSmem / kPerSm, "shared memory");
};

template <int D, int WM, int NQ>
__global__ void __launch_bounds__((Shape<D, WM, NQ>::NT), (Shape<D, WM, NQ>::kPerSm)) attend_kernel(const __grid_constant__ AttendParams p) {
    using S = Shape<D, WM, NQ>;
    constexpr int WN = S::WN, BM = S::BM, NK = S::NK;
    constexpr uint32_t RING = S::kRing;
    extern __shared__ __align__(128) unsigned char smem[];
    volatile uint32_t* valid = reinterpret_cast<uint32_t*>(smem + S::kValid);    // [16][2] which of a tile's 64 keys there are
    volatile uint32_t* fixes = reinterpret_cast<uint32_t*>(smem + S::kFixes);    // [16][2] V of the tile held inf or NaN
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + S::kAnc);                 // [nodes] a node's path from the root
    float2* ml = reinterpret_cast<float2*>(smem + S::kMl);                       // [WN][BM] (max, sum)
    float* os = reinterpret_cast<float*>(smem + S::kOffMeet);                    // [WN][BM][36] 32 columns of O
    uint64_t* ctl = reinterpret_cast<uint64_t*>(smem + S::kCtl);
    uint64_t *full = reinterpret_cast<uint64_t*>(smem + S::kBars), *empty = full + RING, *info = empty + RING;
    const uint32_t sbase = smem_u32(smem), qbase = sbase + S::kOffQ;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const Range range = cta_range<S::NT>(p, ctl, ctl + 2);
    if (range.begin >= range.end) return;
    if (tid == 0) {
        for (uint32_t i = 0; i < RING; ++i) {
            mbar_init(full + i, S::kTeam);
            mbar_init(empty + i, S::kMath / 32);
        }
        for (int i = 0; i < 16; ++i) mbar_init(info + i, S::kTeam);
        mbar_fence_init();
        ctl[2] = range.begin;
    }
    __syncthreads();
    uint64_t u = range.begin, seq_first = range.seq_first;
    const uint64_t u_end = range.end;
    uint32_t b = range.seq;
    // Once a wait has run out the CTA goes on without waiting, so that its barriers still match; the results are
    // rubbish then, and reported.
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity);
    };

    if (tid >= S::kMath) {
        load_stream<D, RING, 1, S::kTeams, S::kTeam, kPieceTiles<NQ>>(p, u, u_end, b, seq_first, warp - S::kMath / 32, smem, full, empty, info, valid, fixes, ok,
                                                     [](uint32_t r, uint32_t c) { return tile_at<D>(r, c); });
        if (!ok) atomicOr(p.status, kDevErrBarrierTimeout);
        return;
    }

    const uint32_t wm = warp / WN, wn = warp % WN, quad = lane >> 2, qc = (lane & 3) * 2;
    uint32_t tile = 0, kslot = 0, phase = 0;                             // tiles so far, their K's slot (V: the next) and its phase
    while (u < u_end) {
        const Piece x = next_piece<kPieceTiles<NQ>>(p, u, u_end, b, seq_first);
        const Seq& sq = x.sq;
        const uint32_t h = x.h, rt = x.rt, t0 = x.t0, n_tiles = x.n_tiles;
        const uint32_t rows = p.nodes * p.group;
        if (sq.bad && tid == 0) atomicOr(p.status, kDevErrBadIndex);

        // q -> NQ bf16 terms in shared memory (rows behind the last one are zero)
#pragma unroll 4
        for (uint32_t i = tid; i < BM * (D / 2); i += S::kMath) {
            const uint32_t r = i / (D / 2), d = (i - r * (D / 2)) * 2, row = rt * BM + r;
            float q0 = 0.0f, q1 = 0.0f;
            if (row < rows && d < p.head_dim) {
                const uint32_t t = row / p.group, g = row - t * p.group;
                if ((int32_t)t < sq.nodes) {
                    const uint64_t at = b * p.q_batch + t * p.q_node + (uint64_t)(h * p.group + g) * p.q_head + d;
                    if constexpr (NQ == 1) {
                        q0 = bf16_to_f32(static_cast<const uint16_t*>(p.q)[at]);
                        q1 = bf16_to_f32(static_cast<const uint16_t*>(p.q)[at + 1]);
                    } else {
                        q0 = static_cast<const float*>(p.q)[at];
                        q1 = static_cast<const float*>(p.q)[at + 1];
                    }
                }
            }
            q0 *= p.q_sign;
            q1 *= p.q_sign;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const uint32_t w = split_pair(q0, q1);
                *reinterpret_cast<uint32_t*>(smem + S::kOffQ + n * (BM * D * 2) + tile_at<D>(r, d >> 3) + (d & 7) * 2) = w;
            }
        }
        if (x.has_nodes && tid < p.nodes) {
            bool bad = false;
            anc[tid] = node_path(p, b, tid, bad);
            if (bad && (int32_t)tid < sq.nodes) atomicOr(p.status, kDevErrBadIndex);
        }
        named_bar_sync(1, S::kMath);

        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        bool fix = false;                                                // a node's V holds inf or NaN

        for (uint32_t i = 0; i < n_tiles; ++i, ++tile) {
            const uint32_t vslot = kslot + 1 == RING ? 0 : kslot + 1, vphase = kslot + 1 == RING ? phase ^ 1 : phase;
            const uint32_t kst = sbase + kslot * S::kSlot, vst = sbase + vslot * S::kSlot;
            const bool own = t0 + i + 1 == sq.tiles;
            wait(info + (tile & 15), (tile >> 4) & 1);
            uint64_t see[2];
            see[0] = see[1] = (uint64_t)valid[(tile & 15) * 2 + 1] << 32 | valid[(tile & 15) * 2];
            if (own) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t t = (rt * BM + wm * 16 + quad + 8 * j) / p.group;
                    if (t < p.nodes) see[j] &= anc[t];
                }
            }
            wait(full + kslot, phase);
            __syncwarp();
            // scores of this warp's keys.  The tensor cores cut off what falls below their accumulator's last bit; with
            // f32 activations the leading term's sum is therefore taken every 32 channels and added in f32.
            float s[NK / 8][4];
#pragma unroll
            for (int j = 0; j < NK / 8; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
            {
                float part[NQ][NK / 8][4];
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int j = 0; j < NK / 8; ++j) part[n][j][0] = part[n][j][1] = part[n][j][2] = part[n][j][3] = 0.0f;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    uint32_t kf[NK / 16][4];
#pragma unroll
                    for (int j = 0; j < NK / 16; ++j)
                        ldsm4(kf[j], kst + tile_at<D>(wn * NK + j * 16 + (lane & 7) + (lane >> 4) * 8, 2 * ks + ((lane >> 3) & 1)));
#pragma unroll
                    for (int n = 0; n < NQ; ++n) {
                        uint32_t a[4];
                        ldsm4(a, qbase + n * (BM * D * 2) + tile_at<D>(wm * 16 + (lane & 15), 2 * ks + (lane >> 4)));
#pragma unroll
                        for (int j = 0; j < NK / 16; ++j) {
                            mma_bf16(NQ == 1 ? s[2 * j] : part[n][2 * j], a, kf[j][0], kf[j][1]);
                            mma_bf16(NQ == 1 ? s[2 * j + 1] : part[n][2 * j + 1], a, kf[j][2], kf[j][3]);
                        }
                    }
                    if (NQ > 1 && (ks & 1)) {
#pragma unroll
                        for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) s[j][e] += part[0][j][e], part[0][j][e] = 0.0f;
                    }
                }
                if constexpr (NQ > 1) {
#pragma unroll
                    for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[j][e] += part[1][j][e] + part[2][j][e];
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + kslot);
            if ((see[0] & see[1]) != ~0ull) {
#pragma unroll
                for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((see[e >> 1] >> (wn * NK + j * 8 + qc + (e & 1))) & 1)) s[j][e] = -INFINITY;
            }
            // Running maximum and sum, in units of log2.  The maximum is rounded once, to m; an exponent is one fused
            // operation from the unscaled score, so its error goes with its distance from the maximum.
            float base[2], corr[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float top = s[0][2 * r];
#pragma unroll
                for (int j = 0; j < NK / 8; ++j) top = fmaxf(top, fmaxf(s[j][2 * r], s[j][2 * r + 1]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(m[r], top * p.scale_log2);
                base[r] = top == -INFINITY ? 0.0f : top;
                corr[r] = exp2_fast(m[r] - base[r]);
                m[r] = top;
                l[r] *= corr[r];
            }
            if (NQ == 1 && __any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
#pragma unroll
                for (int d = 0; d < D / 8; ++d) {
                    o[d][0] *= corr[0];
                    o[d][1] *= corr[0];
                    o[d][2] *= corr[1];
                    o[d][3] *= corr[1];
                }
            }
#pragma unroll
            for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[j][e] = exp2_fast(fmaf(s[j][e], p.scale_log2, -base[e >> 1]));
                    l[e >> 1] += s[j][e];
                }
            wait(full + vslot, vphase);
            __syncwarp();
            if (own) fix = (fixes[(tile & 15) * 2] | (S::kTeam == 2 ? fixes[(tile & 15) * 2 + 1] : 0)) != 0;
            // O = corr O + P V, the tile's product in accumulators of its own for f32 activations (as above)
            uint32_t a[NK / 16][NQ][4];
#pragma unroll
            for (int j = 0; j < NK / 16; ++j)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int w = 0; w < 4; ++w) a[j][n][w] = split_pair(s[2 * j + (w >> 1)][2 * (w & 1)], s[2 * j + (w >> 1)][2 * (w & 1) + 1]);
#pragma unroll
            for (int dt = 0; dt < D / 16; ++dt) {
                float t[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
                for (int j = 0; j < NK / 16; ++j) {
                    uint32_t vf[4];
                    ldsm4_t(vf, vst + tile_at<D>(wn * NK + j * 16 + (lane & 15), 2 * dt + (lane >> 4)));
#pragma unroll
                    for (int n = NQ - 1; n >= 0; --n) {
                        mma_bf16(NQ == 1 ? o[2 * dt] : t[0], a[j][n], vf[0], vf[1]);
                        mma_bf16(NQ == 1 ? o[2 * dt + 1] : t[1], a[j][n], vf[2], vf[3]);
                    }
                }
                if constexpr (NQ > 1) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        o[2 * dt][e] = fmaf(o[2 * dt][e], corr[e >> 1], t[0][e]);
                        o[2 * dt + 1][e] = fmaf(o[2 * dt + 1][e], corr[e >> 1], t[1][e]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + vslot);
            kslot += 2;
            if (kslot >= RING) kslot -= RING, phase ^= 1;
        }

        // the warps of a band meet: common maximum, scaled O through shared memory 32 columns at a time, one sum over the shares
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if ((lane & 3) == 0) ml[wn * BM + wm * 16 + quad + 8 * r] = make_float2(m[r], l[r]);
        }
        named_bar_sync(1, S::kMath);
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * BM + wm * 16 + quad + 8 * r].x);
            f[r] = exp2_fast(m[r] - (top == -INFINITY ? 0.0f : top));
        }
        const Fate to = fate<NQ>(x, u, ctl[2]);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float2*>(os + (wn * BM + wm * 16 + quad + 8 * r) * 36 + j * 8 + qc) = make_float2(o[4 * c + j][2 * r] * f[r], o[4 * c + j][2 * r + 1] * f[r]);
            named_bar_sync(1, S::kMath);
            for (uint32_t i = tid; i < BM * 8; i += S::kMath) {
                const uint32_t r = i >> 3, d = c * 32 + (i & 7) * 4, row = rt * BM + r;
                const uint32_t t = row / p.group, g = row - t * p.group;
                if (row >= rows || (int32_t)t >= sq.nodes || d >= p.head_dim) continue;
                float top = -INFINITY, sum = 0.0f;
#pragma unroll
                for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * BM + r].x);
                const float safe = top == -INFINITY ? 0.0f : top;
                float y[4] = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < WN; ++w) {
                    const float2 e = ml[w * BM + r];
                    sum += e.y * exp2_fast(e.x - safe);
                    const float4 v = *reinterpret_cast<const float4*>(os + (w * BM + r) * 36 + (i & 7) * 4);
                    y[0] += v.x, y[1] += v.y, y[2] += v.z, y[3] += v.w;
                }
                float4* const part = reinterpret_cast<float4*>(p.part_o + ((uint64_t)to.slot * BM + r) * D + d);
                if (NQ == 1 && to.goes_on) {                             // (the same thread wrote it)
                    const float2 e = p.part_ml[(uint64_t)to.slot * BM + r];
                    const float all = fmaxf(top, e.x), base = all == -INFINITY ? 0.0f : all, f0 = exp2_fast(top - base), f1 = exp2_fast(e.x - base);
                    const float4 v = *part;
                    y[0] = y[0] * f0 + v.x * f1, y[1] = y[1] * f0 + v.y * f1, y[2] = y[2] * f0 + v.z * f1, y[3] = y[3] * f0 + v.w * f1;
                    sum = sum * f0 + e.y * f1;
                    top = all;
                }
                if (fix)
                    for (int e = 0; e < 4; ++e) y[e] += nonfinite_sum(p, x, anc[t], d + e);
                if (to.whole) {
                    const float inv = 1.0f / sum;
                    const uint64_t at = b * p.out_batch + t * p.out_node + (uint64_t)(h * p.group + g) * p.out_head + d;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if constexpr (NQ == 1)
                            static_cast<__nv_bfloat16*>(p.out)[at + e] = __float2bfloat16_rn(y[e] * inv);
                        else
                            static_cast<float*>(p.out)[at + e] = y[e] * inv;
                    }
                    if (d == 0 && !(sum > 0.0f)) mark(p, NQ == 1, at);
                } else {
                    *part = make_float4(y[0], y[1], y[2], y[3]);
                    if (NQ > 1 && d == 0) p.part_ml[(uint64_t)to.slot * BM + r] = make_float2(top, sum);
                }
            }
            named_bar_sync(1, S::kMath);                                 // the columns are read (at last: anc and ml, too)
        }
        if (NQ == 1 && !to.whole && tid < BM) {                          // (behind the last use of what pieces before have left)
            float2* const at = p.part_ml + (uint64_t)to.slot * BM + tid;
            const float2 before = to.goes_on ? *at : make_float2(-INFINITY, 0.0f);
            float top = before.x;
#pragma unroll
            for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * BM + tid].x);
            const float base = top == -INFINITY ? 0.0f : top;
            float sum = before.y * exp2_fast(before.x - base);
#pragma unroll
            for (int w = 0; w < WN; ++w) sum += ml[w * BM + tid].y * exp2_fast(ml[w * BM + tid].x - base);
            *at = make_float2(top, sum);
        }
        u += n_tiles;
    }
    if (!ok) atomicOr(p.status, kDevErrBarrierTimeout);
}

// Joins the partials of the items that a CTA border cut, the CTAs in order: W warps per row, which take every W-th of them and
// meet in shared memory (one row's partials may come from every CTA of the grid).  Then looks at every row's result (kMark).
template <int D, int W>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendParams p, uint32_t BM, int bf16_out) {
    constexpr int V = D / 32;
    __shared__ float part[W > 1 ? W : 1][D + 1];                         // O and, behind it, the sum
    const uint32_t lane = threadIdx.x & 31, w = W > 1 ? threadIdx.x >> 5 : 0;
    const uint32_t rows = p.nodes * p.group;
    const uint64_t id = W > 1 ? blockIdx.x : (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    if (id >= (uint64_t)p.batch * p.kv_heads * rows) return;
    const uint32_t row = (uint32_t)(id % rows);
    const uint64_t bh = id / rows;
    const uint32_t h = (uint32_t)(bh % p.kv_heads), b = (uint32_t)(bh / p.kv_heads);
    const uint32_t t = row / p.group, g = row - t * p.group, rt = row / BM, r = row - rt * BM;
    const Seq sq = sequence(p, b);
    if (sq.tiles == 0 || (int32_t)t >= sq.nodes) return;
    uint64_t before, total;
    warp_prefix(p, b, before, total);
    const uint64_t share = cta_share(total, p.grid);
    const uint64_t first = before + ((uint64_t)h * p.row_tiles + rt) * sq.tiles;
    const uint32_t c0 = (uint32_t)(first / share), c1 = (uint32_t)((first + sq.tiles - 1) / share);
    const uint64_t at = b * p.out_batch + t * p.out_node + (uint64_t)(h * p.group + g) * p.out_head + lane * V;
    uint32_t nans = 0;                                                   // this lane's columns that hold a NaN
    auto is_nan = [](uint32_t bits) { return (bits & 0x7fffffffu) > 0x7f800000u; };
    if (c0 == c1) {                                                      // one CTA had it all and wrote it
        if (w > 0) return;
        uint32_t got[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            got[k] = 0;
            if (lane * V + k < p.head_dim) got[k] = bf16_out ? (uint32_t)static_cast<const uint16_t*>(p.out)[at + k] << 16 : static_cast<const uint32_t*>(p.out)[at + k];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) nans |= (uint32_t)is_nan(got[k]) << k;
        if (__shfl_sync(0xffffffffu, got[0], 0) == kMark) {
            if (lane > 0) return;
            if (bf16_out)
                static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(NAN);
            else
                static_cast<float*>(p.out)[at] = NAN;
            return;
        }
    } else {
        // the CTA that has the item's first tile keeps it in its slot 1, the others in slot 0
        float top = -INFINITY;
        for (uint32_t c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.part_ml[(uint64_t)(2 * c + (c == c0)) * BM + r].x);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float safe = top == -INFINITY ? 0.0f : top;
        float acc[V], sum = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = 0.0f;
#pragma unroll 4
        for (uint32_t c = c0 + w; c <= c1; c += W) {
            const uint64_t slot = (uint64_t)(2 * c + (c == c0)) * BM + r;
            const float2 e = p.part_ml[slot];
            const float f = exp2_fast(e.x - safe);
            sum += e.y * f;
            const float* src = p.part_o + slot * D + lane * V;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] += src[k] * f;
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int k = 0; k < V; ++k) part[w][lane * V + k] = acc[k];
            if (lane == 0) part[w][D] = sum;
            __syncthreads();
            if (w > 0) return;
#pragma unroll
            for (int i = 1; i < W; ++i) {
                sum += part[i][D];
#pragma unroll
                for (int k = 0; k < V; ++k) acc[k] += part[i][lane * V + k];
            }
        }
        const float inv = 1.0f / sum;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (lane * V + k >= p.head_dim) break;
            if (bf16_out)
                static_cast<__nv_bfloat16*>(p.out)[at + k] = __float2bfloat16_rn(acc[k] * inv);
            else
                static_cast<float*>(p.out)[at + k] = acc[k] * inv;
            nans |= (uint32_t)(acc[k] != acc[k] && sum > 0.0f) << k;
        }
    }
    for (; nans; nans &= nans - 1) {
        const uint32_t k = __ffs(nans) - 1;
        Piece x;
        x.sq = sq, x.b = b, x.h = h;
        const float y = nonfinite_total(p, x, t, lane * V + k);
        if (y == 0.0f) continue;
        if (bf16_out)
            static_cast<__nv_bfloat16*>(p.out)[at + k] = __float2bfloat16_rn(y);
        else
            static_cast<float*>(p.out)[at + k] = y;
    }
}

template <int D, int WM, int NQ>
cudaError_t run(AttendParams p, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    using S = Shape<D, WM, NQ>;
    static DeviceOnce once;
    auto fn = attend_kernel<D, WM, NQ>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void*>(fn), S::kSmem, once);
    if (e != cudaSuccess) return e;
    p.grid = (uint32_t)(sm_count * S::kPerSm);
    p.row_tiles = (p.nodes * p.group + S::BM - 1) / S::BM;
    if (!attend_workspace(p, ws, S::BM, D)) return cudaSuccess;
    if ((e = attend_launch(fn, dim3(p.grid), S::NT, S::kSmem, use_pdl, s, p)) != cudaSuccess) return e;
    return launch_attend_join(p, S::BM, D, NQ == 1, ws, use_pdl, s);
}

// bf16 activations come here with up to 16 rows, f32 ones with up to 32 and, above a head_dim of 128, with any number (row tiles
// of 32).
template <int D>
cudaError_t run_rows(const AttendParams& p, bool f32, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    if (!f32) return run<D, 1, 1>(p, ws, sm_count, use_pdl, s);
    return p.nodes * p.group <= 16 ? run<D, 1, 3>(p, ws, sm_count, use_pdl, s) : run<D, 2, 3>(p, ws, sm_count, use_pdl, s);
}

template <int W>
auto join_kernel(uint32_t D) {
    return D == 64 ? attend_join_kernel<64, W> : D == 128 ? attend_join_kernel<128, W> : D == 192 ? attend_join_kernel<192, W> : attend_join_kernel<256, W>;
}

}  // namespace

cudaError_t launch_attend_join(const AttendParams& p, uint32_t rows, uint32_t D, bool bf16_out, AttendWorkspace& ws, int use_pdl, cudaStream_t s) {
    // a CTA per row where few rows share the grid's partials, else a warp per row
    const uint64_t all = (uint64_t)p.batch * p.kv_heads * p.nodes * p.group;
    const bool wide = all <= 8ull * p.grid;
    ws.launches = 2;
    return attend_launch(wide ? join_kernel<8>(D) : join_kernel<1>(D), dim3((unsigned)(wide ? all : (all + 7) / 8)), 256, 0, use_pdl, s, p, rows, (int)bf16_out);
}

cudaError_t launch_tree_attention(const lq4_tree_attention_args& a, AttendWorkspace& ws, int32_t* status, int sm_count, int use_pdl, cudaStream_t s) {
    AttendParams p{};
    p.c = cache_view(*a.cache);
    p.q = a.q;
    p.out = a.out;
    p.k = static_cast<const uint16_t*>(a.k);
    p.v = static_cast<const uint16_t*>(a.v);
    p.q_batch = a.q_batch, p.q_node = a.q_node, p.q_head = a.q_head;
    p.out_batch = a.out_batch, p.out_node = a.out_node, p.out_head = a.out_head;
    p.kv_batch = a.kv_batch, p.kv_node = a.kv_node, p.kv_head = a.kv_head;
    p.kv_lens = a.kv_lens;
    p.node_counts = a.node_counts;
    p.parents = a.parents;
    p.batch = a.cache->batch;
    p.nodes = a.nodes;
    p.kv_heads = a.cache->kv_heads;
    p.group = a.q_heads / a.cache->kv_heads;
    p.head_dim = a.cache->head_dim;
    // the scale's sign goes into q (a zero scale too), so that a larger product is a larger score
    p.q_sign = a.scale > 0.0f ? 1.0f : a.scale < 0.0f ? -1.0f : 0.0f;
    p.scale_log2 = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * 1.44269504088896340736f;
    p.status = status;
    const uintptr_t q_at = reinterpret_cast<uintptr_t>(a.q), out_at = reinterpret_cast<uintptr_t>(a.out);
    p.q_vec = !(q_at % 16 || a.q_batch % 8 || a.q_node % 8 || a.q_head % 8);
    p.out_vec = !(out_at % 16 || a.out_batch % 8 || a.out_node % 8 || a.out_head % 8);
    const bool f32 = a.dtype == LQ4_DTYPE_F32;
    ws.need = 0;
    ws.launches = 0;
    if (p.nodes * p.group > (f32 ? kTcMinRowsF32 : kTcMinRows) && (!f32 || p.head_dim <= 128)) return launch_attend_tc(p, f32, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 64) return run_rows<64>(p, f32, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 128) return run_rows<128>(p, f32, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 192) return run_rows<192>(p, f32, ws, sm_count, use_pdl, s);
    return run_rows<256>(p, f32, ws, sm_count, use_pdl, s);
}

}  // namespace lq4
