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
//   loads      cp.async, 16 bytes a lane, ST stages of K and V.  Every key's address is looked up on its own
//              (slot -> page), so pages of any size may end anywhere inside a tile; the lookups run a stage ahead.
//   math       mma.sync m16n8k16 on bf16.  K and V are bf16 in memory and exact.  q and the probabilities are one
//              bf16 term each for bf16 activations (both roundings are of the size of the output's own), and three
//              terms each (24 bits) for f32 ones, so that an f32 result keeps 32-bit accuracy.
//   warps      WM x WN: WM bands of 16 rows, WN shares of the 64 keys.  Each warp keeps its own running maximum,
//              sum and O over its keys; they meet in shared memory once per piece.
//
// A key that a row may not see contributes nothing whatever it holds: its score is replaced by -inf, and a
// non-finite V entry of a node (0 * inf would reach the rows that do not see it) is cleared in shared memory
// and added back at the end for the rows that do see it.
#include "lq4_attend.cuh"

#include <cuda_bf16.h>

#include <atomic>

namespace lq4 {

namespace {

constexpr uint32_t kKeys = 64;                 // keys per tile
constexpr uint32_t kMaxNodes = LQ4_MAX_TREE_NODES;
constexpr uint32_t kMinShare = 1;              // tiles a CTA takes at least

struct AttendParams {
    CacheView c;
    const void* q;
    void* out;
    const uint16_t* k;                         // the nodes' own rows
    const uint16_t* v;
    uint64_t q_batch, q_node, q_head, out_batch, out_node, out_head, kv_batch, kv_node, kv_head;
    const int32_t* kv_lens;
    const int32_t* node_counts;
    const int32_t* parents;
    uint32_t batch, nodes, group, kv_heads, head_dim, row_tiles;
    float scale_log2;                          // scale * log2(e)
    float* part_o;                             // [2 * grid][BM][D]
    float2* part_ml;                           // [2 * grid][BM] (max, sum)
    uint32_t grid;
    int32_t* status;
};

// What the lengths of sequence b come to: committed keys, live nodes, tiles.
struct Seq {
    int32_t len, nodes;
    uint32_t tiles;                            // key tiles of an item, the nodes' own tile last; 0: nothing to do
    bool bad;
};
__device__ __forceinline__ Seq sequence(const AttendParams& p, uint32_t b) {
    Seq s;
    s.len = p.kv_lens[b];
    s.nodes = p.node_counts ? p.node_counts[b] : (int32_t)p.nodes;
    s.bad = false;
    const int64_t cap = (int64_t)p.c.max_pages * p.c.page_size;
    if (s.len > cap) s.len = (int32_t)cap, s.bad = true;
    if (s.nodes > (int32_t)p.nodes) s.nodes = (int32_t)p.nodes, s.bad = true;
    s.tiles = (s.len < 0 || s.nodes <= 0) ? 0 : ((uint32_t)s.len + kKeys - 1) / kKeys + 1;
    return s;
}

// Units (tiles of all items) before sequence b and in all, by one warp.
__device__ __forceinline__ void warp_prefix(const AttendParams& p, uint32_t b, uint64_t& before, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 31;
    uint64_t x = 0, y = 0;
    for (uint32_t i = lane; i < p.batch; i += 32) {
        const uint64_t t = sequence(p, i).tiles;
        y += t;
        if (i < b) x += t;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    const uint64_t items = (uint64_t)p.kv_heads * p.row_tiles;
    before = x * items;
    total = y * items;
}

__device__ __forceinline__ uint64_t cta_share(uint64_t total, uint32_t grid) {
    const uint64_t per = (total + grid - 1) / grid;
    return per < kMinShare ? kMinShare : per;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// (a, b) -> one word of bf16 and what the rounding left of each.
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    a -= __low2float(t);
    b -= __high2float(t);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// Byte offset of 16-byte chunk `c` of row `r` in a tile of D-element bf16 rows: the chunk's low bits are mixed
// with the row's, so that eight rows of one chunk (an ldmatrix) lie in eight different bank groups.
template <int D>
__device__ __forceinline__ uint32_t tile_at(uint32_t r, uint32_t c) { return r * (D * 2) + ((c ^ (r & 7)) << 4); }

template <int D, int WM, int NQ>
struct Shape {
    static constexpr int WN = WM == 4 ? 2 : 4, NT = 32 * WM * WN, BM = 16 * WM;
    static constexpr int NK = kKeys / WN;                                         // keys of a warp
    static constexpr int ST = D == 64 ? 4 : D == 128 ? 3 : NQ * WM < 4 ? 3 : 2;  // stages that fit beside Q
    static constexpr uint32_t kTile = kKeys * D * 2, kStage = 2 * kTile;
    static constexpr uint32_t kQ = NQ * BM * D * 2;
    static constexpr uint32_t kOut = WN * BM * (D + 8) * 4;                       // merge area: stages, then Q
    static constexpr uint32_t kMain = ST * kStage + kQ > kOut ? ST * kStage + kQ : kOut;
    static constexpr uint32_t kOffs = kMain, kValid = kOffs + ST * kKeys * 8, kAnc = kValid + 8 * 8, kMl = kAnc + kMaxNodes * 8;
    static constexpr uint32_t kCtl = kMl + WN * BM * 8, kSmem = kCtl + 64;
    static_assert(kSmem <= (uint32_t)kMaxSmem, "shared memory");
};

template <int D, int WM, int NQ>
__global__ void __launch_bounds__((Shape<D, WM, NQ>::NT), 1) attend_kernel(const __grid_constant__ AttendParams p) {
    using S = Shape<D, WM, NQ>;
    constexpr int WN = S::WN, NT = S::NT, BM = S::BM, NK = S::NK, ST = S::ST, CPR = D / 8;
    extern __shared__ __align__(128) unsigned char smem[];
    uint64_t* offs = reinterpret_cast<uint64_t*>(smem + S::kOffs);      // [ST][64] element offset of a key's row, ~0: none
    uint64_t* valid = reinterpret_cast<uint64_t*>(smem + S::kValid);    // [8] which of the tile's keys there are
    uint64_t* anc = reinterpret_cast<uint64_t*>(smem + S::kAnc);        // [nodes] a node's path from the root
    float2* ml = reinterpret_cast<float2*>(smem + S::kMl);              // [WN][BM]
    uint64_t* ctl = reinterpret_cast<uint64_t*>(smem + S::kCtl);
    const uint32_t sbase = smem_u32(smem), qbase = sbase + ST * S::kStage;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp / WN, wn = warp % WN;
    const uint32_t quad = lane >> 2, qc = (lane & 3) * 2;

    pdl_wait_prior_grids();
    pdl_launch_dependents();
    // this CTA's units, and the sequence the first of them lies in
    const uint64_t items = (uint64_t)p.kv_heads * p.row_tiles;
    uint64_t u, u_end, seq_first;
    uint32_t b;
    {
        uint64_t* wsum = ctl + 2;                                        // (WM * WN <= 8 warps: 8 words would do; 4 used per half)
        const uint32_t per = (p.batch + NT - 1) / NT, i0 = tid * per, i1 = min(i0 + per, p.batch);
        uint64_t mine = 0;
        for (uint32_t i = i0; i < i1; ++i) mine += sequence(p, i).tiles;
        uint64_t incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= (uint32_t)o) incl += t;
        }
        uint64_t* wtot = reinterpret_cast<uint64_t*>(ml);                // one word per warp (ml is free here)
        if (lane == 31) wtot[warp] = incl;
        __syncthreads();
        uint64_t before = incl - mine, total = 0;
        for (uint32_t w = 0; w < (uint32_t)(WM * WN); ++w) {
            if (w < warp) before += wtot[w];
            total += wtot[w];
        }
        total *= items;
        const uint64_t share = cta_share(total, p.grid);
        u = (uint64_t)blockIdx.x * share;
        u_end = min(u + share, total);
        if (u >= u_end) return;                                          // (uniform over the CTA)
        if (u >= before * items && u < (before + mine) * items) {
            uint32_t i = i0;
            for (; i < i1; ++i) {
                const uint64_t t = sequence(p, i).tiles;
                if (u < (before + t) * items) break;
                before += t;
            }
            wsum[0] = i;
            wsum[1] = before * items;
        }
        __syncthreads();
        b = (uint32_t)wsum[0];
        seq_first = wsum[1];
    }

    while (u < u_end) {
        Seq sq = sequence(p, b);
        if (sq.tiles == 0 || u >= seq_first + sq.tiles * items) {        // on to the next sequence
            seq_first += sq.tiles * items;
            ++b;
            continue;
        }
        const uint32_t in_seq_item = (uint32_t)((u - seq_first) / sq.tiles);
        const uint32_t t0 = (uint32_t)((u - seq_first) - (uint64_t)in_seq_item * sq.tiles);
        const uint32_t h = in_seq_item / p.row_tiles, rt = in_seq_item - h * p.row_tiles;
        const uint32_t n_tiles = (uint32_t)min((uint64_t)(sq.tiles - t0), u_end - u);
        const bool has_nodes = t0 + n_tiles == sq.tiles;                 // this piece ends with the nodes' own tile
        const uint32_t rows = p.nodes * p.group;
        if (sq.bad && tid == 0) atomicOr(p.status, kDevErrBadIndex);

        // q -> NQ bf16 terms in shared memory (rows behind the last one are zero)
        for (uint32_t i = tid; i < BM * (D / 2); i += NT) {
            const uint32_t r = i / (D / 2), d = (i - r * (D / 2)) * 2, row = rt * BM + r;
            float x = 0.0f, y = 0.0f;
            if (row < rows && d < p.head_dim) {
                const uint32_t t = row / p.group, g = row - t * p.group;
                if ((int32_t)t < sq.nodes) {
                    const uint64_t at = b * p.q_batch + t * p.q_node + (uint64_t)(h * p.group + g) * p.q_head + d;
                    if constexpr (NQ == 1) {
                        x = bf16_to_f32(static_cast<const uint16_t*>(p.q)[at]);
                        y = bf16_to_f32(static_cast<const uint16_t*>(p.q)[at + 1]);
                    } else {
                        x = static_cast<const float*>(p.q)[at];
                        y = static_cast<const float*>(p.q)[at + 1];
                    }
                }
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const uint32_t w = split_pair(x, y);
                *reinterpret_cast<uint32_t*>(smem + ST * S::kStage + n * (BM * D * 2) + tile_at<D>(r, d >> 3) + (d & 7) * 2) = w;
            }
        }
        if (has_nodes && tid < p.nodes) {
            uint64_t path = 0;
            int32_t at = (int32_t)tid;
            bool bad = false;
            while (at >= 0) {
                path |= 1ull << at;
                int32_t up = p.parents ? p.parents[(uint64_t)b * p.nodes + at] : at - 1;
                if (up < -1 || up >= at) up = -1, bad = (int32_t)tid < sq.nodes;   // a parent comes before its children
                at = up;
            }
            anc[tid] = path;
            if (bad) atomicOr(p.status, kDevErrBadIndex);
        }

        // where the keys of tile `i` of this piece lie; page ids come from memory, so this runs a stage ahead
        auto key_page = [&](uint32_t i) -> int32_t {                     // (threads 0..63)
            const uint32_t key = (t0 + i) * kKeys + tid;
            if (i >= n_tiles || t0 + i + 1 == sq.tiles || key >= (uint32_t)sq.len) return -1;
            return p.c.table[(uint64_t)b * p.c.max_pages + key / p.c.page_size];
        };
        auto put_keys = [&](uint32_t i, int32_t page) {
            const uint32_t key = (t0 + i) * kKeys + tid;
            uint64_t at = ~0ull;
            if (i >= n_tiles) {                                          // (belongs to the next CTA)
            } else if (t0 + i + 1 == sq.tiles) {
                if ((int32_t)tid < sq.nodes) at = b * p.kv_batch + tid * p.kv_node + h * p.kv_head;
            } else if (key < (uint32_t)sq.len) {
                if (page < 0 || (uint32_t)page >= p.c.pages)
                    atomicOr(p.status, kDevErrBadIndex);
                else
                    at = (uint64_t)page * p.c.page_stride + (uint64_t)(key % p.c.page_size) * p.c.slot_stride + h * p.c.head_stride;
            }
            offs[(i % ST) * kKeys + tid] = at;
            const uint32_t bits = __ballot_sync(0xffffffffu, at != ~0ull);
            if (lane == 0) reinterpret_cast<uint32_t*>(valid + (i & 7))[warp] = bits;
        };
        auto load_tile = [&](uint32_t i) {
            if (i < n_tiles) {
                const bool own = t0 + i + 1 == sq.tiles;
                const uint16_t* kb = own ? p.k : p.c.k;
                const uint16_t* vb = own ? p.v : p.c.v;
                const uint32_t stage = sbase + (i % ST) * S::kStage;
#pragma unroll
                for (uint32_t n = 0; n < kKeys * CPR / NT; ++n) {
                    const uint32_t idx = n * NT + tid, r = idx / CPR, c = idx % CPR;
                    const uint64_t at = offs[(i % ST) * kKeys + r];
                    const bool live = at != ~0ull && c * 8 < p.head_dim;
                    const uint32_t dst = stage + tile_at<D>(r, c);
                    cp_async16(dst, live ? kb + at + c * 8 : p.k, live);
                    cp_async16(dst + S::kTile, live ? vb + at + c * 8 : p.k, live);
                }
            }
            cp_commit();
        };
        if (tid < kKeys) {
            int32_t page[ST];
#pragma unroll
            for (int i = 0; i < ST; ++i) page[i] = key_page(i);
#pragma unroll
            for (int i = 0; i < ST; ++i) put_keys(i, page[i]);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) load_tile(i);

        float o[D / 8][4];
#pragma unroll
        for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        bool fix = false;                                                // a node's V holds inf or NaN

        for (uint32_t i = 0; i < n_tiles; ++i) {
            cp_wait<ST - 2>();
            __syncthreads();                                             // tile i is here; everybody is done with tile i - 1
            load_tile(i + ST - 1);
            int32_t page = -1;
            if (tid < kKeys) page = key_page(i + ST);
            const uint32_t kst = sbase + (i % ST) * S::kStage, vst = kst + S::kTile;
            const bool own = t0 + i + 1 == sq.tiles;
            uint64_t see[2];
            see[0] = see[1] = valid[i & 7];
            if (own) {
                bool odd = false;                                        // clear non-finite V entries of the nodes
                for (uint32_t idx = tid; idx < kKeys * CPR; idx += NT) {
                    uint4* w = reinterpret_cast<uint4*>(smem + (vst - sbase) + idx * 16);
                    uint32_t x[4] = {w->x, w->y, w->z, w->w};
                    bool hit = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u, hit = true;
                        if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0x0000ffffu, hit = true;
                    }
                    if (hit) *w = make_uint4(x[0], x[1], x[2], x[3]), odd = true;
                }
                fix = __syncthreads_or(odd);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t t = (rt * BM + wm * 16 + quad + 8 * j) / p.group;
                    if (t < p.nodes) see[j] &= anc[t];
                }
            }
            // scores of this warp's keys
            float s[NK / 8][4];
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
                            mma_bf16(part[n][2 * j], a, kf[j][0], kf[j][1]);
                            mma_bf16(part[n][2 * j + 1], a, kf[j][2], kf[j][3]);
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = part[NQ - 1][j][e];
#pragma unroll
                        for (int n = NQ - 2; n >= 0; --n) x += part[n][j][e];
                        s[j][e] = x * p.scale_log2;
                    }
            }
            if ((see[0] & see[1]) != ~0ull) {
#pragma unroll
                for (int j = 0; j < NK / 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!((see[e >> 1] >> (wn * NK + j * 8 + qc + (e & 1))) & 1)) s[j][e] = -INFINITY;
            }
            // running maximum and sum
            float base[2], corr[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float x = m[r];
#pragma unroll
                for (int j = 0; j < NK / 8; ++j) x = fmaxf(x, fmaxf(s[j][2 * r], s[j][2 * r + 1]));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
                base[r] = x == -INFINITY ? 0.0f : x;
                corr[r] = exp2_fast(m[r] - base[r]);
                m[r] = x;
                l[r] *= corr[r];
            }
            if (__any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f)) {
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
                    s[j][e] = exp2_fast(s[j][e] - base[e >> 1]);
                    l[e >> 1] += s[j][e];
                }
            // O += P V
#pragma unroll
            for (int j = 0; j < NK / 16; ++j) {
                uint32_t a[NQ][4];
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int w = 0; w < 4; ++w) a[n][w] = split_pair(s[2 * j + (w >> 1)][2 * (w & 1)], s[2 * j + (w >> 1)][2 * (w & 1) + 1]);
#pragma unroll
                for (int dt = 0; dt < D / 16; ++dt) {
                    uint32_t vf[4];
                    ldsm4_t(vf, vst + tile_at<D>(wn * NK + j * 16 + (lane & 15), 2 * dt + (lane >> 4)));
#pragma unroll
                    for (int n = NQ - 1; n >= 0; --n) {
                        mma_bf16(o[2 * dt], a[n], vf[0], vf[1]);
                        mma_bf16(o[2 * dt + 1], a[n], vf[2], vf[3]);
                    }
                }
            }
            if (tid < kKeys) put_keys(i + ST, page);
        }
        cp_wait<0>();

        // the warps of a band meet: common maximum, scaled O to shared memory, one sum over the shares
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if ((lane & 3) == 0) ml[wn * BM + wm * 16 + quad + 8 * r] = make_float2(m[r], l[r]);
        }
        __syncthreads();                                                 // (everybody is done with the stages and Q, too)
        float* os = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const uint32_t row = wm * 16 + quad + 8 * r;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * BM + row].x);
            const float f = exp2_fast(m[r] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
            for (int d = 0; d < D / 8; ++d)
                *reinterpret_cast<float2*>(os + (wn * BM + row) * (D + 8) + d * 8 + qc) = make_float2(o[d][2 * r] * f, o[d][2 * r + 1] * f);
        }
        __syncthreads();
        const bool whole = t0 == 0 && has_nodes;
        const uint32_t slot = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);
        for (uint32_t i = tid; i < BM * (D / 4); i += NT) {
            const uint32_t r = i / (D / 4), d = (i - r * (D / 4)) * 4, row = rt * BM + r;
            const uint32_t t = row / p.group, g = row - t * p.group;
            if (row >= rows || (int32_t)t >= sq.nodes || d >= p.head_dim) continue;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < WN; ++w) top = fmaxf(top, ml[w * BM + r].x);
            const float safe = top == -INFINITY ? 0.0f : top;
            float x[4] = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < WN; ++w) {
                const float2 e = ml[w * BM + r];
                sum += e.y * exp2_fast(e.x - safe);
                const float4 y = *reinterpret_cast<const float4*>(os + (w * BM + r) * (D + 8) + d);
                x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
            }
            if (fix) {
                for (uint32_t j = 0; j < (uint32_t)sq.nodes; ++j)
                    if ((anc[t] >> j) & 1)
                        for (int e = 0; e < 4; ++e) {
                            const float y = bf16_to_f32(p.v[b * p.kv_batch + j * p.kv_node + h * p.kv_head + d + e]);
                            if (!isfinite(y)) x[e] += y;
                        }
            }
            if (whole) {
                const float inv = 1.0f / sum;
                const uint64_t at = b * p.out_batch + t * p.out_node + (uint64_t)(h * p.group + g) * p.out_head + d;
                for (int e = 0; e < 4; ++e) {
                    if constexpr (NQ == 1)
                        static_cast<__nv_bfloat16*>(p.out)[at + e] = __float2bfloat16_rn(x[e] * inv);
                    else
                        static_cast<float*>(p.out)[at + e] = x[e] * inv;
                }
            } else {
                *reinterpret_cast<float4*>(p.part_o + ((uint64_t)slot * BM + r) * D + d) = make_float4(x[0], x[1], x[2], x[3]);
                if (d == 0) p.part_ml[(uint64_t)slot * BM + r] = make_float2(top, sum);
            }
        }
        __syncthreads();                                                 // shared memory is free for the next piece
        u += n_tiles;
    }
}

// Joins the partials of the items that a CTA border cut: one warp per row, the CTAs in order.
template <int D, int BM>
__global__ void __launch_bounds__(256) attend_join_kernel(const __grid_constant__ AttendParams p, int bf16_out) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t rows = p.nodes * p.group;
    const uint64_t id = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
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
    if (c0 == c1) return;                                                // one CTA had it all and wrote it
    // the CTA that has the item's first tile keeps it in its slot 1, the others in slot 0
    constexpr int V = D / 32;
    float top = -INFINITY;
    for (uint32_t c = c0 + lane; c <= c1; c += 32) top = fmaxf(top, p.part_ml[(uint64_t)(2 * c + (c == c0)) * BM + r].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float safe = top == -INFINITY ? 0.0f : top;
    float acc[V], sum = 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
#pragma unroll 4
    for (uint32_t c = c0; c <= c1; ++c) {
        const uint64_t slot = (uint64_t)(2 * c + (c == c0)) * BM + r;
        const float2 e = p.part_ml[slot];
        const float f = exp2_fast(e.x - safe);
        sum += e.y * f;
        const float* src = p.part_o + slot * D + lane * V;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += src[k] * f;
    }
    const float inv = 1.0f / sum;
    const uint64_t at = b * p.out_batch + t * p.out_node + (uint64_t)(h * p.group + g) * p.out_head + lane * V;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        if (lane * V + k >= p.head_dim) break;
        if (bf16_out)
            static_cast<__nv_bfloat16*>(p.out)[at + k] = __float2bfloat16_rn(acc[k] * inv);
        else
            static_cast<float*>(p.out)[at + k] = acc[k] * inv;
    }
}

template <int D, int WM, int NQ>
cudaError_t run(AttendParams p, const lq4_tree_attention_args& a, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    using S = Shape<D, WM, NQ>;
    static DeviceOnce once;
    auto fn = attend_kernel<D, WM, NQ>;
    cudaError_t e = opt_in_smem(reinterpret_cast<const void*>(fn), S::kSmem, once);
    if (e != cudaSuccess) return e;
    static std::atomic<int> resident{0};       // CTAs an SM holds at once
    int per_sm = resident.load(std::memory_order_relaxed);
    if (!per_sm) {
        if ((e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fn, S::NT, S::kSmem)) != cudaSuccess) return e;
        if (per_sm < 1) per_sm = 1;
        resident.store(per_sm, std::memory_order_relaxed);
    }
    p.grid = (uint32_t)(sm_count * per_sm);
    p.row_tiles = (p.nodes * p.group + S::BM - 1) / S::BM;
    const size_t slots = (size_t)2 * p.grid * S::BM;
    const size_t need = slots * (D * 4 + 8);
    if (ws.bytes < need) {
        ws.need = need;
        return cudaSuccess;
    }
    p.part_ml = static_cast<float2*>(ws.p);
    p.part_o = reinterpret_cast<float*>(p.part_ml + slots);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.grid);
    cfg.blockDim = dim3(S::NT);
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, fn, p);
    if (e != cudaSuccess) return e;
    const uint64_t warps = (uint64_t)p.batch * p.kv_heads * p.nodes * p.group;
    cfg.gridDim = dim3((unsigned)((warps + 7) / 8));
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, attend_join_kernel<D, S::BM>, p, (int)(NQ == 1));
    ws.launches = 2;
    return e;
}

template <int D, int NQ>
cudaError_t run_rows(const AttendParams& p, const lq4_tree_attention_args& a, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    // bands of 16 rows: as few as hold the rows of an item, at most four (more rows: several row tiles)
    const uint32_t rows = p.nodes * p.group;
    if (rows <= 16) return run<D, 1, NQ>(p, a, ws, sm_count, use_pdl, s);
    if (rows <= 32) return run<D, 2, NQ>(p, a, ws, sm_count, use_pdl, s);
    return run<D, 4, NQ>(p, a, ws, sm_count, use_pdl, s);
}

template <int NQ>
cudaError_t run_dim(const AttendParams& p, const lq4_tree_attention_args& a, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s) {
    if (p.head_dim <= 64) return run_rows<64, NQ>(p, a, ws, sm_count, use_pdl, s);
    if (p.head_dim <= 128) return run_rows<128, NQ>(p, a, ws, sm_count, use_pdl, s);
    return run_rows<256, NQ>(p, a, ws, sm_count, use_pdl, s);
}

}  // namespace

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
    p.scale_log2 = a.scale * 1.44269504088896340736f;
    p.status = status;
    ws.need = 0;
    ws.launches = 0;
    return a.dtype == LQ4_DTYPE_BF16 ? run_dim<1>(p, a, ws, sm_count, use_pdl, s) : run_dim<3>(p, a, ws, sm_count, use_pdl, s);
}

}  // namespace lq4
