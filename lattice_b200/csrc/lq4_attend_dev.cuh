// What the kernels of lq4_tree_attention share: the lengths of the sequences, the cut of the work over the CTAs, small
// wrappers.  Included by lq4_attend.cu and lq4_attend_tc.cu only.
#pragma once

#include "lq4_attend.cuh"
#include "lq4_tc.cuh"

#include <cuda_bf16.h>

namespace lq4 {

constexpr uint32_t kKeys = 64;                 // keys per tile
constexpr uint32_t kMaxNodes = LQ4_MAX_TREE_NODES;
// Tiles of a piece, with bf16 activations.  Every MMA cuts off what falls below its accumulator's last bit, always towards zero:
// some 3e-7 of the sum a tile.  Left to one accumulator, O was 1.1e-3 low after 4096 tiles of tcgen05 and 3.2e-3 after 8192,
// more than the rounding of a bf16 result.  So the sum over a longer run of tiles is taken up in f32, where partials lie
// anyway.  (With f32 activations every tile's product is added up in f32.)
constexpr uint32_t kMaxPiece = 512;
template <int NQ>
constexpr uint32_t kPieceTiles = NQ == 1 ? kMaxPiece : 0xffffffffu;

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
    float q_sign, scale_log2;                  // scale = q_sign * scale_log2 / log2(e), scale_log2 > 0
    float* part_o;                             // [2 * grid][BM][D]
    float2* part_ml;                           // [2 * grid][BM] (max, sum)
    uint32_t grid;
    int32_t* status;
    bool q_vec, out_vec;                       // 16-byte accesses fit q / out
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
    return per ? per : 1;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// (a, b) -> one word of bf16 and what the rounding left of each.
__device__ __forceinline__ uint32_t split_pair(float& a, float& b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    a -= __low2float(t);
    b -= __high2float(t);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// A CTA's share of the range of all tiles, and the sequence its first tile lies in.
struct Range {
    uint64_t begin, end;                       // units; empty: nothing to do
    uint64_t seq_first;                        // unit that sequence `seq` starts at
    uint32_t seq;
};
// Called by all NT threads; `word2` holds two words, `warp_words` one per warp of shared memory, free to overwrite
// until the next barrier.
template <int NT>
__device__ __forceinline__ Range cta_range(const AttendParams& p, uint64_t* word2, uint64_t* warp_words) {
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint64_t items = (uint64_t)p.kv_heads * p.row_tiles;
    const uint32_t per = (p.batch + NT - 1) / NT, i0 = tid * per, i1 = min(i0 + per, p.batch);
    uint64_t mine = 0;
    for (uint32_t i = i0; i < i1; ++i) mine += sequence(p, i).tiles;
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += t;
    }
    if (lane == 31) warp_words[warp] = incl;
    __syncthreads();
    uint64_t before = incl - mine, total = 0;
    for (uint32_t w = 0; w < NT / 32; ++w) {
        if (w < warp) before += warp_words[w];
        total += warp_words[w];
    }
    total *= items;
    const uint64_t share = cta_share(total, p.grid);
    Range r;
    r.begin = min((uint64_t)blockIdx.x * share, total);
    r.end = min(r.begin + share, total);
    r.seq = 0;
    r.seq_first = 0;
    if (r.begin >= r.end) return r;                                      // (uniform over the CTA)
    if (r.begin >= before * items && r.begin < (before + mine) * items) {
        uint32_t i = i0;
        for (; i < i1; ++i) {
            const uint64_t t = sequence(p, i).tiles;
            if (r.begin < (before + t) * items) break;
            before += t;
        }
        word2[0] = i;
        word2[1] = before * items;
    }
    __syncthreads();
    r.seq = (uint32_t)word2[0];
    r.seq_first = word2[1];
    __syncthreads();
    return r;
}

// One piece of a CTA's range: at most kPieceTiles consecutive tiles of one item.
struct Piece {
    Seq sq;
    uint32_t b, h, rt, t0, n_tiles;
    bool has_nodes;                            // it ends with the nodes' own tile
};
// What becomes of a piece that starts at unit u, in the range that starts at unit `begin`.
struct Fate {
    bool whole;                                // the CTA has all of the item, and this is its end: the result
    bool goes_on;                              // the item's pieces before it lie in the slot as a partial
    uint32_t slot;                             // of the CTA's partials: 1 for an item whose first tile it has, else 0
};
template <int NQ>
__device__ __forceinline__ Fate fate(const Piece& x, uint64_t u, uint64_t begin) {
    if (NQ > 1) return {x.t0 == 0 && x.has_nodes, false, 2 * blockIdx.x + (x.t0 == 0 ? 1 : 0)};
    const bool from_first = u - x.t0 >= begin;                           // (the unit of the item's first tile)
    return {from_first && x.has_nodes, x.t0 > 0 && u > begin, 2 * blockIdx.x + (from_first ? 1 : 0)};
}
// The piece that unit `u` starts; moves the sequence cursor (b, seq_first) on to it.
template <uint32_t MOST>
__device__ __forceinline__ Piece next_piece(const AttendParams& p, uint64_t u, uint64_t u_end, uint32_t& b, uint64_t& seq_first) {
    const uint64_t items = (uint64_t)p.kv_heads * p.row_tiles;
    Piece x;
    x.sq = sequence(p, b);
    while (u >= seq_first + x.sq.tiles * items) {                        // (u lies before the end of all units)
        seq_first += x.sq.tiles * items;
        x.sq = sequence(p, ++b);
    }
    const uint32_t item = (uint32_t)((u - seq_first) / x.sq.tiles);
    x.t0 = (uint32_t)((u - seq_first) - (uint64_t)item * x.sq.tiles);
    x.b = b;
    x.h = item / p.row_tiles;
    x.rt = item - x.h * p.row_tiles;
    x.n_tiles = (uint32_t)min((uint64_t)min(x.sq.tiles - x.t0, MOST), u_end - u);
    x.has_nodes = x.t0 + x.n_tiles == x.sq.tiles;
    return x;
}

// A node's path from the root, itself included, as a bit mask; a parent that does not come before its node counts as none.
__device__ __forceinline__ uint64_t node_path(const AttendParams& p, uint32_t b, uint32_t node, bool& bad) {
    uint64_t path = 0;
    int32_t at = (int32_t)node;
    while (at >= 0) {
        path |= 1ull << at;
        int32_t up = p.parents ? p.parents[(uint64_t)b * p.nodes + at] : at - 1;
        if (up < -1 || up >= at) up = -1, bad = true;
        at = up;
    }
    return path;
}

// Clears non-finite entries of eight bf16 values; true if there were any.
__device__ __forceinline__ bool clear_nonfinite(uint4* at) {
    uint32_t x[4] = {at->x, at->y, at->z, at->w};
    bool hit = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if ((x[e] & 0x7f80u) == 0x7f80u) x[e] &= 0xffff0000u, hit = true;
        if ((x[e] & 0x7f800000u) == 0x7f800000u) x[e] &= 0x0000ffffu, hit = true;
    }
    if (hit) *at = make_uint4(x[0], x[1], x[2], x[3]);
    return hit;
}
// What the cleared entries of column d come to for a node with this path.
static __device__ __noinline__ float nonfinite_sum(const AttendParams& p, const Piece& x, uint64_t path, uint32_t d) {
    float sum = 0.0f;
    for (uint32_t j = 0; j < (uint32_t)x.sq.nodes; ++j)
        if ((path >> j) & 1) {
            const float y = bf16_to_f32(p.v[x.b * p.kv_batch + j * p.kv_node + x.h * p.kv_head + d]);
            if (!isfinite(y)) sum += y;
        }
    return sum;
}

// The infinities of cached V.  A weight that is zero in f32 (or in one of the bf16 terms it is split into) makes NaN of an
// infinity that the definition keeps.  attend_join_kernel looks at every result once more and writes what the column has in
// memory where a NaN came out.  A row whose weights are NaN themselves keeps its NaNs: the attention kernels, which write such a
// row whole, mark its first entry with a -NaN that no arithmetic gives.  (Nothing of this is in the loops over the keys.)
constexpr uint32_t kMark = 0xffc10000u;
__device__ __forceinline__ void mark(const AttendParams& p, bool bf16_out, uint64_t at) {
    if (bf16_out)
        static_cast<uint16_t*>(p.out)[at] = kMark >> 16;
    else
        static_cast<uint32_t*>(p.out)[at] = kMark;
}
// What the non-finite entries of column d come to for node t, over all keys that it sees: their sum, or 0 if there are none.
static __device__ __noinline__ float nonfinite_total(const AttendParams& p, const Piece& x, uint32_t t, uint32_t d) {
    constexpr uint32_t kAtATime = 8;
    bool bad = false;
    float sum = nonfinite_sum(p, x, node_path(p, x.b, t, bad), d);
    for (uint32_t key = 0; key < (uint32_t)x.sq.len && sum == sum; key += kAtATime) {
        float y[kAtATime];
#pragma unroll
        for (uint32_t i = 0; i < kAtATime; ++i) {
            const uint32_t k = key + i, entry = k / p.c.page_size;
            const int32_t page = k < (uint32_t)x.sq.len ? p.c.table[(uint64_t)x.b * p.c.max_pages + entry] : -1;
            y[i] = 0.0f;
            if ((uint32_t)page < p.c.pages)
                y[i] = bf16_to_f32(p.c.v[(uint32_t)page * p.c.page_stride + (k - entry * p.c.page_size) * p.c.slot_stride + x.h * p.c.head_stride + d]);
        }
#pragma unroll
        for (uint32_t i = 0; i < kAtATime; ++i)
            if (!isfinite(y[i])) sum += y[i];
    }
    return sum;
}

// ---- loaders --------------------------------------------------------------------
// The K and V rows of all tiles of a CTA's range, through cp.async into RINGS rings of RING slots (K and V of a tile in turn;
// tile n goes to ring n % RINGS), by TEAMS teams of TEAM warps that take the tiles in turn; warp `w` of them.  A lone warp
// pays some five cycles per dependent instruction and waits for its own copies; teams that each look up, copy and hand
// on whole tiles overlap all of it.  A lane holds where its keys lie; table index and slot advance without a division, and
// the page ids are fetched one turn ahead.  A team's next tile is at most a ring ahead of its last one, so that a slot's
// barrier is never two phases off.
//   full, empty   per slot: TEAM arrivals when it is filled; by the readers when it may be filled again
//   info          [16] by tile: TEAM arrivals when `valid` is there (which of the 64 keys there are, [16][2])
//   fixes         [16][2]: non-finite V entries of the nodes' tile were cleared; there when its V is
//   place(r, c)   byte offset of 16-byte chunk c of row r in a slot
template <int D, uint32_t RING, uint32_t RINGS, uint32_t TEAMS, uint32_t TEAM, uint32_t MOST, typename Place>
__device__ __forceinline__ void load_stream(const AttendParams& p, uint64_t u, uint64_t u_end, uint32_t b, uint64_t seq_first, uint32_t w, unsigned char* smem,
                                            uint64_t* full, uint64_t* empty, uint64_t* info, volatile uint32_t* valid, volatile uint32_t* fixes, bool& ok, Place place) {
    constexpr uint32_t CPR = D / 8, kWarps = TEAMS, kOn = kWarps * kKeys, kHold = 2 / TEAM, kCopies = kHold * CPR;
    static_assert(2 * TEAMS / RINGS <= RING && (TEAMS & (TEAMS - 1)) == 0, "a team's next tile is at most a ring ahead of its last one");
    const uint32_t lane = threadIdx.x & 31, sbase = smem_u32(smem);
    const uint32_t lw = w / TEAM, key0 = (w % TEAM) * 32;                // team; this warp's first key of a tile
    uint32_t tile = 0;                                                   // tiles before the current piece
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = mbar_wait(bar, parity);
    };
    struct Ring {
        uint32_t slot, phase;                                        // phase: of `empty` before the slot is filled again
        __device__ __forceinline__ void move(uint32_t groups) {
            slot += groups;
            while (slot >= RING) slot -= RING, phase ^= 1;
        }
    } kr{0, 1}, vr{1, 1};
    kr.move(2 * (lw / RINGS));
    vr.move(2 * (lw / RINGS));
    const uint32_t ring0 = RINGS == 2 ? (lw & 1) * RING : 0;         // (a team's tiles are all even or all odd)
    const uint32_t page_size = p.c.page_size, pages_on = kOn / page_size, slots_on = kOn - pages_on * page_size;
    while (u < u_end) {
        const Piece x = next_piece<MOST>(p, u, u_end, b, seq_first);
        const int32_t* const table = p.c.table + (uint64_t)x.b * p.c.max_pages;
        const uint32_t plain = x.n_tiles - x.has_nodes;              // tiles of cached keys in this piece
        uint32_t i = (lw - tile) & (kWarps - 1);
        struct Key {
            uint32_t key, entry, in_page;
            int32_t page;
        } k2[kHold];
        auto fetch = [&](Key& k) { k.page = i < plain && k.key < (uint32_t)x.sq.len ? table[k.entry] : -1; };
#pragma unroll
        for (uint32_t h = 0; h < kHold; ++h) {
            k2[h].key = (x.t0 + i) * kKeys + key0 + h * 32 + lane;
            k2[h].entry = k2[h].key / page_size;
            k2[h].in_page = k2[h].key - k2[h].entry * page_size;
            fetch(k2[h]);
        }
        while (i < x.n_tiles) {
            const uint32_t n = tile + i;
            const bool own = i == plain;
            uint64_t at[kHold];
            i += kWarps;
#pragma unroll
            for (uint32_t h = 0; h < kHold; ++h) {
                Key& k = k2[h];
                at[h] = ~0ull;
                if (own) {
                    const uint32_t node = key0 + h * 32 + lane;
                    if (node < (uint32_t)x.sq.nodes) at[h] = x.b * p.kv_batch + node * p.kv_node + x.h * p.kv_head;
                } else if (k.key < (uint32_t)x.sq.len) {
                    if ((uint32_t)k.page < p.c.pages)
                        at[h] = (uint32_t)k.page * p.c.page_stride + k.in_page * p.c.slot_stride + x.h * p.c.head_stride;
                    else
                        atomicOr(p.status, kDevErrBadIndex);
                }
                k.key += kOn;
                k.entry += pages_on;
                k.in_page += slots_on;
                if (k.in_page >= page_size) k.in_page -= page_size, ++k.entry;
                fetch(k);
            }
            __syncwarp();
#pragma unroll
            for (uint32_t h = 0; h < kHold; ++h) {
                const uint32_t bits = __ballot_sync(0xffffffffu, at[h] != ~0ull);
                if (lane == 0) valid[(n & 15) * 2 + key0 / 32 + h] = bits;
            }
            if (lane == 0) {
                fixes[(n & 15) * 2 + key0 / 32] = 0;
                mbar_arrive(info + (n & 15));
            }
            auto copy = [&](const uint16_t* base, const Ring& r, uint32_t group) {
                if (group >= RING) wait(empty + ring0 + r.slot, r.phase);
                __syncwarp();
                const uint32_t slot = sbase + (ring0 + r.slot) * (kKeys * D * 2);
#pragma unroll 8
                for (uint32_t c = 0; c < kCopies; ++c) {
                    const uint32_t idx = c * 32 + lane, row = idx / CPR, chunk = idx % CPR;      // (row < 32 or not: the same for all lanes)
                    const uint64_t from = __shfl_sync(0xffffffffu, c < CPR ? at[0] : at[kHold - 1], row & 31);
                    const bool here = from != ~0ull && chunk * 8 < p.head_dim;
                    cp_async16(slot + place(key0 + row, chunk), here ? base + from + chunk * 8 : p.k, here);
                }
                cp_commit();
            };
            copy(own ? p.k : p.c.k, kr, 2 * (n / RINGS));
            copy(own ? p.v : p.c.v, vr, 2 * (n / RINGS) + 1);
            cp_wait<1>();
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + ring0 + kr.slot);
            cp_wait<0>();
            if (own) {                                               // clear non-finite V of the nodes before it is used
                bool odd = false;
                __syncwarp();
                for (uint32_t c = 0; c < kCopies; ++c) {
                    const uint32_t idx = c * 32 + lane;
                    odd |= clear_nonfinite(reinterpret_cast<uint4*>(smem + (ring0 + vr.slot) * (kKeys * D * 2) + place(key0 + idx / CPR, idx % CPR)));
                }
                if (__any_sync(0xffffffffu, odd) && lane == 0) fixes[(n & 15) * 2 + key0 / 32] = 1;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + ring0 + vr.slot);
            kr.move(2 * kWarps / RINGS);
            vr.move(2 * kWarps / RINGS);
        }
        tile += x.n_tiles;
        u += x.n_tiles;
    }
}

// ---- host side --------------------------------------------------------------------
// Points p at the workspace for `grid` CTAs of `rows` rows of D channels; false (and ws.need set) if it is too small.
inline bool attend_workspace(AttendParams& p, AttendWorkspace& ws, uint32_t rows, uint32_t D) {
    const size_t slots = (size_t)2 * p.grid * rows, need = slots * (D * sizeof(float) + sizeof(float2));
    if (ws.bytes < need) {
        ws.need = need;
        return false;
    }
    p.part_ml = static_cast<float2*>(ws.p);
    p.part_o = reinterpret_cast<float*>(p.part_ml + slots);
    return true;
}
// lq4_attend.cu: joins the partials of a launch with items of `rows` rows and D channels; completes ws.launches.
cudaError_t launch_attend_join(const AttendParams& p, uint32_t rows, uint32_t D, bool bf16_out, AttendWorkspace& ws, int use_pdl, cudaStream_t s);
// lq4_attend_tc.cu: items of 128 or 256 rows; f32 activations up to head_dim 128.
cudaError_t launch_attend_tc(const AttendParams& p, bool f32, AttendWorkspace& ws, int sm_count, int use_pdl, cudaStream_t s);

}  // namespace lq4
