// Rotary positions of q / k (with v converted in the same launch) and the append of rows to a paged cache.
//
// Both are passes over memory: every element is read once and written once.
//
// rope_kernel: pair i of a head is a complex number turned by the angle pos * freq[i].  The angle of a far
// position does not fit f32 (at 10^6 radians its step is 2^-4 of a radian), so it is formed in f64 as a number of
// TURNS, its whole part is dropped there, and only the remainder in [-1/2, 1/2] goes to f32 and sincospi:
// three f64 operations per (row, pair), shared by the heads of a CTA through shared memory.  A CTA takes a
// few rows (256 angles, one per thread) and the heads of one tensor, or a slice of them when the rows alone would not
// fill the GPU; a thread keeps its place in the head and has 64 to 128 bytes of several heads under way at a time (V
// pairs per step: both halves are in its registers before it stores, so the call may work in place).  B200, device time: 4099
// rows of 32 heads of 256, bf16, 64 channels turned: 33 us (4.0 TB/s); 2047 rows of 56 heads of 128, f32: 27 us (4.3 TB/s).  What
// bounds it is latency at low occupancy: three CTAs an SM (78 registers, 35 % of the warps), issue active 66 and 40 %, the
// waits for loads and for the instruction before as large as one another, or the loads' alone.
//
// kv_append_kernel: 3 x 4001 rows of 4 heads of 256, f32 to a bf16 cache: 23 us (6.4 TB/s).
#include "lq4_attend.cuh"

#include <cuda_bf16.h>

namespace lq4 {

namespace {

constexpr uint32_t kRopeThreads = 256;

struct RopeParams {
    lq4_rope_part part[LQ4_MAX_ROPE_PARTS];
    uint32_t first_cta[LQ4_MAX_ROPE_PARTS];    // of a part, along grid.y
    uint32_t n_parts, rows, head_dim, half;    // half = rot_dim / 2
    uint32_t rows_per_cta, heads_per_cta;
    uint32_t lanes;                            // threads of a head, a power of two
    const int32_t* positions;
    const double* freq;
    int32_t interleaved;
    float scale;
};

// V consecutive elements of type T (float or bf16 bits): fetched as they lie in memory, and read as f32.
template <typename T, int V>
struct Raw {
    uint32_t w[V * sizeof(T) / 4 ? V * sizeof(T) / 4 : 1];
};
template <typename T, int V>
__device__ __forceinline__ void fetch_vec(const T* p, Raw<T, V>& r) {
    constexpr int kBytes = V * sizeof(T);
    if constexpr (kBytes >= 16) {
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) {
            const uint4 t = reinterpret_cast<const uint4*>(p)[i];
            r.w[4 * i] = t.x, r.w[4 * i + 1] = t.y, r.w[4 * i + 2] = t.z, r.w[4 * i + 3] = t.w;
        }
    } else if constexpr (kBytes == 8) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        r.w[0] = t.x, r.w[1] = t.y;
    } else if constexpr (kBytes == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        r.w[0] = (uint32_t)*reinterpret_cast<const uint16_t*>(p) << 16;
    }
}
template <typename T, int V>
__device__ __forceinline__ void read_vec(const Raw<T, V>& r, float (&v)[V]) {
    if constexpr (sizeof(T) == 4 || V == 1) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.w[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            v[2 * i] = __uint_as_float(r.w[i] << 16);
            v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
        }
    }
}
template <int V>
__device__ __forceinline__ void load_vec(const void* base, int dtype, uint64_t at, float (&v)[V]) {
    if (dtype == LQ4_DTYPE_F32) {
        Raw<float, V> r;
        fetch_vec<float, V>(static_cast<const float*>(base) + at, r);
        read_vec<float, V>(r, v);
    } else {
        Raw<uint16_t, V> r;
        fetch_vec<uint16_t, V>(static_cast<const uint16_t*>(base) + at, r);
        read_vec<uint16_t, V>(r, v);
    }
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&t);
}

template <int V>
__device__ __forceinline__ void store_vec(void* base, int dtype, uint64_t at, const float (&v)[V]) {
    if (dtype == LQ4_DTYPE_F32) {
        float* p = static_cast<float*>(base) + at;
        if constexpr (V >= 4) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i)
                reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        } else {
            p[0] = v[0];
        }
    } else {
        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + at;
        if constexpr (V == 8)
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
        else if constexpr (V == 4)
            *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]));
        else
            p[0] = __float2bfloat16_rn(v[0]);
    }
}

// The heads [head0, head0 + nheads) of one tensor, rows [row0, row0 + nrows): see above.
template <typename T, int V>
__device__ __forceinline__ void rope_heads(const RopeParams& p, const lq4_rope_part& t, const float2* cs, uint32_t row0, uint32_t nrows,
                                           uint32_t head0, uint32_t nheads) {
    constexpr int kItems = sizeof(T) == 4 ? 2 : 4;                        // (row, head) items of a thread at a time
    const bool turns = t.turn != 0;
    // units of a head: half / V pair units of 2V elements, then the copied tail (or all of the head) in units of V
    const uint32_t pair_units = turns ? p.half / V : 0, units = pair_units + (p.head_dim - 2 * V * pair_units) / V;
    const uint32_t step = kRopeThreads / p.lanes, off = p.interleaved ? V : p.half;
    const float sign = t.turn < 0 ? -1.0f : 1.0f;
    const T* const x = static_cast<const T*>(t.x) + row0 * t.x_row + head0 * t.x_head;
    const uint64_t out = row0 * t.out_row + head0 * t.out_head;
    for (uint32_t u = threadIdx.x & (p.lanes - 1); u < units; u += p.lanes) {
        const bool pair = u < pair_units;
        const uint32_t e = pair ? (p.interleaved ? 2 * u * V : u * V) : (u + pair_units) * V;
        uint32_t r = 0, h = threadIdx.x / p.lanes;
        while (h >= nheads) h -= nheads, ++r;
        while (r < nrows) {
            Raw<T, V> first[kItems], second[kItems];
            uint32_t row[kItems], head[kItems];
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                while (h >= nheads) h -= nheads, ++r;
                row[k] = r, head[k] = h;
                if (r < nrows) {
                    const T* src = x + r * t.x_row + h * t.x_head + e;
                    fetch_vec<T, V>(src, first[k]);
                    if (pair) fetch_vec<T, V>(src + off, second[k]);
                }
                h += step;
            }
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                if (row[k] >= nrows) break;
                const uint64_t dst = out + row[k] * t.out_row + head[k] * t.out_head + e;
                float a[V], b[V];
                read_vec<T, V>(first[k], a);
                if (pair) {
                    read_vec<T, V>(second[k], b);
                    const float2* c = cs + row[k] * p.half + u * V;
                    if (p.interleaved) {
                        // pairs (v[2i], v[2i + 1]) over the 2V consecutive elements a | b
                        float v[2 * V];
#pragma unroll
                        for (int j = 0; j < V; ++j) v[j] = a[j], v[V + j] = b[j];
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float cn = c[j].x, sn = c[j].y * sign, x1 = v[2 * j], x2 = v[2 * j + 1];
                            v[2 * j] = x1 * cn - x2 * sn;
                            v[2 * j + 1] = x1 * sn + x2 * cn;
                        }
#pragma unroll
                        for (int j = 0; j < V; ++j) a[j] = v[j], b[j] = v[V + j];
                    } else {
#pragma unroll
                        for (int j = 0; j < V; ++j) {
                            const float cn = c[j].x, sn = c[j].y * sign, x1 = a[j], x2 = b[j];
                            a[j] = x1 * cn - x2 * sn;
                            b[j] = x1 * sn + x2 * cn;
                        }
                    }
                    store_vec<V>(t.out, t.out_dtype, dst + off, b);
                }
                store_vec<V>(t.out, t.out_dtype, dst, a);
            }
            while (h >= nheads) h -= nheads, ++r;
        }
    }
}

template <int V>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const __grid_constant__ RopeParams p) {
    extern __shared__ float2 cs[];                                        // [rows_per_cta][half] (cos, sin), times scale
    uint32_t part = p.n_parts - 1;
    while (blockIdx.y < p.first_cta[part]) --part;
    const lq4_rope_part t = p.part[part];
    const uint32_t row0 = blockIdx.x * p.rows_per_cta, nrows = min(p.rows_per_cta, p.rows - row0);
    const uint32_t head0 = (blockIdx.y - p.first_cta[part]) * p.heads_per_cta, nheads = min(p.heads_per_cta, t.heads - head0);
    pdl_wait_prior_grids();
    if (t.turn != 0) {
        for (uint32_t i = threadIdx.x; i < nrows * p.half; i += kRopeThreads) {
            const uint32_t r = i / p.half, pair = i - r * p.half;
            double turns = (double)p.positions[row0 + r] * p.freq[pair] * 0.15915494309189533577;      // over 2 pi
            turns -= rint(turns);
            float sn, cn;
            sincospif(2.0f * (float)turns, &sn, &cn);
            cs[i] = make_float2(cn * p.scale, sn * p.scale);
        }
        __syncthreads();
    }
    if (t.x_dtype == LQ4_DTYPE_F32)
        rope_heads<float, V>(p, t, cs, row0, nrows, head0, nheads);
    else
        rope_heads<uint16_t, V>(p, t, cs, row0, nrows, head0, nheads);
    pdl_launch_dependents();
}

// One warp per (sequence, row), and per sequence where there are no rows (for the lengths): the page is looked up once, the lanes
// move K then V in 8-element pieces.
struct AppendParams {
    CacheView c;
    const void* k;
    const void* v;
    int32_t dtype;
    uint32_t batch, rows, kv_heads, head_dim;
    uint64_t batch_stride, row_stride, head_stride;
    const int32_t* kv_lens;
    const int32_t* counts;
    const int32_t* index;
    int32_t* new_lens;
    int32_t* status;
};

__global__ void __launch_bounds__(256) kv_append_kernel(const __grid_constant__ AppendParams p) {
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    pdl_wait_prior_grids();
    pdl_launch_dependents();
    const uint32_t per = max(p.rows, 1u);
    if (item >= (uint64_t)p.batch * per) return;
    const uint32_t b = (uint32_t)(item / per), j = (uint32_t)(item - (uint64_t)b * per);
    const int32_t len = p.kv_lens[b];
    int32_t count = p.counts ? p.counts[b] : (int32_t)p.rows;
    const int64_t capacity = (int64_t)p.c.max_pages * p.c.page_size;
    // what the lengths and counts hold out of range is reported, but for a sequence to leave alone
    bool bad = len >= 0 && (len > capacity || count < 0 || count > (int32_t)p.rows);
    count = len < 0 ? 0 : min(max(count, 0), (int32_t)p.rows);
    if (j == 0 && lane == 0 && p.new_lens)
        p.new_lens[b] = len < 0 ? len : (int32_t)min((int64_t)len + count, min(capacity, (int64_t)0x7fffffff));
    if ((int32_t)j < count) {
        const int64_t slot = (int64_t)len + j;
        const int32_t src = p.index ? p.index[item] : (int32_t)j;
        int32_t page = -1;
        if (slot < capacity) page = p.c.table[(uint64_t)b * p.c.max_pages + slot / p.c.page_size];
        if (page < 0 || (uint32_t)page >= p.c.pages || src < 0 || (uint32_t)src >= p.rows) {
            bad = true;
        } else {
            const uint64_t to = (uint64_t)page * p.c.page_stride + (uint64_t)(slot % p.c.page_size) * p.c.slot_stride;
            const uint64_t from = b * p.batch_stride + src * p.row_stride;
            const uint32_t vecs = p.head_dim / 8, total = p.kv_heads * vecs;
            for (uint32_t i = lane; i < total; i += 32) {
                const uint32_t h = i / vecs, e = (i - h * vecs) * 8;
                const uint64_t at = from + h * p.head_stride + e, dst = to + h * p.c.head_stride + e;
                float kx[8], vx[8];
                load_vec<8>(p.k, p.dtype, at, kx);
                load_vec<8>(p.v, p.dtype, at, vx);
                store_vec<8>(p.c.k, LQ4_DTYPE_BF16, dst, kx);
                store_vec<8>(p.c.v, LQ4_DTYPE_BF16, dst, vx);
            }
        }
    }
    if (bad && lane == 0) atomicOr(p.status, kDevErrBadIndex);
}

// Whether every part can be moved `vec` elements at a time.
bool vec_fits(const lq4_rope_args& a, uint32_t half, uint32_t vec) {
    if (half % vec || (a.head_dim - 2 * half) % vec || a.head_dim % vec) return false;
    for (uint32_t i = 0; i < a.n_parts; ++i) {
        const lq4_rope_part& t = a.parts[i];
        if (!t.heads) continue;
        if (t.x_row % vec || t.x_head % vec || t.out_row % vec || t.out_head % vec) return false;
        const uintptr_t xa = t.x_dtype == LQ4_DTYPE_F32 ? 16 : vec * 2, oa = t.out_dtype == LQ4_DTYPE_F32 ? 16 : vec * 2;
        if (reinterpret_cast<uintptr_t>(t.x) % xa || reinterpret_cast<uintptr_t>(t.out) % oa) return false;
    }
    return true;
}

}  // namespace

cudaError_t launch_rope_rows(const lq4_rope_args& a, int sm_count, int use_pdl, cudaStream_t s) {
    RopeParams p{};
    uint32_t heads = 0;
    for (uint32_t i = 0; i < a.n_parts; ++i) {
        if (!a.parts[i].heads) continue;
        p.part[p.n_parts++] = a.parts[i];
        heads += a.parts[i].heads;
    }
    p.rows = a.rows;
    p.head_dim = a.head_dim;
    p.positions = a.positions;
    if (a.rope) {
        p.half = a.rope->rot_dim / 2;
        p.freq = a.rope->freq;
        p.interleaved = a.rope->layout == LQ4_ROPE_INTERLEAVED;
        p.scale = a.rope->scale;
    }
    const uint32_t vec = vec_fits(a, p.half, 8) ? 8 : vec_fits(a, p.half, 4) ? 4 : 1;
    // one angle per thread, at most as many rows as there are; heads are split while the CTAs do not fill the GPU
    // four times over and a CTA still has a unit for every thread
    p.rows_per_cta = p.half ? kRopeThreads / p.half : 4;
    if (p.rows_per_cta == 0) p.rows_per_cta = 1;
    if (p.rows_per_cta > p.rows) p.rows_per_cta = p.rows;
    const uint32_t row_ctas = (p.rows + p.rows_per_cta - 1) / p.rows_per_cta;
    uint32_t splits = (4u * sm_count + row_ctas - 1) / row_ctas;
    const uint32_t units = p.rows_per_cta * heads * (p.head_dim / vec), most = (units + kRopeThreads - 1) / kRopeThreads;
    if (splits > most) splits = most;
    if (splits > heads) splits = heads;
    p.heads_per_cta = (heads + splits - 1) / splits;
    uint32_t ctas = 0;
    for (uint32_t i = 0; i < p.n_parts; ++i) {
        p.first_cta[i] = ctas;
        ctas += (p.part[i].heads + p.heads_per_cta - 1) / p.heads_per_cta;
    }
    p.lanes = 1;
    while (p.lanes < kRopeThreads && p.lanes < a.head_dim / vec) p.lanes <<= 1;
    const dim3 grid(row_ctas, ctas);
    const size_t smem = (size_t)p.rows_per_cta * p.half * sizeof(float2);
    auto fn = vec == 8 ? rope_kernel<8> : vec == 4 ? rope_kernel<4> : rope_kernel<1>;
    return attend_launch(fn, grid, kRopeThreads, smem, use_pdl, s, p);
}

cudaError_t launch_kv_append(const lq4_kv_append_args& a, int32_t* status, int use_pdl, cudaStream_t s) {
    AppendParams p{};
    p.c = cache_view(*a.cache);
    p.k = a.k;
    p.v = a.v;
    p.dtype = a.dtype;
    p.batch = a.cache->batch;
    p.rows = a.rows;
    p.kv_heads = a.cache->kv_heads;
    p.head_dim = a.cache->head_dim;
    p.batch_stride = a.batch_stride;
    p.row_stride = a.row_stride;
    p.head_stride = a.head_stride;
    p.kv_lens = a.kv_lens;
    p.counts = a.counts;
    p.index = a.index;
    p.new_lens = a.new_lens;
    p.status = status;
    const uint64_t items = (uint64_t)p.batch * (p.rows ? p.rows : 1);
    return attend_launch(kv_append_kernel, dim3((unsigned)((items + 7) / 8)), 256, 0, use_pdl, s, p);
}

}  // namespace lq4
