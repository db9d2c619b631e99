// Host-callable launchers of the kernels between the q/k/v projections and o_proj (rotary positions, cache
// append, attention over the cache) and behind lm_head (verification of drafted tokens).
#pragma once

#include "lq4_kernels.cuh"

namespace lq4 {

constexpr int kDevErrBadIndex = 8;      // a page id, length, count, parent or path entry outside its range

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Launches a kernel, with programmatic dependent launch if asked for.
template <typename... Args>
cudaError_t attend_launch(void (*fn)(Args...), dim3 grid, uint32_t threads, size_t smem, int use_pdl, cudaStream_t s, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = use_pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

// ---- lq4_rope.cu ----------------------------------------------------------------
// Arguments are validated by the caller (lq4_api.cu).
cudaError_t launch_rope_rows(const lq4_rope_args& a, int sm_count, int use_pdl, cudaStream_t s);
cudaError_t launch_kv_append(const lq4_kv_append_args& a, int32_t* status, int use_pdl, cudaStream_t s);

// A cache descriptor with its strides filled in.
struct CacheView {
    uint16_t* k;
    uint16_t* v;
    uint64_t page_stride, slot_stride, head_stride;
    const int32_t* table;
    uint32_t pages, page_size, max_pages;
};
inline CacheView cache_view(const lq4_kv_cache& c) {
    CacheView w;
    w.k = static_cast<uint16_t*>(c.k);
    w.v = static_cast<uint16_t*>(c.v);
    w.head_stride = c.head_stride ? c.head_stride : c.head_dim;
    w.slot_stride = c.slot_stride ? c.slot_stride : (uint64_t)c.kv_heads * c.head_dim;
    w.page_stride = c.page_stride ? c.page_stride : (uint64_t)c.page_size * c.kv_heads * c.head_dim;
    w.table = c.page_table;
    w.pages = c.pages;
    w.page_size = c.page_size;
    w.max_pages = c.max_pages;
    return w;
}

// ---- lq4_attend.cu --------------------------------------------------------------
// Partials of the items that are cut between CTAs.  A launch that needs more than `bytes` does nothing and sets
// `need`; its size depends on the device and the number of rows per kv head, not on the lengths.
struct AttendWorkspace {
    void* p;
    size_t bytes, need;
    int launches;
};
cudaError_t launch_tree_attention(const lq4_tree_attention_args& a, AttendWorkspace& ws, int32_t* status, int sm_count,
                                  int use_pdl, cudaStream_t s);

// ---- lq4_verify.cu --------------------------------------------------------------
// The row statistics of a small call (0 bytes: it takes none); `workspace` may be NULL where there is no room for them.
size_t verify_workspace_bytes(const lq4_verify_args& a, int sm_count);
cudaError_t launch_verify_draft(const lq4_verify_args& a, void* workspace, int32_t* status, int sm_count, int use_pdl, cudaStream_t s, int* launches);

}  // namespace lq4
