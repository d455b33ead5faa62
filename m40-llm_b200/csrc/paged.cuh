// The paged cache as the kernels see it, and the checks that its entry points share.
#pragma once
#include "common.cuh"

struct PagedView {
    unsigned char* k;
    unsigned char* v;
    const uint32_t* table;
    uint32_t pages, slots, max_pages, kv_heads, hd;
    uint32_t shift;  // log2 of the entries per page
};

constexpr uint32_t PAGED_NONE = 0xffffffffu;
constexpr uint32_t PAGED_MAX_HEAD_DIM = 512;
constexpr size_t PAGED_SCRATCH_MOST = (size_t)1 << 62;  // bytes that a call may ask for before its size could pass 64 bits; what a device has is less

// Page of entry e of a slot, or PAGED_NONE for one outside the pool; the slot and the entry are inside the cache.
__device__ __forceinline__ uint32_t paged_page(const PagedView& c, uint32_t slot, uint32_t e) {
    const uint32_t page = c.table[(size_t)slot * c.max_pages + (e >> c.shift)];
    return page < c.pages ? page : PAGED_NONE;
}
// Element offset of an entry's row for one kv head.
__device__ __forceinline__ size_t paged_row(const PagedView& c, uint32_t page, uint32_t head, uint32_t e) {
    return ((((size_t)page * c.kv_heads + head) << c.shift) + (e & ((1u << c.shift) - 1u))) * c.hd;
}
__host__ __device__ __forceinline__ uint32_t paged_capacity(const PagedView& c) { return c.max_pages << c.shift; }

// 0 and the view, or the return code for the caller.
static inline int m40_paged_view(const M40llmPagedCache* c, PagedView* out) {
    if (!c || !c->k || !c->v || !c->table) return -1;
    if (c->pages == 0 || c->slots == 0 || c->max_pages == 0 || c->kv_heads == 0 || c->head_dim == 0) return -2;
    if (c->page_tokens == 0 || (c->page_tokens & (c->page_tokens - 1u)) != 0) return -2;
    if (c->elem_dtype != M40LLM_DT_F16 && c->elem_dtype != M40LLM_DT_F32) return -4;
    if (c->page_tokens > 4096u || c->head_dim > PAGED_MAX_HEAD_DIM || c->kv_heads > 65535u ||
        (uint64_t)c->max_pages * c->page_tokens > (1ull << 30))
        return M40LLM_ERR_LIMIT;
    const uintptr_t elem = c->elem_dtype == M40LLM_DT_F16 ? 2u : 4u;
    if ((((uintptr_t)c->k | (uintptr_t)c->v) & (elem - 1u)) != 0) return -2;
    uint32_t shift = 0;
    while ((1u << shift) < c->page_tokens) ++shift;
    *out = PagedView{(unsigned char*)c->k, (unsigned char*)c->v, c->table, c->pages, c->slots, c->max_pages, c->kv_heads, c->head_dim, shift};
    return 0;
}

// Rows of hd elements of `elem` bytes can be moved in 16-byte pieces.
static inline bool m40_paged_vec16(const M40llmPagedCache* c) {
    const uint32_t elem = c->elem_dtype == M40LLM_DT_F16 ? 2u : 4u;
    return ((((uintptr_t)c->k) | ((uintptr_t)c->v)) & 15u) == 0 && (c->head_dim * elem) % 16u == 0;
}
