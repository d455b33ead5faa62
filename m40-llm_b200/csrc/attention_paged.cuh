// What the kernels of attention over a paged cache share: their arguments, and the list of work that resident CTAs take equal runs of.
#pragma once
#include "attention_mma.cuh"
#include "paged.cuh"
#include "paged_list.cuh"

struct PagedAttnArgs {
    PagedView c;
    const float* q;
    float* out;
    const uint32_t* row_slot;
    const uint32_t* row_len;
    const uint32_t* row_begin;
    const float* weights_in;
    float* weights_out;
    float* part_m;  // [rows][q_heads][splits], base 2
    float* part_l;
    float* part_o;  // [rows][q_heads][splits][hd]
    float* scores;  // [rows][q_heads][ld_scores] in base 2, or null
    float* stat;    // [rows][q_heads][2]: maximum, 1 / sum (0 for a row without entries), where scores are kept
    uint32_t* status;
    uint64_t* prefix;  // tiles before each row of the launch, [rows + 1]
    uint32_t rows, q_heads, group, splits, chunk, bound, ld_weights, ld_scores;
    uint32_t row0, heads_at_once, workers, part_warps;  // first row of the launch, q heads of one unit of work, resident CTAs, warps of each
    float scale;  // times log2(e)
};

// The entries [begin, end) of a row; false for a row outside the cache.
__device__ __forceinline__ bool paged_row_range(const PagedAttnArgs& a, uint32_t row, uint32_t* slot, uint32_t* begin, uint32_t* end) {
    *slot = a.row_slot[row];
    *end = a.row_len[row];
    *begin = a.row_begin ? a.row_begin[row] : 0u;
    return *slot < a.c.slots && *end <= a.bound;
}
// 16 bytes by cp.async; zeros where `bytes` is 0 (the source is then not read)
__device__ __forceinline__ void cp_async16_or_zero(uint32_t smem, const void* gmem, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes));
}
// The work of a launch is a list of tiles: rows in order, in a row the units of up to heads_at_once q heads of one kv head, in a unit its tiles of `span`
// entries (from the multiple of span that the row's first entry lies behind). Every resident CTA takes an equal run of the list, so that none starts late and none
// ends early, whatever the lengths. Each warp leaves a part (maximum, sum, output) of every unit that its CTA's run touches, and paged_join_kernel puts the
// parts together: CTA c has part number u + c in unit u of all units, which no other has, as c or u grows from one part of the list to the next.
constexpr uint32_t PAGED_SMEM_MOST = 216u * 1024u;  // dynamic shared memory that the kernels are allowed, whatever a call takes
constexpr uint32_t LIST_ROWS = 256;  // rows of a launch: their ranges stay in shared memory

// The CTA whose run holds tile x of `total`; CTA i of n has [i total / n, (i + 1) total / n).
__device__ __forceinline__ uint64_t quotient(uint64_t x, uint64_t y) {  // most lists are short enough for the fast division
    return (x | y) >> 32 ? x / y : (uint64_t)((uint32_t)x / (uint32_t)y);
}
__device__ __forceinline__ uint32_t cta_of(uint64_t x, uint64_t total, uint32_t n) { return (uint32_t)quotient((x + 1u) * n - 1u, total); }
__device__ __forceinline__ uint32_t ctas_at_work(uint64_t total, uint32_t n) { return total < n ? (uint32_t)total : n; }


struct PagedList {
    uint64_t prefix[LIST_ROWS + 1];  // tiles before each row
    uint32_t slot[LIST_ROWS], begin[LIST_ROWS], end[LIST_ROWS];
};
struct PagedPlace {
    uint32_t row, unit, tile, tiles, t0, t1, first;
};

// By the first warp of a CTA; a barrier has to follow. CTA 0 leaves the prefix for the join.
__device__ __forceinline__ void paged_list_make(const PagedAttnArgs& a, PagedList& s, uint32_t rows, uint32_t span) {
    const uint32_t lane = threadIdx.x & 31u;
    uint64_t before = 0;
    for (uint32_t r0 = 0; r0 < rows; r0 += 32u) {
        const uint32_t r = r0 + lane;
        uint32_t slot = 0, begin = 0, end = 0, n = 0;
        if (r < rows) {
            const bool inside = paged_row_range(a, a.row0 + r, &slot, &begin, &end);
            if (!inside && blockIdx.x == 0) atomicOr(a.status, 1u);
            n = inside && end > begin ? (end - (begin & ~(span - 1u)) + span - 1u) / span : 0u;
        }
        uint64_t sum = n;  // 32 rows of 2^30 entries have 2^32 tiles of 8
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= (uint32_t)o) sum += u;
        }
        if (r < rows) {
            s.slot[r] = slot, s.begin[r] = begin, s.end[r] = end;
            s.prefix[r] = before + sum - n;
            if (blockIdx.x == 0) a.prefix[r] = before + sum - n;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) {
        s.prefix[rows] = before;
        if (blockIdx.x == 0) a.prefix[rows] = before;
    }
}
__device__ __forceinline__ void paged_list_enter(const PagedList& s, PagedPlace& p, uint32_t span) {  // p.row has tiles
    p.t0 = s.begin[p.row], p.t1 = s.end[p.row], p.first = p.t0 & ~(span - 1u);
    p.tiles = (p.t1 - p.first + span - 1u) / span;
}
// Whether the next tile is in another unit.
__device__ __forceinline__ bool paged_list_next(const PagedList& s, PagedPlace& p, uint32_t rows, uint32_t units, uint32_t span) {
    if (++p.tile < p.tiles) return false;
    p.tile = 0;
    if (++p.unit == units) {
        p.unit = 0;
        do ++p.row;
        while (p.row < rows && s.prefix[p.row + 1] == s.prefix[p.row]);
        if (p.row < rows) paged_list_enter(s, p, span);
    }
    return true;
}
__device__ __forceinline__ PagedPlace paged_list_at(const PagedList& s, uint64_t x, uint32_t rows, uint32_t units, uint32_t span) {
    uint32_t l = 0, h = rows;  // the last row that begins at or before x
    while (h - l > 1u) {
        const uint32_t mid = (l + h) / 2u;
        if (s.prefix[mid] * units <= x) l = mid; else h = mid;
    }
    PagedPlace p;
    p.row = l;
    paged_list_enter(s, p, span);
    const uint64_t in_row = x - s.prefix[l] * units;
    p.unit = (uint32_t)quotient(in_row, p.tiles);
    p.tile = (uint32_t)(in_row - (uint64_t)p.unit * p.tiles);
    return p;
}

// paged_lanes_kernel (attention_paged_lanes.cu): whether it takes the cache, how many q heads it takes at a time, its resident CTAs and warps, and one launch for
// the rows from a.row0 on.
struct PagedLanes {
    uint32_t heads_at_once, ctas, warps;
};
bool m40_paged_lanes(const M40llmCudaContext* ctx, const M40llmPagedCache* cache, uint32_t group, PagedLanes* out);
cudaError_t m40_paged_lanes_launch(M40llmCudaContext* ctx, const PagedAttnArgs& a, const PagedLanes& l, bool f32);
